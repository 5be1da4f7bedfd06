// Launch parameters and launchers of the operators around the sparse
// attention: rotation and norms (sfa_rope.hip), attention of a tree of drafted
// tokens (sfa_tree.hip), pages of the cache (sfa_pages.hip).  Their C entry
// points are in sfa_api_ops.hip.
#pragma once

#include <utility>

#include "sfa_common.h"

namespace sfa {

// f(integral_constant i) for i = 0 .. N - 1
template <int... I, class F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each_of(std::make_integer_sequence<int, N>{}, f);
}

// Stores the message for sfa_last_error() and returns code (sfa_api.hip).
int api_fail(int code, const char* msg);
void api_clear();

// ---- rotation and norms ----
// One tensor's heads.  Strides in elements.  Forward: x -> y (append: y is the
// page pool, y_sb / y_ss its page and row strides).  Backward: y is dy.
struct RopeSide {
  const void* x;
  void* y;
  void* dx;
  const void* w;
  void* dw;
  int64_t x_sb, x_ss, x_sh;
  int64_t y_sb, y_ss, y_sh;
  int64_t dx_sb, dx_ss, dx_sh;
  int H, n;    // heads (0: no such tensor), normed dims (0: no norm)
  int groups;  // row groups per token
};
struct RopeParams {
  RopeSide side[2];  // q, k
  const void* v;     // append: the v rows and their pool, or nullptr
  void* v_out;
  int64_t v_sb, v_ss, v_sh, vo_sb, vo_ss, vo_sh;
  int Dv;
  const void* pos;   // [B, S] int32 or int64
  int64_t pos_sb, pos_ss;
  int pos_i64;
  const double* freq;  // [R / 2]
  int w_f32;           // weights are float32 (else of x's type)
  int interleaved;
  int B, S, D, R, off;
  float eps, rope_scale;
  // append
  const int32_t* block_table;  // nullptr: y is a tensor
  int64_t bt_sb;
  const void* slots;
  int64_t slot_sb, slot_ss;
  int slot_i64;
  int max_pages, page_shift, num_pages;
  // geometry (rope_geometry)
  int P, K, chunks;     // lanes a row, 16-byte chunks a lane, chunks a row
  int groups, per, upt; // row groups a token; in blocks of per, upt blocks a token
  int64_t units;        // B * S * groups
  float* part;          // backward: [2][workgroups][1024] partial dw, or nullptr
};
void rope_geometry(RopeParams& p, int esize, bool vec);
int rope_bwd_wgs(const RopeParams& p);
size_t rope_bwd_workspace(const RopeParams& p);
hipError_t launch_rope_fwd(const RopeParams& p, int dtype, bool vec, hipStream_t s);
hipError_t launch_rope_bwd(const RopeParams& p, int dtype, bool vec, hipStream_t s);

// ---- attention of a tree of drafted tokens over a paged cache ----
struct TreeParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* block_table;
  const int32_t* ctx_lens;   // [B]
  const int64_t* tree_mask;  // [B, T]
  const int32_t* tree_lens;  // [B] or nullptr
  const float* sink;
  void* out;
  float* lse;
  int64_t q_sb, q_ss, q_sh;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;  // page, row, head
  int64_t o_sb, o_ss, o_sh, l_sb, l_ss, l_sh;
  int64_t bt_sb, tm_sb, tm_ss;
  int B, T, Hq, Hkv, G, Dqk, Dv;
  int max_pages, page_shift, num_pages, cap;  // cap: max_pages * page_size
  float scale, scale_log2;
  int nrb;                   // row blocks per (sequence, kv head)
  // Key ranges ("slots"): the batch's keys are cut into about `want` ranges of one
  // length (two tiles or more; a tile is a power of two of keys), found on the
  // device; a sequence of several leaves partials per slot.  want = 0: one a sequence.
  int want, tile;
  float* part_o;             // [slots][T * Hq][Dv], normalised by the slot's own sum
  float* part_lse;           // [slots][T * Hq], base-2 (-inf: nothing seen)
  int32_t* seq_slots;        // [B][2] first slot and slots of a sequence
};
struct TreePlan {
  int kernel;
  int rows;       // query rows (token, head) per workgroup
  int want, slots;
  int64_t wgs;    // workgroups of `threads` threads
  int threads;
  bool fits() const { return wgs * threads < (int64_t)1 << 32; }  // one launch
  size_t part_o_bytes, part_lse_bytes, seq_bytes;
  size_t workspace() const { return part_o_bytes + part_lse_bytes + seq_bytes; }
};
TreePlan tree_plan(const TreeParams& p, int dtype, bool vec);
hipError_t launch_tree(const TreeParams& p, const TreePlan& pl, int dtype, hipStream_t s);

// ---- pages of a cache ----
constexpr int kPoolsPerLaunch = 48;
struct PoolList {
  char* base[kPoolsPerLaunch];
  int64_t page_stride[kPoolsPerLaunch];  // bytes
  int64_t page_bytes[kPoolsPerLaunch];
  int n;
};
struct PagesParams {
  int32_t* block_table;
  int64_t bt_sb;
  int32_t* refs;
  int32_t* kv_lens;
  int B, max_pages, num_pages, page_shift;
  int32_t* ws;  // 16 ints, then 3 * num_pages, then 2 * n
};
size_t pages_workspace_ints(int num_pages, int n);
constexpr int kMaxSeqs = 8192;      // sequences of a table that fork and extend plan in one workgroup
constexpr int kMaxPathLen = 64;
hipError_t launch_pages_copy(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* src,
                             const int32_t* dst, int n, bool vec, hipStream_t s);
hipError_t launch_pages_fork(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* parents,
                             const int32_t* children, int n, int32_t* ok, bool vec, hipStream_t s);
hipError_t launch_pages_free(const PagesParams& p, const int32_t* rows, const int32_t* keep_lens, int n, hipStream_t s);
hipError_t launch_pages_extend(const PagesParams& p, const int32_t* new_lens, int32_t* ok, hipStream_t s);
hipError_t launch_pages_compact(const PagesParams& p, const PoolList* pools, int nlists, int32_t* used, bool vec,
                                hipStream_t s);
hipError_t launch_pages_keep(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* ctx_lens,
                             const int32_t* path, int64_t path_sb, int plen, bool vec, hipStream_t s);

}  // namespace sfa

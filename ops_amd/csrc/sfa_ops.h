// Launch parameters and launchers of the operators around the sparse
// attention: rotation and norms (sfa_rope.hip), attention of a tree of drafted
// tokens (sfa_tree.hip), dense attention (sfa_dense*.hip), rows (sfa_read.hip) and
// pages of the cache (sfa_pages.hip).  Their C entry points are in sfa_api_ops.hip.
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
  // append to 8-bit pools (y and v_out of side k are bytes): the rows' exponent bytes
  uint8_t *ks, *vs;
  int64_t ks_sb, ks_ss, ks_sh, vs_sb, vs_ss, vs_sh;
  // geometry (rope_geometry)
  int P, K, chunks;     // lanes a row, 16-byte chunks a lane, chunks a row
  int groups, per, upt; // row groups a token; in blocks of per, upt blocks a token
  int64_t units;        // B * S * groups
  float* part;          // backward: [2][workgroups][1024] partial dw, or nullptr
};
void rope_geometry(RopeParams& p, int esize, bool vec);
int rope_bwd_wgs(const RopeParams& p);
size_t rope_bwd_workspace(const RopeParams& p);
hipError_t launch_rope_fwd(const RopeParams& p, int dtype, bool vec, hipStream_t s);  // p.ks: to 8-bit pools
hipError_t launch_rope_bwd(const RopeParams& p, int dtype, bool vec, hipStream_t s);

// ---- 8-bit rows: e4m3 values times the value of the row's exponent byte ----
struct fp8_t {
  uint8_t x;
};
template <typename T>
__device__ __forceinline__ float value_of(T x) {
  if constexpr (std::is_same<T, fp8_t>::value) return __builtin_amdgcn_cvt_f32_fp8((int)x.x, 0);
  else return to_f32(x);
}
__device__ __forceinline__ float scale_of(uint8_t e) {
  // (2^-127 is no normal number, 255 stands for NaN)
  return __uint_as_float(e == 255 ? 0x7fc00000u : e == 0 ? 0x00400000u : (uint32_t)e << 23);
}

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

// ---- dense attention through a window: a chunk over a paged cache, a sequence ----
struct DenseParams {
  const void* q;
  const void* k;             // pages: pools, else [B, cap]
  const void* v;
  const uint8_t* ks;         // 8-bit pools: exponent bytes, [pages, page, Hkv]
  const uint8_t* vs;
  const int32_t* block_table;  // nullptr: contiguous
  const int32_t* ctx_lens;   // [B] or nullptr: 0
  const int32_t* lens;       // [B] or nullptr: S
  const float* sink;
  void* out;
  float* lse;
  int64_t q_sb, q_ss, q_sh;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;  // (pools: page, row, head)
  int64_t ks_sb, ks_ss, ks_sh, vs_sb, vs_ss, vs_sh;
  int64_t o_sb, o_ss, o_sh, l_sb, l_ss, l_sh;
  int64_t bt_sb;
  int B, S, Hq, Hkv, G, Dqk, Dv;
  int window, first;         // window: up to 2^30, which is more than any distance in a table
  int over;                  // what the caller's has over that (none: 2^31 - 1)
  int page_shift, num_pages, cap;  // cap: rows a sequence can have
  float scale, scale_log2;
  bool vec;                  // rows are whole 16-byte units (8-bit: 8)
  // a launch: row blocks of `rows` query rows, nrb a (sequence, kv head); key tiles of 2^tile_shift
  int rows, nrb, tile_shift;
  int fit, want, min_len, join;  // ranges a kv head that run at once; the most (0: one a row block); tiles of the shortest; of a join
  int slots;                 // of the launch, a kv head
  float* part_o;             // [slots][Hkv][rows][Dv], normalised by the slot's own sum
  float* part_lse;           // [slots][Hkv][rows], base-2 (-inf: nothing seen)
  int32_t* unit_slots;       // [B nrb][2] first slot and slots of a unit
  // backward
  const void* dout;
  void *dq, *dk, *dv;
  int64_t do_sb, do_ss, do_sh, dq_sb, dq_ss, dq_sh, dk_sb, dk_ss, dk_sh, dv_sb, dv_ss, dv_sh;
  const float* dlse;         // lse's strides, or nullptr
  float* dsink;              // [Hq] or nullptr
  // [B][Hkv][S G]: base-2 LSE (+inf: nothing seen) and delta = sum o do - dlse; for the bf16
  // matrix kernels (row_neg) -lse / scale and -delta, which their accumulators start from
  float* row_lse;
  float* row_delta;
  // delta of o before its rounding, which dq leaves for dk, dv and the sink: row_delta again where
  // one workgroup makes a row's dq, else (heads of more than 128 dims) an array that no dq reads
  float* row_exact;
  bool row_neg;
  float* dkv_part;           // partial dK | dV of key blocks cut in chunks: bf16 matrix kernels [B Hkv][dkv_parts]
                             // [kDkvKeys][2 D], others [B Hkv][blocks][dkv_parts][kAnyRows][Dqk + Dv]
  int* dkv_units;            // [units][4] block, chunk, first partial, chunks of the block, in order of the launch
  int chunk, cut0, cut1, cut_chunk;  // query rows a chunk; of the key blocks [cut0, cut1)
  int dkv_parts;             // partials a kv head; others: chunks of a block, at most
};
constexpr int kDenseUnits = 256;  // row blocks of a launch that is cut into ranges, at most
struct DensePlan {
  int kernel;
  int rows, tile_shift, fit, want, min_len, join, slots;
  int64_t wgs;               // workgroups of `threads` threads
  int threads;
  bool fits() const { return wgs * threads < (int64_t)1 << 32; }  // one launch
  size_t part_o_bytes, part_lse_bytes, unit_bytes;
  size_t workspace() const { return part_o_bytes + part_lse_bytes + unit_bytes; }
};
DensePlan dense_plan(const DenseParams& p, int dtype, int kv_dtype);
hipError_t launch_dense(const DenseParams& p, const DensePlan& pl, int dtype, int kv_dtype, hipStream_t s);
constexpr int kDkvKeys = 128;  // keys a block of the dk / dv kernel
struct DenseBwdPlan {
  size_t row_bytes, dkv_bytes, unit_bytes;  // row_lse (row_delta, row_exact: as much each); partial dK | dV; the units
  int row_arrays;
  int chunk, cut0, cut1, cut_chunk, units, parts;  // of the dk / dv kernel: as above; units and partials a kv head
  bool mfma, fits;
  size_t workspace() const { return row_arrays * row_bytes + dkv_bytes + unit_bytes; }
};
DenseBwdPlan dense_bwd_plan(const DenseParams& p, int dtype);
hipError_t launch_dense_bwd(const DenseParams& p, const DenseBwdPlan& pl, int dtype, hipStream_t s);
// any types and head dims (sfa_dense_any.hip)
constexpr int kAnyRows = 64, kAnyShift = 5, kAnyDims = 128;
void launch_dense_any(const DenseParams& p, int dtype, int kv_dtype, hipStream_t s);
void launch_dense_bwd_any(const DenseParams& p, int dtype, hipStream_t s);
// ... up to 128 dims (sfa_dense_held.hip)
void launch_dense_held(const DenseParams& p, int dtype, int kv_dtype, hipStream_t s);
void launch_dense_held_bwd(const DenseParams& p, bool f32, hipStream_t s);

// bf16 queries, head dims 64 and 128, many rows (sfa_dense_wide.hip)
constexpr int kWideRows = 256;
void launch_dense_wide(const DenseParams& p, int kv_dtype, hipStream_t s);

// ... and up to 64 rows a (sequence, kv head) (sfa_dense_few.hip): p.rows 16, 32 or 64
void launch_dense_few(const DenseParams& p, int kv_dtype, hipStream_t s);

// ... and over latent rows (sfa_dense_mla.hip): head dims 576 / 512, V the first dims of K
constexpr int kLatentRows = 64, kLatentQK = 576, kLatentV = 512;
void launch_dense_mla(const DenseParams& p, bool fp8, hipStream_t s);

void launch_dense_bwd_mfma(const DenseParams& p, int units, hipStream_t s);  // (sfa_dense_bwd.hip)

// ---- rows of a cache as contiguous ones (sfa_read.hip) ----
struct ReadParams {
  const void* cache;
  const uint8_t* scale;
  const int32_t* block_table;
  const int32_t* starts;  // nullptr: 0
  const int32_t* lens;
  void* out;
  int64_t c_sb, c_ss, c_sh, s_sb, s_ss, s_sh, o_sb, o_ss, o_sh, bt_sb;
  int B, N, H, D;
  int max_pages, page_shift, num_pages;
};
hipError_t launch_cache_read(const ReadParams& p, int dtype, int cache_dtype, bool vec, hipStream_t s);

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

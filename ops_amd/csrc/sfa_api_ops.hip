// C entry points of the operators around the attention (declared in
// include/sfa.h): argument checks, workspaces, dispatch.  Nothing here
// allocates, frees or synchronises; all work goes onto the caller's stream.

#include <limits.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "sfa_ops.h"

namespace {

constexpr int kMaxHeadDim = 1024;
constexpr int kMaxGridYZ = 65535;

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return sfa::api_fail(code, msg);
}
int done(hipError_t e, const char* what) {
  if (e == hipSuccess) return SFA_OK;
  return fail(SFA_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
template <class... I>
bool mult(int64_t m, I... x) {
  return ((x % m == 0) && ...);
}

int check_pages(const sfa_kv_pages* pg, int B) {
  if (pg == nullptr || pg->block_table == nullptr) return fail(SFA_E_INVALID, "null page table");
  if (pg->flags != 0) return fail(SFA_E_INVALID, "page table flags must be 0");
  if (pg->page_size <= 0 || (pg->page_size & (pg->page_size - 1)) != 0)
    return fail(SFA_E_INVALID, "page_size must be a power of two (got %d)", pg->page_size);
  if (pg->max_pages <= 0 || pg->num_pages <= 0) return fail(SFA_E_INVALID, "max_pages and num_pages must be positive");
  if ((int64_t)pg->num_pages * pg->page_size > INT32_MAX || (int64_t)pg->max_pages * pg->page_size > INT32_MAX)
    return fail(SFA_E_INVALID, "num_pages * page_size and max_pages * page_size must stay below 2^31");
  if (B > 1 && pg->bt_sb < pg->max_pages)
    return fail(SFA_E_INVALID, "block-table row stride %lld is below max_pages %d", (long long)pg->bt_sb, pg->max_pages);
  return SFA_OK;
}

// ---- rotation and norms ----------------------------------------------------------

int check_rope(const sfa_rope_args* a, bool backward, bool append) {
  if (a == nullptr) return fail(SFA_E_INVALID, "null argument struct");
  if (a->dtype != SFA_DTYPE_F32 && a->dtype != SFA_DTYPE_BF16) return fail(SFA_E_INVALID, "unknown dtype %d", a->dtype);
  if (a->w_dtype != SFA_DTYPE_F32 && a->w_dtype != a->dtype)
    return fail(SFA_E_INVALID, "weights must be float32 or of the rows' type");
  if (a->flags != 0) return fail(SFA_E_INVALID, "flags must be 0");
  if (a->B <= 0 || a->S <= 0 || a->Hq < 0 || a->Hkv < 0 || (a->Hq == 0 && a->Hkv == 0))
    return fail(SFA_E_INVALID, "B, S and the heads must be positive");
  if (a->D <= 0 || a->D > kMaxHeadDim) return fail(SFA_E_INVALID, "the head dim must be in [1, %d]", kMaxHeadDim);
  if (a->rotary_dim < 0 || a->rotary_dim % 2 != 0 || a->rope_offset < 0 || a->rotary_dim > a->D ||
      a->rope_offset > a->D - a->rotary_dim)
    return fail(SFA_E_INVALID, "rotated dims [%d, %d + %d) must be an even number within the head's %d", a->rope_offset,
                a->rope_offset, a->rotary_dim, a->D);
  if (a->q_norm < 0 || a->q_norm > a->D || a->k_norm < 0 || a->k_norm > a->D)
    return fail(SFA_E_INVALID, "normed dims must be within the head's %d", a->D);
  if (!(a->eps >= 0.f) || isinf(a->eps)) return fail(SFA_E_INVALID, "eps must be finite and >= 0");
  if (!(a->rope_scale == a->rope_scale) || isinf(a->rope_scale)) return fail(SFA_E_INVALID, "rope_scale must be finite");
  if (a->positions == nullptr || (a->rotary_dim > 0 && a->inv_freq == nullptr)) return fail(SFA_E_INVALID, "null tensor pointer");
  if (a->Hq > 0 && (!a->q_out || (a->q_norm > 0 && !a->q_weight) || ((!backward || a->q_norm > 0) && !a->q)))
    return fail(SFA_E_INVALID, "null tensor pointer");
  if (a->Hkv > 0 && (!a->k_out || (a->k_norm > 0 && !a->k_weight) || ((!backward || a->k_norm > 0) && !a->k)))
    return fail(SFA_E_INVALID, "null tensor pointer");
  if (backward && ((a->Hq > 0 && (!a->dq || (a->q_norm > 0 && !a->dq_weight))) ||
                   (a->Hkv > 0 && (!a->dk || (a->k_norm > 0 && !a->dk_weight)))))
    return fail(SFA_E_INVALID, "null gradient pointer");
  if (append) {
    if (a->Hkv <= 0 || a->slots == nullptr) return fail(SFA_E_INVALID, "append needs k rows and slots");
    if (a->Dv < 0 || a->Dv > kMaxHeadDim) return fail(SFA_E_INVALID, "the v head dim must be in [0, %d]", kMaxHeadDim);
    if (a->Dv > 0 && (!a->v || !a->v_out)) return fail(SFA_E_INVALID, "null tensor pointer");
  }
  // rows and units are counted in 32 bits per launch dimension (and the product itself in 64)
  if ((int64_t)a->B * a->S > INT_MAX / ((int64_t)a->Hq + 2 * (int64_t)a->Hkv))
    return fail(SFA_E_UNSUPPORTED, "more than 2^31 rows");
  return SFA_OK;
}

sfa::RopeParams rope_params(const sfa_rope_args* a, const sfa_kv_pages* pg) {
  sfa::RopeParams p;
  memset(&p, 0, sizeof(p));
  sfa::RopeSide &q = p.side[0], &k = p.side[1];
  q = {a->q, a->q_out, a->dq, a->q_weight, a->dq_weight, a->q_sb, a->q_ss, a->q_sh, a->qo_sb, a->qo_ss, a->qo_sh,
       a->dq_sb, a->dq_ss, a->dq_sh, a->Hq, a->Hq > 0 ? a->q_norm : 0, 0};
  k = {a->k, a->k_out, a->dk, a->k_weight, a->dk_weight, a->k_sb, a->k_ss, a->k_sh, a->ko_sb, a->ko_ss, a->ko_sh,
       a->dk_sb, a->dk_ss, a->dk_sh, a->Hkv, a->Hkv > 0 ? a->k_norm : 0, 0};
  p.pos = a->positions; p.pos_sb = a->p_sb; p.pos_ss = a->p_ss; p.pos_i64 = a->pos_i64;
  p.freq = a->inv_freq;
  p.w_f32 = a->w_dtype == SFA_DTYPE_F32;
  p.interleaved = a->interleaved != 0;
  p.B = a->B; p.S = a->S; p.D = a->D; p.R = a->rotary_dim; p.off = a->rope_offset;
  p.eps = a->eps; p.rope_scale = a->rope_scale;
  if (pg != nullptr) {
    p.block_table = pg->block_table; p.bt_sb = pg->bt_sb;
    p.slots = a->slots; p.slot_sb = a->s_sb; p.slot_ss = a->s_ss; p.slot_i64 = a->slots_i64;
    p.max_pages = pg->max_pages; p.num_pages = pg->num_pages;
    p.page_shift = __builtin_ctz((unsigned)pg->page_size);
    if (a->Dv > 0) {
      p.v = a->v; p.v_out = a->v_out; p.Dv = a->Dv;
      p.v_sb = a->v_sb; p.v_ss = a->v_ss; p.v_sh = a->v_sh;
      p.vo_sb = a->vo_sb; p.vo_ss = a->vo_ss; p.vo_sh = a->vo_sh;
    }
  }
  return p;
}

// Whole 16-byte chunks: rows, strides, and the borders of the normed and
// rotated dims (half layout: the border between the halves too).
bool rope_vec(const sfa_rope_args* a, const sfa::RopeParams& p, bool backward) {
  const int E = a->dtype == SFA_DTYPE_F32 ? 4 : 8;
  if (!mult(E, a->D, a->rope_offset, a->interleaved ? a->rotary_dim : a->rotary_dim / 2)) return false;
  for (int i = 0; i < 2; ++i) {
    const sfa::RopeSide& s = p.side[i];
    if (s.H == 0) continue;
    if (!mult(E, s.n, s.y_sb, s.y_ss, s.y_sh) || !al16(s.y) || (s.n > 0 && !al16(s.w))) return false;
    if ((!backward || s.n > 0) && (!mult(E, s.x_sb, s.x_ss, s.x_sh) || !al16(s.x))) return false;
    if (backward && (!mult(E, s.dx_sb, s.dx_ss, s.dx_sh) || !al16(s.dx))) return false;
  }
  if (p.v != nullptr && (!mult(E, p.Dv, p.v_sb, p.v_ss, p.v_sh, p.vo_sb, p.vo_ss, p.vo_sh) || !al16(p.v) || !al16(p.v_out)))
    return false;
  return true;
}

// ---- drafted trees -----------------------------------------------------------------

int check_tree(const sfa_tree_args* a, const sfa_kv_pages* pg) {
  if (a == nullptr) return fail(SFA_E_INVALID, "null argument struct");
  if (a->dtype != SFA_DTYPE_F32 && a->dtype != SFA_DTYPE_BF16) return fail(SFA_E_INVALID, "unknown dtype %d", a->dtype);
  if (a->flags != 0) return fail(SFA_E_INVALID, "flags must be 0");
  if (a->B <= 0 || a->T <= 0 || a->Hq <= 0 || a->Hkv <= 0) return fail(SFA_E_INVALID, "B, T, Hq, Hkv must be positive");
  if (a->T > 64) return fail(SFA_E_INVALID, "at most 64 drafted tokens a sequence (got %d)", a->T);
  if (a->Hq % a->Hkv != 0) return fail(SFA_E_INVALID, "Hq (%d) must be a multiple of Hkv (%d)", a->Hq, a->Hkv);
  if (a->Dqk <= 0 || a->Dv <= 0 || a->Dqk > kMaxHeadDim || a->Dv > kMaxHeadDim)
    return fail(SFA_E_INVALID, "head dims must be in [1, %d]", kMaxHeadDim);
  if (!a->q || !a->k || !a->v || !a->ctx_lens || !a->tree_mask || !a->out || !a->lse)
    return fail(SFA_E_INVALID, "null tensor pointer");
  if (!(a->scale > 0.f) || isinf(a->scale)) return fail(SFA_E_INVALID, "scale must be finite and > 0");
  const int rc = check_pages(pg, a->B);
  if (rc != SFA_OK) return rc;
  if ((int64_t)pg->max_pages * pg->page_size > (int64_t)1 << 29)
    return fail(SFA_E_UNSUPPORTED, "a table of more than 2^29 rows a sequence");
  if ((int64_t)a->B * a->T > (int64_t)INT_MAX / 4 / a->Hq) return fail(SFA_E_UNSUPPORTED, "more than 2^29 query rows");
  return SFA_OK;
}

sfa::TreeParams tree_params(const sfa_tree_args* a, const sfa_kv_pages* pg) {
  sfa::TreeParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q; p.k = a->k; p.v = a->v;
  p.block_table = pg->block_table; p.bt_sb = pg->bt_sb;
  p.ctx_lens = a->ctx_lens; p.tree_lens = a->tree_lens; p.sink = a->sink;
  p.tree_mask = a->tree_mask; p.tm_sb = a->tm_sb; p.tm_ss = a->tm_ss;
  p.out = a->out; p.lse = a->lse;
  p.q_sb = a->q_sb; p.q_ss = a->q_ss; p.q_sh = a->q_sh;
  p.k_sb = a->k_sb; p.k_ss = a->k_ss; p.k_sh = a->k_sh;
  p.v_sb = a->v_sb; p.v_ss = a->v_ss; p.v_sh = a->v_sh;
  p.o_sb = a->o_sb; p.o_ss = a->o_ss; p.o_sh = a->o_sh;
  p.l_sb = a->l_sb; p.l_ss = a->l_ss; p.l_sh = a->l_sh;
  p.B = a->B; p.T = a->T; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv;
  p.Dqk = a->Dqk; p.Dv = a->Dv;
  p.max_pages = pg->max_pages; p.num_pages = pg->num_pages;
  p.page_shift = __builtin_ctz((unsigned)pg->page_size);
  p.cap = pg->max_pages * pg->page_size;
  p.scale = a->scale;
  p.scale_log2 = a->scale * sfa::kLog2e;
  return p;
}

// 16-byte rows and strides
bool tree_vec(const sfa_tree_args* a) {
  const int E = a->dtype == SFA_DTYPE_F32 ? 4 : 8;
  return mult(E, a->q_sb, a->q_ss, a->q_sh, a->k_sb, a->k_ss, a->k_sh, a->v_sb, a->v_ss, a->v_sh, a->o_sb, a->o_ss,
              a->o_sh) && al16(a->q) && al16(a->k) && al16(a->v) && al16(a->out);
}

// ---- pages ---------------------------------------------------------------------------

constexpr int kMaxPools = 1024;

int check_cache(const sfa_cache* c, bool table, bool refs, bool lens, bool pools) {
  if (c == nullptr) return fail(SFA_E_INVALID, "null argument struct");
  if (c->flags != 0) return fail(SFA_E_INVALID, "flags must be 0");
  if (c->page_size <= 0 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(SFA_E_INVALID, "page_size must be a power of two (got %d)", c->page_size);
  if (c->num_pages <= 0 || (int64_t)c->num_pages * c->page_size > INT32_MAX)
    return fail(SFA_E_INVALID, "num_pages must be positive and num_pages * page_size below 2^31");
  if (c->num_pages > 1 << 30) return fail(SFA_E_UNSUPPORTED, "more than 2^30 pages");
  if (table) {
    if (c->block_table == nullptr) return fail(SFA_E_INVALID, "null page table");
    if (c->B <= 0 || c->max_pages <= 0) return fail(SFA_E_INVALID, "B and max_pages must be positive");
    if ((int64_t)c->max_pages * c->page_size > INT32_MAX)
      return fail(SFA_E_INVALID, "max_pages * page_size must stay below 2^31");
    if (c->B > 1 && c->bt_sb < c->max_pages) return fail(SFA_E_INVALID, "block-table rows overlap");
    if ((int64_t)c->B * c->max_pages > INT32_MAX) return fail(SFA_E_UNSUPPORTED, "a table of more than 2^31 entries");
  }
  if (refs && c->ref_counts == nullptr) return fail(SFA_E_INVALID, "null ref_counts");
  if (lens && c->kv_lens == nullptr) return fail(SFA_E_INVALID, "null kv_lens");
  if (pools) {
    if (c->npools <= 0 || c->npools > kMaxPools || c->pools == nullptr)
      return fail(SFA_E_INVALID, "the number of caches must be in [1, %d]", kMaxPools);
    for (int i = 0; i < c->npools; ++i) {
      const sfa_cache_pool& q = c->pools[i];
      if (q.base == nullptr || q.page_bytes <= 0 || q.page_bytes % c->page_size != 0)
        return fail(SFA_E_INVALID, "cache %d: pages of %lld bytes, %d rows", i, (long long)q.page_bytes, c->page_size);
      if (c->num_pages > 1 && q.page_stride < q.page_bytes) return fail(SFA_E_INVALID, "cache %d: pages overlap", i);
    }
  }
  return SFA_OK;
}

int check_pairs(const sfa_cache* c, int32_t n, void* ws, size_t bytes) {
  if (n < 0 || n > kMaxGridYZ) return fail(SFA_E_INVALID, "the number of pairs must be in [0, %d]", kMaxGridYZ);
  const size_t need = sfa::pages_workspace_ints(c->num_pages, n) * sizeof(int32_t);
  if (ws == nullptr || bytes < need)
    return fail(SFA_E_WORKSPACE, "the call needs %zu workspace bytes (got %zu)", need, bytes);
  return SFA_OK;
}

sfa::PagesParams pages_params(const sfa_cache* c, void* ws) {
  sfa::PagesParams p;
  memset(&p, 0, sizeof(p));
  p.block_table = c->block_table; p.bt_sb = c->bt_sb; p.refs = c->ref_counts; p.kv_lens = c->kv_lens;
  p.B = c->B; p.max_pages = c->max_pages; p.num_pages = c->num_pages;
  p.page_shift = __builtin_ctz((unsigned)c->page_size);
  p.ws = (int32_t*)ws;
  return p;
}

struct Lists {
  sfa::PoolList l[(kMaxPools + sfa::kPoolsPerLaunch - 1) / sfa::kPoolsPerLaunch];
  int n = 0;
  bool vec = true;  // everything that is copied is whole 16-byte units
};
void make_lists(const sfa_cache* c, bool rows, Lists& out) {
  for (int i = 0; i < c->npools; ++i) {
    if (i % sfa::kPoolsPerLaunch == 0) out.l[out.n++].n = 0;
    sfa::PoolList& l = out.l[out.n - 1];
    const sfa_cache_pool& q = c->pools[i];
    l.base[l.n] = (char*)q.base;
    l.page_stride[l.n] = q.page_stride;
    l.page_bytes[l.n] = q.page_bytes;
    ++l.n;
    out.vec = out.vec && al16(q.base) && mult(16, q.page_stride, rows ? q.page_bytes / c->page_size : q.page_bytes);
  }
}

}  // namespace

extern "C" {

int sfa_rope_fwd(const sfa_rope_args* a, const sfa_kv_pages* pages, void* stream) {
  sfa::api_clear();
  int rc = check_rope(a, false, pages != nullptr);
  if (rc == SFA_OK && pages != nullptr) rc = check_pages(pages, a->B);
  if (rc != SFA_OK) return rc;
  sfa::RopeParams p = rope_params(a, pages);
  const bool vec = rope_vec(a, p, false);
  sfa::rope_geometry(p, a->dtype == SFA_DTYPE_F32 ? 4 : 2, vec);
  return done(sfa::launch_rope_fwd(p, a->dtype, vec, (hipStream_t)stream), "sfa_rope_fwd");
}

size_t sfa_rope_bwd_workspace_size(const sfa_rope_args* a) {
  if (check_rope(a, true, false) != SFA_OK) return 0;
  sfa::RopeParams p = rope_params(a, nullptr);
  sfa::rope_geometry(p, a->dtype == SFA_DTYPE_F32 ? 4 : 2, rope_vec(a, p, true));
  return sfa::rope_bwd_workspace(p);
}

int sfa_rope_bwd(const sfa_rope_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  sfa::api_clear();
  const int rc = check_rope(a, true, false);
  if (rc != SFA_OK) return rc;
  sfa::RopeParams p = rope_params(a, nullptr);
  const bool vec = rope_vec(a, p, true);
  sfa::rope_geometry(p, a->dtype == SFA_DTYPE_F32 ? 4 : 2, vec);
  const size_t need = sfa::rope_bwd_workspace(p);
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(SFA_E_WORKSPACE, "sfa_rope_bwd needs %zu workspace bytes (got %zu)", need, workspace_bytes);
    p.part = (float*)workspace;
  }
  return done(sfa::launch_rope_bwd(p, a->dtype, vec, (hipStream_t)stream), "sfa_rope_bwd");
}

size_t sfa_tree_fwd_workspace_size(const sfa_tree_args* a, const sfa_kv_pages* pages) {
  if (check_tree(a, pages) != SFA_OK) return 0;
  const sfa::TreePlan pl = sfa::tree_plan(tree_params(a, pages), a->dtype, tree_vec(a));
  return pl.fits() ? pl.workspace() : 0;
}

int sfa_tree_fwd(const sfa_tree_args* a, const sfa_kv_pages* pages, void* workspace, size_t workspace_bytes,
                 void* stream) {
  sfa::api_clear();
  const int rc = check_tree(a, pages);
  if (rc != SFA_OK) return rc;
  sfa::TreeParams p = tree_params(a, pages);
  const sfa::TreePlan pl = sfa::tree_plan(p, a->dtype, tree_vec(a));
  if (!pl.fits()) return fail(SFA_E_UNSUPPORTED, "more query rows than one launch holds (%lld workgroups)", (long long)pl.wgs);
  const size_t need = pl.workspace();
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need)
      return fail(SFA_E_WORKSPACE, "sfa_tree_fwd needs %zu workspace bytes (got %zu)", need, workspace_bytes);
    p.part_o = (float*)workspace;
    p.part_lse = (float*)((char*)workspace + pl.part_o_bytes);
    p.seq_slots = (int32_t*)((char*)workspace + pl.part_o_bytes + pl.part_lse_bytes);
  }
  return done(sfa::launch_tree(p, pl, a->dtype, (hipStream_t)stream), "sfa_tree_fwd");
}

size_t sfa_cache_workspace_size(const sfa_cache* c, int32_t n) {
  if (check_cache(c, false, false, false, false) != SFA_OK || n < 0 || n > kMaxGridYZ) return 0;
  return sfa::pages_workspace_ints(c->num_pages, n) * sizeof(int32_t);
}

int sfa_cache_copy(const sfa_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* workspace,
                   size_t workspace_bytes, void* stream) {
  sfa::api_clear();
  int rc = check_cache(c, false, false, false, true);
  if (rc == SFA_OK && n == 0) return SFA_OK;
  if (rc == SFA_OK) rc = check_pairs(c, n, workspace, workspace_bytes);
  if (rc != SFA_OK) return rc;
  if (!src || !dst) return fail(SFA_E_INVALID, "null tensor pointer");
  Lists l;
  make_lists(c, false, l);
  return done(sfa::launch_pages_copy(pages_params(c, workspace), l.l, l.n, src, dst, n, l.vec, (hipStream_t)stream),
              "sfa_cache_copy");
}

int sfa_cache_fork(const sfa_cache* c, const int32_t* parents, const int32_t* children, int32_t n, int32_t* ok,
                   void* workspace, size_t workspace_bytes, void* stream) {
  sfa::api_clear();
  int rc = check_cache(c, true, true, true, true);
  if (rc == SFA_OK && n == 0) return SFA_OK;
  if (rc == SFA_OK) rc = check_pairs(c, n, workspace, workspace_bytes);
  if (rc != SFA_OK) return rc;
  if (c->B > sfa::kMaxSeqs) return fail(SFA_E_UNSUPPORTED, "more than %d sequences", sfa::kMaxSeqs);
  if (!parents || !children || !ok) return fail(SFA_E_INVALID, "null tensor pointer");
  Lists l;
  make_lists(c, true, l);
  return done(sfa::launch_pages_fork(pages_params(c, workspace), l.l, l.n, parents, children, n, ok, l.vec,
                                     (hipStream_t)stream), "sfa_cache_fork");
}

int sfa_cache_free(const sfa_cache* c, const int32_t* rows, const int32_t* keep_lens, int32_t n, void* stream) {
  sfa::api_clear();
  const int rc = check_cache(c, true, true, false, false);
  if (rc != SFA_OK) return rc;
  if (n < 0 || n > kMaxGridYZ) return fail(SFA_E_INVALID, "the number of rows must be in [0, %d]", kMaxGridYZ);
  if (n == 0) return SFA_OK;
  if (!rows) return fail(SFA_E_INVALID, "null tensor pointer");
  return done(sfa::launch_pages_free(pages_params(c, nullptr), rows, keep_lens, n, (hipStream_t)stream), "sfa_cache_free");
}

int sfa_cache_extend(const sfa_cache* c, const int32_t* new_lens, int32_t* ok, void* workspace, size_t workspace_bytes,
                     void* stream) {
  sfa::api_clear();
  int rc = check_cache(c, true, true, true, false);
  if (rc == SFA_OK) rc = check_pairs(c, 0, workspace, workspace_bytes);
  if (rc != SFA_OK) return rc;
  if (c->B > sfa::kMaxSeqs) return fail(SFA_E_UNSUPPORTED, "more than %d sequences", sfa::kMaxSeqs);
  if (!new_lens || !ok) return fail(SFA_E_INVALID, "null tensor pointer");
  return done(sfa::launch_pages_extend(pages_params(c, workspace), new_lens, ok, (hipStream_t)stream), "sfa_cache_extend");
}

int sfa_cache_compact(const sfa_cache* c, int32_t* used, void* workspace, size_t workspace_bytes, void* stream) {
  sfa::api_clear();
  int rc = check_cache(c, true, true, false, true);
  if (rc == SFA_OK) rc = check_pairs(c, 0, workspace, workspace_bytes);
  if (rc != SFA_OK) return rc;
  if (!used) return fail(SFA_E_INVALID, "null tensor pointer");
  Lists l;
  make_lists(c, false, l);
  return done(sfa::launch_pages_compact(pages_params(c, workspace), l.l, l.n, used, l.vec, (hipStream_t)stream),
              "sfa_cache_compact");
}

int sfa_cache_keep_path(const sfa_cache* c, const int32_t* ctx_lens, const int32_t* path, int64_t path_sb, int32_t plen,
                        void* stream) {
  sfa::api_clear();
  const int rc = check_cache(c, true, false, false, true);
  if (rc != SFA_OK) return rc;
  if (plen < 0 || plen > sfa::kMaxPathLen) return fail(SFA_E_INVALID, "the path's length must be in [0, %d]", sfa::kMaxPathLen);
  if (plen == 0) return SFA_OK;
  if (c->B > kMaxGridYZ) return fail(SFA_E_UNSUPPORTED, "more than %d sequences", kMaxGridYZ);
  if (!ctx_lens || !path) return fail(SFA_E_INVALID, "null tensor pointer");
  Lists l;
  make_lists(c, true, l);
  return done(sfa::launch_pages_keep(pages_params(c, nullptr), l.l, l.n, ctx_lens, path, path_sb, plen, l.vec,
                                     (hipStream_t)stream), "sfa_cache_keep_path");
}

}  // extern "C"

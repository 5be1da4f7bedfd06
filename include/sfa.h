/*
 * sfa.h — C ABI of libsfa.so, the MI355X (gfx950) top-k sparse flash attention.
 *
 * The boundary replaces the three kernel launches of the reference's autograd
 * host launcher `SparseFlashAttentionTriton` (lilac-me/ops SFA.py:69-306):
 *
 *   sfa_fwd  <- `_attn_fwd[grid](...)`            SFA.py:122-159 (forward, SFA.py:75-164)
 *   sfa_bwd  <- `_attn_bwd_dq_dsink[grid](...)`   SFA.py:199-251
 *             + `_attn_bwd_dk_dv[grid](...)`      SFA.py:266-298 (backward, SFA.py:166-306)
 *
 * plus the workspace sizing the reference does inline with torch.empty
 * (SFA.py:117-120, 188-194, 253-261) and its ValueError paths
 * (SFA.py:52-53, 63-64).
 *
 * Conventions
 *  - Layout is BSHD with element strides for the batch, sequence and head
 *    dimensions; the last (feature) dimension must be contiguous.
 *      q   [B, Sq,  Hq,  Dqk]     k [B, Skv, Hkv, Dqk]     v [B, Skv, Hkv, Dv]
 *      idx [B, Sq,  Hkv, topk]  int32, -1 (or any out-of-range value) = padding
 *      out [B, Sq,  Hq,  Dv]      lse [B, Sq, Hq] float32, natural log
 *    `v` may alias `k` (e.g. MLA: v = k[..., :Dv]); inputs are never written.
 *    Query head h reads KV head h / (Hq / Hkv).
 *  - A slot is valid iff 0 <= idx < bound, bound = kv_lens[b] (if non-NULL,
 *    clamped to Skv) else Skv.  Invalid slots contribute exactly nothing; a
 *    row with no valid slot gives out = 0 and lse = -inf.
 *  - `sink` (optional, float32 [Hq]) adds exp(sink[h]) to every softmax
 *    denominator as SFA.py:469-474 does; NULL means no sink.
 *  - All pointers are device pointers.  The library never allocates, frees
 *    or synchronises: scratch comes from the caller through `workspace`,
 *    whose size the *_workspace_size functions give for the same arguments.
 *    All work is enqueued on `stream` (a hipStream_t; NULL = default stream).
 *  - Return value: 0 on success, a negative SFA_E* code otherwise; the
 *    message for the calling thread is available from sfa_last_error().
 */
#ifndef SFA_H_
#define SFA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SFA_ABI_VERSION 2

#if defined(__GNUC__)
#define SFA_API __attribute__((visibility("default")))
#else
#define SFA_API
#endif

/* Element types of q, k, v, out, dout, dq, dk, dv (F32, BF16), and of the
 * index producer's q / k (BF16, FP8_E4M3: OCP e4m3, one byte). */
enum { SFA_DTYPE_F32 = 0, SFA_DTYPE_BF16 = 1, SFA_DTYPE_FP8_E4M3 = 2 };

/* How the backward produces dK/dV. */
enum {
  SFA_DKV_AUTO = 0,    /* CSR where supported (bf16, d_qk = d_v = 128, G a power of two
                          <= 128, top-k <= 2048, Skv <= 262144) and cheaper: Skv <=
                          64 * top-k and CSR workspace (bitmap, lists, fp32 partials of
                          8 * d bytes per key and chunk of 4 to 64 blocks of 128
                          query-head rows, longer where those would pass 1 GiB)
                          <= 4 GiB; the same scheme at d_qk = d_v = 64 when Skv -
                          min(Sq, Skv) / 2 <= 16 * top-k and the call is large enough
                          (Sq * top-k * ceil(G / 16) >= 32 * Skv, and B * Hkv of those
                          >= 2^18) to repay its extra launches; otherwise ATOMIC          */
  SFA_DKV_ATOMIC = 1,  /* fp32 atomic adds (SFA.py:853) into a workspace accumulator;
                          float32 at d_qk = d_v = 64 or 128 into dk / dv themselves    */
  SFA_DKV_CSR = 2      /* deterministic: membership bitmap inverted into per-key-block
                          lists of referencing query blocks, key-major recompute, fixed-
                          order reduction (index rows that repeat a key take atomics for
                          the repeats); SFA_E_UNSUPPORTED outside the supported shapes
                          (the cost rules of AUTO do not apply).  dsink is reduced in a
                          fixed order in every mode                                     */
};

/* sfa_bwd_args.flags */
#define SFA_BWD_MERGE_KV 1  /* v is the first Dv dims of k's rows (v == k with k's strides, Dv <= Dqk),
                               the reference's single shared kv (SFA.py:88, 116): dk receives the
                               gradient of the shared rows, dK + dV on their first Dv dims, as
                               SFA.py:849-853 sums both into one buffer; dv is not written and may
                               be NULL.  The MLA shape (d_qk 576, d_v 512, 65..128 heads per KV head,
                               bf16) then runs its MFMA backward: AUTO and SFA_DKV_CSR sum per-slot
                               bf16 rows of the shared rows' gradient in a fixed order (Skv <= 65536;
                               slots repeating a key of their row take fp32 atomics), SFA_DKV_ATOMIC
                               adds every slot's fp32 row atomically                              */

/* sfa_fwd_args.flags (the backward ignores them) */
#define SFA_FWD_IDX_SORTED 1  /* every index row lists its valid keys in ascending order before any
                                 padding (what sfa_indexer_topk writes).  Without it the persistent
                                 MLA prefill (the MLA shape, no split-k, >= 4096 work items,
                                 top-k <= 2048, Skv <= 65536; contiguous or paged kv) and MLA prefills of
                                 >= 1024 queries with 8192 <= Skv <= 65536 and top-k <= 2048 (65..128
                                 heads: >= 1024; up to 32 heads: >= 512) first write their rows
                                 in that order into the workspace (valid keys ascending, then -1; a
                                 row that repeats a key is kept as it is) and walks those: the
                                 queries running together on an XCD then gather the same regions
                                 of the prefix at about the same time and share them in its L2.
                                 The result is the same softmax in another summation order
                                 (differences at fp32 rounding).  The flag only skips that pass   */

/* Error codes. */
enum {
  SFA_OK = 0,
  SFA_E_INVALID = -1,   /* bad shape / stride / dtype / null pointer (ValueError) */
  SFA_E_WORKSPACE = -2, /* workspace missing or too small                        */
  SFA_E_UNSUPPORTED = -3,
  SFA_E_HIP = -4        /* a HIP runtime call failed (RuntimeError)               */
};

typedef struct sfa_fwd_args {
  int32_t dtype;                 /* SFA_DTYPE_*                                       */
  int32_t B, Sq, Skv, Hq, Hkv, Dqk, Dv, topk;
  float scale;                   /* softmax scale; <= 0 means 1/sqrt(Dqk) (SFA.py:181-182) */
  const void* q;   int64_t q_sb, q_ss, q_sh;
  const void* k;   int64_t k_sb, k_ss, k_sh;
  const void* v;   int64_t v_sb, v_ss, v_sh;
  const int32_t* idx; int64_t i_sb, i_ss, i_sh;   /* slot stride is 1 */
  const int32_t* kv_lens;        /* [B] or NULL                                        */
  const float* sink;             /* [Hq] or NULL                                       */
  void* out;       int64_t o_sb, o_ss, o_sh;
  float* lse;      int64_t l_sb, l_ss, l_sh;      /* head stride of lse             */
  int32_t num_splits;            /* split-k over the top-k set; 0 = library choice      */
  int32_t flags;                 /* 0 or SFA_FWD_IDX_SORTED                             */
} sfa_fwd_args;

typedef struct sfa_bwd_args {
  sfa_fwd_args fwd;              /* the forward's arguments; out/lse are read here      */
  const void* dout; int64_t do_sb, do_ss, do_sh;
  void* dq;        int64_t dq_sb, dq_ss, dq_sh;
  void* dk;        int64_t dk_sb, dk_ss, dk_sh;
  void* dv;        int64_t dv_sb, dv_ss, dv_sh;
  const float* dlse;             /* gradient w.r.t. lse, float32, lse's strides; NULL = 0 */
  float* dsink;                  /* [Hq] float32, written (not accumulated); NULL if no sink */
  int32_t dkv_mode;              /* SFA_DKV_*                                           */
  int32_t flags;                 /* 0 or SFA_BWD_MERGE_KV                               */
} sfa_bwd_args;

/* Paged KV cache (block table) for sfa_fwd_paged.  k and v then point to
 * page pools [num_pages, page_size, Hkv, D]: k_sb / v_sb are the page strides,
 * k_ss / v_ss the row strides within a page, k_sh / v_sh the head strides.
 * Logical key position i of sequence b (what idx holds) is row
 * i % page_size of page block_table[b * bt_sb + i / page_size].
 * A slot is valid iff 0 <= idx < bound (bound = kv_lens[b] clamped to Skv,
 * else Skv; Skv <= max_pages * page_size) and its page id lies in
 * [0, num_pages); an unmapped page (e.g. -1) makes the slot invalid. */
typedef struct sfa_kv_pages {
  const int32_t* block_table;    /* [B, max_pages] int32 page ids                     */
  int64_t bt_sb;                 /* block-table row stride (elements); the table's
                                    extent, ((B - 1) * bt_sb + max_pages) * 4 bytes,
                                    must stay below 4 GiB                            */
  int32_t max_pages;             /* block-table columns                               */
  int32_t page_size;             /* rows per page, a power of two                     */
  int32_t num_pages;             /* pages in each pool; num_pages * page_size < 2^31  */
  int32_t flags;                 /* reserved, must be 0                               */
} sfa_kv_pages;

/* Top-k index producer (sfa_indexer_topk): creates the index rows sfa_fwd
 * consumes.  The reference takes them as an input (`topk_idxs`, "Sparse
 * indices mapping queries to KV blocks", SFA.py:88-90); the scores are those
 * of DeepSeek-V3.2's lightning indexer:
 *   I[b,t,s] = sum_h w[b,t,h] * max(0, <q[b,t,h,:], k[b,s,:]>)
 * Query t of sequence b may see keys s <= t + L_b - Sq (L_b = kv_lens[b]
 * clamped to Skv, else Skv): causal prefill when Sq = L_b, the whole context
 * for a single decode query.  Row idx[b,t,:] receives the min(topk, allowed)
 * allowed keys with the largest scores (equal scores: the lower key first),
 * in ascending key order, then -1 padding.
 * fp8 (SFA_DTYPE_FP8_E4M3) q / k, as DeepSeek-V3.2 stores them: the score is
 *   I[b,t,s] = k_scale[b,s] * sum_h w[b,t,h] * max(0, <q[b,t,h,:], k[b,s,:]>)
 * with positive per-token k scales (NULL = 1) and the q scales folded into w.
 * Supported: bf16 or fp8 q / k, D = 128, H in {32, 64, 128}, Skv <= 65536. */
typedef struct sfa_indexer_args {
  int32_t B, Sq, Skv, H, D, topk;
  int32_t dtype;                                  /* SFA_DTYPE_BF16 or SFA_DTYPE_FP8_E4M3      */
  const void* q;   int64_t q_sb, q_ss, q_sh;      /* [B, Sq, H, D], unit feature stride       */
  const void* k;   int64_t k_sb, k_ss;            /* [B, Skv, D], unit feature stride         */
  const float* k_scale; int64_t ks_sb;            /* fp8: [B, Skv] positive scales, or NULL   */
  const float* w;  int64_t w_sb, w_ss;            /* [B, Sq, H] float32, unit head stride     */
  const int32_t* kv_lens;                         /* [B] or NULL                              */
  int32_t* idx;    int64_t i_sb, i_ss;            /* [B, Sq, topk] int32 out, unit slot stride */
  float* logits;   int64_t g_sb, g_ss;            /* optional [B, Sq, Skv] float32 out (scores
                                                     of allowed keys; other entries unspecified;
                                                     16-byte aligned rows, g_ss % 4 == 0), or NULL */
  int32_t flags;                                  /* reserved, must be 0                       */
} sfa_indexer_args;

/* ---- rotary positions and per-head norms of q and k -----------------------
 * A row is one head of one token, x[D].  With n normed dims (the first n, 0:
 * none) and R rotated dims from rope_offset, frequencies inv_freq[R / 2]:
 *   u_d = x_d w_d / sqrt(mean_{d < n} x_d^2 + eps)  (d < n), else x_d
 *   y1 = s (u1 cos a - u2 sin a), y2 = s (u2 cos a + u1 sin a),
 *   a = position * inv_freq[i], s = rope_scale,
 * over the pairs (i, i + R/2) of the rotated dims, or (2i, 2i+1) when
 * interleaved.  float32 between load and store, angles reduced in float64.
 * The reference has neither step (its q and kv come ready made, SFA.py:86-94). */
typedef struct sfa_rope_args {
  int32_t dtype;                 /* SFA_DTYPE_F32 or SFA_DTYPE_BF16                   */
  int32_t B, S, D, Hq, Hkv, Dv;  /* Hkv = 0: no k; Dv: the appended v rows (0: none)  */
  int32_t rotary_dim, rope_offset, interleaved;
  int32_t q_norm, k_norm;        /* normed dims (0: no norm)                          */
  int32_t w_dtype;               /* of the weights and their gradients: float32 or dtype */
  int32_t pos_i64, slots_i64;    /* positions / slots are int64 (else int32)          */
  float eps, rope_scale;
  const void* positions; int64_t p_sb, p_ss;       /* [B, S]                          */
  const double* inv_freq;                          /* [rotary_dim / 2]                */
  const void* q;  int64_t q_sb, q_ss, q_sh;        /* [B, S, Hq, D]                   */
  const void* k;  int64_t k_sb, k_ss, k_sh;        /* [B, S, Hkv, D]                  */
  const void* q_weight;  const void* k_weight;     /* [q_norm], [k_norm]              */
  /* forward: written (each may be its input); backward: the gradients of the
   * results, read.  append: k_out is the page pool [num_pages, page_size, Hkv, D]
   * with page, row and head strides                                                 */
  void* q_out;    int64_t qo_sb, qo_ss, qo_sh;
  void* k_out;    int64_t ko_sb, ko_ss, ko_sh;
  const void* v;  int64_t v_sb, v_ss, v_sh;        /* append: [B, S, Hkv, Dv] or NULL */
  void* v_out;    int64_t vo_sb, vo_ss, vo_sh;     /* append: the pool of the v rows  */
  const void* slots; int64_t s_sb, s_ss;           /* append: [B, S] logical cache rows;
                                                      one outside the table or on an
                                                      unmapped page is not written    */
  void* dq;       int64_t dq_sb, dq_ss, dq_sh;     /* backward                        */
  void* dk;       int64_t dk_sb, dk_ss, dk_sh;
  void* dq_weight; void* dk_weight;                /* backward: [q_norm], [k_norm]    */
  int32_t flags;                                   /* reserved, must be 0             */
} sfa_rope_args;

/* ---- attention of a tree of drafted tokens over a paged cache --------------
 * Token t of sequence b sees the cache's rows [0, ctx_lens[b]) and the drafted
 * rows ctx_lens[b] + j, j < tree_lens[b], with bit j of tree_mask[b, t] set.  Rows of
 * unmapped pages are not seen.  A token t >= tree_lens[b] gives out = 0 and
 * lse = -inf, as does one that sees nothing (with a sink its lse is the sink). */
typedef struct sfa_tree_args {
  int32_t dtype;
  int32_t B, T, Hq, Hkv, Dqk, Dv;                  /* T <= 64, head dims <= 1024      */
  float scale;                                     /* > 0                             */
  const void* q;  int64_t q_sb, q_ss, q_sh;        /* [B, T, Hq, Dqk]                 */
  const void* k;  int64_t k_sb, k_ss, k_sh;        /* pools: page, row, head strides  */
  const void* v;  int64_t v_sb, v_ss, v_sh;        /* (v may be the first Dv dims of k) */
  const int32_t* ctx_lens;                         /* [B]                             */
  const int64_t* tree_mask; int64_t tm_sb, tm_ss;  /* [B, T]                          */
  const int32_t* tree_lens;                        /* [B] or NULL: T                  */
  const float* sink;                               /* [Hq] or NULL                    */
  void* out;      int64_t o_sb, o_ss, o_sh;        /* [B, T, Hq, Dv]                  */
  float* lse;     int64_t l_sb, l_ss, l_sh;        /* [B, T, Hq]                      */
  int32_t flags;                                   /* reserved, must be 0             */
} sfa_tree_args;

/* ---- dense attention: a chunk of new tokens over a paged cache, or a sequence --
 * Token t < lens[b] of sequence b stands at row pos = ctx_lens[b] + t and sees the
 * rows j <= pos with j < first or pos - j < window (window 0: all of them); rows of
 * unmapped pages, and rows past the table, are not seen.  With pages the k and v
 * rows are the cache's (the chunk's own among them), else k and v are [B, S, Hkv, D]
 * and ctx_lens NULL.  A token t >= lens[b] gives out = 0 and lse = -inf, as does
 * one that sees nothing (with a sink its lse is the sink).
 * kv_dtype: dtype, or with pages SFA_DTYPE_FP8_E4M3: a row of a head stands for its
 * e4m3 values times 2^(e - 127), e its exponent byte in k_scale / v_scale
 * [num_pages, page_size, Hkv] (255: NaN). */
typedef struct sfa_dense_args {
  int32_t dtype, kv_dtype;
  int32_t B, S, Hq, Hkv, Dqk, Dv;                  /* head dims <= 1024               */
  int32_t window, first;
  float scale;                                     /* > 0                             */
  const void* q;  int64_t q_sb, q_ss, q_sh;        /* [B, S, Hq, Dqk]                 */
  const void* k;  int64_t k_sb, k_ss, k_sh;        /* pools: page, row, head strides  */
  const void* v;  int64_t v_sb, v_ss, v_sh;        /* (v may be the first Dv dims of k) */
  const uint8_t* k_scale; int64_t ks_sb, ks_ss, ks_sh;
  const uint8_t* v_scale; int64_t vs_sb, vs_ss, vs_sh;
  const int32_t* ctx_lens;                         /* [B], or NULL: 0                 */
  const int32_t* lens;                             /* [B], or NULL: S                 */
  const float* sink;                               /* [Hq] or NULL                    */
  void* out;      int64_t o_sb, o_ss, o_sh;        /* [B, S, Hq, Dv]                  */
  float* lse;     int64_t l_sb, l_ss, l_sh;        /* [B, S, Hq]                      */
  int32_t flags;                                   /* reserved, must be 0             */
} sfa_dense_args;
/* Its backward, without pages: out and lse as the forward left them. */
typedef struct sfa_dense_bwd_args {
  sfa_dense_args fwd;
  const void* dout; int64_t do_sb, do_ss, do_sh;
  void* dq;       int64_t dq_sb, dq_ss, dq_sh;
  void* dk;       int64_t dk_sb, dk_ss, dk_sh;
  void* dv;       int64_t dv_sb, dv_ss, dv_sh;
  const float* dlse;                               /* lse's strides, or NULL          */
  float* dsink;                                    /* [Hq], or NULL                   */
  int32_t flags;                                   /* reserved, must be 0             */
} sfa_dense_bwd_args;

/* Exponent bytes of the pools that sfa_rope_append_fp8 writes, with page, row and
 * head strides. */
typedef struct sfa_kv_scales {
  uint8_t* k; int64_t k_sb, k_ss, k_sh;
  uint8_t* v; int64_t v_sb, v_ss, v_sh;            /* NULL without v rows             */
} sfa_kv_scales;

/* Rows of a paged cache, in order: out[b, i] is row starts[b] + i of sequence b, zeros
 * where that is negative, at or past lens[b], or on an unmapped page. */
typedef struct sfa_cache_read_args {
  int32_t dtype, cache_dtype;                      /* of out; of the pool: F32, BF16 or FP8_E4M3 */
  int32_t B, N, H, D;
  const void* cache; int64_t c_sb, c_ss, c_sh;     /* [num_pages, page_size, H, D]    */
  const uint8_t* scale; int64_t s_sb, s_ss, s_sh;  /* FP8_E4M3: exponent bytes        */
  const int32_t* starts;                           /* [B], or NULL: 0                 */
  const int32_t* lens;                             /* [B]                             */
  void* out; int64_t o_sb, o_ss, o_sh;             /* [B, N, H, D]                    */
  int32_t flags;                                   /* reserved, must be 0             */
} sfa_cache_read_args;

/* ---- pages of a cache -------------------------------------------------------
 * block_table [B, max_pages] as in sfa_kv_pages (-1: none), ref_counts
 * [num_pages] the number of entries that map a page: a page is free iff its
 * count is 0, and the pages a call takes are the lowest free ones.  A pool is
 * [num_pages, page_size, ...] with each page contiguous.                      */
typedef struct sfa_cache_pool {
  void* base;
  int64_t page_stride, page_bytes;  /* bytes */
} sfa_cache_pool;
typedef struct sfa_cache {
  const sfa_cache_pool* pools;      /* host array                                     */
  int32_t npools;
  int32_t B, max_pages, page_size, num_pages;
  int32_t flags;                    /* reserved, must be 0                            */
  int32_t* block_table; int64_t bt_sb;
  int32_t* ref_counts;
  int32_t* kv_lens;                 /* [B]                                            */
} sfa_cache;

/* Library ABI version (SFA_ABI_VERSION of the build). */
SFA_API int sfa_abi_version(void);

/* Message describing the last failure on the calling thread ("" if none). */
SFA_API const char* sfa_last_error(void);

/* Bytes of device workspace sfa_fwd needs for `a` (0 when none).
 * Replaces the per-launch workspaces of SFA.py:117-120; what remains: the
 * split-k partial results of the decode shape, and for the persistent MLA
 * prefill (>= 4096 work items) 256 bytes of work-claim counters; for MLA
 * prefills that walk ascending rows, unless SFA_FWD_IDX_SORTED is set, those
 * rows (B * Sq * Hkv * topk int32). */
SFA_API size_t sfa_fwd_workspace_size(const sfa_fwd_args* a);

/* Forward: out = softmax(scale * q k[idx]^T) v[idx], lse = log-sum-exp.
 * Replaces `_attn_fwd` (SFA.py:483-587 via SFA.py:122-159). */
SFA_API int sfa_fwd(const sfa_fwd_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Size of the static per-GPU scratch of sfa_fwd_noalloc (64 MiB). */
#define SFA_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* Forward that allocates nothing and takes no workspace: the same arguments,
 * kernels and results as sfa_fwd.  No counterpart in the reference; it is for
 * callers that cannot allocate device memory (code under HIP-graph capture,
 * tight serving loops, harnesses that forbid hipMalloc).  The workspace of
 * sfa_fwd (sfa_fwd_workspace_size(a) bytes: decode split-k partials, prefill
 * claim counters and sorted index rows) goes to a static device
 * buffer of SFA_NOALLOC_SCRATCH_BYTES that every GPU the library runs on holds
 * until the process ends; a plan that needs more returns SFA_E_WORKSPACE
 * before any device work, with two exceptions.  The kernel for up to 64 heads
 * (and for up to 4 queries of up to 128 with 16384 index slots in all) on MLA
 * rows is split no further than its fp32 partials fit.  The prefill's sorted index rows: when they do not
 * fit, the rows are walked in their own order (the result then equals
 * sfa_fwd's with SFA_FWD_IDX_SORTED set; bitwise equal to sfa_fwd whenever the
 * sorted rows fit or the rows are already ascending).  `stream` must belong to
 * the current device; the first call on a device resolves the buffer's
 * address (make it before any graph capture).  All calls on one GPU share the
 * buffer: calls that may overlap on one GPU (unordered streams) race. */
SFA_API int sfa_fwd_noalloc(const sfa_fwd_args* a, void* stream);

/* Bytes of device workspace sfa_fwd_paged needs for `a` and `pages`. */
SFA_API size_t sfa_fwd_paged_workspace_size(const sfa_fwd_args* a, const sfa_kv_pages* pages);

/* Forward over a paged KV cache: the same result as sfa_fwd on the contiguous
 * cache the block table describes.  The reference has no paged variant (its
 * `_attn_fwd`, SFA.py:483-587, reads one contiguous [S_kv, B, D] kv tensor);
 * this is the serving-side layout of the decode step that precedes it. */
SFA_API int sfa_fwd_paged(const sfa_fwd_args* a, const sfa_kv_pages* pages, void* workspace,
                          size_t workspace_bytes, void* stream);

/* Bytes of device workspace sfa_indexer_topk needs: the fp32 scores of a
 * chunk of queries unless `logits` is given (about 1 GiB, less when all Sq
 * rows take less, more when one block of 512 / H queries of all B sequences
 * takes more), then, when a launch holds few long rows (B x queries < 256,
 * Skv >= 16384: a decode step), the candidate lists of its two-phase
 * selection (8 bytes per candidate, topk rounded up to 4 per segment, at
 * most 8 segments per row).  May be 0. */
SFA_API size_t sfa_indexer_topk_workspace_size(const sfa_indexer_args* a);

/* Scores and top-k selection (no counterpart kernel in the reference, which
 * consumes the result: SFA.py:88-90). */
SFA_API int sfa_indexer_topk(const sfa_indexer_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Bytes of device workspace sfa_bwd needs for `a` (fp32 dK/dV accumulators,
 * delta, the CSR arrays in SFA_DKV_CSR mode).  The MLA backward
 * (SFA_BWD_MERGE_KV at its shape) needs fp32 accumulators of the shared rows
 * (B * Skv * Hkv * Dqk * 4 bytes), delta (B * Sq * Hq * 4 bytes) and one
 * chunk of queries: per query the bf16 P / dS of its slots (about 1 MiB at
 * top-k 2048, G = 128) and, in the deterministic mode, its per-slot bf16
 * gradient rows (top-k * Dqk * 2 bytes) and index maps; a chunk stays within
 * 3.5 GiB in the deterministic mode and 2 GiB with atomics (whole rounds of
 * 256 queries when that many fit, at most 1024 in the deterministic mode,
 * else multiples of 8, at least 8 queries).  The deterministic mode holds
 * the gradient rows and index maps twice (one chunk's reduction reads one
 * set while the next chunk fills the other), so the total is about 5.5 GiB
 * (2 GiB with atomics) plus the accumulators at the full-size shapes.
 * Replaces the workspaces of SFA.py:184-194 and SFA.py:253-261. */
SFA_API size_t sfa_bwd_workspace_size(const sfa_bwd_args* a);

/* Backward: dq, dk, dv (and dsink if requested) from dout, out and lse.
 * Replaces `_attn_bwd_dq_dsink` (SFA.py:856-1002 via SFA.py:199-251) and
 * `_attn_bwd_dk_dv` (SFA.py:1005-1145 via SFA.py:266-298).  dq/dk/dv are
 * fully overwritten (no accumulation into existing contents).  The
 * deterministic MLA backward also enqueues its ordered reductions on a
 * second stream of the device `stream` belongs to (the current device for
 * the null stream), which the library creates on its first such call there
 * (default priority, non-blocking, kept until the process ends) and orders
 * against `stream` with events: when the call returns,
 * `stream` waits for all of that work, and under HIP-graph capture the
 * second stream joins the capture and is joined back.  Such calls on one
 * device enqueue one at a time (a mutex). */
SFA_API int sfa_bwd(const sfa_bwd_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Rotation and norms: q_out and k_out from q and k.  With pages (append) the k
 * rows, and the v rows unchanged, go to the cache rows that `slots` names;
 * pages NULL: k_out is a tensor like k.  Two tokens of a call with the same
 * cache row leave one of them there, which is not specified. */
SFA_API int sfa_rope_fwd(const sfa_rope_args* a, const sfa_kv_pages* pages, void* stream);

/* sfa_rope_fwd with pages whose pools hold e4m3 bytes: the k rows (normed and turned,
 * float32) and the v rows of a's type are quantised as they are written.  Each row
 * of a head is divided by the smallest power of two 2^(e - 127), 16 <= e, that
 * brings its largest finite magnitude to 448 or less, and rounded to the nearest
 * e4m3 value; infinities and NaN become NaN.  k_out / v_out and scales: bytes. */
SFA_API int sfa_rope_append_fp8(const sfa_rope_args* a, const sfa_kv_pages* pages, const sfa_kv_scales* scales,
                                void* stream);

/* dq, dk and the weights' gradients (summed in a fixed order) from the results'
 * gradients in q_out / k_out.  Workspace: 8 KiB per workgroup, up to 8 MiB, with
 * a norm; 0 without. */
SFA_API size_t sfa_rope_bwd_workspace_size(const sfa_rope_args* a);
SFA_API int sfa_rope_bwd(const sfa_rope_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Attention of a drafted tree.  Workspace: float32 partials where the keys are
 * cut into ranges (few query rows on long tables). */
SFA_API size_t sfa_tree_fwd_workspace_size(const sfa_tree_args* a, const sfa_kv_pages* pages);
SFA_API int sfa_tree_fwd(const sfa_tree_args* a, const sfa_kv_pages* pages, void* workspace, size_t workspace_bytes,
                         void* stream);

/* Dense attention.  Workspace: float32 partials where the keys of few query rows are
 * cut into ranges.  pages NULL: contiguous k and v. */
SFA_API size_t sfa_dense_fwd_workspace_size(const sfa_dense_args* a, const sfa_kv_pages* pages);
SFA_API int sfa_dense_fwd(const sfa_dense_args* a, const sfa_kv_pages* pages, void* workspace, size_t workspace_bytes,
                          void* stream);

/* Its gradients (every sum in a fixed order).  Workspace: two floats a query row (three
 * with more than 128 dims), and float32 partials of key blocks that many rows see. */
SFA_API size_t sfa_dense_bwd_workspace_size(const sfa_dense_bwd_args* a);
SFA_API int sfa_dense_bwd(const sfa_dense_bwd_args* a, void* workspace, size_t workspace_bytes, void* stream);

/* Rows of a paged cache as contiguous ones of a's dtype. */
SFA_API int sfa_cache_read(const sfa_cache_read_args* a, const sfa_kv_pages* pages, void* stream);

/* Workspace of the sfa_cache_* calls on n pairs (or sequences). */
SFA_API size_t sfa_cache_workspace_size(const sfa_cache* c, int32_t n);

/* Page src[i] to page dst[i] in every pool.  A pair is left out if a page is
 * outside the pool, if a later pair has its destination, or if its
 * destination is the source of another pair. */
SFA_API int sfa_cache_copy(const sfa_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* workspace,
                           size_t workspace_bytes, void* stream);

/* Row children[i] of the table becomes a fork of row parents[i]: its whole
 * pages are shared (counts raised), the rows of its last page, filled in part,
 * are copied to a free page in every pool; kv_lens[child] = kv_lens[parent].
 * ok[i] = 0 and nothing is written for a pair with a row outside the table,
 * whose child an earlier pair has or any pair has as parent, or that finds no
 * free page.  The child's own pages are not freed (sfa_cache_free first). */
SFA_API int sfa_cache_fork(const sfa_cache* c, const int32_t* parents, const int32_t* children, int32_t n, int32_t* ok,
                           void* workspace, size_t workspace_bytes, void* stream);

/* The entries of rows[i] past the pages of its first keep_lens[i] rows (NULL:
 * all) become -1 and their pages lose a reference. */
SFA_API int sfa_cache_free(const sfa_cache* c, const int32_t* rows, const int32_t* keep_lens, int32_t n, void* stream);

/* Free pages for rows kv_lens[b] .. new_lens[b] - 1 of every sequence where none
 * is mapped: all of a sequence's or none (ok[b] = 0), in order of b while they
 * last (a sequence that needs none is always ok).  kv_lens is not changed. */
SFA_API int sfa_cache_extend(const sfa_cache* c, const int32_t* new_lens, int32_t* ok, void* workspace,
                             size_t workspace_bytes, void* stream);

/* The pages in use moved to the low end of every pool, the table and counts
 * with them; used[0]: how many there are. */
SFA_API int sfa_cache_compact(const sfa_cache* c, int32_t* used, void* workspace, size_t workspace_bytes, void* stream);

/* Row ctx_lens[b] + i becomes what row ctx_lens[b] + path[b, i] was, i < plen <= 64;
 * negative entries leave theirs. */
SFA_API int sfa_cache_keep_path(const sfa_cache* c, const int32_t* ctx_lens, const int32_t* path, int64_t path_sb,
                                int32_t plen, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SFA_H_ */

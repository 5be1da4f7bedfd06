// gfx950 attention of a tree of drafted tokens over a paged cache.
//
// Token t < tree_lens[b] of sequence b sees the cache's rows [0, ctx_b) and
// those drafted rows ctx_b + j, j < tree_lens[b], whose bit j of tree_mask[b][t]
// is set.  out = sum_s softmax_s(scale q.k_s) v_s, lse its log-sum-exp; a sink
// adds exp(sink[h]) to the denominator.  Rows of unmapped pages are not seen;
// a row that sees nothing gives zeros and -inf (with a sink: the sink), a
// token past tree_lens[b] zeros and -inf.
//
// The rows of a (sequence, kv head) are r = t G + h, h < G = Hq / Hkv: its
// keys serve T G query rows.  Work is split over row blocks and over key ranges
// ("slots") of one length for the whole batch, so that ragged contexts give
// even work; the ranges are found on the device from ctx_lens.  A sequence
// of several slots leaves float32 partials that tree_combine_kernel joins.

#include "sfa_lds.h"
#include "sfa_mfma.h"
#include "sfa_ops.h"

namespace sfa {
namespace {

// Base-2 log-sum-exp of 2^m2 l (the logarithm of l's mantissa: its own whole
// part would round the sum once more).
__device__ __forceinline__ float lse2_of(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return m2 + ((float)e + log2f(f));
}
__device__ __forceinline__ float lse_of(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return fmaf(m2, kLn2, fmaf((float)e, kLn2, logf(f)));
}

struct SeqLens {
  int ctx, nodes, keys;  // keys = ctx + nodes, all clamped to the table
};
__device__ __forceinline__ SeqLens seq_lens(const TreeParams& p, int b) {
  SeqLens s;
  s.ctx = min(max(p.ctx_lens[b], 0), p.cap);
  s.nodes = p.tree_lens != nullptr ? min(max(p.tree_lens[b], 0), p.T) : p.T;
  s.keys = (int)min((int64_t)s.ctx + s.nodes, (int64_t)p.cap);
  return s;
}

// A key range of the batch.
struct Slot {
  int b;           // sequence, or -1: none
  int k0, k1;      // its keys
  int first, n;    // the sequence's first slot and how many it has
};
// Length of the ranges, and the sequence of a slot (or the slots of sequence
// `slot` when BY_SEQ).  By one wave; every wave of a workgroup gets the same.
template <bool BY_SEQ>
__device__ Slot find_slot(const TreeParams& p, int slot) {
  const int lane = threadIdx.x & 63;
  int len = 0x7fffffff;  // want = 0: one slot a sequence
  if (p.want > 0) {
    int64_t sum = 0;
    for (int b = lane; b < p.B; b += 64) sum += seq_lens(p, b).keys;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const int64_t l = (sum + p.want - 1) / p.want;
    len = l < p.min_len ? p.min_len : (int)((l + p.tile - 1) / p.tile) * p.tile;
  }
  int before = 0;
  Slot s{-1, 0, 0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const int keys = b < p.B ? seq_lens(p, b).keys : 0;
    int n = b < p.B ? max(1, (int)(((int64_t)keys + len - 1) / len)) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const int first = before + incl - n;
    const bool mine = BY_SEQ ? b == slot : slot >= first && slot < first + n;
    const uint64_t hit = __ballot(mine);
    if (hit != 0) {
      const int w = __builtin_ctzll(hit);
      s.b = b0 + w;
      s.first = __shfl(first, w, 64);
      s.n = __shfl(n, w, 64);
      const int kk = __shfl(keys, w, 64), i = BY_SEQ ? 0 : slot - s.first;
      s.k0 = (int)min((int64_t)i * len, (int64_t)kk);
      s.k1 = (int)min((int64_t)s.k0 + len, (int64_t)kk);
      return s;
    }
    before += __shfl(incl, 63, 64);
  }
  return s;
}

// Element offset of key s of sequence b in a pool of these strides, or -1.
__device__ __forceinline__ int64_t key_row(const TreeParams& p, int b, int s, int64_t page_stride, int64_t row_stride) {
  const int pg = p.block_table[b * p.bt_sb + (s >> p.page_shift)];
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * page_stride + (int64_t)(s & ((1 << p.page_shift) - 1)) * row_stride;
}

// ---- any head dims up to 1024, bf16 or float32: float32 products --------------
constexpr int kGR = 8;     // rows per workgroup
constexpr int kGK = 64;    // keys per tile
constexpr int kGD = 1024;  // largest head dim

// The rows row0 .. row0 + kGR - 1 of (b, g) over keys [k0, k1), by a workgroup of
// 256 threads; emit(i, d, o, l) gets the unnormalised sums and fin(i, m, l) the
// row's maximum (base 2) and sum.
struct GenericScratch {
  float q[kGR][kGD];
  float s[kGR][kGK + 1];
  int64_t krow[kGK], vrow[kGK];
  uint64_t mask[kGR];
  float m[kGR], l[kGR], a[kGR];
};
template <typename T, class Emit, class Fin>
__device__ void generic_rows(const TreeParams& p, int b, int g, int row0, int k0, int k1, GenericScratch& sc, Emit emit,
                             Fin fin) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SeqLens sl = seq_lens(p, b);
  const int R = p.T * p.G;
  for (int i = 0; i < kGR; ++i) {
    const int r = row0 + i;
    const int t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R && t < sl.nodes;
    for (int d = tid; d < p.Dqk; d += 256)
      sc.q[i][d] = live ? to_f32(reinterpret_cast<const T*>(p.q)[b * p.q_sb + t * p.q_ss + h * p.q_sh + d]) : 0.f;
    if (tid == 0) {
      sc.mask[i] = live ? (uint64_t)p.tree_mask[b * p.tm_sb + t * p.tm_ss] : 0;
      sc.m[i] = kNegInf;
      sc.l[i] = 0.f;
    }
  }
  float acc[kGD / 256][kGR];
#pragma unroll
  for (int c = 0; c < kGD / 256; ++c)
#pragma unroll
    for (int i = 0; i < kGR; ++i) acc[c][i] = 0.f;

  for (int j0 = k0; j0 < k1; j0 += kGK) {
    __syncthreads();
    if (tid < kGK) {
      const int s = j0 + tid;
      sc.krow[tid] = s < k1 ? key_row(p, b, s, p.k_sb, p.k_ss) : -1;
      sc.vrow[tid] = s < k1 ? key_row(p, b, s, p.v_sb, p.v_ss) : -1;
    }
    __syncthreads();
    {  // scores: 4 threads a key
      const int key = tid >> 2, part = tid & 3;
      const int64_t ko = sc.krow[key];
      float s[kGR];
#pragma unroll
      for (int i = 0; i < kGR; ++i) s[i] = 0.f;
      if (ko >= 0) {
        const T* kr = reinterpret_cast<const T*>(p.k) + ko + g * p.k_sh;
        for (int d = part; d < p.Dqk; d += 4) {
          const float x = to_f32(kr[d]);
#pragma unroll
          for (int i = 0; i < kGR; ++i) s[i] = fmaf(sc.q[i][d], x, s[i]);
        }
      }
      const int node = j0 + key - sl.ctx;
#pragma unroll
      for (int i = 0; i < kGR; ++i) {
        s[i] += __shfl_xor(s[i], 1, 64);
        s[i] += __shfl_xor(s[i], 2, 64);
        const bool seen = ko >= 0 && (node < 0 || ((sc.mask[i] >> node) & 1));
        if (part == 0) sc.s[i][key] = seen ? s[i] * p.scale_log2 : kNegInf;
      }
    }
    __syncthreads();
    for (int i = wave; i < kGR; i += 4) {  // softmax: a wave a row
      const float s = sc.s[i][lane], m0 = sc.m[i];
      const float m = fmaxf(m0, wave_max(s));
      const float e = s == kNegInf ? 0.f : exp2f(s - m);
      const float sum = wave_sum(e);
      sc.s[i][lane] = e;
      if (lane == 0) {
        const float a = m0 == kNegInf ? 0.f : exp2f(m0 - m);
        sc.a[i] = a;
        sc.m[i] = m;
        sc.l[i] = sc.l[i] * a + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kGD / 256; ++c) {
      const int d = tid + 256 * c;
      if (d >= p.Dv) break;
#pragma unroll
      for (int i = 0; i < kGR; ++i) acc[c][i] *= sc.a[i];
      for (int key = 0; key < kGK; ++key) {
        const int64_t vo = sc.vrow[key];
        if (vo < 0) continue;
        const float x = to_f32(reinterpret_cast<const T*>(p.v)[vo + g * p.v_sh + d]);
#pragma unroll
        for (int i = 0; i < kGR; ++i) {
          const float e = sc.s[i][key];
          if (e != 0.f) acc[c][i] = fmaf(e, x, acc[c][i]);  // (an unseen row's infinities stay out)
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGR; ++i) {
    if (row0 + i >= R) break;
    if (tid == 0) fin(i, sc.m[i], sc.l[i]);
#pragma unroll
    for (int c = 0; c < kGD / 256; ++c) {
      const int d = tid + 256 * c;
      if (d < p.Dv) emit(i, d, acc[c][i], sc.m[i], sc.l[i]);
    }
  }
}

// Row r of (b, g): where its results go.
struct RowOut {
  int t, h, r;  // r: row of the sequence's partials
};
__device__ __forceinline__ RowOut row_out(const TreeParams& p, int g, int r) {
  RowOut o;
  o.t = r / p.G;
  o.h = g * p.G + r % p.G;
  o.r = o.t * p.Hq + o.h;
  return o;
}

// The factor and LSE of a finished row with maximum m (base 2) and sum l.
__device__ __forceinline__ float finish_row(const TreeParams& p, int h, bool live, float m, float l, float& lse) {
  if (!live) {
    lse = kNegInf;
    return 0.f;
  }
  if (l == 0.f) {  // nothing seen
    lse = p.sink ? p.sink[h] : kNegInf;
    return 0.f;
  }
  const float sink2 = p.sink ? p.sink[h] * kLog2e : kNegInf;
  const float mm = fmaxf(m, sink2);
  const float f = m == kNegInf ? 0.f : exp2f(m - mm);
  float x = l * f;
  if (p.sink && mm != kNegInf) x += exp2f(sink2 - mm);
  lse = x > 0.f ? lse_of(mm, x) : x == 0.f ? kNegInf : x;
  return x > 0.f ? f / x : x == 0.f ? 0.f : x;
}

template <typename T>
__global__ __launch_bounds__(256) void tree_generic_kernel(TreeParams p) {
  __shared__ GenericScratch sc;
  int wi = blockIdx.x;
  const int rb = wi % p.nrb;
  wi /= p.nrb;
  const int g = wi % p.Hkv, slot = wi / p.Hkv;
  const Slot sl = find_slot<false>(p, slot);
  if (sl.b < 0) return;
  const int b = sl.b, nodes = seq_lens(p, b).nodes;
  const int64_t pr = (int64_t)slot * p.T * p.Hq;
  const bool partial = sl.n > 1;
  generic_rows<T>(
      p, b, g, rb * kGR, sl.k0, sl.k1, sc,
      [&](int i, int d, float o, float m, float l) {
        const RowOut ro = row_out(p, g, rb * kGR + i);
        if (partial) {
          p.part_o[(pr + ro.r) * p.Dv + d] = l > 0.f ? o / l : l == 0.f ? 0.f : l;
        } else {
          float lse;
          const float f = finish_row(p, ro.h, ro.t < nodes, m, l, lse);
          reinterpret_cast<T*>(p.out)[b * p.o_sb + ro.t * p.o_ss + ro.h * p.o_sh + d] = from_f32<T>(f == 0.f ? 0.f : o * f);
        }
      },
      [&](int i, float m, float l) {
        const RowOut ro = row_out(p, g, rb * kGR + i);
        if (partial) {
          p.part_lse[pr + ro.r] = l > 0.f ? lse2_of(m, l) : l == 0.f ? kNegInf : l;
        } else {
          float lse;
          finish_row(p, ro.h, ro.t < nodes, m, l, lse);
          p.lse[b * p.l_sb + ro.t * p.l_ss + ro.h * p.l_sh] = lse;
        }
      });
}

// ---- joining the slots of a sequence -------------------------------------------
// One wave a row; a slot in which the row sees nothing has LSE -inf.
template <typename T>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), per = (int64_t)p.T * p.Hq;
  if (row >= p.B * per) return;
  const int b = (int)(row / per), r = (int)(row % per), h = r % p.Hq, t = r / p.Hq;
  const Slot sl = find_slot<true>(p, b);
  if (sl.n <= 1) return;
  const float* pl = p.part_lse + sl.first * per + r;
  const float* po = p.part_o + (sl.first * per + r) * p.Dv;
  const bool live = t < seq_lens(p, b).nodes;
  float m = kNegInf;
  bool bad = false;
  for (int i = lane; i < sl.n; i += 64) {
    const float x = pl[i * per];
    bad |= x != x;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  bad = __any(bad);
  float l = 0.f;
  for (int i = lane; i < sl.n; i += 64) {
    const float x = pl[i * per];
    if (x != kNegInf) l += exp2f(x - m);
  }
  l = wave_sum(l);
  if (bad) l = __builtin_nanf("");
  float lse;
  const float f = finish_row(p, h, live, m, l, lse);
  if (lane == 0) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
  T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh;
  for (int d = lane; d < p.Dv; d += 64) {
    float x = 0.f;
    if (f != 0.f)
      for (int i = 0; i < sl.n; ++i) {
        const float e = pl[i * per];
        if (e != kNegInf) x = fmaf(exp2f(e - m), po[i * per * p.Dv + d], x);
      }
    o[d] = from_f32<T>(f == 0.f ? 0.f : x * f);
  }
}

constexpr int kWorkgroups = 1024;  // key ranges are cut until about so many workgroups are in flight

}  // namespace

TreePlan tree_plan(const TreeParams& p, int dtype, bool vec) {
  TreePlan pl{};
  pl.rows = kGR;
  const int64_t nrb = ((int64_t)p.T * p.G + pl.rows - 1) / pl.rows;
  int64_t want = kWorkgroups / (p.Hkv * nrb);
  const int64_t most = ((int64_t)p.cap + 4 * kGK - 1) / (4 * kGK) * p.B;  // at least 4 tiles a slot
  if (want > most) want = most;
  pl.want = want > p.B ? (int)want : 0;
  pl.slots = p.B + pl.want;
  if (pl.want > 0) {
    const size_t rows = (size_t)pl.slots * p.T * p.Hq;
    pl.part_o_bytes = (rows * p.Dv * sizeof(float) + 255) / 256 * 256;
    pl.part_lse_bytes = (rows * sizeof(float) + 255) / 256 * 256;
  }
  return pl;
}

hipError_t launch_tree(const TreeParams& p0, const TreePlan& pl, int dtype, hipStream_t s) {
  TreeParams p = p0;
  p.want = pl.want;
  p.tile = kGK;
  p.min_len = 4 * kGK;
  p.nrb = (p.T * p.G + pl.rows - 1) / pl.rows;
  const unsigned grid = (unsigned)((int64_t)pl.slots * p.Hkv * p.nrb);
  if (dtype == SFA_DTYPE_F32) tree_generic_kernel<float><<<grid, 256, 0, s>>>(p);
  else tree_generic_kernel<bf16><<<grid, 256, 0, s>>>(p);
  if (pl.want > 0) {
    const unsigned cg = (unsigned)(((int64_t)p.B * p.T * p.Hq + 3) / 4);
    if (dtype == SFA_DTYPE_F32) tree_combine_kernel<float><<<cg, 256, 0, s>>>(p);
    else tree_combine_kernel<bf16><<<cg, 256, 0, s>>>(p);
  }
  return hipGetLastError();
}

}  // namespace sfa

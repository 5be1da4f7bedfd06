// gfx950 dense attention through a window (sfa_dense.h), any head dims from 129 up to 1024,
// bf16, float32 or 8-bit pages: every product in float32 on the matrix cores.
//
//   s_ij = scale q_i.k_j,  p = softmax over the rows that i sees,  o_i = sum_j p_ij v_j
//   backward: delta_i = o_i.do_i - dlse_i,  ds_ij = p_ij (do_i.v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Each kernel has columns, 16 a wave (query rows; for dk and dv: keys), and walks over
// entries, 32 at a time (keys; for dk and dv: query rows), whose rows pass through LDS
// as float32, 64 dims at a time.  A score product (16 entries x 16 columns, 16x16x4)
// leaves a lane with 4 entries of one column, which are the second operand of the
// sums' product as they are, its first being the staged rows read down a dim.  A workgroup
// makes 128 dims of its result: wider heads take several, which make the scores again.
// Bound: the float32 matrix rate (153 TFLOP/s), with all rows staged twice or more, each time
// between two barriers that wait for its loads: 16 TFLOP/s over latent rows (512 tokens behind
// 14336, 16 heads: 15.7 ms).

#include "sfa_dense_f32.h"

namespace sfa {
namespace {

constexpr int kC = 64;              // dims staged at a time
constexpr int kPitch = kC + 4;      // (floats; 4 rows apart, the lanes' groups meet different banks)
static_assert(kAnyDims == 2 * kC, "two halves of a workgroup's dims");

// The entries of a tile: element offsets of their rows in two tensors (-1: none)
// and the rows' scales.
struct Entries {
  float t[kE][kPitch];
  int64_t off[2][kE];
  float sc[2][kE];
  float lse[kE], delta[kE];
  int pos[kE];
  uint32_t bad;
};

// 64 dims from c0 of the entries' rows.  SAFE: infinities and NaN are noted as
// bits of e.bad and left out (0 times them would reach columns that do not see them).
template <bool SAFE, typename T>
__device__ __forceinline__ void stage(Entries& e, const T* base, int which, int c0, int D, bool vec) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < kE * kC / 4 / 256; ++i) {
    const int u = tid + 256 * i, row = u / (kC / 4), d = 4 * (u % (kC / 4));
    const int64_t off = e.off[which][row];
    f32x4 x = {};
    if (off >= 0) x = load4(base + off, c0 + d, D, vec);
    if constexpr (sizeof(T) == 1) x = x * e.sc[which][row];
    if constexpr (SAFE) {
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= !(fabsf(x[k]) <= 3.402823466e38f);
      if (bad) {
        atomicOr(&e.bad, 1u << row);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = fabsf(x[k]) <= 3.402823466e38f ? x[k] : 0.f;
      }
    }
    *reinterpret_cast<f32x4*>(&e.t[row][d]) = x;
  }
}

// The lanes' columns: their rows, read again for every tile.
template <typename T>
struct Column {
  const T* p;
  int D;
  bool vec;
  __device__ __forceinline__ Column(const T* p_, int D_, bool vec_) : p(p_), D(D_), vec(vec_) {}
  __device__ __forceinline__ f32x4 at(int c, int hq) const {
    return p != nullptr ? load4(p, 16 * c + 4 * hq, D, vec) : f32x4{};
  }
};

// s[mt] = products of entries 16 mt + 4 hq + k with the lane's column
template <typename TE, typename TC>
__device__ __forceinline__ void scores(Entries& e, const TE* base, int which, int D, bool vec, const Column<TC>& col,
                                       f32x4 (&s)[2], int lt, int hq) {
  s[0] = s[1] = f32x4{};
  for (int c0 = 0; c0 < D; c0 += kC) {
    stage<false>(e, base, which, c0, D, vec);
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x4 b = col.at(c0 / 16 + c, hq);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(&e.t[16 * mt + lt][16 * c + 4 * hq]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], s[mt], 0, 0, 0);
      }
    }
    __syncthreads();
  }
}

// acc[i]: dims d0 + 16 i + 4 hq + k of the lane's column, += sum over the entries
// of their weight w times their row.
template <bool SAFE, typename TE>
__device__ __forceinline__ void sums(Entries& e, const TE* base, int which, int d0, int D, bool vec, const f32x4 (&w)[2],
                                     f32x4 (&acc)[8], int lt, int hq) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (d0 + kC * half >= D) break;
    if constexpr (SAFE) {
      if (threadIdx.x == 0) e.bad = 0;
      __syncthreads();
    }
    stage<SAFE>(e, base, which, d0 + kC * half, D, vec);
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 4; ++o)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          acc[4 * half + o] = __builtin_amdgcn_mfma_f32_16x16x4f32(e.t[16 * mt + 4 * hq + k][16 * o + lt], w[mt][k],
                                                                  acc[4 * half + o], 0, 0, 0);
    if constexpr (SAFE) {  // the columns that see a row with infinities or NaN get what was left out of it
      for (uint32_t bad = e.bad; bad != 0; bad &= bad - 1) {
        const int en = __builtin_ctz(bad), k = en & 3;
        const f32x4 x = en < 16 ? w[0] : w[1];
        const float y = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
        const float we = __shfl(y, lt + 16 * ((en & 15) >> 2), 64);
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          f32x4 v = load4(base + e.off[which][en], d0 + kC * half + 16 * o + 4 * hq, D, vec);
          if constexpr (sizeof(TE) == 1) v = v * e.sc[which][en];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (we != 0.f && !(fabsf(v[q]) <= 3.402823466e38f)) acc[4 * half + o][q] += we * v[q];
        }
      }
    }
    __syncthreads();
  }
}

// The keys of a tile as entries.
template <typename TK>
__device__ __forceinline__ void key_entries(const DenseParams& p, Entries& e, int b, int g, int j0) {
  const int tid = threadIdx.x;
  if (tid < 2 * kE) {
    const int v = tid / kE, i = tid % kE, j = j0 + i;
    const int64_t off = v ? dense_row(p, b, j, p.v_sb, p.v_ss) : dense_row(p, b, j, p.k_sb, p.k_ss);
    e.off[v][i] = off < 0 ? -1 : off + g * (v ? p.v_sh : p.k_sh);
    if constexpr (sizeof(TK) == 1) {
      const int64_t so = v ? dense_row(p, b, j, p.vs_sb, p.vs_ss) : dense_row(p, b, j, p.ks_sb, p.ks_ss);
      e.sc[v][i] = so < 0 ? 0.f : scale_of(v ? p.vs[so + g * p.vs_sh] : p.ks[so + g * p.ks_sh]);
    }
  }
}

template <typename T, typename TK>
__global__ __launch_bounds__(256) void dense_any_fwd_kernel(DenseParams p) {
  __shared__ Entries e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  const int ndc = (p.Dv + kAnyDims - 1) / kAnyDims;
  int wi = gridDim.x - 1 - blockIdx.x;  // (the longest row blocks of a sequence first)
  const int dc = wi % ndc;
  wi /= ndc;
  DenseItem it;
  if (!dense_item(p, wi / p.Hkv, wi % p.Hkv, it)) return;
  const int b = it.b, g = it.g, row = 16 * wave + lt;
  const QRow qr = q_row(p, it.s, g, it.row0 + row);
  const Column<T> q(qr.pos >= 0 ? reinterpret_cast<const T*>(p.q) + b * p.q_sb + qr.t * p.q_ss + qr.h * p.q_sh : nullptr, p.Dqk, p.vec);
  const TK* kp = reinterpret_cast<const TK*>(p.k);
  const TK* vp = reinterpret_cast<const TK*>(p.v);
  f32x4 acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = f32x4{};
  float m = kNegInf, l = 0.f;
  for (int v = it.v0; v < it.v1; ++v) {
    const int j0 = it.tiles.tile(v) << kAnyShift;
    key_entries<TK>(p, e, b, g, j0);
    __syncthreads();
    f32x4 s[2];
    scores(e, kp, 0, p.Dqk, p.vec, q, s, lt, hq);
    float tmax = kNegInf;
    uint32_t seen = 0;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = e.off[0][en] >= 0 && qr.pos >= 0 && dense_seen(p, j0 + en, qr.pos);
        seen |= (uint32_t)ok << (4 * mt + k);
        s[mt][k] = ok ? s[mt][k] * p.scale_log2 : kNegInf;
        tmax = fmaxf(tmax, s[mt][k]);
      }
    tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
    tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
    const float mn = fmaxf(m, tmax), alpha = mn == kNegInf ? 1.f : exp2f(m - mn), moff = mn == kNegInf ? 0.f : mn;
    l *= alpha;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[mt][k] = (seen >> (4 * mt + k)) & 1 ? exp2f(s[mt][k] - moff) : 0.f;
        l += s[mt][k];
      }
    m = mn;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= alpha;
    if (whole_tile(p, it, j0)) sums<false>(e, vp, 1, dc * kAnyDims, p.Dv, p.vec, s, acc, lt, hq);
    else sums<true>(e, vp, 1, dc * kAnyDims, p.Dv, p.vec, s, acc, lt, hq);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!qr.in) return;
  float lse, f;
  if (it.partial) {
    f = dense_part(m, l, lse);
    if (dc == 0 && hq == 0) p.part_lse[it.part + row] = lse;
  } else {
    f = dense_finish(p, qr.h, qr.pos >= 0, m, l, lse);
    if (dc == 0 && hq == 0) p.lse[b * p.l_sb + qr.t * p.l_ss + qr.h * p.l_sh] = lse;
  }
  T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + qr.t * p.o_ss + qr.h * p.o_sh;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = dc * kAnyDims + 16 * i + 4 * hq;
    const f32x4 y = acc[i] * f, x = f == 0.f ? f32x4{} : y;
    if (it.partial) store4(p.part_o + (it.part + row) * p.Dv, d, p.Dv, p.Dv % 4 == 0, x);
    else store4(o, d, p.Dv, p.vec, x);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void dense_any_dq_kernel(DenseParams p) {
  __shared__ Entries e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  const int ndc = (p.Dqk + kAnyDims - 1) / kAnyDims;
  int wi = gridDim.x - 1 - blockIdx.x;
  const int dc = wi % ndc;
  wi /= ndc;
  DenseItem it;
  if (!dense_item(p, wi / p.Hkv, wi % p.Hkv, it)) return;
  const int b = it.b, g = it.g, r = it.row0 + 16 * wave + lt;
  const QRow qr = q_row(p, it.s, g, r);
  const bool live = qr.pos >= 0;
  const Column<T> q(live ? reinterpret_cast<const T*>(p.q) + b * p.q_sb + qr.t * p.q_ss + qr.h * p.q_sh : nullptr, p.Dqk, p.vec);
  const Column<T> go(live ? reinterpret_cast<const T*>(p.dout) + b * p.do_sb + qr.t * p.do_ss + qr.h * p.do_sh : nullptr, p.Dv, p.vec);
  const int64_t rr = ((int64_t)b * p.Hkv + g) * p.S * p.G + r;
  const float lse = live ? p.row_lse[rr] : 0.f, delta = live ? p.row_delta[rr] : 0.f;
  const T* kp = reinterpret_cast<const T*>(p.k);
  const T* vp = reinterpret_cast<const T*>(p.v);
  f32x4 acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = f32x4{};
  float dsum = 0.f;  // sum_j p_ij do_i.v_j: delta again, of o before its rounding
  for (int v = it.v0; v < it.v1; ++v) {
    const int j0 = it.tiles.tile(v) << kAnyShift;
    key_entries<T>(p, e, b, g, j0);
    __syncthreads();
    f32x4 s[2], dp[2];
    scores(e, kp, 0, p.Dqk, p.vec, q, s, lt, hq);
    scores(e, vp, 1, p.Dv, p.vec, go, dp, lt, hq);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = e.off[0][en] >= 0 && live && dense_seen(p, j0 + en, qr.pos);
        const float w = ok ? exp2f(fmaf(s[mt][k], p.scale_log2, -lse)) : 0.f;
        dsum += ok ? w * dp[mt][k] : 0.f;
        s[mt][k] = ok ? w * (dp[mt][k] - delta) : 0.f;
      }
    if (whole_tile(p, it, j0)) sums<false>(e, kp, 0, dc * kAnyDims, p.Dqk, p.vec, s, acc, lt, hq);
    else sums<true>(e, kp, 0, dc * kAnyDims, p.Dqk, p.vec, s, acc, lt, hq);
  }
  dsum += __shfl_xor(dsum, 16, 64);
  dsum = xor32_sum(dsum);
  if (!qr.in) return;
  // (an array of its own: the workgroups of the row's other dims may not have read row_delta yet)
  if (live && hq == 0 && dc == 0) p.row_exact[rr] = dsum - (p.dlse != nullptr ? p.dlse[b * p.l_sb + qr.t * p.l_ss + qr.h * p.l_sh] : 0.f);
  T* o = reinterpret_cast<T*>(p.dq) + b * p.dq_sb + qr.t * p.dq_ss + qr.h * p.dq_sh;
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // (padding: 0 times what the others see)
    const f32x4 y = acc[i] * p.scale, x = live ? y : f32x4{};
    store4(o, dc * kAnyDims + 16 * i + 4 * hq, p.Dqk, p.vec, x);
  }
}

// 64 keys a workgroup, 16 a wave; a chunk of the rows of all heads that see them, in order.
template <typename T>
__global__ __launch_bounds__(256) void dense_any_dkv_kernel(DenseParams p) {
  __shared__ Entries e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  const int dmax = p.Dqk > p.Dv ? p.Dqk : p.Dv, ndc = (dmax + kAnyDims - 1) / kAnyDims;
  const int dc = blockIdx.x % ndc;
  KeyBlock kb;
  if (!key_block(p, blockIdx.x / ndc, kb)) return;
  const DenseSeq s = kb.s;
  const int b = kb.b, g = kb.g, in = 16 * wave + lt, j = kb.kb * kAnyRows + in;
  const bool live = j < s.n;
  const Column<T> kc(live ? reinterpret_cast<const T*>(p.k) + b * p.k_sb + j * p.k_ss + g * p.k_sh : nullptr, p.Dqk, p.vec);
  const Column<T> vc(live ? reinterpret_cast<const T*>(p.v) + b * p.v_sb + j * p.v_ss + g * p.v_sh : nullptr, p.Dv, p.vec);
  const T* qp = reinterpret_cast<const T*>(p.q) + b * p.q_sb;
  const T* dop = reinterpret_cast<const T*>(p.dout) + b * p.do_sb;
  f32x4 dk[8], dv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dk[i] = dv[i] = f32x4{};
  for (int r0 = kb.r0; r0 < kb.r1; r0 += kE) {
    if (tid < kE) {
      const int r = r0 + tid;
      const QRow x = q_row(p, s, g, r < kb.r1 ? r : p.S * p.G);
      const bool in = x.pos >= 0;
      const int64_t rr = ((int64_t)b * p.Hkv + g) * p.S * p.G + r;
      e.off[0][tid] = in ? x.t * p.q_ss + x.h * p.q_sh : -1;
      e.off[1][tid] = in ? x.t * p.do_ss + x.h * p.do_sh : -1;
      e.pos[tid] = x.pos;
      e.lse[tid] = in ? p.row_lse[rr] : 0.f;
      e.delta[tid] = in ? p.row_delta[rr] : 0.f;
    }
    __syncthreads();
    f32x4 w[2], ds[2];
    scores(e, qp, 0, p.Dqk, p.vec, kc, w, lt, hq);
    scores(e, dop, 1, p.Dv, p.vec, vc, ds, lt, hq);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = live && dense_seen(p, j, e.pos[en]);
        w[mt][k] = ok ? exp2f(fmaf(w[mt][k], p.scale_log2, -e.lse[en])) : 0.f;
        ds[mt][k] = ok ? w[mt][k] * (ds[mt][k] - e.delta[en]) : 0.f;
      }
    sums<true>(e, dop, 1, dc * kAnyDims, p.Dv, p.vec, w, dv, lt, hq);
    sums<true>(e, qp, 0, dc * kAnyDims, p.Dqk, p.vec, ds, dk, lt, hq);
  }
  store_dkv<T>(p, kb, in, dc * kAnyDims, dk, dv, hq);
}

// Blocks of several chunks: their sums in order, 4 dims of a key a thread.
template <typename T>
__global__ __launch_bounds__(256) void dense_any_join_kernel(DenseParams p) {
  KeyBlock kb;
  key_block(p, blockIdx.x * p.dkv_parts, kb);
  if (kb.nc <= 1) return;
  const int D = p.Dqk + p.Dv, per = (p.Dqk + 3) / 4 + (p.Dv + 3) / 4;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < kAnyRows * per; i += gridDim.y * 256) {
    const int in = i / per, x = i % per, j = kb.kb * kAnyRows + in;
    const bool isv = x >= (p.Dqk + 3) / 4;
    const int d = 4 * (isv ? x - (p.Dqk + 3) / 4 : x), n = isv ? p.Dv : p.Dqk;
    f32x4 s = {};
#pragma unroll 4
    for (int c = 0; c < kb.nc; ++c)
      s += load4(kb.part + ((int64_t)c * kAnyRows + in) * D + (isv ? p.Dqk : 0), d, n, p.vec);
    if (j >= p.S) continue;
    T* o = isv ? reinterpret_cast<T*>(p.dv) + kb.b * p.dv_sb + j * p.dv_ss + kb.g * p.dv_sh
               : reinterpret_cast<T*>(p.dk) + kb.b * p.dk_sb + j * p.dk_ss + kb.g * p.dk_sh;
    store4(o, d, n, p.vec, isv ? s : s * p.scale);
  }
}

template <typename T, typename TK>
void fwd(const DenseParams& p, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.slots * p.Hkv * ((p.Dv + kAnyDims - 1) / kAnyDims));
  dense_any_fwd_kernel<T, TK><<<grid, 256, 0, s>>>(p);
}
template <typename T>
void bwd(const DenseParams& p, hipStream_t s) {
  const int64_t dmax = p.Dqk > p.Dv ? p.Dqk : p.Dv, blocks = (int64_t)((p.S + kAnyRows - 1) / kAnyRows) * p.B * p.Hkv;
  if (dmax <= kAnyDims) {
    launch_dense_held_bwd(p, sizeof(T) == 4, s);
  } else {
    dense_any_dq_kernel<T><<<(unsigned)((int64_t)p.B * p.nrb * p.Hkv * ((p.Dqk + kAnyDims - 1) / kAnyDims)), 256, 0, s>>>(p);
    DenseParams q = p;
    q.row_delta = p.row_exact;
    dense_any_dkv_kernel<T><<<(unsigned)(blocks * p.dkv_parts * ((dmax + kAnyDims - 1) / kAnyDims)), 256, 0, s>>>(q);
  }
  if (p.dkv_parts > 1) dense_any_join_kernel<T><<<dim3((unsigned)blocks, 4), 256, 0, s>>>(p);
}

}  // namespace

void launch_dense_any(const DenseParams& p, int dtype, int kv_dtype, hipStream_t s) {
  if (p.Dqk <= kAnyDims && p.Dv <= kAnyDims) return launch_dense_held(p, dtype, kv_dtype, s);
  if (kv_dtype == SFA_DTYPE_FP8_E4M3) {
    if (dtype == SFA_DTYPE_F32) fwd<float, fp8_t>(p, s);
    else fwd<bf16, fp8_t>(p, s);
  } else if (dtype == SFA_DTYPE_F32) {
    fwd<float, float>(p, s);
  } else {
    fwd<bf16, bf16>(p, s);
  }
}

void launch_dense_bwd_any(const DenseParams& p, int dtype, hipStream_t s) {
  if (dtype == SFA_DTYPE_F32) bwd<float>(p, s);
  else bwd<bf16>(p, s);
}

}  // namespace sfa

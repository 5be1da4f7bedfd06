// gfx950 dense attention through a window (sfa_dense.h), any head dims up to 128, bf16,
// float32 or 8-bit pages: every product in float32 on the matrix cores.
//
//   s_ij = scale q_i.k_j,  p = softmax over the rows that i sees,  o_i = sum_j p_ij v_j
//   backward: delta_i = o_i.do_i - dlse_i,  ds_ij = p_ij (do_i.v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Each kernel has columns, 16 a wave (query rows; for dk and dv: keys), held in registers, and
// walks over entries, 32 at a time (keys; for dk and dv: query rows), both of whose rows lie
// in LDS as float32.  A score product (16 entries x 16 columns, 16x16x4) leaves a lane with 4
// entries of one column, which are the second operand of the sums' product as they are, its
// first being the same rows read down a dim.  The next tile's rows are loaded to registers
// beside a tile's products.  Bound: the float32 matrix rate (153 TFLOP/s), of which a step of 1948
// tokens, 2 x 16 heads of 64 on one, reaches 37: the LDS reads of one operand a product, and one
// tile's barriers.  (Rows staged anew for each product, 64 dims at a time, as more than 128
// dims need it: 5.1 times as long.)

#include "sfa_dense_f32.h"

namespace sfa {
namespace {

// A tile's rows in two tensors; of tiles in turn: element offsets (-1: none), scales, and for
// dk and dv the rows' positions and statistics.  bad: rows with infinities or NaN.
template <int H>
struct Held {
  float t[2][kE][H + 4];  // (4 rows apart, the lanes' groups meet different banks)
  int64_t off[2][2][kE];
  float sc[2][2][kE];
  float lse[2][kE], delta[2][kE];
  int pos[2][kE];
  uint32_t bad[2][2];
};

template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 type;
  static __device__ __forceinline__ f32x4 value(const f32x4& x) { return x; }
};
template <>
struct Four<bf16> {
  typedef bf16x4 type;
  static __device__ __forceinline__ f32x4 value(const bf16x4& x) { return f32x4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]}; }
};
template <>
struct Four<fp8_t> {
  typedef int type;
  static __device__ __forceinline__ f32x4 value(int x) {
    return f32x4{__builtin_amdgcn_cvt_f32_fp8(x, 0), __builtin_amdgcn_cvt_f32_fp8(x, 1), __builtin_amdgcn_cvt_f32_fp8(x, 2),
                 __builtin_amdgcn_cvt_f32_fp8(x, 3)};
  }
};
// dims d .. d + 3 of a row of D as they are, zeros past its end
template <typename T>
__device__ __forceinline__ typename Four<T>::type raw4(const T* p, int d, int D, bool vec) {
  typename Four<T>::type r = {};
  if (vec) {
    if (d < D) r = *reinterpret_cast<const typename Four<T>::type*>(p + d);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d + e >= D) continue;
      if constexpr (sizeof(T) == 1) r |= (int)p[d + e].x << (8 * e);
      else r[e] = p[d + e];
    }
  }
  return r;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The threads' pieces of the next tile's rows.
template <int H, typename T>
struct Pieces {
  static constexpr int N = kE * H / 4 / 256;
  typename Four<T>::type r[2][N];
  static __device__ __forceinline__ int row(int i) { return (threadIdx.x + 256 * i) / (H / 4); }
  static __device__ __forceinline__ int dim(int i) { return 4 * ((threadIdx.x + 256 * i) % (H / 4)); }
  __device__ __forceinline__ void load(const Held<H>& e, int buf, const T* a, int Da, const T* b, int Db, bool vec) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t off = e.off[buf][w][row(i)];
        r[w][i] = off >= 0 ? raw4((w ? b : a) + off, dim(i), w ? Db : Da, vec) : typename Four<T>::type{};
      }
  }
  __device__ __forceinline__ void store(Held<H>& e, int buf) const {
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f32x4 x = Four<T>::value(r[w][i]);
        if constexpr (sizeof(T) == 1) x = x * e.sc[buf][w][row(i)];
        if (!(finite(x[0]) && finite(x[1]) && finite(x[2]) && finite(x[3]))) atomicOr(&e.bad[buf][w], 1u << row(i));
        *reinterpret_cast<f32x4*>(&e.t[w][row(i)][dim(i)]) = x;
      }
  }
  // Infinities and NaN of the tile in LDS, cleared: 0 times them would reach columns that do not
  // see their rows (add_bad adds them to those that do).
  static __device__ __forceinline__ void clear(Held<H>& e, int w) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f32x4& x = *reinterpret_cast<f32x4*>(&e.t[w][row(i)][dim(i)]);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = finite(x[k]) ? x[k] : 0.f;
    }
  }
};

// A column's row: dims 16 c + 4 hq + 0 .. 3.
template <int H, typename T>
__device__ __forceinline__ void column(const T* p, int D, bool vec, int hq, f32x4 (&r)[H / 16]) {
#pragma unroll
  for (int c = 0; c < H / 16; ++c) r[c] = p != nullptr ? load4(p, 16 * c + 4 * hq, D, vec) : f32x4{};
}

// s[mt] = products of entries 16 mt + 4 hq + k with the lane's column
template <int H>
__device__ __forceinline__ void scores(const float (&t)[kE][H + 4], const f32x4 (&col)[H / 16], f32x4 (&s)[2], int lt, int hq) {
  s[0] = s[1] = f32x4{};
#pragma unroll
  for (int c = 0; c < H / 16; ++c)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(&t[16 * mt + lt][16 * c + 4 * hq]);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], col[c][k], s[mt], 0, 0, 0);
    }
}
// acc[i]: dims 16 i + 4 hq + k of the lane's column, += sum over the entries of weight times row
template <int H>
__device__ __forceinline__ void sums(const float (&t)[kE][H + 4], const f32x4 (&w)[2], f32x4 (&acc)[H / 16], int lt, int hq) {
#pragma unroll
  for (int o = 0; o < H / 16; ++o)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        acc[o] = __builtin_amdgcn_mfma_f32_16x16x4f32(t[16 * mt + 4 * hq + k][16 * o + lt], w[mt][k], acc[o], 0, 0, 0);
}
template <int H, typename T>
__device__ __forceinline__ void add_bad(const Held<H>& e, int buf, int which, const T* base, int D, bool vec, const f32x4 (&w)[2],
                                        f32x4 (&acc)[H / 16], int lt, int hq) {
  for (uint32_t bad = e.bad[buf][which]; bad != 0; bad &= bad - 1) {
    const int en = __builtin_ctz(bad), k = en & 3;
    const f32x4 x = en < 16 ? w[0] : w[1];
    const float y = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
    const float we = __shfl(y, lt + 16 * ((en & 15) >> 2), 64);
#pragma unroll
    for (int o = 0; o < H / 16; ++o) {
      f32x4 v = load4(base + e.off[buf][which][en], 16 * o + 4 * hq, D, vec);
      if constexpr (sizeof(T) == 1) v = v * e.sc[buf][which][en];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (we != 0.f && !finite(v[q])) acc[o][q] += we * v[q];
    }
  }
}

// The keys of a tile as entries: one of K or V a thread, found a tile ahead of its rows.
template <typename TK>
struct KeyEntry {
  int64_t off;
  float sc;
  __device__ __forceinline__ void load(const DenseParams& p, int b, int g, int j0) {
    const int tid = threadIdx.x;
    if (tid >= 2 * kE) return;
    const int v = tid / kE, j = j0 + tid % kE;
    off = v ? dense_row(p, b, j, p.v_sb, p.v_ss) : dense_row(p, b, j, p.k_sb, p.k_ss);
    off = off < 0 ? -1 : off + g * (v ? p.v_sh : p.k_sh);
    if constexpr (sizeof(TK) == 1) {
      const int64_t so = v ? dense_row(p, b, j, p.vs_sb, p.vs_ss) : dense_row(p, b, j, p.ks_sb, p.ks_ss);
      sc = so < 0 ? 0.f : scale_of(v ? p.vs[so + g * p.vs_sh] : p.ks[so + g * p.ks_sh]);
    }
  }
  template <int H>
  __device__ __forceinline__ void store(Held<H>& e, int buf) const {
    const int tid = threadIdx.x;
    if (tid >= 2 * kE) return;
    e.off[buf][tid / kE][tid % kE] = off;
    if constexpr (sizeof(TK) == 1) e.sc[buf][tid / kE][tid % kE] = sc;
  }
};
// The query rows of a tile as entries: those from r0 up to r1.
struct RowEntry {
  int64_t off[2];
  float lse, delta;
  int pos;
  __device__ __forceinline__ void load(const DenseParams& p, const KeyBlock& kb, int r0) {
    const int r = r0 + (int)threadIdx.x;
    if (threadIdx.x >= kE) return;
    const QRow x = q_row(p, kb.s, kb.g, r < kb.r1 ? r : p.S * p.G);
    const bool in = x.pos >= 0;
    const int64_t rr = ((int64_t)kb.b * p.Hkv + kb.g) * p.S * p.G + r;
    off[0] = in ? x.t * p.q_ss + x.h * p.q_sh : -1;
    off[1] = in ? x.t * p.do_ss + x.h * p.do_sh : -1;
    pos = x.pos;
    lse = in ? p.row_lse[rr] : 0.f;
    delta = in ? p.row_delta[rr] : 0.f;
  }
  template <int H>
  __device__ __forceinline__ void store(Held<H>& e, int buf) const {
    const int i = threadIdx.x;
    if (i >= kE) return;
    e.off[buf][0][i] = off[0];
    e.off[buf][1][i] = off[1];
    e.pos[buf][i] = pos;
    e.lse[buf][i] = lse;
    e.delta[buf][i] = delta;
  }
};

// The walk over n tiles: start(i) begins to read a tile's entries, body(i, buf, bad of both
// tensors) is its part.  Between the barriers of a tile the next one's rows are on their way.
template <int H, typename TE, typename Entry, typename Start, typename Body>
__device__ __forceinline__ void walk(const DenseParams& p, Held<H>& e, int n, Entry& ent, const TE* a, int Da, const TE* b, int Db,
                                     Start start, Body body) {
  if (n <= 0) return;
  Pieces<H, TE> next;
  start(0);
  ent.store(e, 0);
  if (threadIdx.x < 4) e.bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  __syncthreads();
  next.load(e, 0, a, Da, b, Db, p.vec);
  if (n > 1) start(1);
  for (int i = 0; i < n; ++i) {
    const int buf = i & 1;
    next.store(e, buf);
    if (i + 1 < n) ent.store(e, buf ^ 1);
    __syncthreads();
    if (threadIdx.x < 2) e.bad[buf ^ 1][threadIdx.x] = 0;
    if (i + 1 < n) next.load(e, buf ^ 1, a, Da, b, Db, p.vec);
    if (i + 2 < n) start(i + 2);
    body(i, buf, e.bad[buf][0] != 0, e.bad[buf][1] != 0);
    __syncthreads();
  }
}

template <typename T, typename TK, int H>
__global__ __launch_bounds__(256, 2) void dense_held_fwd_kernel(DenseParams p) {
  __shared__ Held<H> e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  const int wi = gridDim.x - 1 - blockIdx.x;  // (the longest row blocks of a sequence first)
  DenseItem it;
  if (!dense_item(p, wi / p.Hkv, wi % p.Hkv, it)) return;
  const int b = it.b, g = it.g, row = 16 * wave + lt;
  const QRow qr = q_row(p, it.s, g, it.row0 + row);
  f32x4 q[H / 16];
  column<H>(qr.pos >= 0 ? reinterpret_cast<const T*>(p.q) + b * p.q_sb + qr.t * p.q_ss + qr.h * p.q_sh : nullptr, p.Dqk, p.vec, hq, q);
  const TK* kp = reinterpret_cast<const TK*>(p.k);
  const TK* vp = reinterpret_cast<const TK*>(p.v);
  f32x4 acc[H / 16];
#pragma unroll
  for (int i = 0; i < H / 16; ++i) acc[i] = f32x4{};
  float m = kNegInf, l = 0.f;
  KeyEntry<TK> ent;
  auto at = [&](int i) { return it.tiles.tile(it.v0 + i) << kAnyShift; };
  walk<H>(p, e, it.v1 - it.v0, ent, kp, p.Dqk, vp, p.Dv, [&](int i) { ent.load(p, b, g, at(i)); }, [&](int i, int buf, bool, bool bad) {
    const int j0 = at(i);
    f32x4 s[2];
    scores<H>(e.t[0], q, s, lt, hq);
    float tmax = kNegInf;
    uint32_t seen = 0;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = e.off[buf][0][en] >= 0 && qr.pos >= 0 && dense_seen(p, j0 + en, qr.pos);
        seen |= (uint32_t)ok << (4 * mt + k);
        s[mt][k] = ok ? s[mt][k] * p.scale_log2 : kNegInf;
        tmax = fmaxf(tmax, s[mt][k]);
      }
    tmax = xor32_max(xor16_max(tmax));
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
    for (int i = 0; i < H / 16; ++i) acc[i] *= alpha;
    if (bad) {
      Pieces<H, TK>::clear(e, 1);
      __syncthreads();
    }
    sums<H>(e.t[1], s, acc, lt, hq);
    if (bad) add_bad<H>(e, buf, 1, vp, p.Dv, p.vec, s, acc, lt, hq);
  });
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!qr.in) return;
  float lse, f;
  if (it.partial) {
    f = dense_part(m, l, lse);
    if (hq == 0) p.part_lse[it.part + row] = lse;
  } else {
    f = dense_finish(p, qr.h, qr.pos >= 0, m, l, lse);
    if (hq == 0) p.lse[b * p.l_sb + qr.t * p.l_ss + qr.h * p.l_sh] = lse;
  }
  T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + qr.t * p.o_ss + qr.h * p.o_sh;
#pragma unroll
  for (int i = 0; i < H / 16; ++i) {
    const int d = 16 * i + 4 * hq;
    const f32x4 y = acc[i] * f, x = f == 0.f ? f32x4{} : y;
    if (it.partial) store4(p.part_o + (it.part + row) * p.Dv, d, p.Dv, p.Dv % 4 == 0, x);
    else store4(o, d, p.Dv, p.vec, x);
  }
}

template <typename T, int H>
__global__ __launch_bounds__(256, 2) void dense_held_dq_kernel(DenseParams p) {
  __shared__ Held<H> e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  const int wi = gridDim.x - 1 - blockIdx.x;
  DenseItem it;
  if (!dense_item(p, wi / p.Hkv, wi % p.Hkv, it)) return;
  const int b = it.b, g = it.g, r = it.row0 + 16 * wave + lt;
  const QRow qr = q_row(p, it.s, g, r);
  const bool live = qr.pos >= 0;
  f32x4 q[H / 16], go[H / 16];
  column<H>(live ? reinterpret_cast<const T*>(p.q) + b * p.q_sb + qr.t * p.q_ss + qr.h * p.q_sh : nullptr, p.Dqk, p.vec, hq, q);
  column<H>(live ? reinterpret_cast<const T*>(p.dout) + b * p.do_sb + qr.t * p.do_ss + qr.h * p.do_sh : nullptr, p.Dv, p.vec, hq, go);
  const int64_t rr = ((int64_t)b * p.Hkv + g) * p.S * p.G + r;
  const float lse = live ? p.row_lse[rr] : 0.f, delta = live ? p.row_delta[rr] : 0.f;
  const T* kp = reinterpret_cast<const T*>(p.k);
  f32x4 acc[H / 16];
#pragma unroll
  for (int i = 0; i < H / 16; ++i) acc[i] = f32x4{};
  float dsum = 0.f;  // sum_j p_ij do_i.v_j: delta again, of o before its rounding
  KeyEntry<T> ent;
  auto at = [&](int i) { return it.tiles.tile(it.v0 + i) << kAnyShift; };
  walk<H>(p, e, it.v1 - it.v0, ent, kp, p.Dqk, reinterpret_cast<const T*>(p.v), p.Dv, [&](int i) { ent.load(p, b, g, at(i)); },
          [&](int i, int buf, bool bad, bool) {
    const int j0 = at(i);
    f32x4 s[2], dp[2];
    scores<H>(e.t[0], q, s, lt, hq);
    scores<H>(e.t[1], go, dp, lt, hq);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = e.off[buf][0][en] >= 0 && live && dense_seen(p, j0 + en, qr.pos);
        const float w = ok ? exp2f(fmaf(s[mt][k], p.scale_log2, -lse)) : 0.f;
        dsum += ok ? w * dp[mt][k] : 0.f;
        s[mt][k] = ok ? w * (dp[mt][k] - delta) : 0.f;
      }
    if (bad) {
      __syncthreads();
      Pieces<H, T>::clear(e, 0);
      __syncthreads();
    }
    sums<H>(e.t[0], s, acc, lt, hq);
    if (bad) add_bad<H>(e, buf, 0, kp, p.Dqk, p.vec, s, acc, lt, hq);
  });
  dsum += __shfl_xor(dsum, 16, 64);
  dsum = xor32_sum(dsum);
  if (!qr.in) return;
  if (live && hq == 0) p.row_exact[rr] = dsum - (p.dlse != nullptr ? p.dlse[b * p.l_sb + qr.t * p.l_ss + qr.h * p.l_sh] : 0.f);
  T* o = reinterpret_cast<T*>(p.dq) + b * p.dq_sb + qr.t * p.dq_ss + qr.h * p.dq_sh;
#pragma unroll
  for (int i = 0; i < H / 16; ++i) store4(o, 16 * i + 4 * hq, p.Dqk, p.vec, acc[i] * p.scale);
}

// 64 keys a workgroup, 16 a wave; a chunk of the rows of all heads that see them, in order.
template <typename T, int H>
__global__ __launch_bounds__(256, 2) void dense_held_dkv_kernel(DenseParams p) {
  __shared__ Held<H> e;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lt = lane & 15, hq = lane >> 4;
  KeyBlock kb;
  if (!key_block(p, blockIdx.x, kb)) return;
  const int b = kb.b, g = kb.g, in = 16 * wave + lt, j = kb.kb * kAnyRows + in;
  const bool live = j < kb.s.n;
  f32x4 kc[H / 16], vc[H / 16];
  column<H>(live ? reinterpret_cast<const T*>(p.k) + b * p.k_sb + j * p.k_ss + g * p.k_sh : nullptr, p.Dqk, p.vec, hq, kc);
  column<H>(live ? reinterpret_cast<const T*>(p.v) + b * p.v_sb + j * p.v_ss + g * p.v_sh : nullptr, p.Dv, p.vec, hq, vc);
  const T* qp = reinterpret_cast<const T*>(p.q) + b * p.q_sb;
  const T* dop = reinterpret_cast<const T*>(p.dout) + b * p.do_sb;
  f32x4 dk[H / 16], dv[H / 16];
#pragma unroll
  for (int i = 0; i < H / 16; ++i) dk[i] = dv[i] = f32x4{};
  RowEntry ent;
  const int n = kb.r1 > kb.r0 ? (kb.r1 - kb.r0 + kE - 1) / kE : 0;
  walk<H>(p, e, n, ent, qp, p.Dqk, dop, p.Dv, [&](int i) { ent.load(p, kb, kb.r0 + kE * i); }, [&](int i, int buf, bool badq, bool bado) {
    f32x4 w[2], ds[2];
    scores<H>(e.t[0], kc, w, lt, hq);
    scores<H>(e.t[1], vc, ds, lt, hq);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int en = 16 * mt + 4 * hq + k;
        const bool ok = live && dense_seen(p, j, e.pos[buf][en]);
        w[mt][k] = ok ? exp2f(fmaf(w[mt][k], p.scale_log2, -e.lse[buf][en])) : 0.f;
        ds[mt][k] = ok ? w[mt][k] * (ds[mt][k] - e.delta[buf][en]) : 0.f;
      }
    if (badq || bado) {
      __syncthreads();
      Pieces<H, T>::clear(e, 0);
      Pieces<H, T>::clear(e, 1);
      __syncthreads();
    }
    sums<H>(e.t[1], w, dv, lt, hq);
    sums<H>(e.t[0], ds, dk, lt, hq);
    if (bado) add_bad<H>(e, buf, 1, dop, p.Dv, p.vec, w, dv, lt, hq);
    if (badq) add_bad<H>(e, buf, 0, qp, p.Dqk, p.vec, ds, dk, lt, hq);
  });
  store_dkv<T>(p, kb, in, 0, dk, dv, hq);
}

template <typename T, typename TK>
void fwd(const DenseParams& p, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.slots * p.Hkv);
  if (p.Dqk <= 64 && p.Dv <= 64) dense_held_fwd_kernel<T, TK, 64><<<grid, 256, 0, s>>>(p);
  else dense_held_fwd_kernel<T, TK, 128><<<grid, 256, 0, s>>>(p);
}
template <typename T, int H>
void bwd(const DenseParams& p, hipStream_t s) {
  dense_held_dq_kernel<T, H><<<(unsigned)((int64_t)p.B * p.nrb * p.Hkv), 256, 0, s>>>(p);
  // (row_exact is row_delta: one workgroup a row block reads and writes it)
  dense_held_dkv_kernel<T, H><<<(unsigned)((int64_t)((p.S + kAnyRows - 1) / kAnyRows) * p.B * p.Hkv * p.dkv_parts), 256, 0, s>>>(p);
}

}  // namespace

void launch_dense_held(const DenseParams& p, int dtype, int kv_dtype, hipStream_t s) {
  if (kv_dtype == SFA_DTYPE_FP8_E4M3) {
    if (dtype == SFA_DTYPE_F32) fwd<float, fp8_t>(p, s);
    else fwd<bf16, fp8_t>(p, s);
  } else if (dtype == SFA_DTYPE_F32) {
    fwd<float, float>(p, s);
  } else {
    fwd<bf16, bf16>(p, s);
  }
}

void launch_dense_held_bwd(const DenseParams& p, bool f32, hipStream_t s) {
  const bool small = p.Dqk <= 64 && p.Dv <= 64;
  if (f32 && small) bwd<float, 64>(p, s);
  else if (f32) bwd<float, 128>(p, s);
  else if (small) bwd<bf16, 64>(p, s);
  else bwd<bf16, 128>(p, s);
}

}  // namespace sfa

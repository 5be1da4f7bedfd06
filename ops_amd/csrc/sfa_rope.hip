// gfx950 rotary positions and per-head norms of q and k in one pass: forward
// (into tensors, or the k and v rows straight into the pages of a cache) and
// backward.
//
// A row is one head of one token, x [D].  With n normed dims (the row's first
// n, 0: none), R rotated dims from dim `off`, frequencies f [R / 2]:
//   r = 1 / sqrt(mean_{d < n} x_d^2 + eps),  u_d = x_d r w_d (d < n), else x_d
//   y1 = s (u1 cos a - u2 sin a),  y2 = s (u2 cos a + u1 sin a),  a = pos f_i
// over the pairs (off + i, off + R/2 + i), or (off + 2i, off + 2i + 1) when
// interleaved; other dims pass through.  Backward, from dy:
//   du = s R(-a) dy on the rotated dims,  dw_d = sum_rows du_d xhat_d,
//   dx = r (du w - xhat mean(du w xhat)),  xhat = x r   (d < n), else du.
// Everything between the load and the one rounding at the store is float32,
// except the angle: pos f is reduced to a fraction of a turn in float64 (a
// float32 product is off by 0.06 rad at position 10^6), then sin and cos are
// taken of that fraction.
//
// Bound: HBM, each row read once and written once (backward: x and dy read,
// dx written).  So a row is held in registers, 16 bytes a lane, P lanes a
// row (the power of two that covers it; 8 lanes of 9 chunks for the 576-dim
// latent row), 64 / P heads of one token per wave; the token's angles are
// computed once per wave for all the heads that it takes.  Rows that are not
// whole 16-byte chunks (odd dims, strides, offsets) take the scalar kernels,
// one wave a row.

#include "sfa_ops.h"

namespace sfa {
namespace {

constexpr double kInv2Pi = 0.15915494309189533576888376337251;
constexpr int kMaxD = 1024;
constexpr int kScalarSteps = kMaxD / 64;

template <typename T>
struct Chunk {
  static constexpr int E = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void unpack(const u32x4& r, float (&f)[E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = __uint_as_float(r[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        f[2 * e] = __uint_as_float(r[e] << 16);
        f[2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&f)[E]) {
    if constexpr (sizeof(T) == 4) {
      return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    } else {
      const bf16x8 v = {(bf16)f[0], (bf16)f[1], (bf16)f[2], (bf16)f[3], (bf16)f[4], (bf16)f[5], (bf16)f[6], (bf16)f[7]};
      return __builtin_bit_cast(u32x4, v);
    }
  }
};

__device__ __forceinline__ int64_t load_int(const void* base, int64_t i, int is64) {
  return is64 ? reinterpret_cast<const int64_t*>(base)[i] : (int64_t) reinterpret_cast<const int32_t*>(base)[i];
}

// cos and sin of pos * f, the angle reduced to (-1/2, 1/2] turns in float64
__device__ __forceinline__ void angle(double pos, double f, float& c, float& s) {
  double t = pos * (f * kInv2Pi);
  t -= rint(t);
  sincospif((float)(2.0 * t), &s, &c);
}

template <typename T>
__device__ __forceinline__ float load_w(const RopeParams& p, const void* w, int d) {
  return p.w_f32 ? reinterpret_cast<const float*>(w)[d] : to_f32(reinterpret_cast<const T*>(w)[d]);
}

// Sum over the P lanes of a row (P a power of two, wave-uniform).
__device__ __forceinline__ float row_sum(float x, int P) {
  for (int o = P >> 1; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// A lane's place in the rotation of one 16-byte chunk: whether it is rotated,
// its first frequency, the sign of the partner's sine term (half layout) and
// the chunk that holds the partners.
template <int E>
struct Turn {
  bool on;
  int i0, pair;
  float sgn;
  __device__ __forceinline__ Turn(const RopeParams& p, int c) {
    const int j = c * E - p.off, h = p.R / 2;
    on = j >= 0 && j < p.R;
    if (p.interleaved) {
      i0 = on ? j / 2 : 0;
      pair = c;
      sgn = 1.f;
    } else {
      const bool first = j < h;
      i0 = on ? (first ? j : j - h) : 0;
      pair = on ? (first ? c + h / E : c - h / E) : c;
      sgn = first ? -1.f : 1.f;
    }
  }
  __device__ __forceinline__ void angles(const RopeParams& p, double pos, float (&cs)[E], float (&sn)[E]) const {
    if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) angle(pos, on ? p.freq[i0 + e] : 0.0, cs[e], sn[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) angle(pos, on ? p.freq[i0 + e] : 0.0, cs[e], sn[e]);
    }
    const float s = p.rope_scale;
    if (s != 1.f) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        cs[e] *= s;
        sn[e] *= s;
      }
    }
  }
  // u (own) and o (the partner chunk, half layout) turned by +-a (dir = 1, -1)
  __device__ __forceinline__ void apply(const RopeParams& p, float (&u)[E], const float (&o)[E], const float (&cs)[E],
                                        const float (&sn)[E], float dir) const {
    if (!on) return;
    if (p.interleaved) {
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float a = u[2 * e], b = u[2 * e + 1], sd = dir * sn[e];
        u[2 * e] = a * cs[e] - b * sd;
        u[2 * e + 1] = b * cs[e] + a * sd;
      }
    } else {
      const float q = sgn * dir;
#pragma unroll
      for (int e = 0; e < E; ++e) u[e] = u[e] * cs[e] + q * (o[e] * sn[e]);
    }
  }
};

__device__ __forceinline__ u32x4 shfl16(const u32x4& x, int lane) {
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = (unsigned)__shfl((int)x[e], lane, 64);
  return r;
}

// Byte offset of the cache row that token (b, s) goes to, or -1: slot outside
// the table or page outside the pool.
__device__ __forceinline__ int64_t cache_row(const RopeParams& p, int b, int s, int64_t page_stride, int64_t row_stride) {
  const int64_t slot = load_int(p.slots, b * p.slot_sb + s * p.slot_ss, p.slot_i64);
  if (slot < 0 || slot >= ((int64_t)p.max_pages << p.page_shift)) return -1;
  const int pg = p.block_table[b * p.bt_sb + (slot >> p.page_shift)];
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * page_stride + (slot & ((1 << p.page_shift) - 1)) * row_stride;
}

// Forward.  A wave takes `per` row groups of a token: first the q heads' (64 / P
// rows a group), then the k heads', then (append) 64-chunk groups of the v row.
template <typename T, int K>
__global__ __launch_bounds__(256) void rope_fwd_kernel(RopeParams p) {
  constexpr int E = Chunk<T>::E;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= p.units) return;
  const int64_t tok = unit / p.upt;
  const int b = (int)(tok / p.S), s = (int)(tok % p.S);
  const int P = p.P, rpw = 64 / P, l = lane & (P - 1), rr = lane / P;
  const int g0 = (int)(unit % p.upt) * p.per, g1 = min(g0 + p.per, p.groups);
  const double pos = (double)load_int(p.pos, b * p.pos_sb + s * p.pos_ss, p.pos_i64);

  // the angles of the lane's chunk, for all its rows (rows of several chunks a
  // lane: per chunk and row, where it is rotated)
  const Turn<E> t0(p, l);
  float cs[E], sn[E];
  if constexpr (K == 1) t0.angles(p, pos, cs, sn);

  int held = -1;
  float w[E], wo[E];  // K = 1: the chunk's weights and its partner's
  for (int g = g0; g < g1; ++g) {
    const int si = g < p.side[0].groups ? 0 : g < p.side[0].groups + p.side[1].groups ? 1 : 2;
    if (si == 2) {  // the v row: copied
      const int i = (g - p.side[0].groups - p.side[1].groups) * 64 + lane, cpr = p.Dv / E;
      const int64_t row = cache_row(p, b, s, p.vo_sb, p.vo_ss);
      if (i < p.side[1].H * cpr && row >= 0) {
        const int h = i / cpr, c = i % cpr;
        const T* x = reinterpret_cast<const T*>(p.v) + b * p.v_sb + s * p.v_ss + h * p.v_sh + c * E;
        *reinterpret_cast<u32x4*>(reinterpret_cast<T*>(p.v_out) + row + h * p.vo_sh + c * E) =
            *reinterpret_cast<const u32x4*>(x);
      }
      continue;
    }
    const RopeSide& sd = p.side[si];
    const int h = (si == 0 ? g : g - p.side[0].groups) * rpw + rr;
    const bool live = h < sd.H;
    const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + (int64_t)(live ? h : 0) * sd.x_sh;
    int64_t yo;
    if (si == 1 && p.block_table != nullptr)
      yo = cache_row(p, b, s, sd.y_sb, sd.y_ss);
    else
      yo = b * sd.y_sb + s * sd.y_ss;
    T* y = reinterpret_cast<T*>(sd.y) + yo + (int64_t)(live ? h : 0) * sd.y_sh;
    const bool put = live && yo >= 0;

    u32x4 raw[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      raw[j] = c < p.chunks ? *reinterpret_cast<const u32x4*>(x + c * E) : u32x4{0, 0, 0, 0};
    }
    u32x4 oth[K];  // partner chunks (half layout)
    if (!p.interleaved) {
      if constexpr (K == 1) {
        oth[0] = shfl16(raw[0], (lane & ~(P - 1)) + t0.pair);
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const Turn<E> t(p, j * P + l);
          if (t.on) oth[j] = *reinterpret_cast<const u32x4*>(x + t.pair * E);
        }
      }
    }
    float r = 1.f;
    if (sd.n > 0) {
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        float f[E];
        Chunk<T>::unpack(raw[j], f);
        if ((j * P + l) * E < sd.n) {
          float q4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < E; ++e) q4[e & 3] = fmaf(f[e], f[e], q4[e & 3]);
          q += (q4[0] + q4[1]) + (q4[2] + q4[3]);
        }
      }
      r = 1.f / sqrtf(row_sum(q, P) / (float)sd.n + p.eps);
      if (K == 1 && held != si) {
        held = si;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          w[e] = l * E < sd.n ? load_w<T>(p, sd.w, l * E + e) : 1.f;
          wo[e] = t0.pair * E < sd.n ? load_w<T>(p, sd.w, t0.pair * E + e) : 1.f;
        }
      }
    }
    u32x4 res[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      const Turn<E> t(p, c);
      float u[E], o[E];
      Chunk<T>::unpack(raw[j], u);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
      if (!p.interleaved && t.on) Chunk<T>::unpack(oth[j], o);
      if (c * E < sd.n) {
        const int cw = c;
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] = u[e] * r * (K == 1 ? w[e] : load_w<T>(p, sd.w, cw * E + e));
      }
      if (!p.interleaved && t.on && t.pair * E < sd.n) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * r * (K == 1 ? wo[e] : load_w<T>(p, sd.w, t.pair * E + e));
      }
      if constexpr (K == 1) {
        t.apply(p, u, o, cs, sn, 1.f);
      } else if (t.on) {
        float c2[E], s2[E];
        t.angles(p, pos, c2, s2);
        t.apply(p, u, o, c2, s2, 1.f);
      }
      res[j] = Chunk<T>::pack(u);
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      if (put && c < p.chunks) *reinterpret_cast<u32x4*>(y + c * E) = res[j];
    }
  }
}

// Backward: side.y is dy, side.dx receives dx.  A wave takes a contiguous run of
// (token, row group) units and sums its rows' dw in registers; a workgroup
// writes its sums to partial row blockIdx.x, which rope_dw_kernel adds up in order.
template <typename T, int K>
__global__ __launch_bounds__(256) void rope_bwd_kernel(RopeParams p) {
  constexpr int E = Chunk<T>::E;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int P = p.P, rpw = 64 / P, l = lane & (P - 1), rr = lane / P;
  const int64_t nw = (int64_t)gridDim.x * 4, wv = (int64_t)blockIdx.x * 4 + wave;
  const int64_t u0 = p.units * wv / nw, u1 = p.units * (wv + 1) / nw;
  const Turn<E> t0(p, l);
  float cs[E], sn[E];
  int64_t tok_held = -1;
  int held = -1;
  double pos = 0.0;
  float w[E];
  float dw[2][K][E];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) dw[a][j][e] = 0.f;

  for (int64_t u = u0; u < u1; ++u) {
    const int64_t tok = u / p.groups;
    const int g = (int)(u % p.groups);
    const int b = (int)(tok / p.S), s = (int)(tok % p.S);
    if (tok != tok_held) {
      tok_held = tok;
      pos = (double)load_int(p.pos, b * p.pos_sb + s * p.pos_ss, p.pos_i64);
      if constexpr (K == 1) t0.angles(p, pos, cs, sn);
    }
    const int si = g < p.side[0].groups ? 0 : 1;
    const RopeSide& sd = p.side[si];
    const int h = (si == 0 ? g : g - p.side[0].groups) * rpw + rr;
    const bool live = h < sd.H;
    const int64_t hh = live ? h : 0;
    const T* dy = reinterpret_cast<const T*>(sd.y) + b * sd.y_sb + s * sd.y_ss + hh * sd.y_sh;
    T* dx = reinterpret_cast<T*>(sd.dx) + b * sd.dx_sb + s * sd.dx_ss + hh * sd.dx_sh;
    u32x4 raw[K], xr[K], oth[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      raw[j] = c < p.chunks ? *reinterpret_cast<const u32x4*>(dy + c * E) : u32x4{0, 0, 0, 0};
    }
    if (sd.n > 0) {
      const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + hh * sd.x_sh;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int c = j * P + l;
        xr[j] = c * E < sd.n ? *reinterpret_cast<const u32x4*>(x + c * E) : u32x4{0, 0, 0, 0};
      }
    }
    if (!p.interleaved) {
      if constexpr (K == 1) {
        oth[0] = shfl16(raw[0], (lane & ~(P - 1)) + t0.pair);
      } else {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const Turn<E> t(p, j * P + l);
          if (t.on) oth[j] = *reinterpret_cast<const u32x4*>(dy + t.pair * E);
        }
      }
    }
    if (K == 1 && sd.n > 0 && held != si) {
      held = si;
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = l * E < sd.n ? load_w<T>(p, sd.w, l * E + e) : 1.f;
    }
    float du[K][E];
    float q = 0.f, gx = 0.f;  // sum x^2, sum (du w) x
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      const Turn<E> t(p, c);
      float o[E];
      Chunk<T>::unpack(raw[j], du[j]);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
      if (!p.interleaved && t.on) Chunk<T>::unpack(oth[j], o);
      if constexpr (K == 1) {
        t.apply(p, du[j], o, cs, sn, -1.f);
      } else if (t.on) {
        float c2[E], s2[E];
        t.angles(p, pos, c2, s2);
        t.apply(p, du[j], o, c2, s2, -1.f);
      }
      if (c * E < sd.n) {
        float x[E];
        Chunk<T>::unpack(xr[j], x);
        float q2[2] = {0.f, 0.f}, g2[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float gw = du[j][e] * (K == 1 ? w[e] : load_w<T>(p, sd.w, c * E + e));
          q2[e & 1] = fmaf(x[e], x[e], q2[e & 1]);
          g2[e & 1] = fmaf(gw, x[e], g2[e & 1]);
        }
        q += q2[0] + q2[1];
        gx += g2[0] + g2[1];
      }
    }
    float r = 0.f, m = 0.f;  // 1 / rms, mean of (du w) xhat
    if (sd.n > 0) {
      r = 1.f / sqrtf(row_sum(q, P) / (float)sd.n + p.eps);
      m = row_sum(gx, P) * r / (float)sd.n;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      if (c * E < sd.n) {
        float x[E];
        Chunk<T>::unpack(xr[j], x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float xh = x[e] * r, d = du[j][e];
          const float gw = d * (K == 1 ? w[e] : load_w<T>(p, sd.w, c * E + e));
          if (live) {
            if (si == 0) dw[0][j][e] = fmaf(d, xh, dw[0][j][e]);
            else dw[1][j][e] = fmaf(d, xh, dw[1][j][e]);
          }
          du[j][e] = r * (gw - xh * m);
        }
      }
      if (live && c < p.chunks) *reinterpret_cast<u32x4*>(dx + c * E) = Chunk<T>::pack(du[j]);
    }
  }

  if (p.part == nullptr) return;
  // dw of the workgroup: the row groups of a wave by shuffles, then the waves
  __shared__ float s_w[4][kMaxD];
  for (int a = 0; a < 2; ++a) {
    const int n = p.side[a].n;
    if (n == 0) continue;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x = a == 0 ? dw[0][j][e] : dw[1][j][e];
        for (int o = P; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
        if (rr == 0 && c * E < n) s_w[wave][c * E + e] = x;
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < n; d += 256)
      p.part[((int64_t)a * gridDim.x + blockIdx.x) * kMaxD + d] = (s_w[0][d] + s_w[1][d]) + (s_w[2][d] + s_w[3][d]);
    __syncthreads();
  }
}

// dw [side][n]: the partial rows added in a fixed order, 16 dims and 64 runs of
// rows per workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void rope_dw_kernel(RopeParams p, int nparts) {
  const int a = blockIdx.y, n = p.side[a].n, dc = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + dc;
  __shared__ float s_p[64][17];
  float x = 0.f;
  if (d < n) {
#pragma unroll 4
    for (int i = run; i < nparts; i += 64) x += p.part[((int64_t)a * nparts + i) * kMaxD + d];
  }
  s_p[run][dc] = x;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (run < o) s_p[run][dc] += s_p[run + o][dc];
    __syncthreads();
  }
  if (run == 0 && d < n) {
    if (p.w_f32) reinterpret_cast<float*>(p.side[a].dw)[d] = s_p[0][dc];
    else reinterpret_cast<T*>(p.side[a].dw)[d] = from_f32<T>(s_p[0][dc]);
  }
}

// ---- rows that are not whole 16-byte chunks: one wave a row -----------------

// Dim d's partner and frequency; sgn: the sign of the partner's sine term.
__device__ __forceinline__ bool turn_of(const RopeParams& p, int d, int& pd, int& i, float& sgn) {
  const int j = d - p.off, h = p.R / 2;
  if (j < 0 || j >= p.R) return false;
  const bool first = p.interleaved ? (j & 1) == 0 : j < h;
  i = p.interleaved ? j / 2 : first ? j : j - h;
  pd = p.interleaved ? (first ? d + 1 : d - 1) : first ? d + h : d - h;
  sgn = first ? -1.f : 1.f;
  return true;
}

template <typename T>
__global__ __launch_bounds__(256) void rope_fwd_scalar_kernel(RopeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= p.units) return;
  const int64_t tok = unit / p.groups;
  int h = (int)(unit % p.groups);
  const int b = (int)(tok / p.S), s = (int)(tok % p.S);
  int si = 0;
  while (si < 2 && h >= p.side[si].groups) h -= p.side[si++].groups;
  if (si == 2) {  // one v head
    const int64_t row = cache_row(p, b, s, p.vo_sb, p.vo_ss);
    const T* x = reinterpret_cast<const T*>(p.v) + b * p.v_sb + s * p.v_ss + h * p.v_sh;
    if (row >= 0)
      for (int d = lane; d < p.Dv; d += 64) reinterpret_cast<T*>(p.v_out)[row + h * p.vo_sh + d] = x[d];
    return;
  }
  const RopeSide& sd = p.side[si];
  const double pos = (double)load_int(p.pos, b * p.pos_sb + s * p.pos_ss, p.pos_i64);
  const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + h * sd.x_sh;
  const int64_t yo = si == 1 && p.block_table != nullptr ? cache_row(p, b, s, sd.y_sb, sd.y_ss) : b * sd.y_sb + s * sd.y_ss;
  if (yo < 0) return;
  T* y = reinterpret_cast<T*>(sd.y) + yo + h * sd.y_sh;
  // (own and partner values are all read before any is written: y may be x)
  float v[kScalarSteps], o[kScalarSteps], q = 0.f;
#pragma unroll
  for (int k = 0; k < kScalarSteps; ++k) {
    const int d = lane + 64 * k;
    int pd, i;
    float sgn;
    v[k] = d < p.D ? to_f32(x[d]) : 0.f;
    o[k] = d < p.D && turn_of(p, d, pd, i, sgn) ? to_f32(x[pd]) : 0.f;
    if (d < sd.n) q = fmaf(v[k], v[k], q);
  }
  const float r = sd.n > 0 ? 1.f / sqrtf(wave_sum(q) / (float)sd.n + p.eps) : 1.f;
#pragma unroll
  for (int k = 0; k < kScalarSteps; ++k) {
    const int d = lane + 64 * k;
    if (d >= p.D) continue;
    float u = v[k];
    if (d < sd.n) u = u * r * load_w<T>(p, sd.w, d);
    int pd, i;
    float sgn;
    if (turn_of(p, d, pd, i, sgn)) {
      float uo = o[k], c, sn;
      if (pd < sd.n) uo = uo * r * load_w<T>(p, sd.w, pd);
      angle(pos, p.freq[i], c, sn);
      u = u * (c * p.rope_scale) + sgn * (uo * (sn * p.rope_scale));
    }
    y[d] = from_f32<T>(u);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void rope_bwd_scalar_kernel(RopeParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t nw = (int64_t)gridDim.x * 4, wv = (int64_t)blockIdx.x * 4 + wave;
  const int64_t u0 = p.units * wv / nw, u1 = p.units * (wv + 1) / nw;
  float dw[2][kScalarSteps];
#pragma unroll
  for (int k = 0; k < kScalarSteps; ++k) dw[0][k] = dw[1][k] = 0.f;
  for (int64_t unit = u0; unit < u1; ++unit) {
    const int64_t tok = unit / p.groups;
    int h = (int)(unit % p.groups);
    const int si = h < p.side[0].groups ? 0 : 1;
    if (si == 1) h -= p.side[0].groups;
    const int b = (int)(tok / p.S), s = (int)(tok % p.S);
    const RopeSide& sd = p.side[si];
    const double pos = (double)load_int(p.pos, b * p.pos_sb + s * p.pos_ss, p.pos_i64);
    const T* dy = reinterpret_cast<const T*>(sd.y) + b * sd.y_sb + s * sd.y_ss + h * sd.y_sh;
    const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.x_sb + s * sd.x_ss + h * sd.x_sh;
    T* dx = reinterpret_cast<T*>(sd.dx) + b * sd.dx_sb + s * sd.dx_ss + h * sd.dx_sh;
    float du[kScalarSteps], v[kScalarSteps], q = 0.f, gx = 0.f;
#pragma unroll
    for (int k = 0; k < kScalarSteps; ++k) {
      const int d = lane + 64 * k;
      du[k] = v[k] = 0.f;
      if (d >= p.D) continue;
      float u = to_f32(dy[d]);
      int pd, i;
      float sgn;
      if (turn_of(p, d, pd, i, sgn)) {
        float c, sn;
        angle(pos, p.freq[i], c, sn);
        u = u * (c * p.rope_scale) - sgn * (to_f32(dy[pd]) * (sn * p.rope_scale));
      }
      du[k] = u;
      if (d < sd.n) {
        v[k] = to_f32(x[d]);
        q = fmaf(v[k], v[k], q);
        gx = fmaf(u * load_w<T>(p, sd.w, d), v[k], gx);
      }
    }
    float r = 0.f, m = 0.f;
    if (sd.n > 0) {
      r = 1.f / sqrtf(wave_sum(q) / (float)sd.n + p.eps);
      m = wave_sum(gx) * r / (float)sd.n;
    }
#pragma unroll
    for (int k = 0; k < kScalarSteps; ++k) {
      const int d = lane + 64 * k;
      if (d >= p.D) continue;
      float g = du[k];
      if (d < sd.n) {
        const float xh = v[k] * r;
        if (si == 0) dw[0][k] = fmaf(g, xh, dw[0][k]);
        else dw[1][k] = fmaf(g, xh, dw[1][k]);
        g = r * (g * load_w<T>(p, sd.w, d) - xh * m);
      }
      dx[d] = from_f32<T>(g);
    }
  }
  if (p.part == nullptr) return;
  __shared__ float s_w[4][kMaxD];
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int n = p.side[a].n;
#pragma unroll
    for (int k = 0; k < kScalarSteps; ++k) s_w[wave][lane + 64 * k] = dw[a][k];
    __syncthreads();
    for (int d = threadIdx.x; d < n; d += 256)
      p.part[((int64_t)a * gridDim.x + blockIdx.x) * kMaxD + d] = (s_w[0][d] + s_w[1][d]) + (s_w[2][d] + s_w[3][d]);
    __syncthreads();
  }
}

template <typename T>
void fwd(const RopeParams& p, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)((p.units + 3) / 4));
  if (!vec) rope_fwd_scalar_kernel<T><<<grid, 256, 0, s>>>(p);
  else if (p.K == 1) rope_fwd_kernel<T, 1><<<grid, 256, 0, s>>>(p);
  else if (p.K == 9) rope_fwd_kernel<T, 9><<<grid, 256, 0, s>>>(p);
  else rope_fwd_kernel<T, 4><<<grid, 256, 0, s>>>(p);
}

template <typename T>
void bwd(const RopeParams& p, bool vec, int wgs, hipStream_t s) {
  if (!vec) rope_bwd_scalar_kernel<T><<<wgs, 256, 0, s>>>(p);
  else if (p.K == 1) rope_bwd_kernel<T, 1><<<wgs, 256, 0, s>>>(p);
  else if (p.K == 9) rope_bwd_kernel<T, 9><<<wgs, 256, 0, s>>>(p);
  else rope_bwd_kernel<T, 4><<<wgs, 256, 0, s>>>(p);
  const int n = p.side[0].n > p.side[1].n ? p.side[0].n : p.side[1].n;
  if (n > 0) rope_dw_kernel<T><<<dim3((unsigned)((n + 15) / 16), 2), 1024, 0, s>>>(p, wgs);
}

}  // namespace

// Lanes per row, chunks per lane, row groups (see the kernels).
void rope_geometry(RopeParams& p, int esize, bool vec, bool backward) {
  const int E = 16 / esize;
  p.chunks = p.D / E;
  p.P = 64;
  p.K = 1;
  if (vec) {
    if (p.chunks == 72) {
      p.P = 8;
      p.K = 9;
    } else if (p.chunks > 64) {
      p.K = 4;  // up to 256 chunks: float32 rows of 1024 dims
    } else {
      p.P = 1;
      while (p.P < p.chunks) p.P *= 2;
    }
  }
  const int rpw = vec ? 64 / p.P : 1;
  for (int a = 0; a < 2; ++a) p.side[a].groups = (p.side[a].H + rpw - 1) / rpw;
  int vg = 0;
  if (p.v != nullptr) vg = vec ? (p.side[1].H * (p.Dv / E) + 63) / 64 : p.side[1].H;
  p.groups = p.side[0].groups + p.side[1].groups + vg;
  const int64_t toks = (int64_t)p.B * p.S, all = toks * p.groups;
  p.per = 1;
  p.upt = p.groups;
  p.units = all;
  if (vec && !backward) {
    // enough row groups per wave to share a token's angles, once there are 8192 waves
    int64_t per = all / 8192;
    p.per = (int)(per < 1 ? 1 : per > p.groups ? p.groups : per);
    p.upt = (p.groups + p.per - 1) / p.per;
    p.units = toks * p.upt;
  }
}

// Workgroups of the backward: its partial dw rows are summed, so no more than
// fill the card.
int rope_bwd_wgs(const RopeParams& p) {
  const int64_t w = (p.units + 3) / 4;
  return (int)(w < 1 ? 1 : w > 1024 ? 1024 : w);
}

size_t rope_bwd_workspace(const RopeParams& p) {
  return p.side[0].n > 0 || p.side[1].n > 0 ? (size_t)2 * rope_bwd_wgs(p) * kMaxD * sizeof(float) : 0;
}

hipError_t launch_rope_fwd(const RopeParams& p, int dtype, bool vec, hipStream_t s) {
  if (dtype == SFA_DTYPE_F32) fwd<float>(p, vec, s);
  else fwd<bf16>(p, vec, s);
  return hipGetLastError();
}

hipError_t launch_rope_bwd(const RopeParams& p, int dtype, bool vec, hipStream_t s) {
  const int wgs = rope_bwd_wgs(p);
  if (dtype == SFA_DTYPE_F32) bwd<float>(p, vec, wgs, s);
  else bwd<bf16>(p, vec, wgs, s);
  return hipGetLastError();
}

}  // namespace sfa

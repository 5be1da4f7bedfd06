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
// dx written).  So a row is held in registers, in 16-byte chunks over P lanes
// (half layout over the whole row: two chunks a lane, so that partners meet in
// one lane and share their angles; 8 lanes of 9 chunks for the 576-dim latent
// row), 64 / P heads of one token per wave.  With one or two
// chunks a lane the token's angles are computed once per wave for all the heads
// that it takes (rows of 4 or 9 chunks a lane form them again for every row and
// rotated chunk: registers).  Rows that are not whole 16-byte chunks (odd dims,
// strides, offsets) take the scalar kernels, one wave a row.

#include "sfa_ops.h"

namespace sfa {
namespace {

constexpr double k2Pi4 = 0.63661977236758134307553505349006;  // 2 / pi: quarter turns per radian
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

// Positions, slots and tables through the scalar cache (no kernel here writes
// them): a vector load would wait for all the rows in flight before it.
template <typename I>
__device__ __forceinline__ I load_const(const I* at) {
  return *(const __attribute__((address_space(4))) I*)at;
}
__device__ __forceinline__ int64_t load_int(const void* base, int64_t i, int is64) {
  return is64 ? load_const(reinterpret_cast<const int64_t*>(base) + i)
              : (int64_t)load_const(reinterpret_cast<const int32_t*>(base) + i);
}

// cos and sin of pos * f.  The angle is reduced in float64 to quarter turns q
// and a rest r of at most half a quarter; sin and cos of the rest, x = r pi / 2
// with |x| <= pi / 4, are their Taylor polynomials (the first term left out is
// x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10).
__device__ __forceinline__ void angle(double pos, double f, float& c, float& s) {
  const double u = pos * (f * k2Pi4);
  const double q = rint(u);
  const int n = (int)(q - 4.0 * rint(0.25 * q));  // the quarter, -2 .. 2
  const float x = (float)(u - q) * 1.57079632679489662f, x2 = x * x;
  float a = fmaf(x2, 1.f / 362880.f, -1.f / 5040.f);
  a = fmaf(x2, a, 1.f / 120.f);
  a = fmaf(x2, a, -1.f / 6.f);
  const float sx = fmaf(x * x2, a, x);
  float d = fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f);
  d = fmaf(x2, d, -1.f / 720.f);
  d = fmaf(x2, d, 1.f / 24.f);
  d = fmaf(x2, d, -0.5f);
  const float cx = fmaf(x2, d, 1.f);
  const float s0 = n & 1 ? cx : sx, c0 = n & 1 ? sx : cx;
  s = n & 2 ? -s0 : s0;
  c = (n + 1) & 2 ? -c0 : c0;
}

template <typename T>
__device__ __forceinline__ float load_w(const RopeParams& p, const void* w, int d) {
  return p.w_f32 ? reinterpret_cast<const float*>(w)[d] : to_f32(reinterpret_cast<const T*>(w)[d]);
}

// Sum over the P lanes of a row (lane permutations of the VALU, no LDS trips).
template <int C>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), C, 0xf, 0xf, true));
}
template <int P>
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<0xb1>(x);                          // lane ^ 1
  x += dpp<0x4e>(x);                          // lane ^ 2
  if constexpr (P >= 8) x += dpp<0x141>(x);   // mirror of 8
  if constexpr (P >= 16) x += dpp<0x140>(x);  // mirror of 16
  if constexpr (P >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (P >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
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
  __device__ __forceinline__ void freqs(const RopeParams& p, double (&f)[E]) const {
    each<E>([&](auto ec) {
      constexpr int e = decltype(ec)::value;
      f[e] = on && (e < E / 2 || !p.interleaved) ? p.freq[i0 + e] : 0.0;
    });
  }
  __device__ __forceinline__ void angles(const RopeParams& p, double pos, const double (&f)[E], float (&cs)[E],
                                         float (&sn)[E]) const {
    const float sc = p.rope_scale;
    each<E>([&](auto ec) {
      constexpr int e = decltype(ec)::value;
      float c = 1.f, s = 0.f;
      if (e < E / 2 || !p.interleaved) angle(pos, f[e], c, s);
      cs[e] = c * sc;
      sn[e] = s * sc;
    });
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
  const int pg = load_const(p.block_table + b * p.bt_sb + (slot >> p.page_shift));
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * page_stride + (slot & ((1 << p.page_shift) - 1)) * row_stride;
}

// A row's chunks: lane l of its P lanes holds chunks l, l + P, ..  IN: half
// layout over the whole row in two chunks a lane, so a lane holds both partners;
// else partners are another lane's chunk (K = 1) or read again (K > 2).
template <typename T, int P, int K, bool IN>
struct Row {
  static constexpr int E = Chunk<T>::E;
  static constexpr bool kHeld = IN || K == 1;  // the lane's angles serve all its rows
  u32x4 r[K];
  // (chunks past dim n > 0: the first one again, so that the number of loads in
  // flight does not depend on the lane)
  __device__ __forceinline__ void load(const RopeParams& p, const T* x, int l, int n) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      r[j] = *reinterpret_cast<const u32x4*>(x + (c * E < n ? c * E : 0));
    }
  }
  __device__ __forceinline__ void store(const RopeParams& p, T* y, int l) const {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      if (c >= p.chunks) continue;
      *reinterpret_cast<u32x4*>(y + c * E) = r[j];
    }
  }
  // u(j, own, partner) replaces chunk j by its turned values: pre() makes u of
  // the raw chunk c of this row
  template <class Pre, class Put>
  __device__ __forceinline__ void turn(const RopeParams& p, const T* x, int lane, double pos, const float (&cs)[E],
                                       const float (&sn)[E], float dir, Pre pre, Put put) const {
    const int l = lane & (P - 1);
    if constexpr (IN) {
      float a[E], b[E];
      Chunk<T>::unpack(r[0], a);
      Chunk<T>::unpack(r[1], b);
      pre(0, l, a);
      pre(1, l + P, b);
      float ya[E], yb[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float sd = dir * sn[e];
        ya[e] = a[e] * cs[e] - b[e] * sd;
        yb[e] = b[e] * cs[e] + a[e] * sd;
      }
      put(0, l, ya);
      put(1, l + P, yb);
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if constexpr (K > 2) __builtin_amdgcn_sched_barrier(0);  // (chunk by chunk: registers)
        const int c = j * P + l;
        const Turn<E> t(p, c);
        float u[E], o[E];
        Chunk<T>::unpack(r[j], u);
        pre(j, c, u);
        u32x4 other = {0, 0, 0, 0};
        if (!p.interleaved) {
          if constexpr (K == 1) {
            other = shfl16(r[0], (lane & ~(P - 1)) + t.pair);
          } else {
            if (t.on) other = *reinterpret_cast<const u32x4*>(x + t.pair * E);
          }
        }
        Chunk<T>::unpack(other, o);
        if (!p.interleaved && t.on) pre(K, t.pair, o);
        if constexpr (K == 1) {
          t.apply(p, u, o, cs, sn, dir);
        } else if (t.on) {
          double f2[E];
          float c2[E], s2[E];
          t.freqs(p, f2);
          t.angles(p, pos, f2, c2, s2);
          t.apply(p, u, o, c2, s2, dir);
        }
        put(j, c, u);
      }
    }
  }
};

// The weights of a whole chunk.
template <typename T>
__device__ __forceinline__ void load_chunk_w(const RopeParams& p, const void* w, int c, float (&f)[Chunk<T>::E]) {
  constexpr int E = Chunk<T>::E;
  if (p.w_f32) {
    const float* at = reinterpret_cast<const float*>(w) + c * E;
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(at + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * q + e] = x[e];
    }
  } else {
    Chunk<T>::unpack(*reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(w) + c * E), f);
  }
}
// The weights of the chunks a lane holds (index K: of its partner chunk); rows
// of many chunks read them again for each row.
template <typename T, int P, int K, bool IN>
struct Weights {
  static constexpr int E = Chunk<T>::E;
  static constexpr bool kRegs = K <= 2;
  float w[kRegs ? K + 1 : 1][E];
  __device__ __forceinline__ void load(const RopeParams& p, const RopeSide& sd, int l) {
    if constexpr (kRegs) {
#pragma unroll
      for (int j = 0; j < (IN ? K : K + 1); ++j) {
        const int c = j < K ? j * P + l : Turn<E>(p, l).pair;
#pragma unroll
        for (int e = 0; e < E; ++e) w[j][e] = 1.f;
        if (c * E < sd.n) load_chunk_w<T>(p, sd.w, c, w[j]);
      }
    }
  }
  __device__ __forceinline__ void chunk(const RopeParams& p, const RopeSide& sd, int j, int c, float (&f)[E]) const {
    if constexpr (kRegs) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = w[j][e];
    } else {
      load_chunk_w<T>(p, sd.w, c, f);
    }
  }
};

// A wave's walk over (token, row group) units: blocks of `per` groups of a
// token (p.per, p.upt blocks a token), every nw-th block, so that the waves of the
// card read one window of the tensor at a time.
struct Walk {
  uint32_t blk, nblk, nw;
  int b, s, g, g1;
  __device__ __forceinline__ void at(const RopeParams& p, int groups, int per, int upt) {
    const uint32_t tok = blk / (uint32_t)upt;
    b = (int)(tok / (uint32_t)p.S);
    s = (int)(tok - (uint32_t)b * (uint32_t)p.S);
    g = (int)(blk - tok * (uint32_t)upt) * per;
    g1 = min(g + per, groups);
  }
  __device__ __forceinline__ bool live() const { return blk < nblk; }
  // the next unit; fresh: of another block (another token's, perhaps).  Past the
  // last one the walk is not live and stays at it: its addresses remain good.
  __device__ __forceinline__ bool next(const RopeParams& p, int groups, int per, int upt) {
    if (++g < g1) return false;
    blk += nw;
    if (blk < nblk) at(p, groups, per, upt);
    else g = g1 - 1;
    return true;
  }
};

// Forward.  The units are (token, row group): the q heads' groups (64 / P rows
// each), the k heads', then (append) 64-chunk groups of the v row.  NB units are
// in flight, each in registers of its own that are refilled as soon as its
// results are stored: the next unit's rows handed on from register to register
// are waited for at the copy.  So 8192 tokens of 128 rows of 64 dims take 90 us
// for 162 (caches flushed before the call; a copy of the same rows 81), 2 x 8192
// tokens of 34 normed heads of 128 dims 91 for 119 (285 MB); on inputs that the
// last pass left in the caches 73 and 70.  More in flight gains nothing
// (NB 4 and 6, or 3 of rows in two chunks: 93, 95 us; 112).  Calls of one unit a wave take
// NB = 1 (8.8 us for 11, 64 tokens into the cache: less code to fetch).
template <typename T, int P, int K, bool IN, int NB>
__global__ __launch_bounds__(256, K == 9 ? 2 : K > 2 ? 3 : 4) void rope_fwd_kernel(RopeParams p) {
  typedef Row<T, P, K, IN> R;
  constexpr int E = R::E, rpw = 64 / P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l = lane & (P - 1), rr = lane / P;
  Walk w;
  w.nw = gridDim.x * 4;
  w.blk = blockIdx.x * 4 + wave;
  w.nblk = (uint32_t)p.B * (uint32_t)p.S * (uint32_t)p.upt;
  if (!w.live()) return;
  w.at(p, p.groups, p.per, p.upt);
  const int gq = p.side[0].groups, gk = gq + p.side[1].groups;

  struct Unit {
    R x;
    const T* px;
    T* py;
    int64_t pos;
    int g;
    bool live, fresh, put;
  };
  bool fresh = true;
  auto fill = [&](Unit& u) __attribute__((always_inline)) {  // the walk's unit (past its end: the last one, again)
    u.live = w.live();
    u.fresh = fresh;
    u.g = w.g;
    u.pos = load_int(p.pos, w.b * p.pos_sb + w.s * p.pos_ss, p.pos_i64);
    int64_t yo;
    if (w.g >= gk) {  // of the v row: 64 chunks
      const int i = (w.g - gk) * 64 + lane, cpr = p.Dv / E;
      const bool in = i < p.side[1].H * cpr;
      const int h = in ? i / cpr : 0, c = in ? i % cpr : 0;
      u.px = reinterpret_cast<const T*>(p.v) + w.b * p.v_sb + w.s * p.v_ss + h * p.v_sh + c * E;
#pragma unroll
      for (int j = 0; j < K; ++j) u.x.r[j] = *reinterpret_cast<const u32x4*>(u.px);
      yo = cache_row(p, w.b, w.s, p.vo_sb, p.vo_ss);
      u.put = in && yo >= 0;
      u.py = reinterpret_cast<T*>(p.v_out) + yo + h * p.vo_sh + c * E;
    } else {
      const int si = w.g < gq ? 0 : 1;
      const RopeSide& sd = p.side[si];
      const int h = (si == 0 ? w.g : w.g - gq) * rpw + rr;
      const int64_t hh = h < sd.H ? h : 0;
      u.px = reinterpret_cast<const T*>(sd.x) + w.b * sd.x_sb + w.s * sd.x_ss + hh * sd.x_sh;
      u.x.load(p, u.px, l, p.D);
      if (si == 1 && p.block_table != nullptr) yo = cache_row(p, w.b, w.s, sd.y_sb, sd.y_ss);
      else yo = w.b * sd.y_sb + w.s * sd.y_ss;
      u.put = h < sd.H && yo >= 0;
      u.py = reinterpret_cast<T*>(sd.y) + yo + hh * sd.y_sh;
    }
    if (u.live) fresh = w.next(p, p.groups, p.per, p.upt);
  };
  double freq[E];
  float cs[E], sn[E];
  const Turn<E> lt(p, l);
  if constexpr (R::kHeld) lt.freqs(p, freq);
  Weights<T, P, K, IN> wt[R::kHeld ? 2 : 1];
  if constexpr (R::kHeld) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
      if (p.side[a].n > 0) wt[a].load(p, p.side[a], l);
  }
  auto work = [&](Unit& u) __attribute__((always_inline)) {
    const double pos = (double)u.pos;
    if constexpr (R::kHeld) {
      if (u.fresh) lt.angles(p, pos, freq, cs, sn);
    }
    if (u.g >= gk) {  // v is copied
      if (u.put) *reinterpret_cast<u32x4*>(u.py) = u.x.r[0];
      return;
    }
    const int si = u.g < gq ? 0 : 1;
    const RopeSide& sd = p.side[si];
    float r = 1.f;
    if (sd.n > 0) {
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        float f[E];
        Chunk<T>::unpack(u.x.r[j], f);
        float q4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) q4[e & 3] = fmaf(f[e], f[e], q4[e & 3]);
        if ((j * P + l) * E < sd.n) q += (q4[0] + q4[1]) + (q4[2] + q4[3]);
      }
      r = 1.f / sqrtf(row_sum<P>(q) / (float)sd.n + p.eps);
    }
    u.x.turn(
        p, u.px, lane, pos, cs, sn, 1.f,
        [&](int j, int c, float (&v)[E]) {
          if (c * E < sd.n) {
            float wc[E];
            if constexpr (R::kHeld) {
              float w0[E], w1[E];
              wt[0].chunk(p, sd, j, c, w0);
              wt[1].chunk(p, sd, j, c, w1);
#pragma unroll
              for (int e = 0; e < E; ++e) wc[e] = si == 0 ? w0[e] : w1[e];
            } else {
              wt[0].chunk(p, sd, j, c, wc);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = v[e] * r * wc[e];
          }
        },
        [&](int j, int c, const float (&v)[E]) { u.x.r[j] = Chunk<T>::pack(v); });
    // (every value of the row has been read: y may be x)
    if (u.put) u.x.store(p, u.py, l);
  };
  Unit u[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) fill(u[i]);
  bool more = true;
  while (more) {
    each<NB>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      more = more && u[i].live;
      if (!more) return;
      work(u[i]);
      if (NB == 1 && !w.live()) more = false;
      else fill(u[i]);
    });
  }
}

// Backward of one tensor (blockIdx.y: q or k): side.y is dy, side.dx receives
// dx.  A wave walks over units as in the forward, NB of them in flight, and sums
// its rows' dw in registers; a workgroup writes its sums to partial row
// blockIdx.x, which rope_dw_kernel adds up in order.  NORM: some side is normed.
// (The sizes above, caches flushed: 54 us with NB = 2 for 64, and 109 us, 428 MB,
// with NB = 1, where x and dy keep four loads a lane in flight, 124 with 2; warm
// 49 and 102.)
template <typename T, int P, int K, bool IN, bool NORM, int NB>
__global__ __launch_bounds__(256) void rope_bwd_kernel(RopeParams p) {
  typedef Row<T, P, K, IN> R;
  constexpr int E = R::E, rpw = 64 / P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l = lane & (P - 1), rr = lane / P;
  const int si = blockIdx.y;
  const RopeSide& sd = p.side[si];
  if (sd.H == 0) return;
  const int per = p.per < sd.groups ? p.per : sd.groups, upt = (sd.groups + per - 1) / per;
  Walk w;
  w.nw = gridDim.x * 4;
  w.blk = blockIdx.x * 4 + wave;
  w.nblk = (uint32_t)p.B * (uint32_t)p.S * (uint32_t)upt;

  Weights<T, P, K, IN> wt;
  if (sd.n > 0) wt.load(p, sd, l);
  double freq[E];
  float cs[E], sn[E];
  const Turn<E> lt(p, l);
  if constexpr (R::kHeld) lt.freqs(p, freq);
  float dw[K][E];
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[j][e] = 0.f;

  struct Unit {
    R dy, x;
    const T* py;
    T* px;
    int64_t pos;
    bool on, fresh, live;  // on: a unit of the walk; live: the lane's row is one
  };
  bool fresh = true;
  auto fill = [&](Unit& u) __attribute__((always_inline)) {  // the walk's unit (past its end: the last one, again)
    u.on = w.live();
    u.fresh = fresh;
    u.pos = load_int(p.pos, w.b * p.pos_sb + w.s * p.pos_ss, p.pos_i64);
    const int h = w.g * rpw + rr;
    u.live = h < sd.H;
    const int64_t hh = u.live ? h : 0;
    u.py = reinterpret_cast<const T*>(sd.y) + w.b * sd.y_sb + w.s * sd.y_ss + hh * sd.y_sh;
    u.px = reinterpret_cast<T*>(sd.dx) + w.b * sd.dx_sb + w.s * sd.dx_ss + hh * sd.dx_sh;
    u.dy.load(p, u.py, l, p.D);
    if constexpr (NORM) {  // (a side without a norm: dy again)
      const T* x = sd.n > 0 ? reinterpret_cast<const T*>(sd.x) + w.b * sd.x_sb + w.s * sd.x_ss + hh * sd.x_sh : u.py;
      u.x.load(p, x, l, sd.n > 0 ? sd.n : p.D);
    }
    if (u.on) fresh = w.next(p, sd.groups, per, upt);
  };
  auto work = [&](Unit& u) __attribute__((always_inline)) {
    const double pos = (double)u.pos;
    if constexpr (R::kHeld) {
      if (u.fresh) lt.angles(p, pos, freq, cs, sn);
    }
    float du[K][E];
    float q = 0.f, gx = 0.f;  // sum x^2, sum (du w) x
    u.dy.turn(
        p, u.py, lane, pos, cs, sn, -1.f, [](int, int, float (&)[E]) {},
        [&](int j, int c, const float (&v)[E]) {
#pragma unroll
          for (int e = 0; e < E; ++e) du[j][e] = v[e];
          if constexpr (NORM) {
            if (c * E < sd.n) {
              float x[E], wc[E];
              Chunk<T>::unpack(u.x.r[j], x);
              wt.chunk(p, sd, j, c, wc);
              float q2[2] = {0.f, 0.f}, g2[2] = {0.f, 0.f};
#pragma unroll
              for (int e = 0; e < E; ++e) {
                q2[e & 1] = fmaf(x[e], x[e], q2[e & 1]);
                g2[e & 1] = fmaf(v[e] * wc[e], x[e], g2[e & 1]);
              }
              q += q2[0] + q2[1];
              gx += g2[0] + g2[1];
            }
          }
        });
    R res;
    float r = 0.f, m = 0.f;  // 1 / rms, mean of (du w) xhat
    if (NORM && sd.n > 0) {
      r = 1.f / sqrtf(row_sum<P>(q) / (float)sd.n + p.eps);
      m = row_sum<P>(gx) * r / (float)sd.n;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = j * P + l;
      if constexpr (NORM) {
        if (c * E < sd.n) {
          float x[E], wc[E];
          Chunk<T>::unpack(u.x.r[j], x);
          wt.chunk(p, sd, j, c, wc);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float xh = x[e] * r, d = du[j][e];
            dw[j][e] = fmaf(u.live ? d : 0.f, xh, dw[j][e]);
            du[j][e] = r * (d * wc[e] - xh * m);
          }
        }
      }
      res.r[j] = Chunk<T>::pack(du[j]);
    }
    if (u.live) res.store(p, u.px, l);
  };
  if (w.live()) {
    w.at(p, sd.groups, per, upt);
    Unit u[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) fill(u[i]);
    bool more = true;
    while (more) {
      each<NB>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        more = more && u[i].on;
        if (!more) return;
        work(u[i]);
        if (NB == 1 && !w.live()) more = false;
        else fill(u[i]);
      });
    }
  }

  if (p.part == nullptr || sd.n == 0) return;
  // dw of the workgroup: the row groups of a wave by shuffles, then the waves
  __shared__ float s_w[4][kMaxD];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int c = j * P + l;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float x = dw[j][e];
#pragma unroll
      for (int o = P; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
      if (rr == 0 && c * E < sd.n) s_w[wave][c * E + e] = x;
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < sd.n; d += 256)
    p.part[((int64_t)si * gridDim.x + blockIdx.x) * kMaxD + d] = (s_w[0][d] + s_w[1][d]) + (s_w[2][d] + s_w[3][d]);
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

// (rows from unit `first` on; a loop over them in the kernel held 135 registers
// and scratch for 88)
template <typename T>
__global__ __launch_bounds__(256) void rope_fwd_scalar_kernel(RopeParams p, int64_t first) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = first + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
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

// Workgroups of 4 waves for so many units: no more than stay on the card.
constexpr int kWaves = 4096;
int rope_wgs(int64_t units) {
  const int64_t w = (units + 3) / 4;
  return (int)(w < 1 ? 1 : w > kWaves / 4 ? kWaves / 4 : w);
}

// The kernel of a geometry: f.template operator()<P, K, IN>()
template <class F>
void by_geometry(const RopeParams& p, F f) {
  if (p.K == 2) {
    if (p.P == 4) f.template run<4, 2, true>();
    else if (p.P == 8) f.template run<8, 2, true>();
    else if (p.P == 16) f.template run<16, 2, true>();
    else f.template run<32, 2, true>();
  } else if (p.K == 1) {
    if (p.P == 8) f.template run<8, 1, false>();
    else if (p.P == 16) f.template run<16, 1, false>();
    else if (p.P == 32) f.template run<32, 1, false>();
    else f.template run<64, 1, false>();
  } else if (p.K == 9) {
    f.template run<8, 9, false>();
  } else {
    f.template run<64, 4, false>();
  }
}
template <typename T>
struct Fwd {
  const RopeParams& p;
  hipStream_t s;
  template <int P, int K, bool IN>
  void run() const {
    constexpr int NB = K == 1 ? 3 : K == 2 ? 2 : 1;
    const unsigned grid = (unsigned)rope_wgs(p.units);
    if (NB > 1 && p.units > kWaves) rope_fwd_kernel<T, P, K, IN, NB><<<grid, 256, 0, s>>>(p);
    else rope_fwd_kernel<T, P, K, IN, 1><<<grid, 256, 0, s>>>(p);
  }
};
template <typename T>
struct Bwd {
  const RopeParams& p;
  int wgs;
  hipStream_t s;
  template <int P, int K, bool IN, int NB>
  void launch(dim3 grid) const {
    if (p.side[0].n > 0 || p.side[1].n > 0) rope_bwd_kernel<T, P, K, IN, true, NB><<<grid, 256, 0, s>>>(p);
    else rope_bwd_kernel<T, P, K, IN, false, NB><<<grid, 256, 0, s>>>(p);
  }
  template <int P, int K, bool IN>
  void run() const {
    const dim3 grid((unsigned)wgs, p.side[1].H > 0 ? 2 : 1);
    constexpr int NB = K == 1 ? 2 : 1;
    if (NB > 1 && p.units > kWaves) launch<P, K, IN, NB>(grid);
    else launch<P, K, IN, 1>(grid);
  }
};

template <typename T>
void fwd(const RopeParams& p, bool vec, hipStream_t s) {
  if (vec) {
    by_geometry(p, Fwd<T>{p, s});
    return;
  }
  constexpr int64_t kMost = (int64_t)1 << 23;  // workgroups: a launch has fewer than 2^32 threads
  for (int64_t first = 0; first < p.units; first += 4 * kMost) {
    const int64_t wgs = (p.units - first + 3) / 4;
    rope_fwd_scalar_kernel<T><<<(unsigned)(wgs < kMost ? wgs : kMost), 256, 0, s>>>(p, first);
  }
}

template <typename T>
void bwd(const RopeParams& p, bool vec, int wgs, hipStream_t s) {
  if (!vec) rope_bwd_scalar_kernel<T><<<wgs, 256, 0, s>>>(p);
  else by_geometry(p, Bwd<T>{p, wgs, s});
  const int n = p.side[0].n > p.side[1].n ? p.side[0].n : p.side[1].n;
  if (n > 0) rope_dw_kernel<T><<<dim3((unsigned)((n + 15) / 16), 2), 1024, 0, s>>>(p, wgs);
}

}  // namespace

// Lanes per row, chunks per lane, row groups (see the kernels).
void rope_geometry(RopeParams& p, int esize, bool vec) {
  const int E = 16 / esize;
  p.chunks = p.D / E;
  p.P = 64;
  p.K = 1;
  if (vec) {
    const bool pow2 = (p.chunks & (p.chunks - 1)) == 0;
    if (!p.interleaved && p.off == 0 && p.R == p.D && pow2 && p.chunks >= 8 && p.chunks <= 64) {
      p.P = p.chunks / 2;  // both partners in one lane
      p.K = 2;
    } else if (p.chunks == 72) {
      p.P = 8;
      p.K = 9;
    } else if (p.chunks > 64) {
      p.K = 4;  // up to 256 chunks: float32 rows of 1024 dims
    } else {
      p.P = 8;
      while (p.P < p.chunks) p.P *= 2;
    }
  }
  const int rpw = vec ? 64 / p.P : 1;
  for (int a = 0; a < 2; ++a) p.side[a].groups = (p.side[a].H + rpw - 1) / rpw;
  int vg = 0;
  if (p.v != nullptr) vg = vec ? (p.side[1].H * (p.Dv / E) + 63) / 64 : p.side[1].H;
  p.groups = p.side[0].groups + p.side[1].groups + vg;
  p.units = (int64_t)p.B * p.S * p.groups;
  // blocks of up to 8 groups (a token's angles serve them) once there are 4096 waves of them
  const int64_t per = p.units / kWaves;
  p.per = (int)(per < 1 ? 1 : per > 8 ? 8 : per);
  if (p.per > p.groups) p.per = p.groups;
  p.upt = (p.groups + p.per - 1) / p.per;
}

// Workgroups of the backward: its partial dw rows are summed, so no more than
// fill the card.
int rope_bwd_wgs(const RopeParams& p) {
  const int g = p.side[0].groups > p.side[1].groups ? p.side[0].groups : p.side[1].groups;
  return rope_wgs((int64_t)p.B * p.S * g);
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

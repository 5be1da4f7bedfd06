// Rows of any type and stride of the float32 dense attention kernels, their query rows, and the
// chunks of their dk / dv kernels.
#pragma once

#include "sfa_dense.h"

namespace sfa {

constexpr int kE = 1 << kAnyShift;  // entries a tile
static_assert(kE == 32 && kAnyRows == 64, "four waves of 16 columns, two 16-entry products");

// dims d .. d + 3 of a row of D, zeros past its end
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int d, int D, bool vec) {
  f32x4 r = {};
  if (vec) {  // (whole rows of 4)
    if (d < D) {
      if constexpr (sizeof(T) == 4) {
        r = *reinterpret_cast<const f32x4*>(p + d);
      } else if constexpr (sizeof(T) == 2) {
        const bf16x4 x = *reinterpret_cast<const bf16x4*>(p + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (float)x[e];
      } else {
        const int x = *reinterpret_cast<const int*>(p + d);
        r = f32x4{__builtin_amdgcn_cvt_f32_fp8(x, 0), __builtin_amdgcn_cvt_f32_fp8(x, 1), __builtin_amdgcn_cvt_f32_fp8(x, 2),
                  __builtin_amdgcn_cvt_f32_fp8(x, 3)};
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < D) r[e] = value_of(p[d + e]);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int d, int D, bool vec, const f32x4& x) {
  if (vec && d < D) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(p + d) = x;
    else *reinterpret_cast<bf16x4*>(p + d) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < D) p[d + e] = from_f32<T>(x[e]);
  }
}

// Query row r of (b, g) as a column.
struct QRow {
  int t, h, pos;  // pos: -1: no such row, or a token past the sequence's
  bool in;        // a row of the tensor
};
__device__ __forceinline__ QRow q_row(const DenseParams& p, const DenseSeq& s, int g, int r) {
  QRow x;
  x.t = r / p.G;
  x.h = g * p.G + r % p.G;
  x.in = r < p.S * p.G;
  x.pos = x.in && x.t < s.n ? s.ctx + x.t : -1;
  return x;
}

// A tile that all rows of the block see whole (rows that are not there aside).
__device__ __forceinline__ bool whole_tile(const DenseParams& p, const DenseItem& it, int j0) {
  const int p0 = it.s.ctx + it.row0 / p.G, p1 = it.s.ctx + min((it.row0 + p.rows - 1) / p.G, it.s.n - 1);
  return j0 + kE - 1 <= p0 && (j0 + kE <= p.first || p1 - j0 < p.window);
}

// dk and dv: 64 keys a workgroup, whose rows (of all heads, tokens that see one of the keys) are
// one range, cut in chunks of p.chunk where there are few workgroups; several leave partial
// sums that dense_any_join_kernel adds in order.
struct KeyBlock {
  int b, g, kb, c;  // chunk
  DenseSeq s;
  int r0, r1;       // its rows
  int nc;           // chunks of the block
  float* part;      // the block's first partial sums: [chunk][64][Dqk + Dv]
};
__device__ __forceinline__ bool key_block(const DenseParams& p, int wi, KeyBlock& x) {
  x.c = wi % p.dkv_parts;
  wi /= p.dkv_parts;
  x.g = wi % p.Hkv;
  wi /= p.Hkv;
  x.b = wi % p.B;
  x.kb = wi / p.B;  // (the first keys, which the most rows see, first)
  x.s = dense_seq(p, x.b);
  const int j0 = x.kb * kAnyRows;
  const int t1 = j0 < p.first ? x.s.n : (int)min((int64_t)x.s.n, (int64_t)j0 + kAnyRows - 1 + p.window);
  const int rows = max(t1 - j0, 0) * p.G;
  x.nc = (int)(((int64_t)rows + p.chunk - 1) / p.chunk);
  x.r0 = j0 * p.G + x.c * p.chunk;
  x.r1 = j0 * p.G + (int)min((int64_t)rows, (int64_t)(x.c + 1) * p.chunk);
  const int64_t nkb = (p.S + kAnyRows - 1) / kAnyRows;
  x.part = p.dkv_part + (((int64_t)x.b * p.Hkv + x.g) * nkb + x.kb) * p.dkv_parts * kAnyRows * (p.Dqk + p.Dv);
  return x.c < max(x.nc, 1);
}

// A lane's key (the in-th of its block), dims d0 + 16 i + 4 hq + 0 .. 3.
template <typename T, int N>
__device__ __forceinline__ void store_dkv(const DenseParams& p, const KeyBlock& x, int in, int d0, const f32x4 (&dk)[N],
                                          const f32x4 (&dv)[N], int hq) {
  const int j = x.kb * kAnyRows + in;
  float* part = x.part + ((int64_t)x.c * kAnyRows + in) * (p.Dqk + p.Dv);
  T* ok = reinterpret_cast<T*>(p.dk) + x.b * p.dk_sb + j * p.dk_ss + x.g * p.dk_sh;
  T* ov = reinterpret_cast<T*>(p.dv) + x.b * p.dv_sb + j * p.dv_ss + x.g * p.dv_sh;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = d0 + 16 * i + 4 * hq;
    if (x.nc > 1) {
      store4(part, d, p.Dqk, p.vec, dk[i]);
      store4(part + p.Dqk, d, p.Dv, p.vec, dv[i]);
    } else if (j < p.S) {
      store4(ok, d, p.Dqk, p.vec, dk[i] * p.scale);
      store4(ov, d, p.Dv, p.vec, dv[i]);
    }
  }
}

}  // namespace sfa

// gfx950: rows of a paged cache as contiguous ones, 8-bit rows as the values they
// stand for (e4m3 times a power of two: exact in bf16 and float32).
//
// Bound: HBM, a row read once and written once (655 MB in 139 us, 4.7 TB/s; a copy: 5.14).  A wave takes whole rows (all heads of
// a token), 8 elements a lane, L lanes a row.

#include "sfa_ops.h"

namespace sfa {
namespace {

template <typename T>
__device__ __forceinline__ void read8(const T* p, float scale, float (&f)[8]) {
  if constexpr (sizeof(T) == 1) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i + 0] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * scale;
      f[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * scale;
      f[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * scale;
      f[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * scale;
    }
  } else if constexpr (sizeof(T) == 2) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)x[i];
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * h + i] = x[i];
    }
  }
}
template <typename T>
__device__ __forceinline__ void write8(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<bf16x8*>(p) = bf16x8{(bf16)f[0], (bf16)f[1], (bf16)f[2], (bf16)f[3],
                                           (bf16)f[4], (bf16)f[5], (bf16)f[6], (bf16)f[7]};
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
  }
}
// VEC: 8 elements of a head at a time, else one.
template <typename TI, typename TO, bool VEC>
__global__ __launch_bounds__(256) void cache_read_kernel(ReadParams p, int L) {
  const int lane = threadIdx.x & 63, b = blockIdx.y;
  const int i = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / L) + lane / L;
  if (i >= p.N) return;
  const int64_t at = (p.starts != nullptr ? (int64_t)p.starts[b] : 0) + i;
  int pg = -1;
  if (at >= 0 && at < p.lens[b] && at < (int64_t)p.max_pages << p.page_shift) pg = p.block_table[b * p.bt_sb + (at >> p.page_shift)];
  const bool there = pg >= 0 && pg < p.num_pages;
  const int64_t in = at & ((1 << p.page_shift) - 1);
  const TI* src = reinterpret_cast<const TI*>(p.cache) + (there ? pg * p.c_sb + in * p.c_ss : 0);
  const uint8_t* sc = sizeof(TI) == 1 && there ? p.scale + pg * p.s_sb + in * p.s_ss : nullptr;
  TO* dst = reinterpret_cast<TO*>(p.out) + b * p.o_sb + i * p.o_ss;
  constexpr int E = VEC ? 8 : 1;
  const int per = p.D / E, n = p.H * per;
  for (int c = lane % L; c < n; c += L) {
    const int h = c / per, d = (c - h * per) * E;
    float scale = 1.f;
    if (sizeof(TI) == 1 && there) scale = scale_of(sc[h * p.s_sh]);
    if constexpr (VEC) {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (there) read8(src + h * p.c_sh + d, scale, f);
      write8(dst + h * p.o_sh + d, f);
    } else {
      dst[h * p.o_sh + d] = from_f32<TO>(there ? value_of(src[h * p.c_sh + d]) * scale : 0.f);
    }
  }
}

template <typename TI, typename TO>
void launch(const ReadParams& p, bool vec, hipStream_t s) {
  const int n = p.H * (vec ? p.D / 8 : p.D);
  int L = 1;
  while (L < 64 && L < n) L *= 2;
  const int per = 4 * (64 / L);
  const dim3 grid((unsigned)((p.N + per - 1) / per), (unsigned)p.B);
  if (vec) cache_read_kernel<TI, TO, true><<<grid, 256, 0, s>>>(p, L);
  else cache_read_kernel<TI, TO, false><<<grid, 256, 0, s>>>(p, L);
}
template <typename TO>
void launch_to(const ReadParams& p, int cache_dtype, bool vec, hipStream_t s) {
  if (cache_dtype == SFA_DTYPE_FP8_E4M3) launch<fp8_t, TO>(p, vec, s);
  else if (cache_dtype == SFA_DTYPE_BF16) launch<bf16, TO>(p, vec, s);
  else launch<float, TO>(p, vec, s);
}

}  // namespace

hipError_t launch_cache_read(const ReadParams& p, int dtype, int cache_dtype, bool vec, hipStream_t s) {
  if (dtype == SFA_DTYPE_F32) launch_to<float>(p, cache_dtype, vec, s);
  else launch_to<bf16>(p, cache_dtype, vec, s);
  return hipGetLastError();
}

}  // namespace sfa

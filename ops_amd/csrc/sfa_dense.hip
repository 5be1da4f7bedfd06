// gfx950 dense attention through a window (sfa_dense.h): the choice of kernels,
// the joining of key ranges, and the backward's row sums.

#include "sfa_dense.h"

namespace sfa {
namespace {

// ---- joining the ranges of a row block -------------------------------------------
// A workgroup takes jr rows of a unit, one wave a row; LPR lanes hold it (4 dims each),
// 64 / LPR ranges at a time, jd dims.  A range in which the row sees nothing has LSE -inf.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void dense_combine_kernel(DenseParams p, int jr, int jd) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunks = (p.rows + jr - 1) / jr;
  int wi = blockIdx.x;
  const int row0 = wi % chunks * jr;
  wi /= chunks;
  const int nd = (p.Dv + jd - 1) / jd, dim0 = wi % nd * jd;
  wi /= nd;
  const int g = wi % p.Hkv, u = wi / p.Hkv;
  const int first = p.unit_slots[2 * u], ns = p.unit_slots[2 * u + 1];
  if (ns <= 1) return;
  const int b = u / p.nrb;
  for (int row = row0 + wave; row < min(row0 + jr, p.rows); row += 4) {
    const int r = (u - b * p.nrb) * p.rows + row;
    if (r >= p.S * p.G) return;
    const int t = r / p.G, h = g * p.G + r % p.G;
    const int64_t per = (int64_t)p.Hkv * p.rows, at0 = ((int64_t)first * p.Hkv + g) * p.rows + row;
    const float* pl = p.part_lse + at0;
    const float* po = p.part_o + at0 * p.Dv;
    const bool live = t < dense_seq(p, b).n;
    float m = kNegInf, nan = 0.f;
    for (int k = lane; k < ns; k += 64) {
      const float x = pl[k * per];
      nan += x != x ? x : 0.f;
      m = fmaxf(m, x);
    }
    m = wave_max(m);
    const float moff = m == kNegInf ? 0.f : m;
    float l = 0.f;
    for (int k = lane; k < ns; k += 64) l += exp2f(pl[k * per] - moff);
    l = wave_sum(l + nan);
    float lse;
    const float f = dense_finish(p, h, live, m, l, lse);
    if (lane == 0 && dim0 == 0) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
    T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh;
    const int sub = lane / LPR;
    for (int d0 = dim0; d0 < min(dim0 + jd, p.Dv); d0 += 4 * LPR) {
      const int d = d0 + 4 * (lane % LPR);
      f32x4 x = {};
      if (f != 0.f) {
#pragma unroll 8
        for (int k = sub; k < ns; k += 64 / LPR) {
          const float e = exp2f(pl[k * per] - moff);
          f32x4 v = {};
          const float* at = po + k * per * p.Dv + d;
          if (p.Dv % 4 == 0) {
            if (d < p.Dv) v = *reinterpret_cast<const f32x4*>(at);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = d + q < p.Dv ? at[q] : 0.f;
          }
          x += v * e;
        }
      }
#pragma unroll
      for (int s = LPR; s < 64; s <<= 1)
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] += __shfl_xor(x[q], s, 64);
      if (sub == 0) {
        if (p.vec && d < p.Dv) {
          typedef T t4 __attribute__((ext_vector_type(4)));
          t4 y;
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = from_f32<T>(f == 0.f ? 0.f : x[q] * f);
          *reinterpret_cast<t4*>(o + d) = y;
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (d + q < p.Dv) o[d + q] = from_f32<T>(f == 0.f ? 0.f : x[q] * f);
        }
      }
    }
  }
}
template <typename T>
void combine(const DenseParams& p, hipStream_t s) {
  // Few rows: a wave each (more than 128 dims: for each 128 of them; one row of 512 dims from
  // 56 ranges 14.6 us for 41).  Many: their units often have one range, and then nothing is left
  // to do; a wave takes all dims (8192 rows of 512 dims from 2 ranges: 18 us, 31 with 128 each).
  const int jr = p.rows <= 64 ? 4 : 16;
  const int64_t rows = (int64_t)p.B * p.nrb * p.Hkv * p.rows;
  const int jd = rows < 2048 ? 128 : (p.Dv + 127) / 128 * 128;
  const unsigned grid = (unsigned)(rows / p.rows * ((p.Dv + jd - 1) / jd) * ((p.rows + jr - 1) / jr));
  if (p.Dv <= 64) dense_combine_kernel<T, 16><<<grid, 256, 0, s>>>(p, jr, jd);
  else if (jd <= 128) dense_combine_kernel<T, 32><<<grid, 256, 0, s>>>(p, jr, jd);
  else dense_combine_kernel<T, 64><<<grid, 256, 0, s>>>(p, jr, jd);
}

// ---- backward: per query row its LSE (base 2) and delta = sum o do - dlse (the bf16 matrix
// kernels' dq makes its own) ------------
// 16 lanes a row, from row `first` on.  Rows that see nothing get +inf, which makes every weight 0.
constexpr int64_t kDeltaRows = (int64_t)1 << 27;  // of a launch: fewer than 2^32 threads
template <typename T>
__global__ __launch_bounds__(256) void dense_delta_kernel(DenseParams p, int64_t first) {
  const int64_t rr = first + (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane = threadIdx.x & 15, R = p.S * p.G;
  if (rr >= (int64_t)p.B * p.Hkv * R) return;
  const int b = (int)(rr / ((int64_t)p.Hkv * R)), x = (int)(rr - (int64_t)b * p.Hkv * R), g = x / R, r = x - g * R;
  const int t = r / p.G, h = g * p.G + r % p.G;
  const bool live = t < dense_seq(p, b).n;
  float sum = 0.f;
  if (live) {
    const T* o = reinterpret_cast<const T*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh;
    const T* go = reinterpret_cast<const T*>(p.dout) + b * p.do_sb + t * p.do_ss + h * p.do_sh;
    for (int d = lane; d < p.Dv; d += 16) sum = fmaf(to_f32(o[d]), to_f32(go[d]), sum);
  }
#pragma unroll
  for (int s = 1; s < 16; s <<= 1) sum += __shfl_xor(sum, s, 64);
  if (lane != 0) return;
  const int64_t li = b * p.l_sb + t * p.l_ss + h * p.l_sh;
  const float lse = live ? p.lse[li] : kNegInf;
  const float delta = live ? sum - (p.dlse != nullptr ? p.dlse[li] : 0.f) : 0.f;
  p.row_lse[rr] = lse == kNegInf ? -kNegInf : lse * kLog2e;
  p.row_delta[rr] = delta;
}

// dsink[h] = -sum over the rows of exp(sink - lse) delta, a workgroup a head (from head `first`
// on), in a fixed order.
constexpr int kSinkHeads = 1 << 21;  // of a launch: fewer than 2^32 threads
__global__ __launch_bounds__(1024) void dense_dsink_kernel(DenseParams p, int first) {
  __shared__ float s_x[1024];
  const int h = first + blockIdx.x, g = h / p.G, hl = h % p.G;
  const float sink = p.sink[h] * kLog2e;
  float sum = 0.f;
  for (int b = 0; b < p.B; ++b) {
    const int64_t base = ((int64_t)b * p.Hkv + g) * p.S * p.G;
    const int n = dense_seq(p, b).n;
    for (int t = threadIdx.x; t < n; t += 1024) {
      const int64_t rr = base + (int64_t)t * p.G + hl;
      const float l = p.row_neg ? -p.row_lse[rr] * p.scale_log2 : p.row_lse[rr], d = p.row_delta[rr];
      sum += l == -kNegInf ? 0.f : exp2f(sink - l) * (p.row_neg ? -d : d);
    }
  }
  s_x[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) s_x[threadIdx.x] += s_x[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) p.dsink[h] = -s_x[0];
}

enum { kAny = 0, kWide, kFew16, kFew32, kFew64, kLatent };
struct KernelShape {
  int rows, tile_shift, threads, per_cu;  // per_cu: workgroups on a CU at once
};
constexpr KernelShape kShapes[] = {{kAnyRows, kAnyShift, 256, 4}, {kWideRows, 6, 512, 1}, {16, 7, 256, 2}, {32, 7, 256, 2},
                                   {64, 7, 256, 1}, {kLatentRows, 6, 512, 1}};

void set_launch(DenseParams& p, const DensePlan& pl) {
  p.rows = pl.rows;
  p.tile_shift = pl.tile_shift;
  p.nrb = (int)(((int64_t)p.S * p.G + pl.rows - 1) / pl.rows);
  p.fit = pl.fit;
  p.want = pl.want;
  p.min_len = pl.min_len;
  p.join = pl.join;
  p.slots = pl.slots;
}

}  // namespace

DensePlan dense_plan(const DenseParams& p, int dtype, int kv_dtype) {
  DensePlan pl{};
  pl.kernel = kAny;
  const int64_t R = (int64_t)p.S * p.G;
  if (dtype == SFA_DTYPE_BF16 && p.vec && p.Dqk == p.Dv && (p.Dqk == 64 || p.Dqk == 128))
    pl.kernel = R <= 16 ? kFew16 : R <= 32 ? kFew32 : R <= 64 ? kFew64 : kWide;
  // (e4m3 rows: of whole 16-byte units, as the other rows are, with one scale for both)
  const bool one_scale = kv_dtype == SFA_DTYPE_BF16 ||
                         (p.ks == p.vs && p.ks_sb == p.vs_sb && p.ks_ss == p.vs_ss && p.ks_sh == p.vs_sh && (p.k_sb | p.k_ss | p.k_sh) % 16 == 0);
  if (dtype == SFA_DTYPE_BF16 && p.vec && p.Dqk == kLatentQK && p.Dv == kLatentV && p.v == p.k && p.v_sb == p.k_sb &&
      p.v_ss == p.k_ss && p.v_sh == p.k_sh && one_scale)
    pl.kernel = kLatent;
  const KernelShape& k = kShapes[pl.kernel];
  pl.rows = k.rows;
  pl.tile_shift = k.tile_shift;
  pl.threads = k.threads;
  const int64_t nrb = ((int64_t)p.S * p.G + pl.rows - 1) / pl.rows, units = p.B * nrb;
  const int64_t dims = pl.kernel == kAny ? (p.Dv + kAnyDims - 1) / kAnyDims : 1;
  // Few row blocks: their keys are cut into ranges that fill the card (sfa_dense.h).
  constexpr int64_t kCus = 256;
  const bool few = pl.kernel >= kFew16 && pl.kernel <= kFew64;
  pl.min_len = few ? 2 : 4;
  // A row block's partial results are 128 KB (wide, latent rows): with the joining launch as
  // long as five tiles; of few rows it is the launch.
  pl.join = pl.kernel == kWide || pl.kernel == kLatent ? (int)(R < pl.rows ? 1 + 4 * R / pl.rows : 5) : 1;
  // (LDS of the few rows' kernel: one workgroup a CU with bf16 rows of 128 dims)
  const int per_cu = few && kv_dtype == SFA_DTYPE_BF16 && p.Dqk == 128 ? 1 : k.per_cu;
  const int64_t fit = kCus * per_cu / (p.Hkv * dims);
  pl.fit = (int)(fit > 0 ? fit : 1);
  int64_t want = 2 * ((units > pl.fit ? units : pl.fit));
  const int64_t tiles = ((int64_t)p.cap >> pl.tile_shift) + 1, most = (tiles + pl.min_len - 1) / pl.min_len * units;
  if (want > most) want = most;
  pl.want = units <= kDenseUnits && units <= 2 * pl.fit && want > units ? (int)want : 0;
  pl.slots = (int)(pl.want > 0 ? pl.want : units);
  pl.wgs = (int64_t)pl.slots * p.Hkv * dims;
  if (pl.want > 0) {
    const size_t rows = (size_t)pl.slots * p.Hkv * pl.rows;
    pl.part_o_bytes = (rows * p.Dv * sizeof(float) + 255) / 256 * 256;
    pl.part_lse_bytes = (rows * sizeof(float) + 255) / 256 * 256;
    pl.unit_bytes = (size_t)2 * units * sizeof(int32_t);
  }
  return pl;
}

hipError_t launch_dense(const DenseParams& p0, const DensePlan& pl, int dtype, int kv_dtype, hipStream_t s) {
  DenseParams p = p0;
  set_launch(p, pl);
  if (pl.kernel == kWide) launch_dense_wide(p, kv_dtype, s);
  else if (pl.kernel == kLatent) launch_dense_mla(p, kv_dtype == SFA_DTYPE_FP8_E4M3, s);
  else if (pl.kernel >= kFew16) launch_dense_few(p, kv_dtype, s);
  else launch_dense_any(p, dtype, kv_dtype, s);
  if (pl.want > 0) {
    if (dtype == SFA_DTYPE_F32) combine<float>(p, s);
    else combine<bf16>(p, s);
  }
  return hipGetLastError();
}

DenseBwdPlan dense_bwd_plan(const DenseParams& p, int dtype) {
  DenseBwdPlan pl{};
  const size_t rows = (size_t)p.B * p.Hkv * p.S * p.G;
  // (each a row tile longer: the matrix kernels read whole tiles of them)
  pl.row_bytes = (rows * sizeof(float) + 128 + 255) / 256 * 256;
  pl.row_arrays = 2;
  const int64_t groups = (int64_t)p.B * p.Hkv, most = (int64_t)1 << 32;
  // (its accumulators start from -lse / scale: no infinity while scale is 2^-100 or more)
  pl.mfma = dtype == SFA_DTYPE_BF16 && p.scale >= 0x1p-100f && p.vec && p.Dqk == p.Dv && (p.Dqk == 64 || p.Dqk == 128) &&
            p.k_ss >= 0 && p.v_ss >= 0 && p.k_ss < (int64_t)1 << 24 && p.v_ss < (int64_t)1 << 24;
  if (!pl.mfma) {
    const int64_t dims = ((p.Dqk > p.Dv ? p.Dqk : p.Dv) + kAnyDims - 1) / kAnyDims;
    pl.row_arrays = dims > 1 ? 3 : 2;
    const int64_t nrb = ((int64_t)p.S * p.G + kAnyRows - 1) / kAnyRows, nkb = ((int64_t)p.S + kAnyRows - 1) / kAnyRows;
    // Few key blocks (two workgroups a CU): their rows in chunks, of four times as many
    // workgroups in all (256 tokens, 32 heads on 2: 8 blocks of up to 4096 rows).
    const int64_t blocks = groups * nkb * dims, widest = p.first > 0 || p.window >= p.S ? p.S : (int64_t)p.window + kAnyRows - 1;
    const int64_t rows = (widest < p.S ? widest : p.S) * p.G;
    int64_t chunk = rows;
    if (blocks < 512) chunk = (rows * blocks / 1024 + 128) / 32 * 32;
    if (chunk > rows) chunk = rows;
    pl.chunk = (int)chunk;
    pl.parts = (int)((rows + chunk - 1) / chunk);
    pl.dkv_bytes = pl.parts > 1 ? (size_t)(groups * nkb * pl.parts) * kAnyRows * (p.Dqk + p.Dv) * sizeof(float) : 0;
    pl.fits = groups * nrb * dims * 256 < most && blocks * pl.parts * 256 < most;
    return pl;
  }
  // Key blocks' rows in chunks.  Without a window the first keys are seen by all rows, the
  // last by few; with one, the first tokens by all of them.  Blocks stay whole where
  // there are three or more for two CUs, but for some that are cut in five, for the units
  // left over from whole rounds of 256 (8192 tokens, window 1024: 0.97 of the CUs' time
  // used for 0.84); else every block is cut in chunks of half a CU's share (with the longest
  // first 0.97).  A partial sum costs 128 keys of float32, written and read; a chunk of fewer
  // than 512 rows is mostly its start.  The first tokens' blocks are cut in about four chunks a
  // CU at most, however narrow the window (8192 tokens, window 64, 32 / 8 heads of 128, the first
  // 4096: 1.14 GB of workspace with chunks of the window's blocks, 0.15 so).
  const int64_t nkb = ((int64_t)p.S + kDkvKeys - 1) / kDkvKeys;
  auto block_rows = [&](int64_t kb) {
    const int64_t j0 = kb * kDkvKeys, t1 = j0 < p.first ? p.S : j0 + kDkvKeys - 1 + p.window;
    return ((t1 < p.S ? t1 : (int64_t)p.S) - j0) * p.G;
  };
  constexpr int64_t kCus = 256, kLeast = 512;
  auto up = [&](int64_t x) { return (x < kLeast ? kLeast : x + 31) / 32 * 32; };
  int64_t total = 0, head = 0, widest = 0;  // all rows; of the first tokens' blocks; of a block behind those
  for (int64_t kb = 0; kb < nkb; ++kb) {
    const int64_t r = block_rows(kb);
    total += r;
    if (kb * kDkvKeys < p.first) head += r;
    else if (r > widest) widest = r;
  }
  const int64_t share = total * groups / kCus;
  const bool cut = 3 * widest > 2 * share;
  const int64_t part = head * groups / kCus / 4, chunk = up(cut ? share / 2 : widest > part ? widest : part);
  int64_t units = 0, parts = 0;
  pl.cut0 = pl.cut1 = 0;
  pl.cut_chunk = (int)up(chunk / 5);
  auto count = [&]() {
    units = parts = 0;
    for (int64_t kb = 0; kb < nkb; ++kb) {
      const int64_t c = kb >= pl.cut0 && kb < pl.cut1 ? pl.cut_chunk : chunk, nc = (block_rows(kb) + c - 1) / c;
      units += nc;
      parts += nc > 1 ? nc : 0;
    }
  };
  count();
  const int64_t left = units * groups % kCus;
  if (!cut && left > 0 && 3 * left < 2 * kCus) {
    const int64_t from = ((int64_t)p.first + kDkvKeys - 1) / kDkvKeys;
    const int64_t blocks = (left + groups - 1) / groups;
    if (from + blocks < nkb) {
      pl.cut0 = (int)from;
      pl.cut1 = (int)(from + blocks);
      count();
    }
  }
  pl.chunk = (int)chunk;
  pl.units = (int)units;
  pl.parts = (int)parts;
  pl.dkv_bytes = (size_t)(groups * parts) * kDkvKeys * 2 * p.Dqk * sizeof(float);
  pl.unit_bytes = (size_t)units * 4 * sizeof(int);
  const int64_t nrb = ((int64_t)p.S * p.G + kWideRows - 1) / kWideRows;
  pl.fits = (groups * nrb + 1) * 512 < most && groups * units * 512 < most && groups * nkb * 256 < most;
  return pl;
}

hipError_t launch_dense_bwd(const DenseParams& p0, const DenseBwdPlan& pl, int dtype, hipStream_t s) {
  DenseParams p = p0;
  p.row_neg = pl.mfma;
  DensePlan q{};
  q.rows = pl.mfma ? kWideRows : kAnyRows;
  q.tile_shift = pl.mfma ? 6 : kAnyShift;
  q.slots = p.B * (int)(((int64_t)p.S * p.G + q.rows - 1) / q.rows);
  set_launch(p, q);
  p.chunk = pl.chunk;
  p.cut0 = pl.cut0;
  p.cut1 = pl.cut1;
  p.cut_chunk = pl.cut_chunk;
  p.dkv_parts = pl.parts;
  if (pl.mfma) {  // (whose dq kernel leaves the rows' statistics)
    launch_dense_bwd_mfma(p, pl.units, s);
  } else {
    const int64_t rows = (int64_t)p.B * p.Hkv * p.S * p.G;
    for (int64_t first = 0; first < rows; first += kDeltaRows) {
      const unsigned grid = (unsigned)(((rows - first < kDeltaRows ? rows - first : kDeltaRows) + 15) / 16);
      if (dtype == SFA_DTYPE_F32) dense_delta_kernel<float><<<grid, 256, 0, s>>>(p, first);
      else dense_delta_kernel<bf16><<<grid, 256, 0, s>>>(p, first);
    }
    launch_dense_bwd_any(p, dtype, s);
  }
  p.row_delta = p.row_exact;
  for (int first = 0; p.dsink != nullptr && first < p.Hq; first += kSinkHeads)
    dense_dsink_kernel<<<p.Hq - first < kSinkHeads ? p.Hq - first : kSinkHeads, 1024, 0, s>>>(p, first);
  return hipGetLastError();
}

}  // namespace sfa

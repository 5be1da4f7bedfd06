// gfx950 dense attention through a window (sfa_dense.h) over latent rows: head dims 576 and
// 512, V the first 512 dims of K, bf16 queries, bf16 or e4m3 rows.
//
// Eight waves take 64 query rows and tiles of 64 keys (72 KB of LDS, two stages), and divide
// the two products differently:
//  * S^T = K Q^T (16x16x32): wave (rh, kq) takes 32 rows x 16 keys, its Q in registers; a K
//    operand read from LDS serves 32 rows;
//  * P^T goes through LDS (8 KB) in operand order, and
//  * O^T = V^T P^T (32x32x16): wave w takes dims 64 w .. 64 w + 63 of all 64 rows, so that
//    each V element is read from LDS once.
// A tile is 2176 clocks of products and 356 KB through LDS (2785 clocks): LDS bounds it, then
// the two halves' hand-over (two barriers a tile; without its loads, its scores' or its sums'
// products a launch takes 0.80 to 0.83 of its time, each alone): 512 tokens behind 14336 with 16
// heads 338 us, 0.77 PF/s, with 128 heads 2200 to 2280 us, 0.93 PF/s.  The next tile's rows are
// asked for during S^T.  The running
// maximum is shared: a row's scores are in four waves, so a wave that finds one past the
// maximum by 8 (base 2; 2^8 more at most in a float32 sum) raises a flag, and all of them move
// it after the barrier that publishes P.  P is rounded to bf16 once for its product (2^-8 of a
// weight); sums and statistics are float32.
//
// e4m3 rows (FP8) come to LDS as they are, two stages of 36 KB, and each wave makes bf16 ones
// (times their power of two: exact) of its eight at the start of a step, in one stage of 72 KB:
// a third barrier and 111 KB through LDS a tile (the above: 479 and 3290 us).
//
// No register is free: with bf16 rows 2 spill (4 where pages are shorter than tiles), with e4m3
// ones 14 and 24, and some hundred scalar ones go to lanes of vector registers.

#include "sfa_dense_tiles.h"

namespace sfa {
namespace {

constexpr int kLatentCh = 64, kLatentCr = 8;  // 16-byte chunks of a row's V part, of its rest
constexpr int kLatentRaw = kLatentQK / 16;    // of an e4m3 row

// Chunk c of row r goes to place c ^ at(r) of its row: one chunk of 16 consecutive rows (K)
// meets all 16 bank groups, as do aligned groups of four chunks of four consecutive rows (V,
// transposed).
__device__ __forceinline__ int latent_at(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ int latent_rest_at(int r) { return (r >> 1) & 7; }

// The rows of tiles of 64 keys for 8 waves, 8 rows each: an instruction for a row's first 1024
// bytes, one for the last 128 of all eight.  ONE: a tile's rows have one base and stride
// (contiguous rows, pages of 64 rows or more); else each its own, found a tile ahead.
template <bool ONE, bool FP8>
struct LatentSource {
  uint64_t kbase;
  int64_t kpage, krow;
  const int32_t* trow;
  KeyTiles tiles;
  int v0, n, cap, page_shift, num_pages, wave, lane;
  int pg;                // page ids: of 64 tiles by lane; of the next tile's row `lane`
  uint64_t base, mask;   // the tile begin() was called for: its (ONE) or the lane's row's address, rows that are there
  int64_t step;
  int left;
  const uint8_t* ks;     // FP8: exponents, and that of row wave * 8 + lane / 8 of begin()'s tile
  int64_t ks_sb, ks_ss;
  int exponent;

  __device__ __forceinline__ LatentSource(const DenseParams& p, const DenseItem& it, int wave_, int lane_)
      : tiles(it.tiles), v0(it.v0), n(it.v1 - it.v0), cap(p.cap), page_shift(p.page_shift), num_pages(p.num_pages), wave(wave_),
        lane(lane_) {
    constexpr int64_t E = FP8 ? 1 : 2;
    kbase = (uint64_t)(uintptr_t)p.k + (uint64_t)(E * it.g * p.k_sh);
    kpage = E * p.k_sb;
    krow = E * p.k_ss;
    if constexpr (FP8) {
      ks = p.ks + it.g * p.ks_sh;
      ks_sb = p.ks_sb;
      ks_ss = p.ks_ss;
    }
    trow = nullptr;
    if (p.block_table != nullptr) {
      trow = p.block_table + it.b * p.bt_sb;
    } else {  // one page of all rows
      kbase += (uint64_t)(it.b * kpage);
      page_shift = 30;
      num_pages = 1;
    }
    ids(0);
  }
  __device__ __forceinline__ int at(int i) const { return tiles.tile(v0 + max(min(i, n - 1), 0)) * kWideKeys; }
  __device__ __forceinline__ int entry(int j) const { return trow == nullptr ? 0 : trow[min(j, cap - 1) >> page_shift]; }
  __device__ __forceinline__ void ids(int i) { pg = entry(ONE ? at(i + lane) : at(i) + lane); }

  // (past the range: zeros)
  __device__ __forceinline__ void begin(int i) {
    const bool on = i < n;
    const int j0 = at(i), in_page = (1 << page_shift) - 1;
    const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
    if constexpr (ONE) {
      const int id = __builtin_amdgcn_readlane(pg, i & 63), rows = cap - j0;
      const bool ok = on && id >= 0 && id < num_pages;
      base = ok ? kbase + (uint64_t)(id * kpage + (j0 & in_page) * krow) : zero;
      step = ok ? krow : 0;
      left = ok ? rows : kWideKeys;
      mask = !ok ? 0 : rows >= kWideKeys ? ~0ull : (1ull << rows) - 1;
      if constexpr (FP8) {
        const int r = wave * 8 + (lane >> 3);
        exponent = ok && r < rows ? ks[id * ks_sb + ((j0 & in_page) + r) * ks_ss] : 127;
      }
      if (((i + 1) & 63) == 0) ids(i + 1);
    } else {
      const int j = j0 + lane;
      const bool ok = on && j < cap && pg >= 0 && pg < num_pages;
      base = ok ? kbase + (uint64_t)(pg * kpage + (j & in_page) * krow) : zero;
      mask = __ballot(ok);
      if constexpr (FP8) {
        const int r = wave * 8 + (lane >> 3), id = __shfl(pg, r, 64);
        exponent = (mask >> r) & 1 ? ks[id * ks_sb + ((j0 + r) & in_page) * ks_ss] : 127;
      }
    }
  }
  // FP8: the wave's rows as they are
  __device__ __forceinline__ void raw(u32x4* dst, int ln) const {
    u32x4* const mine = dst + wave * 8 * kLatentRaw;
#pragma unroll
    for (int k = 0; k < (8 * kLatentRaw + 63) / 64; ++k) {
      const int i = 64 * k + ln, r = min(wave * 8 + i / kLatentRaw, kWideKeys - 1);
      uint64_t a;
      if constexpr (ONE) {
        a = row_at(r);
      } else {
        a = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(base >> 32), r, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)base, r, 64);
      }
      if (i < 8 * kLatentRaw) dense_dma16(mine + 64 * k, a + (uint64_t)(16 * (i % kLatentRaw)));
    }
  }
  // ... and as bf16 in their places of a tile
  __device__ __forceinline__ void widen(const u32x4* src, u32x4* kt, u32x4* rt, float scale, int ln) const {
    const int r = wave * 8 + (ln >> 3);
    const u32x4* const row = src + r * kLatentRaw;
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      const int c = (ln & 7) + 8 * i;
      if (c >= kLatentRaw) break;
      const u32x4 x = row[c];
      u32x4 y[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        y[w >> 1][2 * (w & 1)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[w], scale, false));
        y[w >> 1][2 * (w & 1) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[w], scale, true));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (i < 4) kt[r * kLatentCh + ((2 * c + h) ^ latent_at(r))] = y[h];
        else rt[r * kLatentCr + ((2 * c + h - kLatentCh) ^ latent_rest_at(r))] = y[h];
      }
    }
  }
  __device__ __forceinline__ uint64_t row_at(int row) const {  // (ONE; rows past the last: row 0, which no row of theirs sees)
    return base + (row < left ? (uint64_t)(row * step) : 0);
  }
  __device__ __forceinline__ void row(int k, u32x4* kt, int ln) const {  // the k-th of the wave's eight
    const int r = wave * 8 + k;
    uint64_t a;
    if constexpr (ONE) {
      a = row_at(r);
    } else {
      a = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(base >> 32), r) << 32) |
          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)base, r);
    }
    dense_dma16(kt + r * kLatentCh, a, 16u * (uint32_t)(ln ^ latent_at(r)));
  }
  __device__ __forceinline__ void rest(u32x4* rt, int ln) const {
    const int r = wave * 8 + (ln >> 3);
    uint64_t a;
    if constexpr (ONE) {
      a = row_at(r);
    } else {
      a = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(base >> 32), r, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)base, r, 64);
    }
    dense_dma16(rt + wave * 8 * kLatentCr, a + (uint64_t)(16 * (kLatentCh + ((ln & 7) ^ latent_rest_at(r)))));
  }
};

template <bool ONE, bool FP8>
__global__ __launch_bounds__(512, 2) void dense_mla_kernel(DenseParams p) {
  typedef Mfma<16> M16;
  typedef Mfma<32> M;
  constexpr int CH = kLatentCh, CR = kLatentCr, KT = kWideKeys, STEPS = kLatentQK / 32, QR = 16;  // steps of Q in registers
  constexpr int LAST = FP8 ? 0 : 1;       // the last stage
  __shared__ u32x4 s_k[LAST + 1][KT * CH];  // dims 0 .. 511 (K and V)
  __shared__ u32x4 s_r[LAST + 1][KT * CR];  // dims 512 .. 575
  __shared__ u32x4 s_raw[2][FP8 ? KT * kLatentRaw : 1];
  __shared__ u32x4 s_p[4][2][kLatentRows];  // P of 16 keys: [lane half][row] keys 4 half + 0 .. 3, 8 + 4 half + 0 .. 3
  __shared__ u32x4 s_q[4][kLatentRows];   // Q's last 32 dims: [8 of them][row]
  __shared__ u32x4 s_q1[4][32];           // the 32 before them, of rows 16 .. 31 and 48 .. 63
  __shared__ float s_m[kLatentRows];      // running maxima (base 2)
  __shared__ float s_x[4][kLatentRows];   // per key quarter: row maxima, then row sums
  __shared__ int s_over[2];
  __shared__ unsigned long long s_bad[2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rh = wave & 1, kq = wave >> 1;

  int slot, g;
  dense_place(p, slot, g);
  DenseItem it;
  if (!dense_item(p, slot, g, it)) return;
  const int b = it.b, R = p.S * p.G;
  // what all rows of the block see of a tile without a look at each
  const int p0 = it.s.ctx + it.row0 / p.G, p1 = it.s.ctx + min((it.row0 + p.rows - 1) / p.G, it.s.n - 1);

  // The rows of Q come through LDS, where a tile goes later (straight from global memory each
  // load touches 16 rows and four waves load the same: 6 us a workgroup).
  {
    const int r0 = it.row0 + 8 * wave;
    int t = r0 / p.G, h = r0 - t * p.G;
    const uint64_t qbase = (uint64_t)(uintptr_t)p.q + (uint64_t)(2 * (b * p.q_sb + g * p.G * p.q_sh)), zero = (uint64_t)(uintptr_t)kZeroRow;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int row = 8 * wave + k;
      const uint64_t a = r0 + k < R && t < it.s.n ? qbase + (uint64_t)(2 * (t * p.q_ss + h * p.q_sh)) : zero;
      dense_dma16(&s_k[LAST][row * CH], a, 16u * (uint32_t)(lane ^ latent_at(row)));
      if (++h == p.G) {
        h = 0;
        ++t;
      }
    }
    const int row = 8 * wave + (lane >> 3), r = it.row0 + row;
    t = r / p.G;
    h = r - t * p.G;
    const uint64_t a = r < R && t < it.s.n ? qbase + (uint64_t)(2 * (t * p.q_ss + h * p.q_sh)) : zero;
    dense_dma16(&s_r[LAST][8 * wave * CR], a + (uint64_t)(16 * (CH + ((lane & 7) ^ latent_rest_at(row)))));
  }
  if (tid < kLatentRows) {
    s_m[tid] = kNegInf;
    if (tid < 2) {
      s_over[tid] = 0;
      s_bad[tid] = 0;
    }
  }

  LatentSource<ONE, FP8> src(p, it, wave, lane);
  const int ntiles = it.v1 - it.v0;
  src.begin(0);
  uint64_t mask = src.mask;
  if constexpr (FP8) {
    src.raw(s_raw[0], lane);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) src.row(k, s_k[0], lane);
    src.rest(s_r[0], lane);
  }
  if constexpr (!ONE) src.ids(1);

  bf16x8 q[2][QR], q16;  // (Q's last one and a half steps in LDS: there is no register to spare)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  dense_barrier();
  {
    const int lt = lane & 15, hq = lane >> 4;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int row = 32 * rh + 16 * n + lt;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const bf16x8 y = s < 16 ? __builtin_bit_cast(bf16x8, s_k[LAST][row * CH + ((4 * s + hq) ^ latent_at(lt))])
                                : __builtin_bit_cast(bf16x8, s_r[LAST][row * CR + ((4 * (s - 16) + hq) ^ latent_rest_at(lt))]);
        if (s < QR) q[n][s < QR ? s : 0] = y;
        else if (s == QR && n == 0) q16 = y;
        else if (kq == 0 && s == QR) s_q1[hq][16 * rh + lt] = __builtin_bit_cast(u32x4, y);
        else if (kq == 0) s_q[hq][row] = __builtin_bit_cast(u32x4, y);
      }
    }
  }

  f32x16 oacc[2][2];  // [32 dims][32 rows]
#pragma unroll
  for (int o = 0; o < 2; ++o)
#pragma unroll
    for (int n = 0; n < 2; ++n) oacc[o][n] = f32x16{};
  float m_used[2] = {kNegInf, kNegInf}, l_part[2] = {0.f, 0.f};
  int nbad = 0;

  for (int j = 0; j < ntiles; ++j) {
    u32x4 *kt = s_k[j & LAST], *rt = s_r[j & LAST];
    u32x4 *kn = s_k[(j + 1) & LAST], *rn = s_r[(j + 1) & LAST];
    // (lane constants are formed per tile: held across the loop they spill)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    int lt = ln & 15, hq = ln >> 4;
    const uint32_t ka = lds_addr(kt) + (uint32_t)((16 * kq + lt) * CH) * 16u, kx = 16u * (uint32_t)(hq ^ latent_at(lt));
    const uint32_t kr = lds_addr(rt) + (uint32_t)((16 * kq + lt) * CR) * 16u, rx = 16u * (uint32_t)(hq ^ latent_rest_at(lt));
    // tile j has landed for all waves; tile j - 1 and its P are read
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (FP8) {
      const float scale = scale_of((uint8_t)src.exponent);
      src.begin(j + 1);
      src.raw(s_raw[(j + 1) & 1], ln);
      src.widen(s_raw[j & 1], kt, rt, scale, ln);
      dense_barrier();
    }
    // contraction steps in order, the one with Q in LDS first
    auto order = [](int i) { return i == 0 ? STEPS - 1 : i - 1; };
    auto read_k = [&](int s) {
      return s < 16 ? lds_b128_at(ka + (kx ^ (uint32_t)(64 * s))) : lds_b128_at(kr + (rx ^ (uint32_t)(64 * (s - 16))));
    };
    bf16x8 kf[3], ql[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) ql[n] = __builtin_bit_cast(bf16x8, s_q[hq][32 * rh + 16 * n + lt]);
#pragma unroll
    for (int i = 0; i < 2; ++i) kf[i] = read_k(order(i));
    if constexpr (!FP8) src.begin(j + 1);
    if (tid == 0) s_over[(j + 1) & 1] = 0;
    f32x4 sc[2];
    each<STEPS>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i + 2 < STEPS) kf[(i + 2) % 3] = read_k(order(i + 2));
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if constexpr (i == 0) sc[n] = M16::mma(kf[0], ql[n], f32x4{});
        else if constexpr (i <= QR) sc[n] = M16::mma(kf[i % 3], q[n][(i + QR - 1) % QR], sc[n]);
        else sc[n] = M16::mma(kf[i % 3], n == 0 ? q16 : ql[0], sc[n]);
      }
      if constexpr (i == 14) ql[0] = __builtin_bit_cast(bf16x8, s_q1[hq][16 * rh + lt]);
      // the next tile's rows
      if constexpr (!FP8 && i % 2 == 1 && i / 2 < 8) src.row(i / 2, kn, ln);
      else if constexpr (!FP8 && i == 17) src.rest(rn, ln);
    });
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!ONE) src.ids(j + 2);

    // the lane's keys 16 kq + 4 hq + e of its rows
    const int j0 = src.at(j);
    const bool masked = !(j0 + KT - 1 <= p0 && (j0 + KT <= p.first || p1 - j0 < p.window) && mask == ~0ull);
    if (masked) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        // (formed here: held they spill)
        const int r = it.row0 + 32 * rh + 16 * n + lt, t = r / p.G, pos = r < R && t < it.s.n ? it.s.ctx + t : -1;
        const uint32_t bits = (uint32_t)((seen_of(p, pos, j0) & mask) >> (16 * kq + 4 * hq));
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = (bits >> e) & 1 ? sc[n][e] : kNegInf;
      }
    }
    bool over = false;
    float tmax[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      tmax[n] = fmaxf(fmaxf(sc[n][0], sc[n][1]), fmaxf(sc[n][2], sc[n][3])) * p.scale_log2;
      over |= tmax[n] > m_used[n] + 8.f;
    }
    if (__any(over) && ln == 0) s_over[j & 1] = 1;
    char* const pw = reinterpret_cast<char*>(&s_p[kq][hq & 1][32 * rh + lt]) + 8 * (hq >> 1);
    auto weights = [&](float (&sum)[2]) {  // P^T of the lane's keys into LDS
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float moff = m_used[n] == kNegInf ? 0.f : -m_used[n];
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(sc[n][e], p.scale_log2, moff));
        *reinterpret_cast<bf16x4*>(pw + n * 16 * 16) = bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
        sum[n] = (x[0] + x[1]) + (x[2] + x[3]);
      }
    };
    float sum[2];
    weights(sum);

    // operands of the sums: V rows 16 kk + 4 half + (lane % 16) / 4 and 8 further, 16 dims by lane / 16 % 2
    asm volatile("" : "+v"(ln));  // (what the second half needs is formed now)
    const int lr = ln & 31, half = ln >> 5, l16 = ln & 15, vrow = 4 * half + (l16 >> 2);
    const int vc = 8 * wave + 2 * ((ln >> 4) & 1) + ((l16 & 3) >> 1);
    const uint32_t va = lds_addr(kt) + (uint32_t)(vrow * CH * 16) + (uint32_t)(l16 & 1) * 8u;
    const uint32_t vx = 16u * (uint32_t)(vc ^ latent_at(vrow)), vy = 16u * (uint32_t)(vc ^ latent_at(vrow + 8)) + 8u * CH * 16u;
    auto read_v = [&](int u) {  // product pair u: 16 keys, 32 dims
      const uint32_t off = (uint32_t)(u / 2 * 16 * CH * 16), x = 64u * (uint32_t)(u % 2);
      const bf16x4 lo = lds_tr16_at(va + (vx ^ x) + off), hi = lds_tr16_at(va + (vy ^ x) + off);
      return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    bf16x8 a[3], pb[2][2];
    a[0] = read_v(0);
    a[1] = read_v(1);
    dense_barrier();  // P and the flag are there
    if (s_over[j & 1] != 0) {
      const int lt = ln & 15, hq = ln >> 4;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float t = xor32_max(xor16_max(tmax[n]));
        if (hq == 0) s_x[kq][32 * rh + 16 * n + lt] = t;
      }
      dense_barrier();
      auto moved = [&](int row, float& alpha) {
        const float m = s_m[row];
        const float mn = fmaxf(fmaxf(m, fmaxf(s_x[0][row], s_x[1][row])), fmaxf(s_x[2][row], s_x[3][row]));
        alpha = mn == kNegInf ? 1.f : exp2f(m - mn);
        return mn;
      };
      float alpha;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        moved(32 * n + lr, alpha);
        oacc[0][n] *= alpha;
        oacc[1][n] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        m_used[n] = moved(32 * rh + 16 * n + lt, alpha);
        l_part[n] *= alpha;
      }
      weights(sum);
      dense_barrier();
      if (kq == 0 && hq == 0) {
        s_m[32 * rh + lt] = m_used[0];
        s_m[32 * rh + 16 + lt] = m_used[1];
      }
    }
    l_part[0] += sum[0];
    l_part[1] += sum[1];

    uint64_t bad = 0;
    if (masked) {
      // Infinities and NaN of V in rows that not every row sees: noted and cleared, as 0 times
      // them would reach rows that do not see them.  (Two words in turn: the other one's
      // readers have passed a step's barrier.)
      const int w = nbad & 1;
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        u32x4& x = s_k[j & LAST][(wave * 8 + i) * CH + ln];
        u32x4 m;
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = bad16(x[e]);
        if ((m[0] | m[1] | m[2] | m[3]) != 0) {
          x = x & ~m;
          atomicOr(&s_bad[w], 1ull << (wave * 8 + i));
        }
      }
      dense_barrier();
      bad = s_bad[w];
      ++nbad;
      if (tid == 0) s_bad[nbad & 1] = 0;
      a[0] = read_v(0);
      a[1] = read_v(1);
    }
    // O^T += V^T P^T over the wave's 64 dims
    auto read_p = [&](int kk, int n) { return __builtin_bit_cast(bf16x8, s_p[kk][half][32 * n + lr]); };
    pb[0][0] = read_p(0, 0);
    pb[0][1] = read_p(0, 1);
    each<8>([&](auto uc) {
      constexpr int u = decltype(uc)::value, kk = u / 2, o = u % 2;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (u + 2 < 8) a[(u + 2) % 3] = read_v(u + 2);
      if constexpr (o == 0 && kk < 3) {
        pb[(kk + 1) & 1][0] = read_p(kk + 1, 0);
        pb[(kk + 1) & 1][1] = read_p(kk + 1, 1);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) oacc[o][n] = M::mma(a[u % 3], pb[kk & 1][n], oacc[o][n]);
    });
    __builtin_amdgcn_sched_barrier(0);
    for (; bad != 0; bad &= bad - 1) {  // to the rows that see them
      const int key = __builtin_ctzll(bad);
      const int64_t at = dense_row(p, b, j0 + key, p.k_sb, p.k_ss);
      if (at < 0) continue;
      const int64_t v = at + g * p.k_sh + 64 * wave + 4 * half;
      float vs = 1.f;
      if constexpr (FP8) vs = scale_of(p.ks[dense_row(p, b, j0 + key, p.ks_sb, p.ks_ss) + g * p.ks_sh]);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float e = (float)reinterpret_cast<const bf16*>(&s_p[key >> 4][(key >> 2) & 1][32 * n + lr])[4 * ((key >> 3) & 1) + (key & 3)];
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4 xf;
            bf16x4 xb;
            if constexpr (FP8) {
              const int w = *reinterpret_cast<const int*>(reinterpret_cast<const uint8_t*>(p.k) + v + 32 * o + 8 * i);
              xf = f32x4{__builtin_amdgcn_cvt_f32_fp8(w, 0), __builtin_amdgcn_cvt_f32_fp8(w, 1), __builtin_amdgcn_cvt_f32_fp8(w, 2),
                         __builtin_amdgcn_cvt_f32_fp8(w, 3)} * vs;
            } else {
              xb = *reinterpret_cast<const bf16x4*>(reinterpret_cast<const bf16*>(p.k) + v + 32 * o + 8 * i);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float y = FP8 ? xf[c] : (float)xb[c];
              if (e != 0.f && !(fabsf(y) <= 3.402823466e38f)) oacc[o][n][4 * i + c] += e * y;
            }
          }
      }
    }
    mask = src.mask;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- row sums over the key quarters; results: lane holds rows 32 n + lr, dims
  // 64 wave + 32 o + 8 i + 4 half + 0 .. 3 -----------------------------------------------
  {
    const int lt = lane & 15, hq = lane >> 4;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float l = l_part[n];
      l += __shfl_xor(l, 16, 64);
      l = xor32_sum(l);
      if (hq == 0) s_x[kq][32 * rh + 16 * n + lt] = l;
    }
  }
  dense_barrier();
  const int lr = lane & 31, half = lane >> 5;
  static_assert(sizeof(s_k) >= (FP8 ? 1 : 2) * 8 * 32 * 16 * 16, "32 float32 rows of 64 dims a wave, or all 64");
  u32x4* const rows = &s_k[0][0];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int row = 32 * n + lr, r = it.row0 + row, t = r / p.G, h = g * p.G + r % p.G;
    const bool in = r < R, first = in && wave == 0 && half == 0;
    const float l = (s_x[0][row] + s_x[1][row]) + (s_x[2][row] + s_x[3][row]);
    float lse, f;
    if (it.partial) {
      f = dense_part(s_m[row], l, lse);
      if (first) p.part_lse[it.part + row] = lse;
    } else {
      f = dense_finish(p, h, in && t < it.s.n, s_m[row], l, lse);
      if (first) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
    }
    auto results = [&](auto put) {
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = f == 0.f ? 0.f : oacc[o][n][4 * i + e] * f;
          put(32 * o + 8 * i + 4 * half, x);
        }
    };
    if (it.partial) {
      const RowsOut<16> out{rows + (FP8 ? wave : 2 * wave + n) * 32 * 16};
      results([&](int d, f32x4 x) { out.put(lr, d, x); });
      out.store(in ? (uint64_t)(uintptr_t)(p.part_o + (it.part + row) * p.Dv + 64 * wave) : 0, lane);
    } else {
      const RowsOut<8> out{rows + (FP8 ? wave : 2 * wave + n) * 32 * 8};
      results([&](int d, f32x4 x) { out.put(lr, d, bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]}); });
      out.store(in ? (uint64_t)(uintptr_t)(reinterpret_cast<bf16*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh + 64 * wave) : 0,
                lane);
    }
  }
}

}  // namespace

void launch_dense_mla(const DenseParams& p, bool fp8, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.slots * p.Hkv);
  const bool one = dense_one_base(p, fp8 ? 1 : 2, 6);
  if (fp8 && one) dense_mla_kernel<true, true><<<grid, 512, 0, s>>>(p);
  else if (fp8) dense_mla_kernel<false, true><<<grid, 512, 0, s>>>(p);
  else if (one) dense_mla_kernel<true, false><<<grid, 512, 0, s>>>(p);
  else dense_mla_kernel<false, false><<<grid, 512, 0, s>>>(p);
}

}  // namespace sfa

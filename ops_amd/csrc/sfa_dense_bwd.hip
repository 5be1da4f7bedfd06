// gfx950 backward of dense attention through a window (sfa_dense.h), head dims 64 and
// 128 in bf16.
//
//   p_ij = exp(scale q_i.k_j - lse_i),  ds_ij = p_ij (do_i.v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Two kernels, each of which makes the scores again, so that every sum has a fixed
// order without atomics: seven products for the five that are needed.  Products of 32 x
// 32 (32x32x16): a lane holds 16 scores of one column (dq: a query row; dk, dv: a key),
// which rounded to bf16 are the second operand of the sums' products as they are;
// the first is read from LDS transposed.  A step makes the scores of the next 32 entries
// beside the weights of this one's, then its sums.  Each wave reads every entry's rows
// as rows and again transposed: a kilobyte of LDS a product, as much as four SIMDs can
// take at once, which bounds both kernels together with the products.  p and ds are
// rounded to bf16 once for their products (2^-8 of each); sums are float32.

#include "sfa_dense_tiles.h"

namespace sfa {
namespace {

typedef Mfma<32> M;
typedef f32x16 acc_t;

// ---- dq: eight waves of 32 query rows, tiles of 64 keys -------------------------------
template <int D>
__global__ __launch_bounds__(512, 2) void dense_dq_kernel(DenseParams p) {
  typedef Tile<D> L;
  constexpr int NW = 8, KT = kWideKeys, KS = D / 16, OT = D / 32, NS = 4;
  __shared__ u32x4 s_kv[NS][2][L::SLOTS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hq = lane >> 5;
  int slot, g;
  if (!dense_place(p, slot, g)) return;
  DenseItem it;
  if (!dense_item(p, slot, g, it)) return;
  const int b = it.b, r = it.row0 + 32 * wave + lr;
  const int t = r / p.G, h = g * p.G + r % p.G;
  const bool in = r < p.S * p.G, live = in && t < it.s.n;
  const int pos = live ? t : -1;
  const int p0 = it.row0 / p.G, p1 = min((it.row0 + p.rows - 1) / p.G, it.s.n - 1);
  const int64_t rr = ((int64_t)b * p.Hkv + g) * p.S * p.G + r;

  bf16x8 qb[KS], ob[KS];
  {
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
    const bf16* o = reinterpret_cast<const bf16*>(p.dout) + b * p.do_sb + (live ? t * p.do_ss + h * p.do_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 16 * s), y = *reinterpret_cast<const bf16x8*>(o + 16 * s);
      qb[s] = live ? x : bf16x8{};
      ob[s] = live ? y : bf16x8{};
    }
  }
  const float moff = live ? p.row_lse[rr] * p.scale_log2 : kNegInf, ndelta = live ? p.row_delta[rr] : 0.f;

  TileSource<D, NW, false, true> src(p, it, wave, lane);
  const int n = it.v1 - it.v0;
  acc_t dq[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) dq[o] = acc_t{};

  constexpr int FLIP = D == 128 ? 6 : 5;
  const int l16 = lane & 15, trow = 4 * hq + (l16 >> 2), tc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
  const uint32_t kx = 16u * (uint32_t)L::at(lr), k0a = 16u * (uint32_t)(L::slot(lr, L::at(lr)) + hq);
  const uint32_t tx = 16u * (uint32_t)(L::at(trow) ^ tc), t0a = 16u * (uint32_t)L::slot(trow, L::at(trow)) + (uint32_t)(l16 & 1) * 8u;

  uint64_t mask[NS + 1];
#pragma unroll
  for (int i = 0; i < NS; ++i) mask[i] = src.load(i, s_kv[i][0], s_kv[i][1]);
  src.template wait<0>();
  dense_barrier();

  // A half step's products: those of the next 32 keys' scores and of do.v in turn, then the sums.
  constexpr int NQ = 2 * KS, NM = NQ + 2 * OT;
  // (i even: K, odd: V; rows 32 kb ..)
  auto read_row = [&](uint32_t k, uint32_t v, uint32_t x, int i, int kb) {
    const int c = i >> 1;
    return lds_b128_at((i & 1 ? v : k) + (x ^ ((uint32_t)(D == 128 ? c >> 1 : c) << FLIP)) +
                       (uint32_t)((D == 128 ? 32 * (c & 1) : 0) + L::rows(32 * kb)));
  };
  auto read_t = [&](uint32_t a, uint32_t x, int i, int kb) {
    const uint32_t at = a + (x ^ (uint32_t)(64 * (i % OT))) + (uint32_t)L::rows(32 * kb + 16 * (i / OT));
    const bf16x4 lo = lds_tr16_at(at), hi = lds_tr16_at(at + (uint32_t)L::rows(8));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  acc_t sa, sb, da, db;
  bf16x8 op[4];
  {
    const uint32_t k = lds_addr(s_kv[0][0]) + k0a, v = lds_addr(s_kv[0][1]) + k0a;
    sa = da = acc_t{};
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const bf16x8 x = read_row(k, v, kx, i, 0);
      if (i & 1) da = M::mma(x, ob[i >> 1], da);
      else sa = M::mma(x, qb[i >> 1], sa);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = read_row(k, v, kx, i, 1);
  }

  int st = 0;
  // half 0: sums of keys 0 .. 31 of tile j, scores of its keys 32 .. 63; half 1: sums of
  // those, scores of tile j + 1's first 32
  auto half = [&](int j, auto hc, acc_t& cs, acc_t& cd, acc_t& ns, acc_t& nd) {
    constexpr int H = decltype(hc)::value;
    const int st1 = (st + 1) & (NS - 1);
    uint32_t xf = kx, tf = tx;
    asm volatile("" : "+v"(xf), "+v"(tf));
    const uint32_t kt = lds_addr(s_kv[st][0]) + t0a;
    const uint32_t kn = lds_addr(s_kv[H ? st1 : st][0]) + k0a, vn = lds_addr(s_kv[H ? st1 : st][1]) + k0a;
    const uint32_t kn2 = lds_addr(s_kv[st1][0]) + k0a, vn2 = lds_addr(s_kv[st1][1]) + k0a;
    const int j0 = src.at(j);
    const bool whole = mask[0] == ~0ull && j0 + KT - 1 <= p0 && (j0 + KT <= p.first || p1 - j0 < p.window);
    uint32_t seen = ~0u;
    if (!whole) {
      // infinities and NaN of keys that not every row sees: 0 times them would reach those
      // that do not (those that do have weights that are no numbers)
      clear_rows<D, NW>(s_kv[st][0], 32 * H, wave, lane);
      seen = (uint32_t)((seen_of(p, pos, j0) & mask[0]) >> (32 * H)) >> (4 * hq);
    }
    bf16x8 pb[2];
    float ex = 0.f;
    each<NM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i < NQ) {
        constexpr int c = i >> 1;
        if constexpr (i & 1) nd = M::mma(op[i & 3], ob[c], c == 0 ? acc_t{} : nd);
        else ns = M::mma(op[i & 3], qb[c], c == 0 ? acc_t{} : ns);
      } else {
        constexpr int o = (i - NQ) % OT;
        dq[o] = M::mma(op[i & 3], pb[(i - NQ) / OT], dq[o]);
      }
      if constexpr (H == 1 && i == NM - 4) {
        src.template wait<1>();  // (tile j + 2 has landed; this one is read)
        dense_barrier();
      }
      if constexpr (i + 4 < NQ) op[i & 3] = read_row(kn, vn, xf, i + 4, 1 - H);
      else if constexpr (i + 4 < NM) op[i & 3] = read_t(kt, tf, i + 4 - NQ, H);
      else op[i & 3] = read_row(kn2, vn2, xf, i + 4 - NM, H);
      // ds, evenly before the last 16 keys' sums
      each<16>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (e * (NM - OT) / 16 == i) {
          const float w = __builtin_amdgcn_exp2f(fmaf(cs[e], p.scale_log2, moff));
          float x = w * (cd[e] + ndelta);
          x = (seen >> (8 * (e >> 2) + (e & 3))) & 1 ? x : 0.f;
          if constexpr (e & 1) {
            pb[e >> 3][(e & 7) - 1] = (bf16)ex;
            pb[e >> 3][e & 7] = (bf16)x;
          }
          ex = x;
        }
      });
      if constexpr (H == 1 && i == NM - 2) mask[NS] = src.load(j + 4, s_kv[st][0], s_kv[st][1]);
    });
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (H == 1) {
#pragma unroll
      for (int i = 0; i < NS; ++i) mask[i] = mask[i + 1];
      st = st1;
    }
  };
  for (int j = 0; j < n; ++j) {
    half(j, std::integral_constant<int, 0>{}, sa, da, sb, db);
    half(j, std::integral_constant<int, 1>{}, sb, db, sa, da);
  }
  src.template wait<0>();
  if (!in) return;
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dq[o][4 * i + e] * p.scale;
      *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(p.dq) + b * p.dq_sb + t * p.dq_ss + h * p.dq_sh + 32 * o + 8 * i + 4 * hq) =
          bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
    }
}

// ---- dk and dv: four waves of 32 keys, tiles of 32 query rows of all heads ---------------
// A key block's rows are one range of r = t G + h; blocks that many rows see are cut in
// chunks of p.chunk rows, which leave partial sums that dense_dkv_join_kernel adds in order.
struct DkvUnit {
  int kb;          // key block, or -1: none
  int r0, r1;      // its rows (of the longest sequence)
  int part, nc;    // first partial of the block (if nc > 1), chunks
  int c;
};
__device__ __forceinline__ int dkv_tokens(const DenseParams& p, int j0) {  // tokens that see a key of the block at j0
  return j0 < p.first ? p.S : (int)min((int64_t)p.S, (int64_t)j0 + kDkvKeys - 1 + p.window);
}
__device__ __forceinline__ int dkv_chunks(const DenseParams& p, int kb) {
  const int j0 = kb * kDkvKeys;
  const int64_t rows = (int64_t)(dkv_tokens(p, j0) - j0) * p.G;
  return (int)((rows + p.chunk - 1) / p.chunk);
}
// of unit u of a (sequence, kv head)
__device__ __forceinline__ DkvUnit dkv_unit(const DenseParams& p, int u) {
  const int lane = threadIdx.x & 63, nkb = (p.S + kDkvKeys - 1) / kDkvKeys;
  int before = 0, parts = 0;
  for (int k0 = 0; k0 < nkb; k0 += 64) {
    const int kb = k0 + lane, nc = kb < nkb ? dkv_chunks(p, kb) : 0, np = nc > 1 ? nc : 0;
    int incl = nc, pin = np;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64), z = __shfl_up(pin, o, 64);
      if (lane >= o) {
        incl += y;
        pin += z;
      }
    }
    const int first = before + incl - nc;
    const uint64_t hit = __ballot(u >= first && u < first + nc);
    if (hit != 0) {
      const int w = __builtin_ctzll(hit);
      DkvUnit x;
      x.kb = k0 + w;
      x.nc = __builtin_amdgcn_readlane(nc, w);
      x.c = u - __builtin_amdgcn_readlane(first, w);
      x.part = __builtin_amdgcn_readlane(parts + pin - np, w);
      const int j0 = x.kb * kDkvKeys;
      x.r0 = j0 * p.G + x.c * p.chunk;
      x.r1 = (int)min((int64_t)x.r0 + p.chunk, (int64_t)dkv_tokens(p, j0) * p.G);
      return x;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
    parts += __builtin_amdgcn_readlane(pin, 63);
  }
  return DkvUnit{-1, 0, 0, 0, 0, 0};
}

template <int D>
__global__ __launch_bounds__(256, D == 128 ? 1 : 2) void dense_dkv_kernel(DenseParams p, int units) {
  typedef Tile<D> L;
  constexpr int NW = 4, RT = 32, KS = D / 16, OT = D / 32, NS = 4, CH = D / 8, RPI = L::RPI, NI = RT / RPI / NW;
  constexpr int SLOTS = RT / RPI * L::GROUP, LOADS = 2 * NI + 1;
  static_assert(NI >= 1, "a load instruction a wave");
  __shared__ u32x4 s_row[NS][2][SLOTS];     // Q, dO
  __shared__ float s_c[NS][NW][2][RT];      // -lse / scale, -delta (a copy a wave)

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hq = lane >> 5;
  const int groups = p.B * p.Hkv, gi = blockIdx.x % groups;
  const int b = gi / p.Hkv, g = gi % p.Hkv;
  const DkvUnit un = dkv_unit(p, blockIdx.x / groups);
  if (un.kb < 0) return;
  const int kb = __builtin_amdgcn_readfirstlane(un.kb);
  const DenseSeq sq = dense_seq(p, b);
  const int end = min(__builtin_amdgcn_readfirstlane(un.r1), sq.n * p.G), begin = __builtin_amdgcn_readfirstlane(un.r0);
  const int j0 = kb * kDkvKeys, key = j0 + 32 * wave + lr;
  const int n = end > begin ? (end - begin + RT - 1) / RT : 0;

  // ---- the keys' rows as second operands ----
  bf16x8 kf[KS], vf[KS];
  {
    const bool live = key < sq.n;
    const bf16* k = reinterpret_cast<const bf16*>(p.k) + b * p.k_sb + (live ? key * p.k_ss : 0) + g * p.k_sh + 8 * hq;
    const bf16* v = reinterpret_cast<const bf16*>(p.v) + b * p.v_sb + (live ? key * p.v_ss : 0) + g * p.v_sh + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(k + 16 * s), y = *reinterpret_cast<const bf16x8*>(v + 16 * s);
      kf[s] = live ? x : bf16x8{};
      vf[s] = live ? y : bf16x8{};
    }
  }

  // ---- loads: rows begin + 32 i .. as (token, head) pairs that advance with the tiles ----
  int lt[NI], lh[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int r = begin + (wave * NI + k) * RPI + lane / CH;
    lt[k] = r / p.G;
    lh[k] = r - lt[k] * p.G;
  }
  const int dt = RT / p.G, dh = RT - dt * p.G;
  const uint64_t qbase = (uint64_t)(uintptr_t)p.q + (uint64_t)(2 * (b * p.q_sb + g * p.G * p.q_sh));
  const uint64_t obase = (uint64_t)(uintptr_t)p.dout + (uint64_t)(2 * (b * p.do_sb + g * p.G * p.do_sh));
  const int64_t r_all = ((int64_t)b * p.Hkv + g) * p.S * p.G;
  const int last_row = p.S * p.G - 1;
  auto load = [&](int i) {  // tile i, in order of i
    const int st = i & (NS - 1);
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const int q = wave * NI + k;
      const uint32_t c = 16u * (uint32_t)((lane % CH) ^ L::at(lane / CH));
      const bool ok = i < n && lt[k] < sq.n;
      const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
      const uint64_t qa = ok ? qbase + (uint64_t)(2 * (lt[k] * p.q_ss + lh[k] * p.q_sh)) : zero;
      const uint64_t oa = ok ? obase + (uint64_t)(2 * (lt[k] * p.do_ss + lh[k] * p.do_sh)) : zero;
      dense_dma16(&s_row[st][0][q * L::GROUP], qa + c);
      dense_dma16(&s_row[st][1][q * L::GROUP], oa + c);
      lt[k] += dt;
      lh[k] += dh;
      if (lh[k] >= p.G) {
        lh[k] -= p.G;
        ++lt[k];
      }
    }
    const int r = min(begin + i * RT + (lane & 31), last_row);
    dense_dma4(&s_c[st][wave][0][0], (uint64_t)(uintptr_t)((lane < 32 ? p.row_lse : p.row_delta) + r_all + r));
  };
#pragma unroll
  for (int i = 0; i < NS; ++i) load(i);

  acc_t dk[OT], dv[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) dk[o] = dv[o] = acc_t{};

  constexpr int FLIP = D == 128 ? 6 : 5;
  const int l16 = lane & 15, trow = 4 * hq + (l16 >> 2), tc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
  const uint32_t kx = 16u * (uint32_t)L::at(lr), k0a = 16u * (uint32_t)(L::slot(lr, L::at(lr)) + hq);
  const uint32_t tx = 16u * (uint32_t)(L::at(trow) ^ tc), t0a = 16u * (uint32_t)L::slot(trow, L::at(trow)) + (uint32_t)(l16 & 1) * 8u;
  constexpr int NQ = 2 * KS, NM = NQ + 4 * OT;
  // (i even: Q, odd: dO)
  auto read_row = [&](uint32_t q, uint32_t o, uint32_t x, int i) {
    const int c = i >> 1;
    return lds_b128_at((i & 1 ? o : q) + (x ^ ((uint32_t)(D == 128 ? c >> 1 : c) << FLIP)) + (uint32_t)(D == 128 ? 32 * (c & 1) : 0));
  };
  // dO transposed by 16 rows, then Q
  auto read_t = [&](uint32_t q, uint32_t o, uint32_t x, int i) {
    const uint32_t at = (i < 2 * OT ? o : q) + (x ^ (uint32_t)(64 * (i % OT))) + (uint32_t)L::rows(16 * (i / OT % 2));
    const bf16x4 lo = lds_tr16_at(at), hi = lds_tr16_at(at + (uint32_t)L::rows(8));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // the accumulators' start values: the lane's rows 8 x + 4 hq + 0 .. 3 (no VALU for either)
  auto start = [&](const float* c) {
    acc_t a;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(c + 8 * x + 4 * hq);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * x + e] = y[e];
    }
    return a;
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  dense_barrier();
  acc_t sa, sb, da, db;
  bf16x8 op[4];
  {
    const uint32_t q = lds_addr(s_row[0][0]) + k0a, o = lds_addr(s_row[0][1]) + k0a;
    sa = start(s_c[0][wave][0]);
    da = start(s_c[0][wave][1]);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const bf16x8 x = read_row(q, o, kx, i);
      if (i & 1) da = M::mma(x, vf[i >> 1], da);
      else sa = M::mma(x, kf[i >> 1], sa);
    }
    const uint32_t q1 = lds_addr(s_row[1][0]) + k0a, o1 = lds_addr(s_row[1][1]) + k0a;
#pragma unroll
    for (int i = 0; i < 4; ++i) op[i] = read_row(q1, o1, kx, i);
  }

  auto step = [&](int i0, acc_t& cs, acc_t& cd, acc_t& ns, acc_t& nd) {
    const int st = i0 & (NS - 1), st1 = (i0 + 1) & (NS - 1), st2 = (i0 + 2) & (NS - 1);
    uint32_t xf = kx, tf = tx;
    asm volatile("" : "+v"(xf), "+v"(tf));
    const uint32_t qt = lds_addr(s_row[st][0]) + t0a, ot = lds_addr(s_row[st][1]) + t0a;
    const uint32_t qn = lds_addr(s_row[st1][0]) + k0a, on = lds_addr(s_row[st1][1]) + k0a;
    const uint32_t qn2 = lds_addr(s_row[st2][0]) + k0a, on2 = lds_addr(s_row[st2][1]) + k0a;
    // rows that see all keys of the block, or not
    const int r0 = begin + i0 * RT, t0 = r0 / p.G, t1 = (r0 + RT - 1) / p.G;
    const bool whole = r0 + RT <= end && j0 + kDkvKeys - 1 <= t0 && (j0 + kDkvKeys <= p.first || t1 - j0 < p.window);
    uint32_t seen = ~0u;
    if (!whole) {
      clear_rows<D, NW>(s_row[st][0], 0, wave, lane);
      clear_rows<D, NW>(s_row[st][1], 0, wave, lane);
      // row 8 x + 4 hq + e of the tile sees the lane's key
      seen = 0;
      int t = (r0 + 4 * hq) / p.G, h = r0 + 4 * hq - t * p.G;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int r = r0 + 8 * (x >> 2) + 4 * hq + (x & 3);
        seen |= (uint32_t)(r < end && dense_seen(p, key, t)) << (8 * (x >> 2) + (x & 3));
        const int by = (x & 3) == 3 ? 5 : 1;
        h += by;
        while (h >= p.G) {
          h -= p.G;
          ++t;
        }
      }
    }
    bf16x8 pb[2], db2[2];
    float ep = 0.f, es = 0.f;
    ns = start(s_c[st1][wave][0]);
    nd = start(s_c[st1][wave][1]);
    each<NM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i < NQ) {
        if constexpr (i & 1) nd = M::mma(op[i & 3], vf[i >> 1], nd);
        else ns = M::mma(op[i & 3], kf[i >> 1], ns);
      } else {
        constexpr int u = i - NQ, o = u % OT, k = u / OT % 2;
        if constexpr (u < 2 * OT) dv[o] = M::mma(op[i & 3], pb[k], dv[o]);
        else dk[o] = M::mma(op[i & 3], db2[k], dk[o]);
      }
      if constexpr (i == NM - 4) {
        // tile i0 + 2 has landed (behind it: i0 + 3), this one is read
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
        dense_barrier();
      }
      if constexpr (i + 4 < NQ) op[i & 3] = read_row(qn, on, xf, i + 4);
      else if constexpr (i + 4 < NM) op[i & 3] = read_t(qt, ot, tf, i + 4 - NQ);
      else op[i & 3] = read_row(qn2, on2, xf, i + 4 - NM);
      // p and ds, evenly before the first sums
      each<16>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (e * (NQ + OT) / 16 == i) {
          const bool ok = (seen >> (8 * (e >> 2) + (e & 3))) & 1;
          float w = __builtin_amdgcn_exp2f(cs[e] * p.scale_log2), x = w * cd[e];
          w = ok ? w : 0.f;
          x = ok ? x : 0.f;
          if constexpr (e & 1) {
            pb[e >> 3][(e & 7) - 1] = (bf16)ep;
            pb[e >> 3][e & 7] = (bf16)w;
            db2[e >> 3][(e & 7) - 1] = (bf16)es;
            db2[e >> 3][e & 7] = (bf16)x;
          }
          ep = w;
          es = x;
        }
      });
      if constexpr (i == NM - 2) load(i0 + 4);
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  int i = 0;
  for (; i + 1 < n; i += 2) {
    step(i, sa, da, sb, db);
    step(i + 1, sb, db, sa, da);
  }
  if (i < n) step(i, sa, da, sb, db);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- results: the lane's key, dims 32 o + 8 x + 4 hq + 0 .. 3 ----
  if (un.nc > 1) {
    float* out = p.dkv_part + (((int64_t)gi * p.dkv_parts + un.part + un.c) * kDkvKeys + 32 * wave + lr) * (2 * D);
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int d = 32 * o + 8 * x + 4 * hq;
        *reinterpret_cast<f32x4*>(out + d) = f32x4{dk[o][4 * x], dk[o][4 * x + 1], dk[o][4 * x + 2], dk[o][4 * x + 3]};
        *reinterpret_cast<f32x4*>(out + D + d) = f32x4{dv[o][4 * x], dv[o][4 * x + 1], dv[o][4 * x + 2], dv[o][4 * x + 3]};
      }
    return;
  }
  if (key >= p.S) return;
  bf16* ok = reinterpret_cast<bf16*>(p.dk) + b * p.dk_sb + key * p.dk_ss + g * p.dk_sh;
  bf16* ov = reinterpret_cast<bf16*>(p.dv) + b * p.dv_sb + key * p.dv_ss + g * p.dv_sh;
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      bf16x4 a, c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = (bf16)(dk[o][4 * x + e] * p.scale);
        c[e] = (bf16)dv[o][4 * x + e];
      }
      const int d = 32 * o + 8 * x + 4 * hq;
      *reinterpret_cast<bf16x4*>(ok + d) = a;
      *reinterpret_cast<bf16x4*>(ov + d) = c;
    }
}

// The chunks of key blocks that have several, added in order: 4 dims of a key a lane.
template <int D>
__global__ __launch_bounds__(256) void dense_dkv_join_kernel(DenseParams p) {
  const int nkb = (p.S + kDkvKeys - 1) / kDkvKeys;
  const int gi = blockIdx.x % (p.B * p.Hkv), kb = blockIdx.x / (p.B * p.Hkv);
  // (the block's first partial: the chunks before it)
  const int lane = threadIdx.x & 63;
  const int nc = dkv_chunks(p, kb);
  if (kb >= nkb || nc <= 1) return;
  int part = 0;
  for (int k = lane; k < kb; k += 64) {
    const int x = dkv_chunks(p, k);
    part += x > 1 ? x : 0;
  }
  part = dense_lanes_sum(part);
  const int b = gi / p.Hkv, g = gi % p.Hkv;
  constexpr int PER = 2 * D / 4;  // pieces a key
  const float* src = p.dkv_part + ((int64_t)gi * p.dkv_parts + part) * kDkvKeys * 2 * D;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < kDkvKeys * PER; i += gridDim.y * 256) {
    const int k = i / PER, d = 4 * (i % PER), key = kb * kDkvKeys + k;
    f32x4 s = {};
#pragma unroll 4
    for (int c = 0; c < nc; ++c) s += *reinterpret_cast<const f32x4*>(src + ((int64_t)c * kDkvKeys + k) * 2 * D + d);
    if (key >= p.S) continue;
    const bool isv = d >= D;
    const float f = isv ? 1.f : p.scale;
    bf16* o = isv ? reinterpret_cast<bf16*>(p.dv) + b * p.dv_sb + key * p.dv_ss + g * p.dv_sh + d - D
                  : reinterpret_cast<bf16*>(p.dk) + b * p.dk_sb + key * p.dk_ss + g * p.dk_sh + d;
    *reinterpret_cast<bf16x4*>(o) = bf16x4{(bf16)(s[0] * f), (bf16)(s[1] * f), (bf16)(s[2] * f), (bf16)(s[3] * f)};
  }
}

template <int D>
void launch(const DenseParams& p, int units, hipStream_t s) {
  dense_dq_kernel<D><<<(unsigned)((int64_t)p.B * p.nrb * p.Hkv), 512, 0, s>>>(p);
  dense_dkv_kernel<D><<<(unsigned)((int64_t)units * p.B * p.Hkv), 256, 0, s>>>(p, units);
  if (p.dkv_parts > 0)
    dense_dkv_join_kernel<D><<<dim3((unsigned)((p.S + kDkvKeys - 1) / kDkvKeys * p.B * p.Hkv), 4), 256, 0, s>>>(p);
}

}  // namespace

void launch_dense_bwd_mfma(const DenseParams& p, int units, hipStream_t s) {
  if (p.Dqk == 64) launch<64>(p, units, s);
  else launch<128>(p, units, s);
}

}  // namespace sfa

// gfx950 backward of dense attention through a window (sfa_dense.h), head dims 64 and
// 128 in bf16.
//
//   p_ij = exp(scale q_i.k_j - lse_i),  ds_ij = p_ij (do_i.v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// Two kernels, each of which makes the scores again, so that every sum has a fixed
// order without atomics: seven products for the five that are needed.
//
// dq: products of 32 x 32 (32x32x16) leave a lane with 16 scores of its query row, which
// rounded to bf16 are the second operand of the sums' product as they are; the first is read
// from LDS transposed.  A step makes the scores of the next 32 keys beside the weights of this
// one's, then its sums.  Each wave reads every key's rows as rows and K's again transposed: a
// kilobyte of LDS a product, as much as four SIMDs can take at once, which bounds it together
// with the products.  dk, dv: see there.  p and ds are rounded to bf16 once for their products
// (2^-8 of each: dk and dv up to 0.0025 rms from float64 where their own rounding is 0.0017; two
// parts would be half of the products again); dq's delta takes o as it was rounded to bf16 (dq
// 0.0026 to 0.0028: another would need o's other half kept).  Sums are float32.
//
// 8192 tokens, window 1024, 32 / 8 heads of 128: dq 272 us (0.71 PF/s of its three products), dk
// and dv 422 (0.61 PF/s of their four); 2 x 4096 tokens without a window, 32 / 2 heads: 406, 700.
// (In long runs; 292 and 491, 432 and 768 in the first passes.)

#include "sfa_dense_tiles.h"

namespace sfa {
namespace {

typedef Mfma<32> M;
typedef f32x16 acc_t;

// ---- units of the dk / dv kernel -----------------------------------------------------------
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
__device__ __forceinline__ int dkv_chunk(const DenseParams& p, int kb) {
  return kb >= p.cut0 && kb < p.cut1 ? p.cut_chunk : p.chunk;
}
__device__ __forceinline__ int dkv_chunks(const DenseParams& p, int kb) {
  const int j0 = kb * kDkvKeys, chunk = dkv_chunk(p, kb);
  const int64_t rows = (int64_t)(dkv_tokens(p, j0) - j0) * p.G;
  return (int)((rows + chunk - 1) / chunk);
}
// Chunk c of key block kb.  Chunks are counted from the last row that sees the block, so
// that without a window those of all blocks begin and end at the same rows.
__device__ __forceinline__ void dkv_rows(const DenseParams& p, DkvUnit& x) {
  const int j0 = x.kb * kDkvKeys, chunk = dkv_chunk(p, x.kb);
  const int64_t first = (int64_t)j0 * p.G, last = (int64_t)dkv_tokens(p, j0) * p.G, end = last - (int64_t)x.c * chunk;
  x.r1 = (int)end;
  x.r0 = (int)max(first, end - chunk);
}
// The units of a (sequence, kv head), in the order of their launch: the longest first, so that the
// card's last ones are short; those of a full chunk in order of the chunk, then of the block, so
// that what runs at once reads the same rows (a block's chunks after one another: 0.26 of the
// reads in L2).  One workgroup beside those of dq counts for each unit how many come before it
// (in each workgroup of the dk / dv kernel the search took 54 of its 530 us).  More blocks than
// kSorted: in order of the blocks.
constexpr int kSorted = 4096;
__device__ __forceinline__ void dkv_units(const DenseParams& p, int* lds) {
  const int nkb = (p.S + kDkvKeys - 1) / kDkvKeys, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* const s_whole = lds;            // chunks of the block's full size
  int* const s_rest = lds + kSorted;   // rows of its shorter one
  int* const s_sum = lds + 2 * kSorted;  // [8 waves][2]
  int* const s_at = s_sum + 16;          // of 512 blocks: the first unit, the first partial, chunks
  const bool sorted = nkb <= kSorted;
  auto cut = [&](int kb) { return kb >= p.cut0 && kb < p.cut1; };
  if (sorted) {
    for (int kb = tid; kb < nkb; kb += 512) {
      const int j0 = kb * kDkvKeys, chunk = dkv_chunk(p, kb);
      const int64_t rows = (int64_t)(dkv_tokens(p, j0) - j0) * p.G;
      s_whole[kb] = (int)(rows / chunk);
      s_rest[kb] = (int)(rows - rows / chunk * chunk);
    }
    dense_barrier();
  }
  auto place = [&](int kb, int c0, int step, const int* at0) {
    const int nc = at0[2];
    for (int c = c0; c < nc; c += step) {
      int at = at0[0] + c;
      if (sorted) {
        const bool full = c < s_whole[kb], mine = cut(kb);
        const int size = full ? dkv_chunk(p, kb) : s_rest[kb];
        at = full && mine ? c : 0;
#pragma unroll 4
        for (int k = 0; k < nkb; ++k) {
          const int whole = s_whole[k], rest = s_rest[k];
          if (!cut(k)) at += full && !mine ? min(whole, c) + (k < kb && whole > c ? 1 : 0) : whole;
          else if (!full || mine) at += full ? (k < kb ? whole : 0) : p.cut_chunk >= size ? whole : 0;
          if (!full || mine) at += rest > size || (!full && rest == size && k < kb) ? 1 : 0;
        }
      }
      *reinterpret_cast<int4*>(p.dkv_units + 4 * (int64_t)at) = int4{kb, c, at0[1], nc};
    }
  };
  int before = 0, parts = 0;  // of the blocks so far
  for (int k0 = 0; k0 < nkb; k0 += 512) {
    const int kb = k0 + tid, nc = kb < nkb ? dkv_chunks(p, kb) : 0, np = nc > 1 ? nc : 0;
    int x = nc, y = np;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int xx = __shfl_up(x, o, 64), yy = __shfl_up(y, o, 64);
      x += lane >= o ? xx : 0;
      y += lane >= o ? yy : 0;
    }
    if (lane == 63) {
      s_sum[2 * wave] = x;
      s_sum[2 * wave + 1] = y;
    }
    dense_barrier();
    int first = before + x - nc, part = parts + y - np;
    for (int w = 0; w < 8; ++w) {
      first += w < wave ? s_sum[2 * w] : 0;
      part += w < wave ? s_sum[2 * w + 1] : 0;
      before += s_sum[2 * w];
      parts += s_sum[2 * w + 1];
    }
    s_at[3 * tid] = first;
    s_at[3 * tid + 1] = part;
    s_at[3 * tid + 2] = nc;
    dense_barrier();
    // (as many threads a block as there are)
    const int blocks = min(512, nkb - k0), sub = 512 / blocks, in = tid / sub;
    if (in < blocks) place(k0 + in, tid % sub, sub, s_at + 3 * in);  // (s_at: written again behind the next scan's barrier)
  }
}

// ---- dq: eight waves of 32 query rows, tiles of 64 keys -------------------------------
template <int D>
__global__ __launch_bounds__(512, 2) void dense_dq_kernel(DenseParams p) {
  typedef Tile<D> L;
  constexpr int NW = 8, KT = kWideKeys, KS = D / 16, OT = D / 32, NS = 4;
  __shared__ u32x4 s_kv[NS][2][L::SLOTS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hq = lane >> 5;
  static_assert(sizeof(s_kv) >= (2 * kSorted + 16 + 3 * 512) * sizeof(int), "the units' counts");
  if (blockIdx.x == gridDim.x - 1) return dkv_units(p, reinterpret_cast<int*>(s_kv));
  int slot, g;
  dense_place(p, slot, g);
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
  // The row's statistics, which the dk / dv kernel's accumulators start from: -lse / scale
  // (nothing seen: -inf, which makes every weight 0) and -delta.
  float moff = kNegInf, ndelta = 0.f;
  {
    const bf16* o = reinterpret_cast<const bf16*>(p.out) + b * p.o_sb + (live ? t * p.o_ss + h * p.o_sh : 0) + 8 * hq;
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(o + 16 * s);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e & 1] = fmaf((float)x[e], (float)ob[s][e], sum[e & 1]);
    }
    const float all = xor32_sum(sum[0] + sum[1]);
    if (live) {
      const int64_t li = b * p.l_sb + t * p.l_ss + h * p.l_sh;
      const float lse = p.lse[li];
      moff = lse == kNegInf ? kNegInf : -lse / p.scale;
      ndelta = (p.dlse != nullptr ? p.dlse[li] : 0.f) - all;
    }
    if (in && hq == 0) {
      p.row_lse[rr] = moff;
      p.row_delta[rr] = ndelta;
    }
    moff *= p.scale_log2;
  }

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
  // sum_j p_ij do_i.v_j: delta again, but of o before its rounding to bf16 (of dsink, a float32
  // sum, that rounding is most of the error: 0.003 of it)
  float dsum = 0.f;
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
    if (!whole) {
      // infinities and NaN of keys that not every row sees: 0 times them would reach those
      // that do not (those that do have weights that are no numbers).  Another wave may still be
      // reading these rows for its scores: half 0 ends without a barrier, as do the first scores;
      // the first 32 rows of later tiles are read before half 1's.
      if (H == 1 || j == 0) dense_barrier();
      clear_rows<D, NW>(s_kv[st][0], 32 * H, wave, lane);
      const uint32_t seen = (uint32_t)((seen_of(p, pos, j0) & mask[0]) >> (32 * H)) >> (4 * hq);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool ok = (seen >> (8 * (e >> 2) + (e & 3))) & 1;
        cs[e] = ok ? cs[e] : kNegInf;
        cd[e] = ok ? cd[e] : 0.f;
      }
      // (opaque: otherwise the other path copies each score to where this one left it)
      asm volatile("" : "+v"(cs), "+v"(cd));
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
          const float x = w * (cd[e] + ndelta);
          dsum = fmaf(w, cd[e], dsum);
          asm volatile("" : "+v"(dsum));  // (added here: all weights held for one sum at the end spill)
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
  dense_barrier();  // the tiles are read
  dsum = xor32_sum(dsum);
  if (live && hq == 0) p.row_exact[rr] = (p.dlse != nullptr ? p.dlse[b * p.l_sb + t * p.l_ss + h * p.l_sh] : 0.f) - dsum;
  const RowsOut<D / 8> out{&s_kv[0][0][0] + wave * 32 * (D / 8)};
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (bf16)(live ? dq[o][4 * i + e] * p.scale : 0.f);  // (padding: 0 times what the others see)
      out.put(lr, 32 * o + 8 * i + 4 * hq, x);
    }
  out.store(in ? (uint64_t)(uintptr_t)(reinterpret_cast<bf16*>(p.dq) + b * p.dq_sb + t * p.dq_ss + h * p.dq_sh) : 0, lane);
}

// ---- dk and dv: 128 keys, tiles of 32 query rows of all heads ----------------------------
// Waves 0 .. 3 make p and ds of 32 rows x 128 keys (each 16 rows x 64 keys, 16x16x32: an
// operand of Q or dO read from LDS serves 64 keys) and leave them in LDS as bf16, in operand
// order; waves 4 .. 7, one on each SIMD beside one of those, take the last step's for the
// sums of 64 keys x half of the dims.  So no wave holds both the keys' rows and the
// sums (all in one wave are 320 registers: 929 us at 8192 tokens, window 1024, 32 / 8
// heads of 128, where this took 505 in as short a run), the products of one cover the weights of the other, and
// LDS moves 112 KB a step of 1024 clocks' products.  The waves of sums load the rows, five
// tiles ahead: they have the registers for the addresses (by all waves it was 626, with
// spills).
template <int D>
__global__ __launch_bounds__(512, 2) void dense_dkv_kernel(DenseParams p) {
  typedef Tile<D> L;
  typedef Mfma<16> M16;
  constexpr int NW = 8, RT = 32, NS = 7, CH = D / 8, RPI = L::RPI;
  constexpr int GROUPS = RT / RPI, PER = 2 * GROUPS / 4, LOADS = PER + 1;  // load instructions a tensor; a wave of sums
  constexpr int SLOTS = GROUPS * L::GROUP;
  __shared__ u32x4 s_row[NS][2][SLOTS];        // Q, dO
  __shared__ u32x4 s_pd[2][2][2][2][kDkvKeys]; // [step][p, ds][16 rows][lane half][key]: 8 rows
  __shared__ float s_c[NS][NW / 2][2][RT];     // -lse / scale, -delta (a copy for each wave of weights)

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = p.B * p.Hkv, gi = blockIdx.x % groups;
  const int b = gi / p.Hkv, g = gi % p.Hkv;
  const int4 unit = *reinterpret_cast<const int4*>(p.dkv_units + 4 * (int64_t)(blockIdx.x / groups));
  DkvUnit un{unit.x, 0, 0, unit.z, unit.w, unit.y};
  dkv_rows(p, un);
  const int kb = __builtin_amdgcn_readfirstlane(un.kb);
  const DenseSeq sq = dense_seq(p, b);
  const int end = min(__builtin_amdgcn_readfirstlane(un.r1), sq.n * p.G), begin = __builtin_amdgcn_readfirstlane(un.r0);
  const int nc = __builtin_amdgcn_readfirstlane(un.nc), part = __builtin_amdgcn_readfirstlane(un.part + un.c);
  const int j0 = kb * kDkvKeys;
  const int n = end > begin ? (end - begin + RT - 1) / RT : 0;
  // Blocks that are whole go through their rows from a multiple of the chunk on and around, so
  // that blocks that run at once and overlap read the same rows at a time.
  const int turn = nc == 1 && p.window < p.S ? (p.chunk - begin % p.chunk) % p.chunk / RT : 0, from = turn < n ? turn : 0;

  // ---- loads (by the waves of sums, which have registers for it): addresses that advance ----
  const int lw = wave & 3;
  const bool is_do = lw >= 2;
  const int dt = RT / p.G, dh_step = RT - dt * p.G;
  const int64_t x_ss = 2 * (is_do ? p.do_ss : p.q_ss), x_sh = 2 * (is_do ? p.do_sh : p.q_sh);
  const uint64_t xbase = is_do ? (uint64_t)(uintptr_t)p.dout + (uint64_t)(2 * (b * p.do_sb + g * p.G * p.do_sh))
                               : (uint64_t)(uintptr_t)p.q + (uint64_t)(2 * (b * p.q_sb + g * p.G * p.q_sh));
  const uint64_t by = (uint64_t)(dt * x_ss + dh_step * x_sh), by_wrap = by + (uint64_t)(x_ss - p.G * x_sh);
  uint64_t xa[PER];  // of the lane's rows of the next tile
  int xh[PER];       // their heads
  auto start_rows = [&](int tile) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = begin + tile * RT + (lw * PER + k) % GROUPS * RPI + lane / CH, t = r / p.G;
      xh[k] = r - t * p.G;
      xa[k] = xbase + (uint64_t)(t * x_ss + xh[k] * x_sh) + 16u * (uint32_t)((lane % CH) ^ L::at(lane / CH));
    }
  };
  const uint64_t c_at = (uint64_t)(uintptr_t)((lane < 32 ? p.row_lse : p.row_delta) + ((int64_t)b * p.Hkv + g) * p.S * p.G + begin + (lane & 31));
  int ls = 0, lpos = from;  // the next tile's place in LDS and among the unit's
  auto load = [&](int i) {  // the i-th tile, in order of i
    const int st = ls, left = i < n ? end - begin - lpos * RT : 0;
    ls = ls == NS - 1 ? 0 : ls + 1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int q = (lw * PER + k) % GROUPS;
      dense_dma16(&s_row[st][is_do][q * L::GROUP], q * RPI + lane / CH < left ? xa[k] : (uint64_t)(uintptr_t)kZeroRow);
      xh[k] += dh_step;
      const bool wrap = xh[k] >= p.G;
      xh[k] -= wrap ? p.G : 0;
      xa[k] += wrap ? by_wrap : by;
    }
    // (up to 31 rows behind the last, whose tiles are masked: the array is that much longer)
    dense_dma4(&s_c[st][lw][0][0], c_at + (uint64_t)(4 * RT) * (uint64_t)lpos);
    if (++lpos >= n) {
      lpos = 0;
      start_rows(0);
    }
  };
  // The tile a step is at: its number, place, first row's token and head (divisions are long).
  struct At {
    int i, st, pos, t, h;
    bool whole;  // its rows all see all keys of the block
  };
  const int tb = begin / p.G, hb = begin - tb * p.G;  // (of the first)
  const int dt31 = (RT - 1) / p.G, dh31 = RT - 1 - dt31 * p.G;
  auto settle = [&](At& a) {
    const int t1 = a.t + dt31 + (a.h + dh31 >= p.G ? 1 : 0);
    a.whole = begin + a.pos * RT + RT <= end && j0 + kDkvKeys - 1 <= a.t && (j0 + kDkvKeys <= p.first || t1 - j0 < p.window);
  };
  auto advance = [&](At& a) {
    ++a.i;
    a.st = a.st == NS - 1 ? 0 : a.st + 1;
    a.t += dt;
    a.h += dh_step;
    if (a.h >= p.G) {
      a.h -= p.G;
      ++a.t;
    }
    if (++a.pos == n) {
      a.pos = 0;
      a.t = tb;
      a.h = hb;
    }
    settle(a);
  };
  At at{0, 0, from, (begin + from * RT) / p.G, 0, false};
  at.h = begin + from * RT - at.t * p.G;
  settle(at);
  // Between the steps: what the sums are about to read of a tile whose rows do not see all
  // keys is cleared of infinities and NaN (0 times them would reach the keys they do not see).
  auto clear = [&](int st, bool is_whole) {
    if (!is_whole) {
      clear_rows<D, NW>(s_row[st][0], 0, wave, lane);
      clear_rows<D, NW>(s_row[st][1], 0, wave, lane);
    }
  };
  // In step i the sums read tile i - 1, the weights are made of tile i and their next operands
  // read of tile i + 1; tile i + 5 goes where tile i - 2 was.  At its end tile i + 2 has landed
  // (behind it i + 3 .. i + 5), what the step read is read.

  if (wave < 4) {
    // ---- weights: rows 16 rh + .., keys 64 kg + .. ----
    constexpr int KS = D / 32;
    const int lt = lane & 15, hq = lane >> 4, kg = wave & 1, rh = wave >> 1;
    bf16x8 kf[4][KS], vf[4][KS];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = j0 + 64 * kg + 16 * j + lt;
      const bool live = key < sq.n;
      const bf16* k = reinterpret_cast<const bf16*>(p.k) + b * p.k_sb + (live ? key * p.k_ss : 0) + g * p.k_sh + 8 * hq;
      const bf16* v = reinterpret_cast<const bf16*>(p.v) + b * p.v_sb + (live ? key * p.v_ss : 0) + g * p.v_sh + 8 * hq;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(k + 32 * s), y = *reinterpret_cast<const bf16x8*>(v + 32 * s);
        kf[j][s] = live ? x : bf16x8{};
        vf[j][s] = live ? y : bf16x8{};
      }
    }
    const int row = 16 * rh + lt;
    const uint32_t x0 = 16u * (uint32_t)(hq ^ L::at(row)), a0 = 16u * (uint32_t)L::slot(row, L::at(row));
    // A tile's operands are held: 16 keys after 16 keys, their scores and do.v in turn, beside
    // the weights of the 16 before.
    bf16x8 op[2][KS];
    f32x4 c0, c1;  // its rows' start values
    auto read_op = [&](int st, int w, int c) {
      return lds_b128_at(lds_addr(s_row[st][w]) + a0 + (x0 ^ (uint32_t)(64 * c)));
    };
    auto read_c = [&](int st) {
      c0 = *reinterpret_cast<const f32x4*>(&s_c[st][wave][0][16 * rh + 4 * hq]);
      c1 = *reinterpret_cast<const f32x4*>(&s_c[st][wave][1][16 * rh + 4 * hq]);
    };
    dense_barrier();
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      op[0][c] = read_op(0, 0, c);
      op[1][c] = read_op(0, 1, c);
    }
    read_c(0);
    int prev_st = 0;
    bool prev_whole = true;
    auto step = [&](auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      if (at.i > 0) clear(prev_st, prev_whole);
      // tokens of the lane's rows (-1: none)
      int tok[4];
      if constexpr (MASKED) {
        const int r0 = begin + at.pos * RT + 16 * rh + 4 * hq;
        int t = r0 / p.G, h = r0 - t * p.G;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          tok[e] = r0 + e < end ? t : -1;
          if (++h == p.G) {
            h = 0;
            ++t;
          }
        }
      }
      const int st1 = at.st == NS - 1 ? 0 : at.st + 1;
      char* const out = reinterpret_cast<char*>(&s_pd[at.i & 1][0][rh][hq & 1][64 * kg + lt]) + 8 * (hq >> 1);
      constexpr int WHICH = (int)sizeof(s_pd[0][0]), NJ = 2 * KS;  // products of 16 keys
      f32x4 s[2], d[2], w;
      bf16x4 dw;
      // four weights in four stages, some products apart
      auto weights = [&](int j, int stage) {
        f32x4 &cs = s[j & 1], &cd = d[j & 1];
        if (stage == 0) {
          if constexpr (MASKED) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool ok = dense_seen(p, j0 + 64 * kg + 16 * j + lt, tok[e]);
              // (do.v that is no number makes the weight none: its row is cleared for the sums)
              cs[e] = ok ? fmaf(0.f, cd[e], cs[e]) : kNegInf;
              cd[e] = ok ? cd[e] : 0.f;
            }
          }
          w = cs * p.scale_log2;
        } else if (stage == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(w[e]);
        } else if (stage == 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) dw[e] = (bf16)(w[e] * cd[e]);
        } else {
          *reinterpret_cast<bf16x4*>(out + 16 * 16 * j) = bf16x4{(bf16)w[0], (bf16)w[1], (bf16)w[2], (bf16)w[3]};
          *reinterpret_cast<bf16x4*>(out + WHICH + 16 * 16 * j) = dw;
        }
      };
      each<4 * NJ>([&](auto uc) {
        constexpr int u = decltype(uc)::value, j = u / NJ, i = u % NJ, c = i >> 1;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (i & 1) d[j & 1] = M16::mma(op[1][c], vf[j][c], c == 0 ? c1 : d[j & 1]);
        else s[j & 1] = M16::mma(op[0][c], kf[j][c], c == 0 ? c0 : s[j & 1]);
        if constexpr (j == 3) op[i & 1][c] = read_op(st1, i & 1, c);
        if constexpr (j > 0 && i % (NJ / 4) == 0) weights(j - 1, i / (NJ / 4));
      });
      __builtin_amdgcn_sched_barrier(0);
      read_c(st1);
#pragma unroll
      for (int k = 0; k < 4; ++k) weights(3, k);
      prev_st = at.st;
      prev_whole = at.whole;
      advance(at);
      dense_barrier();
    };
    for (int i = 0; i < n; ++i) {
      if (at.whole) step(std::false_type{});
      else step(std::true_type{});
    }
    if (n > 0) clear(prev_st, prev_whole);
    return;
  }

  // ---- sums: keys 64 kg + 32 m + .., dims DW dh + .. ----
  constexpr int DW = D / 2, DT = DW / 32;
  const int lr = lane & 31, hq = lane >> 5, kg = wave & 1, dh = (wave >> 1) & 1;
  f32x16 dk[DT][2], dv[DT][2];
#pragma unroll
  for (int o = 0; o < DT; ++o)
#pragma unroll
    for (int m = 0; m < 2; ++m) dk[o][m] = dv[o][m] = f32x16{};
  const int l16 = lane & 15, trow = 4 * hq + (l16 >> 2), tc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
  const uint32_t tx = 16u * (uint32_t)(L::at(trow) ^ tc), t0a = 16u * (uint32_t)L::slot(trow, L::at(trow)) + (uint32_t)(l16 & 1) * 8u;
  start_rows(from);
#pragma unroll
  for (int i = 0; i < 5; ++i) load(i);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  dense_barrier();
  for (int i = 0; i <= n; ++i) {  // (step 0 has no weights yet; at: tile i - 1)
    if (i < n) load(i + 5);
    if (i > 0) {
      clear(at.st, at.whole);
      const int st = at.st;
      const uint32_t q = lds_addr(s_row[st][0]) + t0a, o = lds_addr(s_row[st][1]) + t0a;
      const uint32_t pd = lds_addr(&s_pd[at.i & 1][0][0][hq][64 * kg + lr]);
      constexpr int WHICH = (int)sizeof(s_pd[0][0]), HALF = (int)sizeof(s_pd[0][0][0]);
      // products u: [dv, dk][16 rows][32 dims][32 keys]
      constexpr int NU = 2 * 2 * DT;
      auto read_t = [&](int u) {
        const int which = u / (2 * DT), ks = u / DT % 2, t = u % DT;
        const uint32_t at = (which ? q : o) + (tx ^ (uint32_t)(2 * (DW * dh + 32 * t))) + (uint32_t)L::rows(16 * ks);
        const bf16x4 lo = lds_tr16_at(at), hi = lds_tr16_at(at + (uint32_t)L::rows(8));
        return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      auto read_w = [&](int u, int m) {
        return lds_b128_at(pd + (uint32_t)(u / (2 * DT) * WHICH + u / DT % 2 * HALF + 32 * 16 * m));
      };
      bf16x8 a[3], w[2][2];
      a[0] = read_t(0);
      a[1] = read_t(1);
      w[0][0] = read_w(0, 0);
      w[0][1] = read_w(0, 1);
      each<NU>([&](auto uc) {
        constexpr int u = decltype(uc)::value, which = u / (2 * DT), t = u % DT, k = u / DT;
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (u + 2 < NU) a[(u + 2) % 3] = read_t(u + 2);
        if constexpr (t == 0 && u + DT < NU) {
          w[(k + 1) & 1][0] = read_w(u + DT, 0);
          w[(k + 1) & 1][1] = read_w(u + DT, 1);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if constexpr (which == 0) dv[t][m] = M::mma(a[u % 3], w[k & 1][m], dv[t][m]);
          else dk[t][m] = M::mma(a[u % 3], w[k & 1][m], dk[t][m]);
        }
      });
      __builtin_amdgcn_sched_barrier(0);
      advance(at);
    }
    if (i < n) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(3 * LOADS) : "memory");
      dense_barrier();
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- results: the lane's keys, dims DW dh + 32 o + 8 x + 4 hq + 0 .. 3 ----
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int in = 64 * kg + 32 * m + lr, key = j0 + in;
    if (nc > 1) {
      float* out = p.dkv_part + (((int64_t)gi * p.dkv_parts + part) * kDkvKeys + in) * (2 * D);
#pragma unroll
      for (int o = 0; o < DT; ++o)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int d = DW * dh + 32 * o + 8 * x + 4 * hq;
          *reinterpret_cast<f32x4*>(out + d) = f32x4{dk[o][m][4 * x], dk[o][m][4 * x + 1], dk[o][m][4 * x + 2], dk[o][m][4 * x + 3]};
          *reinterpret_cast<f32x4*>(out + D + d) = f32x4{dv[o][m][4 * x], dv[o][m][4 * x + 1], dv[o][m][4 * x + 2], dv[o][m][4 * x + 3]};
        }
      continue;
    }
    if (key >= p.S) continue;
    bf16* ok = reinterpret_cast<bf16*>(p.dk) + b * p.dk_sb + key * p.dk_ss + g * p.dk_sh;
    bf16* ov = reinterpret_cast<bf16*>(p.dv) + b * p.dv_sb + key * p.dv_ss + g * p.dv_sh;
#pragma unroll
    for (int o = 0; o < DT; ++o)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        bf16x4 a, c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = (bf16)(dk[o][m][4 * x + e] * p.scale);
          c[e] = (bf16)dv[o][m][4 * x + e];
        }
        const int d = DW * dh + 32 * o + 8 * x + 4 * hq;
        *reinterpret_cast<bf16x4*>(ok + d) = a;
        *reinterpret_cast<bf16x4*>(ov + d) = c;
      }
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
  dense_dq_kernel<D><<<(unsigned)((int64_t)p.B * p.nrb * p.Hkv + 1), 512, 0, s>>>(p);
  dense_dkv_kernel<D><<<(unsigned)((int64_t)units * p.B * p.Hkv), 512, 0, s>>>(p);
  if (p.dkv_parts > 0)
    dense_dkv_join_kernel<D><<<dim3((unsigned)((p.S + kDkvKeys - 1) / kDkvKeys * p.B * p.Hkv), 4), 256, 0, s>>>(p);
}

}  // namespace

void launch_dense_bwd_mfma(const DenseParams& p, int units, hipStream_t s) {
  if (p.Dqk == 64) launch<64>(p, units, s);
  else launch<128>(p, units, s);
}

}  // namespace sfa

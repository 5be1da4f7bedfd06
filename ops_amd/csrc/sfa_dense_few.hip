// gfx950 dense attention through a window (sfa_dense.h), head dims 64 and 128 in
// bf16, up to 64 query rows a (sequence, kv head): a decode step, a few tokens.
//
// Bound: HBM, the keys' rows.  A workgroup of four waves takes a range of 128-key tiles,
// 32 keys a wave; each wave brings its own rows to LDS, without a barrier among
// them, K two tiles ahead of its use and V as well: a tile's place is loaded over as
// soon as its last operand is read.  8-bit rows come as they are and become bf16 at
// their operand reads (e4m3 is exact in bf16); their powers of two go onto the scores
// and the weights.  S^T = K Q^T (16 keys x 16 rows a product), Q in registers; P^T is
// the operand of O^T = V^T P^T as it is.  The weights are multiplied in two bf16
// parts, which is hidden under the loads: results are as near the exact ones as their
// own rounding.  The waves' sums meet in LDS at the end, float32.  A step of ragged contexts
// (2.2 GB of bf16 rows, 32 / 8 heads of 128) takes 443 us, 4.99 TB/s; of e4m3 rows (0.8 GB, one
// workgroup's conversions under the other's loads) 170 us, 4.73 TB/s; a copy reaches 5.14.

#include "sfa_dense_tiles.h"

namespace sfa {
namespace {

constexpr int kFewKeys = 32;  // a wave's part of a tile

// Places of a row's 16-byte chunks in LDS, c ^ at(r): 16 rows at one chunk (K), and the
// rows of two lane groups at a chunk or a pair of chunks (V, transposed), lie in
// different banks.
template <int ROW>  // bytes a row
struct FewSwz {
  static __device__ __forceinline__ int bf16_at(int r) {
    if constexpr (ROW == 256) return ((r & 7) << 1) | ((r >> 3) & 1);
    else return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  }
  static __device__ __forceinline__ int fp8_at(int r) {
    if constexpr (ROW == 128) return ((r >> 1) & 3) | ((((r >> 4) ^ (r >> 3)) & 1) << 2);
    else return (r >> 2) & 3;
  }
};

__device__ __forceinline__ uint32_t bad8(uint32_t w) {  // bytes of w that are NaN: their masks
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= (w & (0x7fu << (8 * i))) == (0x7fu << (8 * i)) ? 0xffu << (8 * i) : 0u;
  return m;
}
// Infinities and NaN of bf16 elements as the largest finite values: for the weights' second
// parts, which are 0 or of either sign and would make no number of the first ones' infinities
// (1% of a step: 438 -> 443 us, 32 contexts of 1K to 32K).
__device__ __forceinline__ bf16x8 no_infinities(bf16x8 x) {
  typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  // (positive ones are the upper end of signed 16 bits, negative ones of unsigned)
  const i16x8 p = __builtin_elementwise_min(__builtin_bit_cast(i16x8, x), i16x8(0x7f7f));
  return __builtin_bit_cast(bf16x8, __builtin_elementwise_min(__builtin_bit_cast(u16x8, p), u16x8(0xff7f)));
}
// at most N of the wave's loads in flight, its LDS reads done
template <int N>
__device__ __forceinline__ void few_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <int D, int NG, bool FP8, bool ONE>
__global__ __launch_bounds__(256, NG == 4 ? 1 : 2) void dense_few_kernel(DenseParams p) {
  typedef Mfma<16> M;
  typedef f32x4 acc_t;
  constexpr int WK = 4, KT = kFewKeys, KS = D / 32, OT = D / 16, ROWS = 16 * NG;
  constexpr int ROW = FP8 ? D : 2 * D, CH = ROW / 16, RPI = 64 / CH, NI = KT / RPI;  // rows and instructions of a load
  constexpr int PART = KT * CH;                        // 16-byte chunks of a tile's K or V
  constexpr int LOADS = FP8 ? NI + 1 : NI;             // a K or V part's loads in flight
  constexpr int STAGES = 2;
  constexpr int MERGE = 2 * NG * OT * 64, SLOTS = STAGES * WK * 2 * PART > MERGE ? STAGES * WK * 2 * PART : MERGE;

  __shared__ u32x4 s_kv[SLOTS];
  __shared__ int s_id[WK][2][64];
  __shared__ uint32_t s_sc[FP8 ? WK : 1][STAGES][2][64];  // exponents of K and V rows (lanes 32 .. 63 repeat them)
  __shared__ float s_ml[WK][2][ROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wk = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lt = lane & 15, hq = lane >> 4;

  const int g = blockIdx.x % p.Hkv;
  DenseItem it;
  if (!dense_item(p, blockIdx.x / p.Hkv, g, it)) return;
  const int b = it.b, n = it.v1 - it.v0;

  // ---- rows ----
  bf16x8 qb[NG][KS];
  int pos[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int r = it.row0 + 16 * i + lt, t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < p.S * p.G && t < it.s.n;
    pos[i] = live ? it.s.ctx + t : -1;
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 32 * s);
      qb[i][s] = live ? x : bf16x8{};
    }
  }
  const int p0 = it.s.ctx + it.row0 / p.G, p1 = it.s.ctx + min((it.row0 + p.rows - 1) / p.G, it.s.n - 1);

  // ---- loads ----
  const int64_t esz = FP8 ? 1 : 2;
  const bool paged = p.block_table != nullptr;
  const int shift = paged ? p.page_shift : 30, npages = paged ? p.num_pages : 1, in_page = (1 << shift) - 1;
  const int32_t* trow = paged ? p.block_table + b * p.bt_sb : nullptr;
  const uint64_t kbase = (uint64_t)(uintptr_t)p.k + (uint64_t)(esz * (g * p.k_sh + (paged ? 0 : b * p.k_sb)));
  const uint64_t vbase = (uint64_t)(uintptr_t)p.v + (uint64_t)(esz * (g * p.v_sh + (paged ? 0 : b * p.v_sb)));
  const int64_t kpage = esz * p.k_sb, vpage = esz * p.v_sb, krow = esz * p.k_ss, vrow = esz * p.v_ss;
  // first key of the wave's i-th tile (past the range: its last tile's)
  auto key_at = [&](int i) { return it.tiles.tile(it.v0 + max(min(i, n - 1), 0)) * (WK * KT) + wk * KT; };
  // Table entries come in batches of 64, npt a tile, through LDS: the loop has no load
  // that the compiler would wait for (and every load before it with it).
  const int lg = ONE || shift >= 5 ? 0 : 5 - shift, npt = 1 << lg, tpb = 64 >> lg;
  // (the batch behind the one that tile i is in, in every step: the number of loads is constant)
  auto fetch_ids = [&](int batch) {
    const int i = batch * tpb + (lane >> lg), j = min(key_at(i) + ((lane & (npt - 1)) << shift), p.cap - 1);
    dense_dma4(s_id[wk][batch & 1], paged ? (uint64_t)(uintptr_t)(trow + (j >> shift)) : (uint64_t)(uintptr_t)kZeroRow);
  };
  // id of row r of the i-th tile
  auto id_of = [&](int i, int r) {
    if (!paged) return 0;
    return s_id[wk][(i / tpb) & 1][(i & (tpb - 1)) * npt + (ONE ? 0 : r >> min(shift, 5))];
  };
  // One part (K or V) of the i-th tile; its rows that are there.
  auto load_part = [&](int i, bool v, u32x4* dst) {
    const int j0 = key_at(i);
    const bool on = i < n;
    const uint64_t base = v ? vbase : kbase, zero = (uint64_t)(uintptr_t)kZeroRow;
    const int64_t page = v ? vpage : kpage, row = v ? vrow : krow;
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (lane constants are formed per part)
    const int sub = ln / CH;
    uint64_t mask;
    auto at = [&](int r) { return FP8 ? FewSwz<ROW>::fp8_at(r) : FewSwz<ROW>::bf16_at(r); };
    const uint8_t* sc = v ? p.vs : p.ks;
    const int64_t s_sb = v ? p.vs_sb : p.ks_sb, s_ss = v ? p.vs_ss : p.ks_ss, s_sh = v ? p.vs_sh : p.ks_sh;
    if constexpr (ONE) {
      const int id = __builtin_amdgcn_readfirstlane(id_of(i, 0)), in = j0 & in_page, left = p.cap - j0;
      const bool ok = on && left > 0 && id >= 0 && id < npages;
      const uint64_t tb = ok ? base + (uint64_t)(id * page + in * row) : zero;
#pragma unroll
      for (int q = 0; q < NI; ++q) {
        const int r = q * RPI + sub;
        const uint32_t c = 16u * (uint32_t)((ln % CH) ^ at(r));
        dense_dma16(dst + q * 64, tb, (ok && r < left ? (uint32_t)(r * (int)row) : 0u) + c);
      }
      if constexpr (FP8) {
        const int r = ln & 31;
        const bool there = ok && r < left;
        dense_dma1(&s_sc[wk][i & 1][v][0], there ? (uint64_t)(uintptr_t)(sc + id * s_sb + (in + r) * s_ss + g * s_sh) : zero);
      }
      mask = !ok ? 0 : left >= KT ? ~0ull : (1ull << left) - 1;
    } else {
#pragma unroll
      for (int q = 0; q < NI; ++q) {
        const int r = q * RPI + sub, j = j0 + r, id = id_of(i, r);
        const bool ok = on && j < p.cap && id >= 0 && id < npages;
        const uint64_t a = ok ? base + (uint64_t)(id * page + (j & in_page) * row) : zero;
        dense_dma16(dst + q * 64, a + 16u * (uint32_t)((ln % CH) ^ at(r)));
      }
      const int r = ln & 31, j = j0 + r, id = id_of(i, r);
      const bool ok = on && j < p.cap && id >= 0 && id < npages;
      if constexpr (FP8)
        dense_dma1(&s_sc[wk][i & 1][v][0], ok ? (uint64_t)(uintptr_t)(sc + id * s_sb + (j & in_page) * s_ss + g * s_sh) : zero);
      mask = __ballot(ok);
    }
    return (uint32_t)mask;
  };
  auto part_at = [&](int i, bool v) { return s_kv + ((i & 1) * WK + wk) * (2 * PART) + (v ? PART : 0); };

  // ---- operands ----
  const uint32_t pitch = ROW;
  // K: row lt (+ 16), 8 dims at 32 s + 8 hq; V: transposed, by 16 dims
  const int ksz = FP8 ? FewSwz<ROW>::fp8_at(lt) : FewSwz<ROW>::bf16_at(lt);
  const int ksz16 = FP8 ? FewSwz<ROW>::fp8_at(lt + 16) : FewSwz<ROW>::bf16_at(lt + 16);
  auto as_bf16 = [&](uint32_t w0, uint32_t w1) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.f, true));
    return __builtin_bit_cast(bf16x8, r);
  };
  auto read_k = [&](uint32_t kt, int mt, int s) {
    const uint32_t row = kt + (uint32_t)(16 * mt + lt) * pitch;
    const int z = mt ? ksz16 : ksz;
    if constexpr (FP8) {
      const uint32_t a = row + (uint32_t)(((2 * s + (hq >> 1)) ^ z) * 16 + (hq & 1) * 8);
      const u32x2 w = *(const __attribute__((address_space(3))) u32x2*)(uintptr_t)a;
      return as_bf16(w[0], w[1]);
    } else {
      return lds_b128_at(row + (uint32_t)(((4 * s + hq) ^ z) * 16));
    }
  };
  auto read_v = [&](uint32_t vt, int ot) {
    if constexpr (FP8) {
      // 8 rows x 16 dims: rows 4 hq + 0 .. 3 and 16 further, two lanes a row
      const int i = lt >> 1, r = 4 * hq + (i & 3) + 16 * (i >> 2);
      const uint32_t a = vt + (uint32_t)r * pitch + (uint32_t)((ot ^ FewSwz<ROW>::fp8_at(r)) * 16 + (lt & 1) * 8);
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
      const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uintptr_t)a);
      return as_bf16((uint32_t)w[0], (uint32_t)w[1]);
    } else {
      // 4 rows x 16 dims, four lanes a row; then the rows 16 further
      const int r = 4 * hq + (lt >> 2), c = 2 * ot + ((lt & 3) >> 1);
      const uint32_t a = vt + (uint32_t)r * pitch + (uint32_t)((lt & 1) * 8);
      const bf16x4 lo = lds_tr16_at(a + (uint32_t)((c ^ FewSwz<ROW>::bf16_at(r)) * 16));
      const bf16x4 hi = lds_tr16_at(a + 16u * pitch + (uint32_t)((c ^ FewSwz<ROW>::bf16_at(r + 16)) * 16));
      return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  };

  acc_t oacc[NG][OT];
  float m_used[NG], l_part[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    m_used[i] = kNegInf;
    l_part[i] = 0.f;
#pragma unroll
    for (int o = 0; o < OT; ++o) oacc[i][o] = acc_t{};
  }

  // Infinities and NaN of a V part whose rows not every query row sees, as bits; cleared in
  // LDS, as 0 times them would reach rows that do not see them, and added by hand to those that do.
  auto clear_bad = [&](u32x4* v) {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const u32x4 w = v[64 * i + lane];
      u32x4 m;
#pragma unroll
      for (int e = 0; e < 4; ++e) m[e] = FP8 ? bad8(w[e]) : bad16(w[e]);
      const bool any = (m[0] | m[1] | m[2] | m[3]) != 0;
      if (any) v[64 * i + lane] = w & ~m;
      for (uint64_t l = __ballot(any); l != 0; l &= l - 1) bad |= 1u << (RPI * i + __builtin_ctzll(l) / CH);
    }
    return bad;
  };
  auto add_bad = [&](uint32_t bad, int j0, const bf16x8 (&pb)[NG], const bf16x8 (&pr)[NG]) {
    const DenseParams& p = late_params();
    for (; bad != 0; bad &= bad - 1) {
      const int key = __builtin_ctz(bad), at = 4 * (key >> 4) + (key & 3);
      const int64_t vo = dense_row(p, b, j0 + key, p.v_sb, p.v_ss);
      if (vo < 0) continue;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float own = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) own = e == at ? (float)pb[i][e] + (float)pr[i][e] : own;
        const float w = __shfl(own, lt + 16 * ((key & 15) >> 2), 64);
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t d = vo + g * p.v_sh + 16 * o + 4 * hq + e;
            float v;
            if constexpr (FP8) v = __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(p.v)[d], 0);
            else v = (float)reinterpret_cast<const bf16*>(p.v)[d];
            if (w != 0.f && !(fabsf(v) <= 3.402823466e38f)) oacc[i][o][e] += w * v;
          }
      }
    }
  };

  fetch_ids(0);
  fetch_ids(1);
  few_wait<0>();
  uint32_t mk[3];  // rows that are there, of tiles j, j + 1, j + 2
  mk[0] = load_part(0, false, part_at(0, false));
  load_part(0, true, part_at(0, true));
  fetch_ids(1);
  mk[1] = load_part(1, false, part_at(1, false));
  load_part(1, true, part_at(1, true));

  for (int j = 0; j < n; ++j) {
    const int j0 = key_at(j);
    const uint32_t kt = lds_addr(part_at(j, false)), vt = lds_addr(part_at(j, true));
    few_wait<3 * LOADS + 1>();  // K of tile j: behind it V of j, ids, both of j + 1
    // ---- scores: the lane's row, keys 16 mt + 4 hq + e ----
    acc_t sc[NG][2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8 kf = read_k(kt, mt, s);
#pragma unroll
        for (int i = 0; i < NG; ++i) sc[i][mt] = M::mma(kf, qb[i][s], s == 0 ? acc_t{} : sc[i][mt]);
      }
    f32x4 vsc[2];
    if constexpr (FP8) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const u32x4 e = *reinterpret_cast<const u32x4*>(&s_sc[wk][j & 1][0][16 * mt + 4 * hq]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float k = scale_of((uint8_t)e[x]);
#pragma unroll
          for (int i = 0; i < NG; ++i) sc[i][mt][x] *= k;
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's place is read
    fetch_ids((j + 2) / tpb + 1);
    mk[2] = load_part(j + 2, false, part_at(j, false));
    const uint32_t mask = mk[0];
    // ---- softmax ----
    const bool whole = mask == 0xffffffffu && j0 + KT - 1 <= p0 && (j0 + KT <= p.first || p1 - j0 < p.window);
    bf16x8 pb[NG], pr[NG];
    bool over = false;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (!whole) {
        const uint32_t seen = ((uint32_t)seen_of(p, pos[i], j0) & mask) >> (4 * hq);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[i][mt][x] = (seen >> (16 * mt + x)) & 1 ? sc[i][mt][x] : kNegInf;
      }
      float t = fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3]));
      t = fmaxf(t, fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
      over |= t * p.scale_log2 > m_used[i] + 8.f;
    }
    if (__any(over)) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float t = fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3]));
        t = fmaxf(t, fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
        const float mn = fmaxf(m_used[i], xor32_max(xor16_max(t)) * p.scale_log2);
        const float alpha = mn == kNegInf ? 1.f : exp2f(m_used[i] - mn);
        l_part[i] *= alpha;
#pragma unroll
        for (int o = 0; o < OT; ++o) oacc[i][o] *= alpha;
        m_used[i] = mn;
      }
    }
    few_wait<3 * LOADS + 2>();  // V of tile j: behind it ids, both of j + 1, ids, K of j + 2
    if constexpr (FP8) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const u32x4 e = *reinterpret_cast<const u32x4*>(&s_sc[wk][j & 1][1][16 * mt + 4 * hq]);
#pragma unroll
        for (int x = 0; x < 4; ++x) vsc[mt][x] = scale_of((uint8_t)e[x]);
      }
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const float moff = m_used[i] == kNegInf ? 0.f : -m_used[i];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float w = __builtin_amdgcn_exp2f(fmaf(sc[i][mt][x], p.scale_log2, moff));
          l_part[i] += w;
          if constexpr (FP8) w = whole || w != 0.f ? w * vsc[mt][x] : 0.f;  // (a row of NaN that is not seen)
          pb[i][4 * mt + x] = (bf16)w;
          pr[i][4 * mt + x] = (bf16)(w - (float)pb[i][4 * mt + x]);
        }
    }
    // ---- sums ----
    uint32_t bad = 0;
    if (!whole) bad = clear_bad(part_at(j, true));
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const bf16x8 a = read_v(vt, o), af = FP8 ? a : no_infinities(a);  // (e4m3 has none)
#pragma unroll
      for (int i = 0; i < NG; ++i) oacc[i][o] = M::mma(af, pr[i], M::mma(a, pb[i], oacc[i][o]));
    }
    if (bad != 0) add_bad(bad, j0, pb, pr);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V's place is read
    load_part(j + 2, true, part_at(j, true));
    mk[0] = mk[1];
    mk[1] = mk[2];
  }
  few_wait<0>();

  // ---- the waves' sums joined in halves through LDS, and the results ----
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    l_part[i] += __shfl_xor(l_part[i], 16, 64);
    l_part[i] = xor32_sum(l_part[i]);
  }
#pragma unroll
  for (int half = WK / 2; half > 0; half >>= 1) {
    dense_barrier();
    f32x4* mine = reinterpret_cast<f32x4*>(s_kv) + (wk % half) * (NG * OT * 64);
    if (wk >= half && wk < 2 * half) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
#pragma unroll
        for (int o = 0; o < OT; ++o) mine[(i * OT + o) * 64 + lane] = oacc[i][o];
        if (hq == 0) {
          s_ml[wk][0][16 * i + lt] = m_used[i];
          s_ml[wk][1][16 * i + lt] = l_part[i];
        }
      }
    }
    dense_barrier();
    if (wk < half) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const float m2 = s_ml[wk + half][0][16 * i + lt], l2 = s_ml[wk + half][1][16 * i + lt];
        const float m = fmaxf(m_used[i], m2);
        // (a row without a finite maximum has sums that are zero or NaN)
        const float a1 = m_used[i] == kNegInf ? 1.f : exp2f(m_used[i] - m), a2 = m2 == kNegInf ? 1.f : exp2f(m2 - m);
        l_part[i] = l_part[i] * a1 + l2 * a2;
#pragma unroll
        for (int o = 0; o < OT; ++o) oacc[i][o] = oacc[i][o] * a1 + mine[(i * OT + o) * 64 + lane] * a2;
        m_used[i] = m;
      }
    }
  }
  if (wk != 0) return;
  const DenseParams& pe = late_params();
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const int row = 16 * i + lt, r = it.row0 + row, t = r / pe.G, h = g * pe.G + r % pe.G;
    if (r >= pe.S * pe.G) continue;
    float lse, f;
    if (it.partial) {
      f = dense_part(m_used[i], l_part[i], lse);
      if (hq == 0) pe.part_lse[it.part + row] = lse;
    } else {
      f = dense_finish(pe, h, pos[i] >= 0, m_used[i], l_part[i], lse);
      if (hq == 0) pe.lse[b * pe.l_sb + t * pe.l_ss + h * pe.l_sh] = lse;
    }
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const f32x4 y = oacc[i][o] * f, x = f == 0.f ? f32x4{} : y;
      const int d = 16 * o + 4 * hq;
      if (it.partial) {
        *reinterpret_cast<f32x4*>(pe.part_o + (it.part + row) * D + d) = x;
      } else {
        *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(pe.out) + b * pe.o_sb + t * pe.o_ss + h * pe.o_sh + d) =
            bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
      }
    }
  }
}

template <int D, int NG>
void launch(const DenseParams& p, bool fp8, unsigned grid, hipStream_t s) {
  const bool one = dense_one_base(p, fp8 ? 1 : 2, 5);
  if (fp8 && one) dense_few_kernel<D, NG, true, true><<<grid, 256, 0, s>>>(p);
  else if (fp8) dense_few_kernel<D, NG, true, false><<<grid, 256, 0, s>>>(p);
  else if (one) dense_few_kernel<D, NG, false, true><<<grid, 256, 0, s>>>(p);
  else dense_few_kernel<D, NG, false, false><<<grid, 256, 0, s>>>(p);
}
template <int D>
void by_rows(const DenseParams& p, bool fp8, unsigned grid, hipStream_t s) {
  if (p.rows == 16) launch<D, 1>(p, fp8, grid, s);
  else if (p.rows == 32) launch<D, 2>(p, fp8, grid, s);
  else launch<D, 4>(p, fp8, grid, s);
}

}  // namespace

void launch_dense_few(const DenseParams& p, int kv_dtype, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.slots * p.Hkv);
  if (p.Dqk == 64) by_rows<64>(p, kv_dtype == SFA_DTYPE_FP8_E4M3, grid, s);
  else by_rows<128>(p, kv_dtype == SFA_DTYPE_FP8_E4M3, grid, s);
}

}  // namespace sfa

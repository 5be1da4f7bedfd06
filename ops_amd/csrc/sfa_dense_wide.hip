// gfx950 dense attention through a window (sfa_dense.h), head dims 64 and 128 in
// bf16, many query rows: a chunk of a prompt, a training step's forward.
//
// Eight waves of 32 query rows share tiles of 64 keys in LDS.  S^T = K Q^T (32 keys x
// 32 rows a product, 32x32x16, Q in registers) leaves a lane with 16 keys of
// its row; in bf16 they are the second operand of O^T = V^T P^T as they are, whose
// first is read from LDS transposed.  A step makes the scores of tile j + 1 beside
// the softmax of tile j, then the sums of tile j.  The running maximum moves only
// when a score passes it by 8 (base 2; 2^8 more at most in a float32 sum), so a tile
// needs no maximum across lanes.  P is rounded to bf16 once for its product (2^-8 of
// a weight, as much as the result's own rounding); sums and statistics are float32.
//
// Bound: the products and the softmax's instructions beside them: 2048 tokens behind 14336, 32 /
// 8 heads of 128, 510 us, 1.01 PF/s (a large product reaches 1.19 on this card), matrix units
// busy 0.48; of 64 dims a score's exponential takes as long as its products.  Short ranges pay
// 13 us a workgroup for the rows' way in and out (8192 tokens, window 1024: 190 us, 0.68 PF/s).
//
// e4m3 rows come to registers one product before a step's end and go from there to LDS, so a
// step waits for their loads with nothing to cover them: 381 us for 320 over bf16 pages (4 x
// 1000 tokens, window 4096, 64 / 8 heads of 64), 781 for 522 with 128 dims (the prompt above),
// where the bytes and their scales spill as well (32 registers; 20 with small pages, 8 of bf16).

#include "sfa_dense_tiles.h"

namespace sfa {
namespace {

template <int D, bool FP8, bool ONE>
__global__ __launch_bounds__(512, 2) void dense_wide_kernel(DenseParams p) {
  typedef Mfma<32> M;
  typedef f32x16 acc_t;
  constexpr int NW = 8, KT = kWideKeys, KS = D / 16, OT = D / 32, NS = 4;
  __shared__ u32x4 s_kv[NS][2][Tile<D>::SLOTS];
  __shared__ unsigned long long s_bad[2];
  static_assert(sizeof(s_kv) >= 256 * D * 4, "the results' rows");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, hq = lane >> 5;

  int slot, g;
  dense_place(p, slot, g);
  DenseItem it;
  if (!dense_item(p, slot, g, it)) return;
  const int b = it.b, row = 32 * wave + lr, r = it.row0 + row;
  const int t = r / p.G, h = g * p.G + r % p.G;
  const bool in = r < p.S * p.G, live = in && t < it.s.n;
  const int pos = live ? it.s.ctx + t : -1;
  // what all rows of the block see of a tile without a look at each
  const int p0 = it.s.ctx + it.row0 / p.G, p1 = it.s.ctx + min((it.row0 + p.rows - 1) / p.G, it.s.n - 1);

  bf16x8 qb[KS];
  {
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 16 * s);
      qb[s] = live ? x : bf16x8{};
    }
  }

  TileSource<D, NW, FP8, ONE> src(p, it, wave, lane);
  const int n = it.v1 - it.v0;
  acc_t oacc[OT];
#pragma unroll
  for (int o = 0; o < OT; ++o) oacc[o] = acc_t{};
  float m_used = kNegInf, l_part = 0.f;

  // Operand addresses.  K: row lr, chunk 2 s + hq; V: rows 4 hq + (lane % 16) / 4, 16 dims
  // by lane / 16 % 2.  The places of a row's chunks differ by rows in bits 2 and 3 (D = 64: 1
  // and 2) of the chunk's number, which a step flips in its copy of the address.
  typedef Tile<D> L;
  constexpr int FLIP = D == 128 ? 6 : 5;  // the first of those bits, in bytes
  const int l16 = lane & 15, vrow = 4 * hq + (l16 >> 2), vc = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
  const uint32_t kx = 16u * (uint32_t)L::at(lr), k0a = 16u * (uint32_t)(L::slot(lr, L::at(lr)) + hq);
  const uint32_t vx = 16u * (uint32_t)(L::at(vrow) ^ vc) , v0a = 16u * (uint32_t)L::slot(vrow, L::at(vrow)) + (uint32_t)(l16 & 1) * 8u;

  uint64_t mask[NS + 1];  // rows that are there, of tiles j, j + 1, ..
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    mask[i] = src.load(i, s_kv[i][0], s_kv[i][1]);
    src.store(s_kv[i][0], s_kv[i][1]);
  }
  if (tid < 2) s_bad[tid] = 0;
  src.template wait<0>();
  dense_barrier();

  // A step's products: NQ of the next tile's scores, 32 keys at a time, then the
  // sums' by 16 keys; each takes one operand from LDS, read four products ahead.
  constexpr int NQ = 2 * KS, NM = NQ + 4 * OT;
  bf16x8 op[4];
  // (a, x: the address of place 0 of the lane's row, the flips; i: the product)
  auto read_k = [&](uint32_t a, uint32_t x, int i) {
    const int c = i % KS, kb = i / KS;
    return lds_b128_at(a + (x ^ ((uint32_t)(D == 128 ? c >> 1 : c) << FLIP)) + (uint32_t)((D == 128 ? 32 * (c & 1) : 0) + L::rows(32 * kb)));
  };
  auto read_v = [&](uint32_t a, uint32_t x, int i) {
    const uint32_t at = a + (x ^ (uint32_t)(64 * (i % OT)));
    const bf16x4 lo = lds_tr16_at(at + (uint32_t)L::rows(16 * (i / OT))), hi = lds_tr16_at(at + (uint32_t)L::rows(16 * (i / OT) + 8));
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // the largest of a lane's 32 scores, in 16 steps of two
  auto max_step = [&](const acc_t (&c)[2], float (&x)[2], auto tc) {
    constexpr int t = decltype(tc)::value, k = t & 1, e = 2 * (t >> 1);
    x[k] = t < 2 ? max_raw(c[k][0], c[k][1]) : max3_raw(x[k], c[k][e], c[k][e + 1]);
  };
  auto max_of = [&](const acc_t (&c)[2]) {
    float x[2];
    each<16>([&](auto tc) { max_step(c, x, tc); });
    return max_raw(x[0], x[1]);
  };
  acc_t sa[2], sb[2];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    sa[kb] = acc_t{};
#pragma unroll
    for (int c = 0; c < KS; ++c) sa[kb] = M::mma(read_k(lds_addr(s_kv[0][0]) + k0a, kx, kb * KS + c), qb[c], sa[kb]);
  }
  M::drain_v1(sa[0]);  // (max_of reads them in inline asm: a step's come many products later)
  M::drain_v1(sa[1]);
  float tmax = max_of(sa);
#pragma unroll
  for (int i = 0; i < 4; ++i) op[i] = read_k(lds_addr(s_kv[1][0]) + k0a, kx, i);

  // (a lane's key e of block kb is 32 kb + 8 (e / 4) + 4 hq + e % 4)
  auto add_bad = [&](uint64_t bad, int j0, const bf16x8 (&pb)[4]) {
    for (; bad != 0; bad &= bad - 1) {
      const int key = __builtin_ctzll(bad), e = 4 * ((key & 31) >> 3) + (key & 3);
      uint32_t word = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32x4 x = __builtin_bit_cast(u32x4, pb[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) word = 8 * k + 2 * i == ((key >> 5) * 16 + e) - (e & 1) ? x[i] : word;
      }
      const float own = __uint_as_float(e & 1 ? word & 0xffff0000u : word << 16);
      const float w = __shfl(own, lr + 32 * ((key >> 2) & 1), 64);
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[4];
          src.value4(j0 + key, 32 * o + 8 * i + 4 * hq, v);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (w != 0.f && !(fabsf(v[q]) <= 3.402823466e38f)) oacc[o][4 * i + q] += w * v[q];
        }
    }
  };
  int st = 0, nbad = 0;
  auto whole = [&](int j) {
    const int j0 = src.at(j);
    return j0 + KT - 1 <= p0 && (j0 + KT <= p.first || p1 - j0 < p.window);
  };
  auto step = [&](int j, acc_t (&cur)[2], acc_t (&nxt)[2]) {
    const int st1 = (st + 1) & (NS - 1), st2 = (st + 2) & (NS - 1);
    // (opaque: the flipped addresses are formed at their reads, not held)
    uint32_t kf = kx, vf = vx;
    asm volatile("" : "+v"(kf), "+v"(vf));
    const uint32_t kn = lds_addr(s_kv[st1][0]) + k0a, kn2 = lds_addr(s_kv[st2][0]) + k0a, vt = lds_addr(s_kv[st][1]) + v0a;
    uint64_t bad = 0;
    if (!(whole(j) && mask[0] == ~0ull)) {
      // (two words in turn: the other one's readers have passed a step's barrier)
      bad = clear_bad<D, NW>(s_kv[st][1], &s_bad[nbad & 1], wave, lane);
      ++nbad;
      if (tid == 0) s_bad[nbad & 1] = 0;
      // the rows that the lane's row sees, as bits from its first key on
      const uint64_t seen = seen_of(p, pos, src.at(j)) & mask[0];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const uint32_t bits = (uint32_t)(seen >> (32 * kb)) >> (4 * hq);
#pragma unroll
        for (int e = 0; e < 16; ++e) cur[kb][e] = (bits >> (8 * (e >> 2) + (e & 3))) & 1 ? cur[kb][e] : kNegInf;
      }
      tmax = max_of(cur);
      // (opaque: otherwise the other path copies each score to where this one left it)
      asm volatile("" : "+v"(cur[0]), "+v"(cur[1]));
    }
    if (__any(tmax * p.scale_log2 > m_used + 8.f)) {
      const float mn = fmaxf(m_used, xor32_max(tmax * p.scale_log2));
      const float alpha = mn == kNegInf ? 1.f : exp2f(m_used - mn);
      l_part *= alpha;
#pragma unroll
      for (int o = 0; o < OT; ++o) oacc[o] *= alpha;
      m_used = mn;
    }
    const float moff = m_used == kNegInf ? 0.f : -m_used;

    bf16x8 pb[4];
    float ex[2], arg = fmaf(cur[0][0], p.scale_log2, moff), mx[2];
    each<NM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i < NQ) {
        constexpr int kb = i / KS, c = i % KS;
        nxt[kb] = M::mma(op[i & 3], qb[c], c == 0 ? acc_t{} : nxt[kb]);
      } else {
        constexpr int k = (i - NQ) / OT, o = (i - NQ) % OT;
        oacc[o] = M::mma(op[i & 3], pb[k], oacc[o]);
      }
      if constexpr (i == NM - 4) {
        // This tile's V and the next one's K are read: once tile j + 2 has landed (of those in
        // flight the last but one that was asked for), tile j + 4 may take this one's place.
        src.template wait<1>();
        dense_barrier();
      }
      if constexpr (i + 4 < NQ) op[i & 3] = read_k(kn, kf, i + 4);
      else if constexpr (i + 4 < NM) op[i & 3] = read_v(vt, vf, i + 4 - NQ);
      else op[i & 3] = read_k(kn2, kf, i + 4 - NM);
      // the weights, evenly before the last keys' sums; each is used when the next one is made
      each<32>([&](auto ec) {
        constexpr int e = decltype(ec)::value;
        if constexpr (e * (NM - OT) / 32 == i) {
          const float x = __builtin_amdgcn_exp2f(arg);
          if constexpr (e < 31) arg = fmaf(cur[(e + 1) >> 4][(e + 1) & 15], p.scale_log2, moff);
          if constexpr (e > 0) l_part += ex[(e - 1) & 1];
          if constexpr (e > 0 && e % 2 == 0) {
            pb[(e - 2) >> 3][(e - 2) & 7] = (bf16)ex[0];
            pb[(e - 2) >> 3][(e - 1) & 7] = (bf16)ex[1];
          }
          ex[e & 1] = x;
          if constexpr (e == 31) {
            l_part += x;
            pb[3][6] = (bf16)ex[0];
            pb[3][7] = (bf16)ex[1];
          }
          asm volatile("" : "+v"(l_part));  // (added here: all weights held for one sum at the end spill)
        }
      });
      // the next tile's maxima
      each<16>([&](auto tc) {
        constexpr int t = decltype(tc)::value, i0 = NQ + 3;
        if constexpr (i0 + t * (NM - i0) / 16 == i) max_step(nxt, mx, tc);
      });
      if constexpr (i == NM - 2) {
        mask[NS] = src.load(j + 4, s_kv[st][0], s_kv[st][1]);
      }
    });
    __builtin_amdgcn_sched_barrier(0);
    tmax = max_raw(mx[0], mx[1]);
    if (bad != 0) add_bad(bad, src.at(j), pb);
    src.store(s_kv[st][0], s_kv[st][1]);
#pragma unroll
    for (int i = 0; i < NS; ++i) mask[i] = mask[i + 1];
    st = st1;
  };
  int j = 0;
  for (; j + 1 < n; j += 2) {
    step(j, sa, sb);
    step(j + 1, sb, sa);
  }
  if (j < n) step(j, sa, sb);
  src.template wait<0>();

  // ---- results: lane holds row lr, dims 32 o + 8 i + 4 hq + 0 .. 3 --------------------
  dense_barrier();  // the tiles are read
  {  // (what follows is formed now: held across the loop it spills)
    const DenseParams& p = late_params();
    int ln = lane;
    asm volatile("" : "+v"(ln));
    const int lr = ln & 31, hq = ln >> 5, row = 32 * wave + lr, r = it.row0 + row, t = r / p.G, h = g * p.G + r % p.G;
    const bool in = r < p.S * p.G, live = in && t < it.s.n;
    const float l = xor32_sum(l_part);
    float lse, f;
    if (it.partial) {
      f = dense_part(m_used, l, lse);
      if (in && hq == 0) p.part_lse[it.part + row] = lse;
    } else {
      f = dense_finish(p, h, live, m_used, l, lse);
      if (in && hq == 0) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
    }
    u32x4* const rows = &s_kv[0][0][0];
    auto results = [&](auto put) {
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = f == 0.f ? 0.f : oacc[o][4 * i + e] * f;
          put(32 * o + 8 * i + 4 * hq, x);
        }
    };
    if (it.partial) {
      const RowsOut<D / 4> out{rows + wave * 32 * (D / 4)};
      results([&](int d, f32x4 x) { out.put(lr, d, x); });
      out.store(in ? (uint64_t)(uintptr_t)(p.part_o + (it.part + row) * D) : 0, ln);
    } else {
      const RowsOut<D / 8> out{rows + wave * 32 * (D / 8)};
      results([&](int d, f32x4 x) { out.put(lr, d, bf16x4{(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]}); });
      out.store(in ? (uint64_t)(uintptr_t)(reinterpret_cast<bf16*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh) : 0, ln);
    }
  }
}

template <int D>
void launch(const DenseParams& p, bool fp8, unsigned grid, hipStream_t s) {
  const bool one = dense_one_base(p, fp8 ? 1 : 2, 6);
  if (fp8 && one) dense_wide_kernel<D, true, true><<<grid, 512, 0, s>>>(p);
  else if (fp8) dense_wide_kernel<D, true, false><<<grid, 512, 0, s>>>(p);
  else if (one) dense_wide_kernel<D, false, true><<<grid, 512, 0, s>>>(p);
  else dense_wide_kernel<D, false, false><<<grid, 512, 0, s>>>(p);
}

}  // namespace

void launch_dense_wide(const DenseParams& p, int kv_dtype, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.slots * p.Hkv);
  if (p.Dqk == 64) launch<64>(p, kv_dtype == SFA_DTYPE_FP8_E4M3, grid, s);
  else launch<128>(p, kv_dtype == SFA_DTYPE_FP8_E4M3, grid, s);
}

}  // namespace sfa

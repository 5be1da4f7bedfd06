// gfx950 attention of a tree of drafted tokens over a paged cache.
//
// Token t < tree_lens[b] of sequence b sees the cache's rows [0, ctx_b) and
// those drafted rows ctx_b + j, j < tree_lens[b], whose bit j of tree_mask[b][t]
// is set.  out = sum_s softmax_s(scale q.k_s) v_s, lse its log-sum-exp; a sink
// adds exp(sink[h]) to the denominator.  Rows of unmapped pages are not seen;
// a row that sees nothing gives zeros and -inf (with a sink: the sink), a
// token past tree_lens[b] zeros and -inf.
//
// The rows of a (sequence, kv head) are r = t G + h, h < G = Hq / Hkv: its
// keys serve T G query rows.  Work is split over row blocks and over key ranges
// ("slots") of one length for the whole batch, so that ragged contexts give
// even work; the ranges are found on the device from ctx_lens.  A sequence
// of several slots leaves float32 partials that tree_combine_kernel joins.

#include "sfa_lds.h"
#include "sfa_mfma.h"
#include "sfa_ops.h"

namespace sfa {
namespace {

// Base-2 log-sum-exp of 2^m2 l (the logarithm of l's mantissa: its own whole
// part would round the sum once more).
__device__ __forceinline__ float lse2_of(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return m2 + ((float)e + log2f(f));
}
__device__ __forceinline__ float lse_of(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return fmaf(m2, kLn2, fmaf((float)e, kLn2, logf(f)));
}

struct SeqLens {
  int ctx, nodes, keys;  // keys = ctx + nodes, all clamped to the table
};
__device__ __forceinline__ SeqLens seq_lens(const TreeParams& p, int b) {
  SeqLens s;
  s.ctx = min(max(p.ctx_lens[b], 0), p.cap);
  s.nodes = p.tree_lens != nullptr ? min(max(p.tree_lens[b], 0), p.T) : p.T;
  s.keys = (int)min((int64_t)s.ctx + s.nodes, (int64_t)p.cap);
  return s;
}

// A key range of the batch.
struct Slot {
  int b;           // sequence, or -1: none
  int k0, k1;      // its keys
  int first, n;    // the sequence's first slot and how many it has
};
// Length of the ranges, and the sequence of a slot (or the slots of sequence
// `slot` when BY_SEQ).  By one wave; every wave of a workgroup gets the same.
template <bool BY_SEQ>
__device__ Slot find_slot(const TreeParams& p, int slot) {
  const int lane = threadIdx.x & 63;
  int len = 0x7fffffff;  // want = 0: one slot a sequence
  if (p.want > 0) {
    int64_t sum = 0;
    for (int b = lane; b < p.B; b += 64) sum += seq_lens(p, b).keys;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    const int64_t l = (sum + p.want - 1) / p.want;
    len = l < p.min_len ? p.min_len : (int)((l + p.tile - 1) / p.tile) * p.tile;
    // ranges of that length are up to B more than wanted: longer ones, so that
    // all of them run at once (a few steps come within a tile of the best)
    for (int i = 0; i < 6 && p.want > p.B; ++i) {
      int64_t n = 0;
      for (int b = lane; b < p.B; b += 64) n += max(1, (int)(((int64_t)seq_lens(p, b).keys + len - 1) / len));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
      if (n <= p.want) break;
      const int64_t up = (len * n / p.want + p.tile - 1) / p.tile * p.tile;
      len = (int)min((int64_t)0x7fffffff / p.tile * p.tile, up > len ? up : (int64_t)len + p.tile);
    }
  }
  int before = 0;
  Slot s{-1, 0, 0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane;
    const int keys = b < p.B ? seq_lens(p, b).keys : 0;
    int n = b < p.B ? max(1, (int)(((int64_t)keys + len - 1) / len)) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const int first = before + incl - n;
    const bool mine = BY_SEQ ? b == slot : slot >= first && slot < first + n;
    const uint64_t hit = __ballot(mine);
    if (hit != 0) {
      const int w = __builtin_ctzll(hit);
      s.b = b0 + w;
      s.first = __shfl(first, w, 64);
      s.n = __shfl(n, w, 64);
      const int kk = __shfl(keys, w, 64), i = BY_SEQ ? 0 : slot - s.first;
      s.k0 = (int)min((int64_t)i * len, (int64_t)kk);
      s.k1 = (int)min((int64_t)s.k0 + len, (int64_t)kk);
      return s;
    }
    before += __shfl(incl, 63, 64);
  }
  return s;
}

// Element offset of key s of sequence b in a pool of these strides, or -1.
__device__ __forceinline__ int64_t key_row(const TreeParams& p, int b, int s, int64_t page_stride, int64_t row_stride) {
  const int pg = p.block_table[b * p.bt_sb + (s >> p.page_shift)];
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * page_stride + (int64_t)(s & ((1 << p.page_shift) - 1)) * row_stride;
}

// ---- any head dims up to 1024, bf16 or float32: float32 products --------------
constexpr int kGR = 8;     // rows per workgroup
constexpr int kGK = 64;    // keys per tile
constexpr int kGD = 1024;  // largest head dim

// The rows row0 .. row0 + kGR - 1 of (b, g) over keys [k0, k1), by a workgroup of
// 256 threads; emit(i, d, o, l) gets the unnormalised sums and fin(i, m, l) the
// row's maximum (base 2) and sum.
struct GenericScratch {
  float q[kGR][kGD];
  float s[kGR][kGK + 1];
  int64_t krow[kGK], vrow[kGK];
  uint64_t mask[kGR];
  float m[kGR], l[kGR], a[kGR];
};
template <typename T, class Emit, class Fin>
__device__ void generic_rows(const TreeParams& p, int b, int g, int row0, int k0, int k1, GenericScratch& sc, Emit emit,
                             Fin fin) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const SeqLens sl = seq_lens(p, b);
  const int R = p.T * p.G;
  for (int i = 0; i < kGR; ++i) {
    const int r = row0 + i;
    const int t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R && t < sl.nodes;
    for (int d = tid; d < p.Dqk; d += 256)
      sc.q[i][d] = live ? to_f32(reinterpret_cast<const T*>(p.q)[b * p.q_sb + t * p.q_ss + h * p.q_sh + d]) : 0.f;
    if (tid == 0) {
      sc.mask[i] = live ? (uint64_t)p.tree_mask[b * p.tm_sb + t * p.tm_ss] : 0;
      sc.m[i] = kNegInf;
      sc.l[i] = 0.f;
    }
  }
  float acc[kGD / 256][kGR];
#pragma unroll
  for (int c = 0; c < kGD / 256; ++c)
#pragma unroll
    for (int i = 0; i < kGR; ++i) acc[c][i] = 0.f;

  for (int j0 = k0; j0 < k1; j0 += kGK) {
    __syncthreads();
    if (tid < kGK) {
      const int s = j0 + tid;
      sc.krow[tid] = s < k1 ? key_row(p, b, s, p.k_sb, p.k_ss) : -1;
      sc.vrow[tid] = s < k1 ? key_row(p, b, s, p.v_sb, p.v_ss) : -1;
    }
    __syncthreads();
    {  // scores: 4 threads a key
      const int key = tid >> 2, part = tid & 3;
      const int64_t ko = sc.krow[key];
      float s[kGR];
#pragma unroll
      for (int i = 0; i < kGR; ++i) s[i] = 0.f;
      if (ko >= 0) {
        const T* kr = reinterpret_cast<const T*>(p.k) + ko + g * p.k_sh;
        for (int d = part; d < p.Dqk; d += 4) {
          const float x = to_f32(kr[d]);
#pragma unroll
          for (int i = 0; i < kGR; ++i) s[i] = fmaf(sc.q[i][d], x, s[i]);
        }
      }
      const int node = j0 + key - sl.ctx;
#pragma unroll
      for (int i = 0; i < kGR; ++i) {
        s[i] += __shfl_xor(s[i], 1, 64);
        s[i] += __shfl_xor(s[i], 2, 64);
        const bool seen = ko >= 0 && (node < 0 || ((sc.mask[i] >> node) & 1));
        if (part == 0) sc.s[i][key] = seen ? s[i] * p.scale_log2 : kNegInf;
      }
    }
    __syncthreads();
    for (int i = wave; i < kGR; i += 4) {  // softmax: a wave a row
      const float s = sc.s[i][lane], m0 = sc.m[i];
      const float m = fmaxf(m0, wave_max(s));
      const float e = s == kNegInf ? 0.f : exp2f(s - m);
      const float sum = wave_sum(e);
      sc.s[i][lane] = e;
      if (lane == 0) {
        const float a = m0 == kNegInf ? 0.f : exp2f(m0 - m);
        sc.a[i] = a;
        sc.m[i] = m;
        sc.l[i] = sc.l[i] * a + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kGD / 256; ++c) {
      const int d = tid + 256 * c;
      if (d >= p.Dv) break;
#pragma unroll
      for (int i = 0; i < kGR; ++i) acc[c][i] *= sc.a[i];
      for (int key = 0; key < kGK; ++key) {
        const int64_t vo = sc.vrow[key];
        if (vo < 0) continue;
        const float x = to_f32(reinterpret_cast<const T*>(p.v)[vo + g * p.v_sh + d]);
#pragma unroll
        for (int i = 0; i < kGR; ++i) {
          const float e = sc.s[i][key];
          if (e != 0.f) acc[c][i] = fmaf(e, x, acc[c][i]);  // (an unseen row's infinities stay out)
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGR; ++i) {
    if (row0 + i >= R) break;
    if (tid == 0) fin(i, sc.m[i], sc.l[i]);
#pragma unroll
    for (int c = 0; c < kGD / 256; ++c) {
      const int d = tid + 256 * c;
      if (d < p.Dv) emit(i, d, acc[c][i], sc.m[i], sc.l[i]);
    }
  }
}

// Row r of (b, g): where its results go.
struct RowOut {
  int t, h, r;  // r: row of the sequence's partials
};
__device__ __forceinline__ RowOut row_out(const TreeParams& p, int g, int r) {
  RowOut o;
  o.t = r / p.G;
  o.h = g * p.G + r % p.G;
  o.r = o.t * p.Hq + o.h;
  return o;
}

// The factor and LSE of a finished row with maximum m (base 2) and sum l.
__device__ __forceinline__ float finish_row(const TreeParams& p, int h, bool live, float m, float l, float& lse) {
  if (!live) {
    lse = kNegInf;
    return 0.f;
  }
  if (l == 0.f) {  // nothing seen
    lse = p.sink ? p.sink[h] : kNegInf;
    return 0.f;
  }
  const float sink2 = p.sink ? p.sink[h] * kLog2e : kNegInf;
  const float mm = fmaxf(m, sink2);
  const float f = m == kNegInf ? 0.f : exp2f(m - mm);
  float x = l * f;
  if (p.sink && mm != kNegInf) x += exp2f(sink2 - mm);
  lse = x > 0.f ? lse_of(mm, x) : x == 0.f ? kNegInf : x;
  return x > 0.f ? f / x : x == 0.f ? 0.f : x;
}

template <typename T>
__global__ __launch_bounds__(256) void tree_generic_kernel(TreeParams p) {
  __shared__ GenericScratch sc;
  int wi = blockIdx.x;
  const int rb = wi % p.nrb;
  wi /= p.nrb;
  const int g = wi % p.Hkv, slot = wi / p.Hkv;
  const Slot sl = find_slot<false>(p, slot);
  if (sl.b < 0) return;
  const int b = sl.b, nodes = seq_lens(p, b).nodes;
  const int64_t pr = (int64_t)slot * p.T * p.Hq;
  const bool partial = sl.n > 1;
  generic_rows<T>(
      p, b, g, rb * kGR, sl.k0, sl.k1, sc,
      [&](int i, int d, float o, float m, float l) {
        const RowOut ro = row_out(p, g, rb * kGR + i);
        if (partial) {
          p.part_o[(pr + ro.r) * p.Dv + d] = l > 0.f ? o / l : l == 0.f ? 0.f : l;
        } else {
          float lse;
          const float f = finish_row(p, ro.h, ro.t < nodes, m, l, lse);
          reinterpret_cast<T*>(p.out)[b * p.o_sb + ro.t * p.o_ss + ro.h * p.o_sh + d] = from_f32<T>(f == 0.f ? 0.f : o * f);
        }
      },
      [&](int i, float m, float l) {
        const RowOut ro = row_out(p, g, rb * kGR + i);
        if (partial) {
          p.part_lse[pr + ro.r] = l > 0.f ? lse2_of(m, l) : l == 0.f ? kNegInf : l;
        } else {
          float lse;
          finish_row(p, ro.h, ro.t < nodes, m, l, lse);
          p.lse[b * p.l_sb + ro.t * p.l_ss + ro.h * p.l_sh] = lse;
        }
      });
}

// ---- head dims 64 and 128 on the matrix cores, bf16 ------------------------------
// A workgroup of WR x WK waves takes 64 WR rows (wave column wr its NG groups
// of 16; NG < 4 only for WR = 1) of one key range; wave row wk takes every
// WK-th tile of 32 keys.  So a tile is read from HBM once for up to 256 rows,
// and a short row set still spreads its keys over the waves of a CU:
//  * K and V rows go straight into LDS (16 bytes a lane, PD tiles ahead), in
//    an order of chunks that both operand reads find without bank conflicts
//    (Swz); the page ids go the same way, 2 PD tiles ahead, so that the loop has
//    no load that the compiler would wait for;
//  * S^T = K Q^T, 16 keys x 16 rows a product (16x16x32), Q in registers: a K
//    operand read from LDS serves 16 NG rows.  A lane holds 8 keys of a row;
//  * base-2 softmax against a running maximum that moves only when a score
//    passes it by 8 (2^8 more at most in a float32 sum), so that a tile needs no
//    maximum across lanes; P^T in bf16 is already the operand of
//    O^T = V^T P^T, whose V^T operands are transposing reads.
// Unmapped rows and rows past the range read zeros.  Rounding P to bf16 adds
// 2^-9 sum p |v| / sqrt(keys) or so, as much as the result's own rounding;
// sums, maxima and partials are float32.

template <int D>
struct Swz {  // position of chunk c of row r: c ^ at(r)
  static __device__ __forceinline__ int at(int r) {
    // 16 rows at one chunk (K) and 8 rows at one pair of chunks (V, transposing)
    // lie in different banks
    if constexpr (D == 128) return ((r & 7) << 1) | ((r >> 3) & 1);
    else return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  }
};

// lane l: 16 (4) bytes from its address to dst + 16 l (4 l); not seen by the
// compiler: the kernel waits for vmcnt itself
__device__ __forceinline__ void dma16(const void* lds, uint64_t addr) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(d), "v"(addr) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* lds, uint64_t addr) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(d), "v"(addr) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {  // at most N of this wave's loads in flight, all its LDS reads done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D, int NG, int WR, int WK, int PD>
__global__ __launch_bounds__(64 * WR * WK, 2) void tree_mfma_kernel(TreeParams p) {
  using M = Mfma<16>;
  typedef M::acc_t acc_t;
  static_assert(NG == 4 || WR == 1, "whole waves of rows");
  constexpr int NW = WR * WK, KT = 32, CH = D / 8, KS = D / 32, OT = D / 16;
  constexpr int RPI = 64 / CH, ROWI = KT / RPI;        // rows per load instruction, instructions per K (or V) tile
  constexpr int NI = 2 * ROWI / WR;                    // instructions per wave and tile
  constexpr int TILE = 2 * KT * CH, NS = PD + 1;       // 16-byte slots of a K and V tile, stages
  constexpr int WROWS = 16 * NG;
  constexpr int MERGE = WK > 1 ? (WK / 2) * WR * NG * OT * 64 : 0;
  constexpr int SLOTS = NS * WK * TILE > MERGE ? NS * WK * TILE : MERGE;

  __shared__ u32x4 s_kv[SLOTS];
  __shared__ int s_page[NW][NS * 64];
  __shared__ uint64_t s_mask[WR * WROWS];
  __shared__ float s_ml[NW][2][WROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % WR, wk = wave / WR;
  const int lt = lane & 15, hq = lane >> 4;

  // ---- work item: the row blocks of one range and kv head on one XCD ------------
  int wi = blockIdx.x, rb;
  const int nitems = gridDim.x / p.nrb;
  if (nitems % 8 == 0) {
    const int x = wi % 8, r = wi / 8;
    rb = r % p.nrb;
    wi = (r / p.nrb) * 8 + x;
  } else {
    rb = wi % p.nrb;
    wi /= p.nrb;
  }
  const int g = wi % p.Hkv, slot = wi / p.Hkv;
  const Slot sl = find_slot<false>(p, slot);
  if (sl.b < 0) return;
  const int b = __builtin_amdgcn_readfirstlane(sl.b);
  const int k0 = __builtin_amdgcn_readfirstlane(sl.k0), k1 = __builtin_amdgcn_readfirstlane(sl.k1);
  const SeqLens len = seq_lens(p, b);
  const int ctx = __builtin_amdgcn_readfirstlane(len.ctx), nodes = __builtin_amdgcn_readfirstlane(len.nodes);
  const int R = p.T * p.G, row0 = rb * WR * WROWS;
  const int niter = (k1 - k0 + WK * KT - 1) / (WK * KT);

  // ---- rows: Q^T operands (lane: row 16 n + lt, dims 32 s + 8 hq ..), tree masks ----
  bf16x8 qb[NG][KS];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = row0 + wr * WROWS + 16 * n + lt, t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R;
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 32 * s);
      qb[n][s] = live ? x : bf16x8{};
    }
  }
  for (int i = tid; i < WR * WROWS; i += 64 * NW) {
    const int r = row0 + i;
    s_mask[i] = r < R ? (uint64_t)p.tree_mask[b * p.tm_sb + (r / p.G) * p.tm_ss] : 0;
  }

  // ---- loads -------------------------------------------------------------------------
  // lanes 0..31 hold the K row addresses of a tile, lanes 32..63 the V rows'
  const bool vside = lane >= 32;
  const uint64_t side_base = vside ? (uint64_t)(uintptr_t)p.v + (uint64_t)(2 * g * p.v_sh)
                                   : (uint64_t)(uintptr_t)p.k + (uint64_t)(2 * g * p.k_sh);
  const int64_t page_bytes = 2 * (vside ? p.v_sb : p.k_sb), row_bytes = 2 * (vside ? p.v_ss : p.k_ss);
  const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
  const int32_t* trow = p.block_table + b * p.bt_sb;
  const int last_key = p.cap - 1;
  auto key_of = [&](int j) { return k0 + (j * WK + wk) * KT + (lane & 31); };
  auto page_addr = [&](int j) {  // (past the range: any entry, not used)
    return (uint64_t)(uintptr_t)(trow + (min(key_of(j), last_key) >> p.page_shift));
  };
  // rows of tile j with page ids pg into stage st; returns the mask of rows that are there
  auto load_tile = [&](int j, int pg, int st) -> uint32_t {
    const int s = key_of(j);
    const bool ok = s < k1 && pg >= 0 && pg < p.num_pages;
    const uint64_t a = ok ? side_base + (uint64_t)((int64_t)pg * page_bytes + (int64_t)(s & ((1 << p.page_shift) - 1)) * row_bytes)
                          : zero;
    const uint32_t mask = (uint32_t)__ballot(ok);
    const int lo = (int)(uint32_t)a, hi = (int)(uint32_t)(a >> 32);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = wr * NI + i, v = q >= ROWI ? 1 : 0;
      const int row = (q - v * ROWI) * RPI + lane / CH;
      const int src = v * 32 + row;
      const uint64_t ra = ((uint64_t)(uint32_t)__shfl(hi, src, 64) << 32) | (uint32_t)__shfl(lo, src, 64);
      dma16(&s_kv[(st * WK + wk) * TILE + q * 64], ra + (uint64_t)(16 * ((lane % CH) ^ Swz<D>::at(row))));
    }
    return mask;
  };

  uint32_t vm[NS];  // rows that are there, of tiles j, j + 1, ..
  {
    int pg[2 * PD];
#pragma unroll
    for (int j = 0; j < 2 * PD; ++j) pg[j] = *reinterpret_cast<const int32_t*>(page_addr(j));
#pragma unroll
    for (int j = PD; j < 2 * PD; ++j) s_page[wave][(j % NS) * 64 + lane] = pg[j];
#pragma unroll
    for (int j = 0; j < PD; ++j) vm[j] = load_tile(j, pg[j], j);
  }
  wait_vm<(PD - 1) * NI>();  // tile 0 (its page ids are not in the loop's count yet)
  wg_barrier();              // the masks are staged

  // ---- operand addresses ---------------------------------------------------------------
  const uint32_t pitch = CH * 16;
  const uint32_t ka = (uint32_t)lt * pitch + (uint32_t)((hq ^ Swz<D>::at(lt)) << 4);
  const int rr = lt >> 2, cc = lt & 3, vr = 4 * hq + rr;
  const uint32_t va = (uint32_t)vr * pitch + (uint32_t)(((cc >> 1) ^ Swz<D>::at(vr)) << 4) + (uint32_t)(cc & 1) * 8u;

  acc_t oacc[NG][OT];
  float m_used[NG], l_part[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    m_used[n] = kNegInf;
    l_part[n] = 0.f;
#pragma unroll
    for (int i = 0; i < OT; ++i) oacc[n][i] = acc_t{};
  }

  int st = 0, st_new = PD;  // stage of tile j, of tile j + PD
  for (int j = 0; j < niter; ++j) {
    wait_vm<(PD - 1) * (NI + 1)>();  // tile j and the page ids of tile j + PD have landed
    if constexpr (WR > 1) asm volatile("s_barrier" ::: "memory");  // ... for all its waves; stage st_new is read
    {
      const int pg = s_page[wave][st_new * 64 + lane];
      // (page ring: tile j + 2 PD takes the place of tile j + PD - 1, read at j - 1)
      const int ring = st_new == 0 ? NS - 1 : st_new - 1;
      dma4(&s_page[wave][ring * 64], page_addr(j + 2 * PD));
      vm[PD] = load_tile(j + PD, pg, st_new);
    }
    const u32x4* kt = &s_kv[(st * WK + wk) * TILE];
    const u32x4* vt = kt + KT * CH;
    const int base = k0 + (j * WK + wk) * KT;
    const uint32_t mask = vm[0];
    // drafted rows in this step's tiles (any of the workgroup's)
    const bool tail = k0 + (j + 1) * WK * KT > ctx;
    uint32_t bad = 0;  // drafted rows whose V holds infinities or NaN: out of the product, added by hand
    if (tail) {
      uint32_t x = 0;
#pragma unroll
      for (int c = 0; c < CH / 2; ++c) {
        const u32x4 w = vt[(lane >> 1) * CH + (lane & 1) * (CH / 2) + c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x |= (w[e] & 0x7f80u) == 0x7f80u;
          x |= (w[e] & 0x7f800000u) == 0x7f800000u;
        }
      }
      const uint64_t rows2 = __ballot(x != 0 && base + (lane >> 1) >= ctx);
      // (bit r: row r)
      const uint64_t any2 = rows2 | (rows2 >> 1);
      for (int r = 0; r < 32; ++r) bad |= (uint32_t)((any2 >> (2 * r)) & 1) << r;
      if constexpr (WR > 1) wg_barrier();
      if (bad != 0 && wr == 0) {
        for (int i = lane; i < KT * CH; i += 64)
          if ((bad >> (i / CH)) & 1) const_cast<u32x4*>(vt)[i] = u32x4{0, 0, 0, 0};
      }
      if constexpr (WR > 1) wg_barrier();
    }
    const bool plain = mask == 0xffffffffu && !tail;

    // by 16 keys (half the scores in registers): S^T, then its softmax; a lane
    // holds keys 16 mt + 4 hq + e of its row
    bf16x8 pb[NG];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      acc_t sacc[NG];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8 kf = lds_read_b128(kt, (ka ^ (uint32_t)(64 * s)) + (uint32_t)(16 * mt) * pitch);
#pragma unroll
        for (int n = 0; n < NG; ++n) sacc[n] = M::mma(kf, qb[n][s], s == 0 ? acc_t{} : sacc[n]);
      }
      if (!plain) {
        // bits of the lane's 4 keys: there, and context or a node the row sees
        const int key = 16 * mt + 4 * hq, node = base + key - ctx, back = min(max(-node, 0), 4);
        const uint32_t there = mask >> key;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const uint64_t tm = s_mask[wr * WROWS + 16 * n + lt];
          const uint32_t drafted = node > 63 ? 0u : (uint32_t)(tm >> (max(node, 0) & 63));
          const uint32_t seen = there & ((drafted << back) | ((1u << back) - 1u));
          const float x0 = seen & 1u ? sacc[n][0] : kNegInf, x1 = seen & 2u ? sacc[n][1] : kNegInf;
          const float x2 = seen & 4u ? sacc[n][2] : kNegInf, x3 = seen & 8u ? sacc[n][3] : kNegInf;
          sacc[n] = acc_t{x0, x1, x2, x3};
        }
      }
      bool over = false;
#pragma unroll
      for (int n = 0; n < NG; ++n)
        over |= fmaxf(fmaxf(sacc[n][0], sacc[n][1]), fmaxf(sacc[n][2], sacc[n][3])) * p.scale_log2 > m_used[n] + 8.f;
      if (__any(over)) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float tmax = fmaxf(fmaxf(sacc[n][0], sacc[n][1]), fmaxf(sacc[n][2], sacc[n][3]));
          tmax = xor32_max(xor16_max(tmax)) * p.scale_log2;
          const float m_new = fmaxf(m_used[n], tmax);
          const float alpha = m_new == kNegInf ? 1.f : exp2f(m_used[n] - m_new);
          l_part[n] *= alpha;
#pragma unroll
          for (int i = 0; i < OT; ++i) oacc[n][i] *= alpha;
          if (mt == 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pb[n][i] = (bf16)((float)pb[n][i] * alpha);
          }
          m_used[n] = m_new;
        }
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float moff = m_used[n] == kNegInf ? 0.f : -m_used[n];
        float ex[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ex[i] = __builtin_amdgcn_exp2f(fmaf(sacc[n][i], p.scale_log2, moff));
          pb[n][4 * mt + i] = (bf16)ex[i];
        }
        l_part[n] += (ex[0] + ex[1]) + (ex[2] + ex[3]);
        for (uint32_t left = bad & (0xffffu << (16 * mt)); left != 0; left &= left - 1) {
          const int key = __builtin_ctz(left);
          float e = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) e = (key & 3) == i ? ex[i] : e;
          e = __shfl(e, lt + 16 * ((key & 15) >> 2), 64);
          const int64_t vo = key_row(p, b, base + key, p.v_sb, p.v_ss);
          if (vo < 0) continue;
          const bf16* v = reinterpret_cast<const bf16*>(p.v) + vo + g * p.v_sh + 4 * hq;
#pragma unroll
          for (int ot = 0; ot < OT; ++ot)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (e != 0.f) oacc[n][ot][i] = fmaf(e, (float)v[16 * ot + i], oacc[n][ot][i]);
        }
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      const uint32_t off = va ^ (uint32_t)(32 * ot);
      const bf16x4 lo = lds_read_tr16(vt, off), hi = lds_read_tr16(vt, off + 16u * pitch);
      const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (int n = 0; n < NG; ++n) oacc[n][ot] = M::mma(a, pb[n], oacc[n][ot]);
    }
#pragma unroll
    for (int i = 0; i < PD; ++i) vm[i] = vm[i + 1];
    st = st + 1 == NS ? 0 : st + 1;
    st_new = st_new + 1 == NS ? 0 : st_new + 1;
  }
  wait_vm<0>();  // the loads past the range have landed before LDS is used for anything else

  // ---- row sums; the wave rows' results joined in halves ----------------------------
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    l_part[n] += __shfl_xor(l_part[n], 16, 64);
    l_part[n] = xor32_sum(l_part[n]);
  }
#pragma unroll
  for (int half = WK / 2; half > 0; half >>= 1) {
    wg_barrier();
    f32x4* mine = reinterpret_cast<f32x4*>(s_kv) + (size_t)((wk % half) * WR + wr) * (NG * OT * 64);
    if (wk >= half && wk < 2 * half) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int ot = 0; ot < OT; ++ot) mine[(n * OT + ot) * 64 + lane] = oacc[n][ot];
        if (hq == 0) {
          s_ml[wave][0][16 * n + lt] = m_used[n];
          s_ml[wave][1][16 * n + lt] = l_part[n];
        }
      }
    }
    wg_barrier();
    if (wk < half) {
      const int other = wave + half * WR;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float m2 = s_ml[other][0][16 * n + lt], l2 = s_ml[other][1][16 * n + lt];
        const float m = fmaxf(m_used[n], m2);
        const float a1 = m_used[n] == kNegInf ? 0.f : exp2f(m_used[n] - m), a2 = m2 == kNegInf ? 0.f : exp2f(m2 - m);
        // (a row without a finite maximum has sums that are zero or NaN)
        l_part[n] = (m_used[n] == kNegInf ? l_part[n] : l_part[n] * a1) + (m2 == kNegInf ? l2 : l2 * a2);
#pragma unroll
        for (int ot = 0; ot < OT; ++ot) {
          const f32x4 o2 = mine[(n * OT + ot) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x1 = m_used[n] == kNegInf ? oacc[n][ot][i] : oacc[n][ot][i] * a1;
            const float x2 = m2 == kNegInf ? o2[i] : o2[i] * a2;
            oacc[n][ot][i] = x1 + x2;
          }
        }
        m_used[n] = m;
      }
    }
  }
  if (wk != 0) return;

  // ---- results: lane holds row lt, dims 16 ot + 4 hq + e ------------------------------
  const int64_t pr = (int64_t)slot * p.T * p.Hq;
  const bool partial = sl.n > 1;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = row0 + wr * WROWS + 16 * n + lt;
    if (r >= R) continue;
    const RowOut ro = row_out(p, g, r);
    const float m = m_used[n], l = l_part[n];
    float f, lse;
    if (partial) {
      f = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      lse = l > 0.f ? lse2_of(m, l) : l == 0.f ? kNegInf : l;
      if (hq == 0) p.part_lse[pr + ro.r] = lse;
    } else {
      f = finish_row(p, ro.h, ro.t < nodes, m, l, lse);
      if (hq == 0) p.lse[b * p.l_sb + ro.t * p.l_ss + ro.h * p.l_sh] = lse;
    }
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      f32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f == 0.f ? 0.f : oacc[n][ot][i] * f;
      if (partial) {
        *reinterpret_cast<f32x4*>(p.part_o + (pr + ro.r) * D + 16 * ot + 4 * hq) = o;
      } else {
        const bf16x4 o4 = {(bf16)o[0], (bf16)o[1], (bf16)o[2], (bf16)o[3]};
        *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(p.out) + b * p.o_sb + ro.t * p.o_ss + ro.h * p.o_sh + 16 * ot +
                                   4 * hq) = o4;
      }
    }
  }
}

// ---- joining the slots of a sequence -------------------------------------------
// One wave a row; a slot in which the row sees nothing has LSE -inf.
template <typename T>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), per = (int64_t)p.T * p.Hq;
  if (row >= p.B * per) return;
  const int b = (int)(row / per), r = (int)(row % per), h = r % p.Hq, t = r / p.Hq;
  const Slot sl = find_slot<true>(p, b);
  if (sl.n <= 1) return;
  const float* pl = p.part_lse + sl.first * per + r;
  const float* po = p.part_o + (sl.first * per + r) * p.Dv;
  const bool live = t < seq_lens(p, b).nodes;
  float m = kNegInf;
  bool bad = false;
  for (int i = lane; i < sl.n; i += 64) {
    const float x = pl[i * per];
    bad |= x != x;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  bad = __any(bad);
  float l = 0.f;
  for (int i = lane; i < sl.n; i += 64) {
    const float x = pl[i * per];
    if (x != kNegInf) l += exp2f(x - m);
  }
  l = wave_sum(l);
  if (bad) l = __builtin_nanf("");
  float lse;
  const float f = finish_row(p, h, live, m, l, lse);
  if (lane == 0) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
  T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh;
  for (int d = lane; d < p.Dv; d += 64) {
    float x = 0.f;
    if (f != 0.f)
      for (int i = 0; i < sl.n; ++i) {
        const float e = pl[i * per];
        if (e != kNegInf) x = fmaf(exp2f(e - m), po[i * per * p.Dv + d], x);
      }
    o[d] = from_f32<T>(f == 0.f ? 0.f : x * f);
  }
}

// Kernels by query rows per (sequence, kv head): rows a workgroup, tile keys, waves.
enum { kGeneric = 0, kRows16, kRows32, kRows64, kRows128, kRows256 };
struct KernelShape {
  int rows, tile;
};
constexpr KernelShape kShapes[] = {{kGR, kGK}, {16, 128}, {32, 128}, {64, 128}, {128, 128}, {256, 64}};
constexpr int kWorkgroups = 256;  // key ranges are cut until about so many workgroups (one a CU) are in flight

template <int D>
void launch_mfma(const TreeParams& p, int kernel, unsigned grid, hipStream_t s) {
  switch (kernel) {
    case kRows16: tree_mfma_kernel<D, 1, 1, 4, 1><<<grid, 256, 0, s>>>(p); break;
    case kRows32: tree_mfma_kernel<D, 2, 1, 4, 1><<<grid, 256, 0, s>>>(p); break;
    case kRows64: tree_mfma_kernel<D, 4, 1, 4, 1><<<grid, 256, 0, s>>>(p); break;
    case kRows128: tree_mfma_kernel<D, 4, 2, 4, 1><<<grid, 512, 0, s>>>(p); break;
    default: tree_mfma_kernel<D, 4, 4, 2, 2><<<grid, 512, 0, s>>>(p);
  }
}

}  // namespace

TreePlan tree_plan(const TreeParams& p, int dtype, bool vec) {
  TreePlan pl{};
  const int64_t R = (int64_t)p.T * p.G;
  if (dtype == SFA_DTYPE_BF16 && vec && p.Dqk == p.Dv && (p.Dqk == 64 || p.Dqk == 128))
    pl.kernel = R <= 16 ? kRows16 : R <= 32 ? kRows32 : R <= 64 ? kRows64 : R <= 128 ? kRows128 : kRows256;
  pl.rows = kShapes[pl.kernel].rows;
  const int64_t nrb = (R + pl.rows - 1) / pl.rows, min_len = 2 * kShapes[pl.kernel].tile;
  int64_t want = (pl.kernel == kGeneric ? 4 : 1) * kWorkgroups / (p.Hkv * nrb);
  const int64_t most = ((int64_t)p.cap + min_len - 1) / min_len * p.B;
  if (want > most) want = most;
  pl.want = want > p.B ? (int)want : 0;
  pl.slots = p.B + pl.want;
  if (pl.want > 0) {
    const size_t rows = (size_t)pl.slots * p.T * p.Hq;
    pl.part_o_bytes = (rows * p.Dv * sizeof(float) + 255) / 256 * 256;
    pl.part_lse_bytes = (rows * sizeof(float) + 255) / 256 * 256;
  }
  return pl;
}

hipError_t launch_tree(const TreeParams& p0, const TreePlan& pl, int dtype, hipStream_t s) {
  TreeParams p = p0;
  p.want = pl.want;
  p.tile = kShapes[pl.kernel].tile;
  p.min_len = 2 * p.tile;
  p.nrb = (p.T * p.G + pl.rows - 1) / pl.rows;
  const unsigned grid = (unsigned)((int64_t)pl.slots * p.Hkv * p.nrb);
  if (pl.kernel != kGeneric) {
    if (p.Dqk == 64) launch_mfma<64>(p, pl.kernel, grid, s);
    else launch_mfma<128>(p, pl.kernel, grid, s);
  } else if (dtype == SFA_DTYPE_F32) {
    tree_generic_kernel<float><<<grid, 256, 0, s>>>(p);
  } else {
    tree_generic_kernel<bf16><<<grid, 256, 0, s>>>(p);
  }
  if (pl.want > 0) {
    const unsigned cg = (unsigned)(((int64_t)p.B * p.T * p.Hq + 3) / 4);
    if (dtype == SFA_DTYPE_F32) tree_combine_kernel<float><<<cg, 256, 0, s>>>(p);
    else tree_combine_kernel<bf16><<<cg, 256, 0, s>>>(p);
  }
  return hipGetLastError();
}

}  // namespace sfa

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

// Sums over the 64 lanes (row rotations and lane swaps: no LDS trips).
__device__ __forceinline__ int lanes_sum(int x) {
  x += __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true);  // row_ror:8
  x += __builtin_amdgcn_mov_dpp(x, 0x124, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x122, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x121, 0xf, 0xf, true);
  const auto a = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
  x = (int)(a[0] + a[1]);
  const auto c = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
  return (int)(c[0] + c[1]);
}

// A key range of the batch.
struct Slot {
  int b;           // sequence, or -1: none
  int k0, k1;      // its keys
  int first, n;    // the sequence's first slot and how many it has
};
// The range of a slot; every wave finds the same.  Lengths are multiples of
// the tile: ceil(all tiles / want) of them first, which gives up to B ranges more
// than wanted, then longer ones until they are `want` or fewer, so that all
// run at once (a few steps come within a tile of the best).
__device__ Slot find_slot(const TreeParams& p, int slot) {
  if (p.want == 0)  // one range a sequence
    return slot < p.B ? Slot{slot, 0, seq_lens(p, slot).keys, slot, 1} : Slot{-1, 0, 0, 0, 0};
  const int lane = threadIdx.x & 63, shift = 31 - __builtin_clz(p.tile);
  auto tiles_of = [&](int b) { return b < p.B ? (seq_lens(p, b).keys + p.tile - 1) >> shift : 0; };
  const int mine = tiles_of(lane);  // (of the first 64 sequences)
  int64_t sum = lanes_sum(mine);
  for (int b0 = 64; b0 < p.B; b0 += 64) sum += lanes_sum(tiles_of(b0 + lane));
  int len = max(2, (int)((sum + p.want - 1) / p.want));  // in tiles
  for (int i = 0; i < 6; ++i) {
    auto ranges = [&](int t, int b) { return b < p.B ? max(1, (t + len - 1) / len) : 0; };
    int n = lanes_sum(ranges(mine, lane));
    for (int b0 = 64; b0 < p.B; b0 += 64) n += lanes_sum(ranges(tiles_of(b0 + lane), b0 + lane));
    if (n <= p.want) break;
    len = max(len + 1, (int)((int64_t)len * n / p.want));
  }
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + lane, t = b0 == 0 ? mine : tiles_of(b);
    const int n = b < p.B ? max(1, (t + len - 1) / len) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const int first = before + incl - n;
    const uint64_t hit = __ballot(slot >= first && slot < first + n);
    if (hit != 0) {
      const int w = __builtin_ctzll(hit);
      Slot s;
      s.b = b0 + w;
      s.first = __builtin_amdgcn_readlane(first, w);
      s.n = __builtin_amdgcn_readlane(n, w);
      const int keys = seq_lens(p, s.b).keys;
      const int64_t k0 = (int64_t)(slot - s.first) * len << shift;
      s.k0 = (int)min(k0, (int64_t)keys);
      s.k1 = (int)min(k0 + ((int64_t)len << shift), (int64_t)keys);
      return s;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return Slot{-1, 0, 0, 0, 0};
}

// Element offset of key s of sequence b in a pool of these strides, or -1.
__device__ __forceinline__ int64_t key_row(const TreeParams& p, int b, int s, int64_t page_stride, int64_t row_stride) {
  const int pg = p.block_table[b * p.bt_sb + (s >> p.page_shift)];
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * page_stride + (int64_t)(s & ((1 << p.page_shift) - 1)) * row_stride;
}

// A sequence's slots, for tree_combine_kernel.
__device__ __forceinline__ void note_slots(const TreeParams& p, int slot, const Slot& sl) {
  if (p.want > 0 && slot == sl.first && threadIdx.x == 0) {
    p.seq_slots[2 * sl.b] = sl.first;
    p.seq_slots[2 * sl.b + 1] = sl.n;
  }
}

// ---- any head dims up to 1024, bf16 or float32: float32 products --------------
constexpr int kGR = 8;     // rows per workgroup
constexpr int kGK = 64;    // keys per tile
constexpr int kGD = 1024;  // largest head dim

// The rows row0 .. row0 + kGR - 1 of (b, g) over keys [k0, k1), by a workgroup of
// 256 threads; fin(i, m, l) gets a row's maximum (base 2) and sum, emit(i, d, o, m, l)
// its unnormalised sum of dim d with them.  Far from its floor: the keys are read
// again for every 8 rows, and a score is a scalar product of four threads (4 x 4K
// float32 keys of 128 dims, 8 tokens, 16 / 4 heads: 188 us, the bytes alone 15).
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
  const Slot sl = find_slot(p, slot);
  if (sl.b < 0) return;
  const int b = sl.b, nodes = seq_lens(p, b).nodes;
  if (rb == 0 && g == 0) note_slots(p, slot, sl);
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
// tree_mfma_kernel: a workgroup of four waves takes 16 NG rows of one key range,
// wave w every fourth tile of 32 keys, so that a short row set still spreads its
// keys over a CU.  tree_pipe_kernel (below): WR x WK waves, wave column wr with
// rows 16 NG wr .., wave row wk with every WK-th tile, which is read from HBM once
// for up to 256 rows.  In both
//  * K and V rows go straight into LDS (16 bytes a lane, a tile or more ahead), in
//    an order of chunks that both operand reads find without bank conflicts
//    (Swz); the page ids go the same way, further ahead, so that the loop has
//    no load that the compiler would wait for;
//  * S^T = K Q^T, 16 keys x 16 rows a product (16x16x32), Q in registers: a K
//    operand read from LDS serves 16 NG rows.  A lane holds 8 keys of a row;
//  * base-2 softmax against a running maximum that moves only when a score
//    passes it by 8 (2^8 more at most in a float32 sum), so that a tile needs no
//    maximum across lanes; P^T in bf16 is already the operand of
//    O^T = V^T P^T, whose V^T operands are transposing reads.
// Unmapped rows and rows past the range read zeros.  Sums, maxima and partials
// are float32.  P is rounded to bf16 for the product: tree_mfma_kernel multiplies
// what that left in a second one (2^-16 of a weight), tree_pipe_kernel does not
// (2^-8, which adds 2^-9 sum p |v| / sqrt(keys) or so, as much as the result's own
// rounding).

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
// ... from a wave-uniform base and 32-bit lane offsets
__device__ __forceinline__ void dma16(const void* lds, uint64_t base, uint32_t off) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(d), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* lds, uint64_t base, uint32_t off) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, %2" ::"s"(d), "v"(off), "s"(base) : "memory", "m0");
}
// the wait states between the last MFMA that wrote any of these AGPRs and a VALU read
__device__ __forceinline__ void drain_all(f32x4 (&c)[4]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]));
}
__device__ __forceinline__ void drain_all(f32x4 (&c)[8]) {
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
               : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]));
}
template <int N>
__device__ __forceinline__ void wait_vm() {  // at most N of this wave's loads in flight, all its LDS reads done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wg_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- work item: the row blocks of one range and kv head on one XCD ------------
struct WorkItem {
  int b, g, rb, k0, k1, ctx, nodes, slot;
  bool partial;
};
__device__ __forceinline__ bool work_item(const TreeParams& p, WorkItem& it) {
  int wi = blockIdx.x;
  const int nitems = gridDim.x / p.nrb, x = wi % 8;
  if (nitems % 8 == 0) {
    it.rb = (wi / 8) % p.nrb;
    wi = wi / 8 / p.nrb * 8 + x;
  } else if ((nitems == 1 || nitems == 2 || nitems == 4) && p.nrb % 8 == 0) {  // an item on 8 / nitems of them
    const int per = 8 / nitems;
    it.rb = wi / 8 * per + x % per;
    wi = x / per;
  } else {
    it.rb = wi % p.nrb;
    wi /= p.nrb;
  }
  it.g = wi % p.Hkv;
  it.slot = wi / p.Hkv;
  const Slot sl = find_slot(p, it.slot);
  if (sl.b < 0) return false;
  if (it.rb == 0 && it.g == 0) note_slots(p, it.slot, sl);
  it.b = __builtin_amdgcn_readfirstlane(sl.b);
  it.k0 = __builtin_amdgcn_readfirstlane(sl.k0);
  it.k1 = __builtin_amdgcn_readfirstlane(sl.k1);
  it.partial = sl.n > 1;
  const SeqLens len = seq_lens(p, it.b);
  it.ctx = __builtin_amdgcn_readfirstlane(len.ctx);
  it.nodes = __builtin_amdgcn_readfirstlane(len.nodes);
  return true;
}

// The rows of a wave row's tiles into LDS: lanes 0..31 hold the K row addresses
// of a tile, lanes 32..63 the V rows', and hand them to the lanes that load.
template <int D, int WR, int WK>
struct TileLoads {
  static constexpr int KT = 32, CH = D / 8, RPI = 64 / CH, ROWI = KT / RPI, NI = 2 * ROWI / WR;
  uint64_t side_base;
  int64_t page_bytes, row_bytes;
  const int32_t* trow;
  int key0, k1, last_key, page_shift, num_pages, wr, lane;
  __device__ __forceinline__ TileLoads(const TreeParams& p, int b, int g, int k0, int k1_, int wr_, int wk, int lane_)
      : k1(k1_), last_key(p.cap - 1), page_shift(p.page_shift), num_pages(p.num_pages), wr(wr_), lane(lane_) {
    const bool vside = lane >= 32;
    side_base = vside ? (uint64_t)(uintptr_t)p.v + (uint64_t)(2 * g * p.v_sh)
                      : (uint64_t)(uintptr_t)p.k + (uint64_t)(2 * g * p.k_sh);
    page_bytes = 2 * (vside ? p.v_sb : p.k_sb);
    row_bytes = 2 * (vside ? p.v_ss : p.k_ss);
    trow = p.block_table + b * p.bt_sb;
    key0 = k0 + wk * KT + (lane & 31);
  }
  __device__ __forceinline__ uint64_t page_addr(int j) const {  // (past the range: any entry, not used)
    return (uint64_t)(uintptr_t)(trow + (min(key0 + j * WK * KT, last_key) >> page_shift));
  }
  // rows of tile j with page ids pg to dst; returns the mask of rows that are there
  __device__ __forceinline__ uint32_t load(int j, int pg, u32x4* dst) const {
    const int s = key0 + j * WK * KT;
    const bool ok = s < k1 && pg >= 0 && pg < num_pages;
    const uint64_t a = ok ? side_base + (uint64_t)((int64_t)pg * page_bytes + (int64_t)(s & ((1 << page_shift) - 1)) * row_bytes)
                          : (uint64_t)(uintptr_t)kZeroRow;
    const uint32_t mask = (uint32_t)__ballot(ok);
    const int lo = (int)(uint32_t)a, hi = (int)(uint32_t)(a >> 32);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = wr * NI + i, v = q >= ROWI ? 1 : 0;
      const int row = (q - v * ROWI) * RPI + lane / CH;
      const int src = v * 32 + row;
      const uint64_t ra = ((uint64_t)(uint32_t)__shfl(hi, src, 64) << 32) | (uint32_t)__shfl(lo, src, 64);
      dma16(dst + q * 64, ra + (uint64_t)(16 * ((lane % CH) ^ Swz<D>::at(row))));
    }
    return mask;
  }
};

// The same where a tile lies within one page (pages of 32 rows or more): the
// wave's rows have one base, and a load instruction costs one select.
template <int D, int WR, int WK>
struct PageLoads {
  static constexpr int KT = 32, CH = D / 8, RPI = 64 / CH, ROWI = KT / RPI, NI = 2 * ROWI / WR;
  uint64_t kbase, vbase;
  int64_t kpage, vpage, krow, vrow;
  const int32_t* trow;
  uint32_t off[NI];  // lane offsets of the wave's instructions
  int key0, k1, last_key, page_shift, num_pages, wr, lane;
  // tile `next`, as begin() found it
  uint64_t kb, vb;
  bool ok;
  __device__ __forceinline__ PageLoads(const TreeParams& p, int b, int g, int k0, int k1_, int wr_, int wk, int lane_)
      : kbase((uint64_t)(uintptr_t)p.k + (uint64_t)(2 * g * p.k_sh)), vbase((uint64_t)(uintptr_t)p.v + (uint64_t)(2 * g * p.v_sh)),
        kpage(2 * p.k_sb), vpage(2 * p.v_sb), krow(2 * p.k_ss), vrow(2 * p.v_ss), trow(p.block_table + b * p.bt_sb),
        key0(k0 + wk * KT), k1(k1_), last_key(p.cap - 1), page_shift(p.page_shift), num_pages(p.num_pages), wr(wr_),
        lane(lane_) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int q = wr * NI + i, v = q >= ROWI ? 1 : 0, row = (q - v * ROWI) * RPI + lane / CH;
      off[i] = (uint32_t)(row * (int)(v ? vrow : krow)) + 16u * (uint32_t)((lane % CH) ^ Swz<D>::at(row));
    }
  }
  // page id of tile j to ring slot dst (every lane the same one)
  __device__ __forceinline__ void fetch_page(int j, int* dst) const {
    dma4(dst, (uint64_t)(uintptr_t)(trow + (min(key0 + j * WK * KT, last_key) >> page_shift)), 0u);
  }
  // tile j with its page id; returns the mask of rows that are there
  __device__ __forceinline__ uint32_t begin(int j, int pg) {
    const int s = key0 + j * WK * KT, n = k1 - s, in = s & ((1 << page_shift) - 1);
    ok = n > 0 && pg >= 0 && pg < num_pages;
    const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
    kb = ok ? kbase + (uint64_t)(pg * kpage + in * krow) : zero;
    vb = ok ? vbase + (uint64_t)(pg * vpage + in * vrow) : zero;
    return !ok ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  }
  __device__ __forceinline__ void issue(int i, u32x4* dst) const {
    const int q = wr * NI + i;
    dma16(dst + q * 64, q >= ROWI ? vb : kb, ok ? off[i] : 16u * (uint32_t)lane);
  }
};

// Bits of the 4 keys from `key` of a tile: there, and context or a node that the
// row with tree mask tm sees (past: the tile's first key minus the context's length).
template <bool TAIL>
__device__ __forceinline__ uint32_t seen4(uint32_t mask, uint64_t tm, int key, int past) {
  uint32_t seen = mask >> key;
  if constexpr (TAIL) {
    const int node = past + key, back = min(max(-node, 0), 4);
    const uint32_t drafted = node > 63 ? 0u : (uint32_t)(tm >> (max(node, 0) & 63));
    seen &= (drafted << back) | ((1u << back) - 1u);
  }
  return seen;
}

// Drafted rows of a V tile that hold infinities or NaN, as bits; they are
// cleared in LDS (0 times them would reach rows that do not see them) and
// added by add_bad_rows to the rows that do.
template <int D, int WR>
__device__ __forceinline__ uint32_t bad_rows(u32x4* vt, int base, int ctx, int wr, int lane) {
  constexpr int KT = 32, CH = D / 8;
  uint32_t x = 0, bad = 0;
#pragma unroll
  for (int c = 0; c < CH / 2; ++c) {
    const u32x4 w = vt[(lane >> 1) * CH + (lane & 1) * (CH / 2) + c];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x |= (w[e] & 0x7f80u) == 0x7f80u;
      x |= (w[e] & 0x7f800000u) == 0x7f800000u;
    }
  }
  uint64_t rows2 = __ballot(x != 0 && base + (lane >> 1) >= ctx);
  for (; rows2 != 0; rows2 &= rows2 - 1) bad |= 1u << (__builtin_ctzll(rows2) >> 1);
  if constexpr (WR > 1) wg_barrier();
  if (bad != 0 && wr == 0) {
    for (int i = lane; i < KT * CH; i += 64)
      if ((bad >> (i / CH)) & 1) vt[i] = u32x4{0, 0, 0, 0};
  }
  if constexpr (WR > 1) wg_barrier();
  return bad;
}
template <int D, int NG, class Add>
__device__ __forceinline__ void add_bad_rows(const TreeParams& p, int b, int g, int base, uint32_t bad,
                                             const bf16x8 (&pb)[NG], int lt, int hq, Add add) {
  for (; bad != 0; bad &= bad - 1) {
    const int key = __builtin_ctz(bad), i = 4 * (key >> 4) + (key & 3);
    const int64_t vo = key_row(p, b, base + key, p.v_sb, p.v_ss);
    if (vo < 0) continue;
    const bf16* v = reinterpret_cast<const bf16*>(p.v) + vo + g * p.v_sh + 4 * hq;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const u32x4 w = __builtin_bit_cast(u32x4, pb[n]);
      const uint32_t word = i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3];
      const float e = __shfl(__uint_as_float(i & 1 ? word & 0xffff0000u : word << 16), lt + 16 * ((key & 15) >> 2), 64);
#pragma unroll
      for (int ot = 0; ot < D / 16; ++ot) {
        const bf16x4 x = *reinterpret_cast<const bf16x4*>(v + 16 * ot);
        // (rows that do not see the key keep its infinities out)
        const f32x4 y = {e * (float)x[0], e * (float)x[1], e * (float)x[2], e * (float)x[3]};
        add(n, ot, e != 0.f ? y : f32x4{});
      }
    }
  }
}

// The wave rows' sums joined in halves through LDS, and the results.
template <int D, int NG, int WR, int WK>
__device__ __forceinline__ void finish_rows(const TreeParams& p, const WorkItem& it, int row0, u32x4* s_kv, float* s_ml,
                                            f32x4 (&oacc)[NG][D / 16], float (&m_used)[NG], float (&l_part)[NG], int wave,
                                            int lane) {
  constexpr int OT = D / 16, WROWS = 16 * NG;
  const int wr = wave % WR, wk = wave / WR, lt = lane & 15, hq = lane >> 4;
  const int b = it.b, g = it.g, R = p.T * p.G;
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
          s_ml[(2 * wave + 0) * WROWS + 16 * n + lt] = m_used[n];
          s_ml[(2 * wave + 1) * WROWS + 16 * n + lt] = l_part[n];
        }
      }
    }
    wg_barrier();
    if (wk < half) {
      const int other = wave + half * WR;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float m2 = s_ml[(2 * other + 0) * WROWS + 16 * n + lt], l2 = s_ml[(2 * other + 1) * WROWS + 16 * n + lt];
        const float m = fmaxf(m_used[n], m2);
        // (a row without a finite maximum has sums that are zero or NaN)
        const float a1 = m_used[n] == kNegInf ? 1.f : exp2f(m_used[n] - m), a2 = m2 == kNegInf ? 1.f : exp2f(m2 - m);
        l_part[n] = l_part[n] * a1 + l2 * a2;
#pragma unroll
        for (int ot = 0; ot < OT; ++ot) oacc[n][ot] = oacc[n][ot] * a1 + mine[(n * OT + ot) * 64 + lane] * a2;
        m_used[n] = m;
      }
    }
  }
  if (wk != 0) return;

  // ---- results: lane holds row lt, dims 16 ot + 4 hq + e ------------------------------
  const int64_t pr = (int64_t)it.slot * p.T * p.Hq;
  const bool partial = it.partial;
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
      f = finish_row(p, ro.h, ro.t < it.nodes, m, l, lse);
      if (hq == 0) p.lse[b * p.l_sb + ro.t * p.l_ss + ro.h * p.l_sh] = lse;
    }
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      const f32x4 of = oacc[n][ot] * f, o = f == 0.f ? f32x4{} : of;
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

template <int D, int NG>
__global__ __launch_bounds__(256, 1) void tree_mfma_kernel(TreeParams p) {
  using M = Mfma<16>;
  typedef M::acc_t acc_t;
  constexpr int WK = 4, KT = 32, CH = D / 8, KS = D / 32, OT = D / 16;
  constexpr int TILE = 2 * KT * CH, NS = 2;  // 16-byte slots of a K and V tile, stages
  constexpr int ROWS = 16 * NG;
  constexpr int MERGE = (WK / 2) * NG * OT * 64;
  constexpr int SLOTS = NS * WK * TILE > MERGE ? NS * WK * TILE : MERGE;

  __shared__ u32x4 s_kv[SLOTS];
  __shared__ int s_page[WK][NS * 64];
  __shared__ uint64_t s_mask[ROWS];
  __shared__ float s_ml[WK][2][ROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wk = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lt = lane & 15, hq = lane >> 4;

  WorkItem it;
  if (!work_item(p, it)) return;
  const int b = it.b, g = it.g, k0 = it.k0, k1 = it.k1, ctx = it.ctx;
  const int R = p.T * p.G, row0 = it.rb * ROWS;
  const int niter = (k1 - k0 + WK * KT - 1) / (WK * KT);

  // ---- rows: Q^T operands (lane: row 16 n + lt, dims 32 s + 8 hq ..), tree masks ----
  bf16x8 qb[NG][KS];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = row0 + 16 * n + lt, t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R;
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 32 * s);
      qb[n][s] = live ? x : bf16x8{};
    }
  }
  for (int i = tid; i < ROWS; i += 256) {
    const int r = row0 + i;
    s_mask[i] = r < R ? (uint64_t)p.tree_mask[b * p.tm_sb + (r / p.G) * p.tm_ss] : 0;
  }

  TileLoads<D, 1, WK> ld(p, b, g, k0, k1, 0, wk, lane);
  uint32_t mask;  // rows of tile j that are there
  {
    const int pg = *reinterpret_cast<const int32_t*>(ld.page_addr(0)), pg1 = *reinterpret_cast<const int32_t*>(ld.page_addr(1));
    s_page[wk][64 + lane] = pg1;
    mask = ld.load(0, pg, &s_kv[wk * TILE]);
  }
  wait_vm<0>();
  wg_barrier();  // the masks are staged

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

  int st = 0;  // stage of tile j; tile j + 1 goes to the other
  auto step = [&](int j, auto with_drafts) {
    constexpr bool TAIL = decltype(with_drafts)::value;
    wait_vm<0>();  // tile j and the page ids of tile j + 1 have landed (a wave loads what it alone reads)
    // (the page ids of tile j + 2 take the place of tile j's, read at j - 1)
    const int pg = s_page[wk][(st ^ 1) * 64 + lane];
    dma4(&s_page[wk][st * 64], ld.page_addr(j + 2));
    const uint32_t mask_next = ld.load(j + 1, pg, &s_kv[((st ^ 1) * WK + wk) * TILE]);
    u32x4* kt = &s_kv[(st * WK + wk) * TILE];
    u32x4* vt = kt + KT * CH;
    const int base = k0 + (j * WK + wk) * KT;
    uint32_t bad = 0;  // drafted rows whose V holds infinities or NaN: out of the product, added by hand
    if constexpr (TAIL) bad = bad_rows<D, 1>(vt, base, ctx, 0, lane);

    // by 16 keys (half the scores in registers): S^T, then its softmax; a lane
    // holds keys 16 mt + 4 hq + e of its row
    // weights, and what their rounding left: a second product costs 3 % where the
    // keys' rows bound the call, and results are as near the exact ones as their own
    // rounding (0.0017 rms relative; 0.0021 to 0.0026 with one rounded weight)
    bf16x8 pb[NG], pr[NG];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      acc_t sacc[NG];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8 kf = lds_read_b128(kt, (ka ^ (uint32_t)(64 * s)) + (uint32_t)(16 * mt) * pitch);
#pragma unroll
        for (int n = 0; n < NG; ++n) sacc[n] = M::mma(kf, qb[n][s], s == 0 ? acc_t{} : sacc[n]);
      }
      if (TAIL || mask != 0xffffffffu) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const uint32_t seen = seen4<TAIL>(mask, TAIL ? s_mask[16 * n + lt] : 0, 16 * mt + 4 * hq, base - ctx);
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
            for (int i = 0; i < 4; ++i) {
              const float x = ((float)pb[n][i] + (float)pr[n][i]) * alpha;
              pb[n][i] = (bf16)x;
              pr[n][i] = (bf16)(x - (float)pb[n][i]);
            }
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
          pr[n][4 * mt + i] = (bf16)(ex[i] - (float)pb[n][4 * mt + i]);
        }
        l_part[n] += (ex[0] + ex[1]) + (ex[2] + ex[3]);
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      const uint32_t off = va ^ (uint32_t)(32 * ot);
      const bf16x4 lo = lds_read_tr16(vt, off), hi = lds_read_tr16(vt, off + 16u * pitch);
      const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (int n = 0; n < NG; ++n) oacc[n][ot] = M::mma(a, pr[n], M::mma(a, pb[n], oacc[n][ot]));
    }
    if constexpr (TAIL)
      add_bad_rows<D, NG>(p, b, g, base, bad, pb, lt, hq, [&](int n, int ot, const acc_t& y) { oacc[n][ot] += y; });
    mask = mask_next;
    st ^= 1;
  };
  // steps without a drafted row in any of the workgroup's tiles, then the others
  const int whole = min(max(ctx - k0, 0) / (WK * KT), niter);
  int j = 0;
  for (; j < whole; ++j) step(j, std::false_type{});
  for (; j < niter; ++j) step(j, std::true_type{});
  wait_vm<0>();  // the loads past the range have landed before LDS is used for anything else

  finish_rows<D, NG, 1, WK>(p, it, row0, s_kv, &s_ml[0][0][0], oacc, m_used, l_part, wk, lane);
}

// ---- more than 64 rows: two waves a SIMD, scores a tile ahead ---------------------
// 32 rows a wave, and each wave overlaps its own work too: a step issues the
// products S^T of tile j + 1 and O^T of tile j, and between them, one score
// after every second product or so, the softmax of tile j, which depends on
// neither.  Sums and Q stay in AGPRs (inline asm: the compiler would copy Q to
// VGPRs for every product); sched_barrier keeps the order that is written here.
// 16 sequences of 4K-32K keys, 256 rows (one of 128K keys, 8 kv heads): 115 (180) us,
// the matrix cores busy 0.35 (0.39) of the time, 4.5 VALU instructions a product.
// 64 rows a wave read half as much from LDS and took 132 (198) us with one wave a
// SIMD, 256 (406) us with two, which spill; without the overlap 163 (248) us.
// PAGE: tiles of 32 keys lie within one page, whose rows have one base and stride
// (198 us for 208 with an address per row, 128K keys, 64 rows a wave; with 32 rows a
// wave it is 112 and 181 us in pages of 64 rows, 108 and 188 with an address per row
// in pages of 16, which spills one register).
template <int D, int NG, int WR, int WK, int NS, bool PAGE>
__global__ __launch_bounds__(64 * WR * WK, WR * WK / 4) void tree_pipe_kernel(TreeParams p) {
  using M = Mfma16A;
  typedef M::acc_t acc_t;
  constexpr int NW = WR * WK, KT = 32, CH = D / 8, KS = D / 32, OT = D / 16;
  constexpr int RPI = 64 / CH, ROWI = KT / RPI, NI = 2 * ROWI / WR;
  constexpr int TILE = 2 * KT * CH, WROWS = 16 * NG, RING = 4;  // NS stages of a K and V tile
  constexpr int MERGE = WK > 1 ? (WK / 2) * WR * NG * OT * 64 : 0;
  constexpr int SLOTS = NS * WK * TILE > MERGE ? NS * WK * TILE : MERGE;
  static_assert(NG % 2 == 0, "drain_v4");
  static_assert(NS >= 3 && NS <= RING + 1, "page ids of NS - 1 tiles are held");

  __shared__ u32x4 s_kv[SLOTS];
  __shared__ int s_page[NW][(RING + 1) * 64];  // (and one slot for ids that are not used)
  __shared__ uint64_t s_mask[WR * WROWS];
  __shared__ float s_ml[NW][2][WROWS];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave % WR, wk = wave / WR;
  const int lt = lane & 15, hq = lane >> 4;

  WorkItem it;
  if (!work_item(p, it)) return;
  const int b = it.b, g = it.g, k0 = it.k0, k1 = it.k1, ctx = it.ctx;
  const int R = p.T * p.G, row0 = it.rb * WR * WROWS;
  const int niter = (k1 - k0 + WK * KT - 1) / (WK * KT);

  bf16x8 qb[NG][KS];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = row0 + wr * WROWS + 16 * n + lt, t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R;
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 32 * s);
      qb[n][s] = M::to_agpr(live ? x : bf16x8{});
    }
  }
  for (int i = tid; i < WR * WROWS; i += 64 * NW) {
    const int r = row0 + i;
    s_mask[i] = r < R ? (uint64_t)p.tree_mask[b * p.tm_sb + (r / p.G) * p.tm_ss] : 0;
  }

  typedef typename std::conditional<PAGE, PageLoads<D, WR, WK>, TileLoads<D, WR, WK>>::type Loads;
  Loads ld(p, b, g, k0, k1, wr, wk, lane);
  // Loads go out in groups, tile t's page id for tile t + NS - 2 before its own rows;
  // group t goes out in step t - NS (0 .. NS - 1 here).
  uint32_t vm[NS + 1];  // rows that are there, of tiles j, j + 1, ..
  auto group_page = [&](int t) {
    int* ring = &s_page[wave][(t < 2 ? RING : (t + NS - 2) % RING) * 64];
    if constexpr (PAGE) ld.fetch_page(t + NS - 2, ring);
    else dma4(ring, ld.page_addr(t + NS - 2));
  };
  {
    int pg[NS];
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      if constexpr (PAGE) pg[t] = ld.trow[min(ld.key0 + t * WK * KT, ld.last_key) >> ld.page_shift];
      else pg[t] = *reinterpret_cast<const int32_t*>(ld.page_addr(t));
    }
#pragma unroll
    for (int t = 0; t < NS; ++t) {
      u32x4* dst = &s_kv[(t * WK + wk) * TILE];
      group_page(t);
      if constexpr (PAGE) {
        vm[t] = ld.begin(t, __builtin_amdgcn_readfirstlane(pg[t]));
#pragma unroll
        for (int i = 0; i < NI; ++i) ld.issue(i, dst);
      } else {
        vm[t] = ld.load(t, pg[t], dst);
      }
    }
    vm[NS] = 0;
  }
  wait_vm<(NS - 2) * (NI + 1)>();  // tiles 0 and 1
  wg_barrier();

  const uint32_t pitch = CH * 16;
  const uint32_t ka = (uint32_t)lt * pitch + (uint32_t)((hq ^ Swz<D>::at(lt)) << 4);
  const int rr = lt >> 2, cc = lt & 3, vr = 4 * hq + rr;
  const uint32_t va = (uint32_t)vr * pitch + (uint32_t)(((cc >> 1) ^ Swz<D>::at(vr)) << 4) + (uint32_t)(cc & 1) * 8u;

  acc_t oacc[NG][OT];
  float m_used[NG], l_part[NG];
  float thr[NG], moff[NG];  // the raw score that moves the maximum, and -maximum (0 while there is none)
  const float inv_scale = 1.f / p.scale_log2;
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    m_used[n] = thr[n] = kNegInf;
    l_part[n] = moff[n] = 0.f;
#pragma unroll
    for (int i = 0; i < OT; ++i) {
      acc_t z = acc_t{};
      asm volatile("" : "+a"(z));
      oacc[n][i] = z;
    }
  }

  // S^T product i of a tile: contraction step i / 2 NG, keys 16 (i / NG % 2) .., rows 16 (i % NG) ..
  constexpr int NSM = 2 * NG * KS, NPV = NG * OT, NM = NSM + NPV, NF = 2 * KS;
  auto read_k = [&](const u32x4* kt, int f) {
    return lds_read_b128(kt, (ka ^ (uint32_t)(64 * (f >> 1))) + (uint32_t)(16 * (f & 1)) * pitch);
  };
  acc_t sca[NG][2], scb[NG][2];
  float tmax[NG];
  {
    const u32x4* kt = &s_kv[wk * TILE];
    bf16x8 prev_k = {};
    each<NSM>([&](auto ic) {
      constexpr int i = decltype(ic)::value, s = i / (2 * NG), mt = (i / NG) & 1, n = i % NG;
      const bf16x8 kf = read_k(kt, i / NG);
      if constexpr (s == 0) M::mma_v0_ba(kf, qb[n][s], sca[n][mt], prev_k);
      else M::mma_v_ba(kf, qb[n][s], sca[n][mt], prev_k);
      prev_k = kf;
    });
    M::tail1(prev_k);
#pragma unroll
    for (int n = 0; n < NG; n += 2) M::drain_v4(sca[n][0], sca[n][1], sca[n + 1][0], sca[n + 1][1]);
  }
  constexpr int PK = NF < 3 ? NF : 3;  // K operands read ahead
  bf16x8 kf[4];                        // the first of tile j + 1 at the start of step j
#pragma unroll
  for (int f = 0; f < PK; ++f) kf[f] = read_k(&s_kv[((1 % NS) * WK + wk) * TILE], f);
  auto max_of = [&](const acc_t (&sc)[2]) {
    return max_raw(max3_raw(max3_raw(sc[0][0], sc[0][1], sc[0][2]), sc[0][3], sc[1][0]), max3_raw(sc[1][1], sc[1][2], sc[1][3]));
  };
#pragma unroll
  for (int n = 0; n < NG; ++n) tmax[n] = max_of(sca[n]);

  int st = 0;
  auto step = [&](int j, acc_t (&cur)[NG][2], acc_t (&nxt)[NG][2], auto with_drafts) {
    constexpr bool TAIL = decltype(with_drafts)::value;
    const int st1 = st + 1 == NS ? 0 : st + 1, st2 = st1 + 1 == NS ? 0 : st1 + 1;
    u32x4* vt = &s_kv[(st * WK + wk) * TILE] + KT * CH;
    const u32x4* kn = &s_kv[(st1 * WK + wk) * TILE];
    const u32x4* kn2 = &s_kv[(st2 * WK + wk) * TILE];
    u32x4* dst = &s_kv[(st * WK + wk) * TILE];
    int pg = 0;
    const int base = k0 + (j * WK + wk) * KT;
    const uint32_t mask = vm[0];
    uint32_t bad = 0;  // drafted rows whose V holds infinities or NaN: out of the product, added by hand
    if constexpr (TAIL) bad = bad_rows<D, WR>(vt, base, ctx, wr, lane);
    if (TAIL || mask != 0xffffffffu) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const uint64_t tm = TAIL ? s_mask[wr * WROWS + 16 * n + lt] : 0;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint32_t seen = seen4<TAIL>(mask, tm, 16 * mt + 4 * hq, base - ctx);
          const float x0 = seen & 1u ? cur[n][mt][0] : kNegInf, x1 = seen & 2u ? cur[n][mt][1] : kNegInf;
          const float x2 = seen & 4u ? cur[n][mt][2] : kNegInf, x3 = seen & 8u ? cur[n][mt][3] : kNegInf;
          cur[n][mt] = acc_t{x0, x1, x2, x3};
        }
        tmax[n] = max_of(cur[n]);
      }
    }
    bool over = false;
#pragma unroll
    for (int n = 0; n < NG; ++n) over |= tmax[n] > thr[n];
    if (__any(over)) {
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const float m_new = fmaxf(m_used[n], xor32_max(xor16_max(tmax[n])) * p.scale_log2);
        const float alpha = m_new == kNegInf ? 1.f : exp2f(m_used[n] - m_new);
        l_part[n] *= alpha;
        m_used[n] = m_new;
        thr[n] = (m_new + 8.f) * inv_scale;
        moff[n] = m_new == kNegInf ? 0.f : -m_new;
        drain_all(oacc[n]);
#pragma unroll
        for (int i = 0; i < OT; ++i) {
          acc_t x = oacc[n][i] * alpha;
          asm volatile("" : "+a"(x));
          oacc[n][i] = x;
        }
      }
    }

    bf16x8 vf[OT], pb[NG];
    uint32_t pw[NG][4];
    float ex[2] = {0.f, 0.f}, arg = fmaf(cur[0][0][0], p.scale_log2, moff[0]);
    bf16x8 pa = {}, pp = {};
    each<NM>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i < NSM) {
        constexpr int f = i / NG, s = f >> 1, mt = f & 1, n = i % NG;
        if constexpr (s == 0) M::mma_v0_ba(kf[f & 3], qb[n][s], nxt[n][mt], pa);
        else M::mma_v_ba(kf[f & 3], qb[n][s], nxt[n][mt], pa);
        pa = kf[f & 3];
        if constexpr (n == 1 && f + 3 < NF) kf[(f + 3) & 3] = read_k(kn, f + 3);
        if constexpr (i % (NSM / OT) == (NSM / OT) / 2) {
          constexpr int o = i / (NSM / OT);
          const uint32_t off = va ^ (uint32_t)(32 * o);
          const bf16x4 lo = lds_read_tr16(vt, off), hi = lds_read_tr16(vt, off + 16u * pitch);
          vf[o] = bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
      } else {
        constexpr int n = (i - NSM) / OT, o = (i - NSM) % OT;
        if constexpr (o == 0) pb[n] = __builtin_bit_cast(bf16x8, u32x4{pw[n][0], pw[n][1], pw[n][2], pw[n][3]});
        M::template mma<o == 0>(vf[o], pb[n], oacc[n][o], pa, pp);
        pa = vf[o];
        pp = pb[n];
      }
      // the softmax's scores, evenly over the products before the last row group's
      constexpr int NE = 8 * NG;
      each<NE>([&](auto ec) {
        constexpr int e = decltype(ec)::value, n = e >> 3, k = e & 7;
        if constexpr (e * (NM - OT) / NE == i) {
          const float x = __builtin_amdgcn_exp2f(arg);
          if constexpr (e < NE - 1) {
            constexpr int n1 = (e + 1) >> 3, k1_ = (e + 1) & 7;
            arg = fmaf(cur[n1][k1_ >> 2][k1_ & 3], p.scale_log2, moff[n1]);
          }
          l_part[n] += x;
          ex[k & 1] = x;
          if constexpr (k & 1) {
            const bf16x2 w = {(bf16)ex[0], (bf16)ex[1]};
            pw[n][k >> 1] = __builtin_bit_cast(uint32_t, w);
          }
        }
      });
      // Once tile j's operands are all in registers: wait for tile j + 2, let the
      // other waves finish with tile j, then load tile j + NS over it and read
      // the first K operands of tile j + 2.
      constexpr int BAR = NM - 20 > NSM ? NM - 20 : NSM;
      static_assert(BAR + 5 + NI <= NM, "the step's loads fit");
      if constexpr (i == BAR) {
        wait_vm<(NS - 3) * (NI + 1)>();
        if constexpr (WR > 1) asm volatile("s_barrier" ::: "memory");
        pg = s_page[wave][((j + NS) % RING) * 64 + lane];
      }
      if constexpr (i > BAR && i - BAR - 1 < PK) kf[i - BAR - 1] = read_k(kn2, i - BAR - 1);
      if constexpr (i == BAR + 4) {
        group_page(j + NS);
        if constexpr (PAGE) vm[NS] = ld.begin(j + NS, __builtin_amdgcn_readfirstlane(pg));
        else vm[NS] = ld.load(j + NS, pg, dst);
      }
      if constexpr (PAGE) {
        if constexpr (i > BAR + 4 && i - BAR - 5 < NI) ld.issue(i - BAR - 5, dst);
      }
      // ... and the next tile's maxima after them
      if constexpr (i >= NM - OT && (i - (NM - OT)) % (OT / NG) == 0) {
        constexpr int n = (i - (NM - OT)) / (OT / NG);
        tmax[n] = max_of(nxt[n]);
      }
    });
    M::tail(pa, pp);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (TAIL) {
      add_bad_rows<D, NG>(p, b, g, base, bad, pb, lt, hq, [&](int n, int o, const acc_t& y) {
        M::drain(oacc[n][o]);
        acc_t x = oacc[n][o] + y;
        asm volatile("" : "+a"(x));
        oacc[n][o] = x;
      });
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) vm[i] = vm[i + 1];
    st = st1;
  };
  // steps without a drafted row in any of the workgroup's tiles, then the others
  const int whole = min(max(ctx - k0, 0) / (WK * KT), niter);
  int j = 0;
  for (; j + 1 < whole; j += 2) {
    step(j, sca, scb, std::false_type{});
    step(j + 1, scb, sca, std::false_type{});
  }
  for (; j < niter; ++j) {
    step(j, sca, scb, std::true_type{});
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sca[n][0] = scb[n][0];
      sca[n][1] = scb[n][1];
    }
  }
  wait_vm<0>();  // the loads past the range have landed before LDS is used for anything else
#pragma unroll
  for (int n = 0; n < NG; ++n) drain_all(oacc[n]);
  finish_rows<D, NG, WR, WK>(p, it, row0, s_kv, &s_ml[0][0][0], oacc, m_used, l_part, wave, lane);
}

// ---- latent rows: d_qk = 576, d_v = 512, V the first 512 dims of K, bf16 ----------
// One workgroup of 8 waves takes 64 rows of one key range, in tiles of 64
// keys (72 KB of LDS, two stages), and divides the two products differently:
//  * S^T = K Q^T: wave (rh, kq) takes 32 rows x 16 keys, its Q in 144 AGPRs; a K
//    operand read from LDS serves 32 rows;
//  * P^T goes through LDS (8 KB) in the operand order, and
//  * O^T = V^T P^T: wave w takes dims 64 w .. 64 w + 63 of all 64 rows (64
//    accumulators), so each V element is read from LDS once.
// Per tile LDS moves 356 KB (2785 clocks), the products take 2176 clocks of
// every SIMD.  The next tile's rows are loaded during S^T, a load after every
// fourth product.  The running maximum is shared: a row's scores are in four
// waves, so a wave that finds one past the maximum by 8 (base 2) raises a flag,
// and all of them move it together after the barrier that publishes P.
// P is rounded to bf16 once (2^-8 of a weight; results 0.0019 rms from float64 where
// float32 weights leave the result's own 0.0017): what that left would make half of
// the products again and needs 8 KB that LDS, 163.6 KB full, does not have.
struct MlaTree {
  static constexpr int kDqk = 576, kDv = 512, kKeys = 64, kSteps = kDqk / 32;
  static constexpr int kCh = kDv / 8, kCr = (kDqk - kDv) / 8;  // 16-byte chunks of the two parts of a row
};

// PAGE: tiles lie within one page (64 rows or more), whose rows have one base: 245 to
// 252 us, with an address per row 245 to 256 in pages of 16 and 32 rows (4 sequences
// of 8K to 32K keys, 8 tokens, 128 heads).
template <bool PAGE>
__global__ __launch_bounds__(512, 2) void tree_mla_kernel(TreeParams p) {
  typedef MlaTree C;
  typedef Mfma16A MA;
  typedef Mfma<16> M;
  typedef f32x4 acc_t;
  constexpr int CH = C::kCh, CR = C::kCr, KEYS = C::kKeys, STEPS = C::kSteps, RPW = KEYS / 8;

  __shared__ u32x4 s_k[2][KEYS * CH];  // dims 0 .. 511 (K and V), swizzled as rows of 128
  __shared__ u32x4 s_r[2][KEYS * CR];  // dims 512 .. 575, as rows of 64
  __shared__ u32x4 s_p[2 * 64 * 4];  // [32-key half][hq][row] 8 keys
  __shared__ u32x4 s_q[64 * 4];      // [hq][row] Q's last 32 dims
  __shared__ u32x4 s_q1[32 * 4];     // [hq][16 rh + lt] the 32 before them, of row group 1
  __shared__ uint64_t s_mask[64];
  __shared__ float s_m[64];          // running maxima (base 2)
  __shared__ float s_x[4][64];       // per key quarter: row maxima, then row sums
  __shared__ int s_over[2];
  __shared__ unsigned long long s_bad;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rh = wave & 1, kq = wave >> 1;
  const int lt = lane & 15, hq = lane >> 4;

  WorkItem it;
  if (!work_item(p, it)) return;
  const int b = it.b, g = it.g, k0 = it.k0, k1 = it.k1, ctx = it.ctx;
  const int R = p.T * p.G, row0 = it.rb * 64;
  const int ntiles = (k1 - k0 + KEYS - 1) / KEYS;

  // ---- rows ----------------------------------------------------------------------
  // (Q's last one and a half contraction steps in LDS: 128 AGPRs, and no VGPR to spare)
  bf16x8 qa[2][16], q16;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int r = row0 + 32 * rh + 16 * n + lt, t = r / p.G, h = g * p.G + r % p.G;
    const bool live = r < R;
    const bf16* q = reinterpret_cast<const bf16*>(p.q) + b * p.q_sb + (live ? t * p.q_ss + h * p.q_sh : 0) + 8 * hq;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const bf16x8 x = *reinterpret_cast<const bf16x8*>(q + 32 * s), y = live ? x : bf16x8{};
      if (s < 16) qa[n][s < 16 ? s : 0] = MA::to_agpr(y);
      else if (s == 16 && n == 0) q16 = y;
      else if (s == 16 && kq == 0) s_q1[hq * 32 + 16 * rh + lt] = __builtin_bit_cast(u32x4, y);
      else if (s == 17 && kq == 0) s_q[hq * 64 + 32 * rh + 16 * n + lt] = __builtin_bit_cast(u32x4, y);
    }
  }
  if (tid < 64) {
    const int r = row0 + tid;
    s_mask[tid] = r < R ? (uint64_t)p.tree_mask[b * p.tm_sb + (r / p.G) * p.tm_ss] : 0;
    s_m[tid] = kNegInf;
    if (tid < 2) s_over[tid] = 0;
    if (tid == 2) s_bad = 0;
  }

  // ---- loads: the wave's 8 rows of a tile, one instruction each for their first
  // 1024 bytes and one for the last 128 of all; lane l finds the address of row l
  const uint64_t kbase = (uint64_t)(uintptr_t)p.k + 2 * (int64_t)g * p.k_sh;
  const int32_t* trow = p.block_table + b * p.bt_sb;
  const int last_key = p.cap - 1;
  auto page_of = [&](int j, int ln) { return trow[min(k0 + j * KEYS + ln, last_key) >> p.page_shift]; };
  auto row_addr = [&](int j, int pg, int ln, bool& ok) {
    const int s = k0 + j * KEYS + ln;
    ok = s < k1 && pg >= 0 && pg < p.num_pages;
    const uint64_t a = kbase + (uint64_t)((int64_t)pg * (2 * p.k_sb) + (int64_t)(s & ((1 << p.page_shift) - 1)) * (2 * p.k_ss));
    return ok ? a : (uint64_t)(uintptr_t)kZeroRow;
  };
  auto load_row = [&](int i, uint64_t ra, u32x4* dst, int ln) {
    const int row = wave * RPW + i;
    const uint64_t base = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(ra >> 32), row) << 32) |
                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)ra, row);
    dma16(dst + row * CH, base, 16u * (uint32_t)(ln ^ Swz<128>::at(row)));
  };
  auto load_tails = [&](uint64_t ra, u32x4* dst, int ln) {
    const int row = wave * RPW + (ln >> 3);
    const uint64_t a = ((uint64_t)(uint32_t)__shfl((int)(uint32_t)(ra >> 32), row, 64) << 32) |
                       (uint32_t)__shfl((int)(uint32_t)ra, row, 64);
    dma16(dst + wave * RPW * CR, a + (uint64_t)(16 * (CH + ((ln & 7) ^ Swz<64>::at(row)))));
  };
  // PAGE: the tile's base and row stride (a tile that is not there: zeros, stride 0)
  const int64_t krow_bytes = 2 * p.k_ss;
  struct TileBase {
    uint64_t base;
    int64_t row;
    uint64_t mask;
  };
  auto page_tile = [&](int j, int pg) {
    const int s = k0 + j * KEYS, n = k1 - s;
    const bool ok = n > 0 && pg >= 0 && pg < p.num_pages;
    TileBase t;
    t.base = ok ? kbase + (uint64_t)((int64_t)pg * (2 * p.k_sb) + (int64_t)(s & ((1 << p.page_shift) - 1)) * krow_bytes)
                : (uint64_t)(uintptr_t)kZeroRow;
    t.row = ok ? krow_bytes : 0;
    t.mask = !ok ? 0 : n >= KEYS ? ~0ull : (1ull << n) - 1;
    return t;
  };
  auto page_row = [&](int i, const TileBase& t, u32x4* dst, int ln) {
    const int row = wave * RPW + i;
    dma16(dst + row * CH, t.base + (uint64_t)(row * t.row), 16u * (uint32_t)(ln ^ Swz<128>::at(row)));
  };
  auto page_tails = [&](const TileBase& t, u32x4* dst, int ln) {
    const int row = wave * RPW + (ln >> 3);
    dma16(dst + wave * RPW * CR, t.base + (uint64_t)(wave * RPW * t.row),
          (uint32_t)((ln >> 3) * (int)t.row) + 16u * (uint32_t)(CH + ((ln & 7) ^ Swz<64>::at(row))));
  };
  uint64_t mask;  // the rows of tile j that are there
  if constexpr (PAGE) {
    const TileBase t = page_tile(0, __builtin_amdgcn_readfirstlane(page_of(0, 0)));
    mask = t.mask;
#pragma unroll
    for (int i = 0; i < RPW; ++i) page_row(i, t, s_k[0], lane);
    page_tails(t, s_r[0], lane);
  } else {
    bool ok;
    const uint64_t ra = row_addr(0, page_of(0, lane), lane, ok);
    mask = __ballot(ok);
#pragma unroll
    for (int i = 0; i < RPW; ++i) load_row(i, ra, s_k[0], lane);
    load_tails(ra, s_r[0], lane);
  }
  int pg_next = page_of(1, PAGE ? 0 : lane);

  acc_t oacc[4][4];  // [16 dims][16 rows]
#pragma unroll
  for (int o = 0; o < 4; ++o)
#pragma unroll
    for (int n = 0; n < 4; ++n) oacc[o][n] = acc_t{};
  float m_used[2] = {kNegInf, kNegInf}, l_part[2] = {0.f, 0.f};

  auto step = [&](int j, auto with_drafts) {
    constexpr bool TAIL = decltype(with_drafts)::value;
    const u32x4 *kt = s_k[j & 1], *rt = s_r[j & 1];
    // (lane constants are formed per tile: held across the loop they spill)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    int lt = ln & 15, hq = ln >> 4;
    // operand addresses (rows are whole multiples of 128 bytes: a chunk's bits
    // can be flipped in place)
    const int krow = 16 * kq + lt, fr = Swz<128>::at(lt);
    const uint32_t ka = (uint32_t)(krow * CH + (hq ^ fr)) * 16u;
    const uint32_t kr = (uint32_t)(krow * CR + (hq ^ Swz<64>::at(lt))) * 16u;
    // tile j has landed for all waves; tile j - 1 and its P are read
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // contraction steps in order, the one with Q in LDS first
    auto order = [](int i) { return i == 0 ? STEPS - 1 : i - 1; };
    bf16x8 kf[3], ql[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) ql[n] = lds_read_b128(s_q, (uint32_t)((hq * 64 + 32 * rh + 16 * n + lt) * 16));
    auto read_k = [&](int s) {
      return s < 16 ? lds_read_b128(kt, ka ^ (uint32_t)(64 * s)) : lds_read_b128(rt, kr ^ (uint32_t)(64 * (s - 16)));
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) kf[s] = read_k(order(s));
    uint64_t ra = 0, mask_next;
    TileBase tb = {};
    if constexpr (PAGE) {
      tb = page_tile(j + 1, __builtin_amdgcn_readfirstlane(pg_next));
      mask_next = tb.mask;
    } else {
      bool ok;
      ra = row_addr(j + 1, pg_next, ln, ok);
      mask_next = __ballot(ok);
    }
    if (tid == 0) s_over[(j + 1) & 1] = 0;

    // S^T of 16 keys x 32 rows
    acc_t sacc[2];
    bf16x8 pk = {};
    each<STEPS>([&](auto ic) {
      constexpr int i = decltype(ic)::value, s = i - 1;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (i + 2 < STEPS) kf[(i + 2) % 3] = read_k(i + 1);
      if constexpr (i == 0) {
        MA::mma_v0(kf[0], ql[0], sacc[0], pk);
        MA::mma_v0(kf[0], ql[1], sacc[1], pk);
      } else if constexpr (s < 16) {
        MA::mma_v_ba(kf[i % 3], qa[0][s], sacc[0], pk);
        MA::mma_v_ba(kf[i % 3], qa[1][s], sacc[1], pk);
      } else {
        MA::mma_v(kf[i % 3], q16, sacc[0], pk);
        MA::mma_v(kf[i % 3], ql[0], sacc[1], pk);
      }
      pk = kf[i % 3];
      if constexpr (i == 14) ql[0] = lds_read_b128(s_q1, (uint32_t)((hq * 32 + 16 * rh + lt) * 16));
      // the next tile's rows
      if constexpr (i % 2 == 1 && i / 2 < RPW) {
        if constexpr (PAGE) page_row(i / 2, tb, s_k[(j + 1) & 1], ln);
        else load_row(i / 2, ra, s_k[(j + 1) & 1], ln);
      } else if constexpr (i == 17) {
        if constexpr (PAGE) page_tails(tb, s_r[(j + 1) & 1], ln);
        else load_tails(ra, s_r[(j + 1) & 1], ln);
      }
    });
    __builtin_amdgcn_sched_barrier(0);
    pg_next = page_of(j + 2, PAGE ? 0 : ln);
    MA::tail1(pk);
    MA::drain_v1(sacc[0]);
    MA::drain_v1(sacc[1]);
    asm volatile("" : "+v"(ln));  // (what the second half needs is formed now)
    lt = ln & 15;
    hq = ln >> 4;
    const int rr = lt >> 2, cc = lt & 3, vrow = 4 * hq + rr;
    const uint32_t va =
        (uint32_t)(vrow * CH + ((8 * wave + (cc >> 1)) ^ Swz<128>::at(vrow))) * 16u + (uint32_t)(cc & 1) * 8u;
    char* const pw = reinterpret_cast<char*>(s_p) + (((kq >> 1) * 4 + hq) * 64 + 32 * rh + lt) * 16 + (kq & 1) * 8;

    // the lane's keys 16 kq + 4 hq + e of its rows
    if (TAIL || mask != ~0ull) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t seen = seen4<TAIL>((uint32_t)(mask >> (16 * kq)), TAIL ? s_mask[32 * rh + 16 * n + lt] : 0, 4 * hq,
                                          k0 + j * KEYS + 16 * kq - ctx);
        const float x0 = seen & 1u ? sacc[n][0] : kNegInf, x1 = seen & 2u ? sacc[n][1] : kNegInf;
        const float x2 = seen & 4u ? sacc[n][2] : kNegInf, x3 = seen & 8u ? sacc[n][3] : kNegInf;
        sacc[n] = acc_t{x0, x1, x2, x3};
      }
    }
    bool over = false;
    float tmax[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      tmax[n] = max_raw(max3_raw(sacc[n][0], sacc[n][1], sacc[n][2]), sacc[n][3]);
      over |= tmax[n] * p.scale_log2 > m_used[n] + 8.f;
    }
    if (__any(over) && lane == 0) s_over[j & 1] = 1;
    auto weights = [&](float (&sum)[2]) {  // P^T of the lane's keys into LDS
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float moff = m_used[n] == kNegInf ? 0.f : -m_used[n];
        float ex[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ex[e] = __builtin_amdgcn_exp2f(fmaf(sacc[n][e], p.scale_log2, moff));
        const bf16x4 w = {(bf16)ex[0], (bf16)ex[1], (bf16)ex[2], (bf16)ex[3]};
        *reinterpret_cast<bf16x4*>(pw + n * 16 * 16) = w;
        sum[n] = (ex[0] + ex[1]) + (ex[2] + ex[3]);
      }
    };
    float sum[2];
    weights(sum);
    if constexpr (TAIL) {
      // drafted rows whose V holds infinities or NaN (the wave's 8 rows)
      const int row = wave * RPW + (ln >> 3);
      uint32_t x = 0;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        const u32x4 w = kt[row * CH + (ln & 7) * 8 + c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x |= (w[e] & 0x7f80u) == 0x7f80u;
          x |= (w[e] & 0x7f800000u) == 0x7f800000u;
        }
      }
      if (x != 0 && k0 + j * KEYS + row >= ctx) atomicOr(&s_bad, 1ull << row);
    }
    wg_barrier();  // P, the flag (and the rows with infinities) are there
    if (s_over[j & 1] != 0) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float t = xor32_max(xor16_max(tmax[n])) * p.scale_log2;
        if (hq == 0) s_x[kq][32 * rh + 16 * n + lt] = t;
      }
      wg_barrier();
      auto moved = [&](int row, float& alpha) {
        const float m = s_m[row];
        const float mn = fmaxf(fmaxf(m, fmaxf(s_x[0][row], s_x[1][row])), fmaxf(s_x[2][row], s_x[3][row]));
        alpha = mn == kNegInf ? 1.f : exp2f(m - mn);
        return mn;
      };
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float alpha;
        moved(16 * n + lt, alpha);
#pragma unroll
        for (int o = 0; o < 4; ++o) oacc[o][n] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float alpha;
        m_used[n] = moved(32 * rh + 16 * n + lt, alpha);
        l_part[n] *= alpha;
      }
      weights(sum);
      wg_barrier();
      if (kq == 0 && hq == 0) {
        s_m[32 * rh + lt] = m_used[0];
        s_m[32 * rh + 16 + lt] = m_used[1];
      }
    }
    l_part[0] += sum[0];
    l_part[1] += sum[1];

    uint64_t bad = 0;
    if constexpr (TAIL) {
      bad = s_bad;
      if (bad != 0) {  // out of the product: 0 times them would reach rows that do not see them
        for (int i = ln; i < RPW * CH; i += 64)
          if ((bad >> (wave * RPW + i / CH)) & 1) s_k[j & 1][wave * RPW * CH + i] = u32x4{0, 0, 0, 0};
        wg_barrier();
      }
    }
    // O^T += V^T P^T over the wave's 64 dims
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      bf16x8 pb[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) pb[n] = lds_read_b128(s_p, (uint32_t)(((kk * 4 + hq) * 64 + 16 * n + lt) * 16));
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        if (o % 2 == 0) __builtin_amdgcn_sched_barrier(0);
        const uint32_t off = (va ^ (uint32_t)(32 * o)) + (uint32_t)(32 * kk * CH) * 16u;
        const bf16x4 lo = lds_read_tr16(kt, off), hi = lds_read_tr16(kt, off + 16u * CH * 16u);
        const bf16x8 a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int n = 0; n < 4; ++n) oacc[o][n] = M::mma(a, pb[n], oacc[o][n]);
      }
    }
    if constexpr (TAIL) {
      if (bad != 0) {  // the rows that see them
        for (uint64_t left = bad; left != 0; left &= left - 1) {
          const int key = __builtin_ctzll(left);
          const int64_t vo = key_row(p, b, k0 + j * KEYS + key, p.k_sb, p.k_ss);
          if (vo < 0) continue;
          const bf16* v = reinterpret_cast<const bf16*>(p.k) + vo + g * p.k_sh + 64 * wave + 4 * hq;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            // (the key's place in the operand order: half, lane group, then 4 + 4)
            const int at = (((key >> 5) * 4 + ((key & 15) >> 2)) * 64 + 16 * n + lt) * 8 + ((key >> 4) & 1) * 4 + (key & 3);
            const float e = (float)reinterpret_cast<const bf16*>(s_p)[at];
#pragma unroll
            for (int o = 0; o < 4; ++o) {
              __builtin_amdgcn_sched_barrier(0);
              const bf16x4 x = *reinterpret_cast<const bf16x4*>(v + 16 * o);
              const acc_t y = {e * (float)x[0], e * (float)x[1], e * (float)x[2], e * (float)x[3]};
              oacc[o][n] += e != 0.f ? y : acc_t{};
            }
          }
        }
        wg_barrier();
        if (tid == 0) s_bad = 0;
      }
    }
    mask = mask_next;
  };
  const int whole = min(max(ctx - k0, 0) / KEYS, ntiles);
  int j = 0;
  for (; j < whole; ++j) step(j, std::false_type{});
  for (; j < ntiles; ++j) step(j, std::true_type{});
  wait_vm<0>();

  // ---- row sums over the key quarters; results ------------------------------------------
  wg_barrier();
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float l = l_part[n];
    l += __shfl_xor(l, 16, 64);
    l = xor32_sum(l);
    if (hq == 0) s_x[kq][32 * rh + 16 * n + lt] = l;
  }
  wg_barrier();
  const int64_t pr = (int64_t)it.slot * p.T * p.Hq;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = 16 * n + lt, r = row0 + row;
    if (r >= R) continue;
    const RowOut ro = row_out(p, g, r);
    const float m = s_m[row], l = (s_x[0][row] + s_x[1][row]) + (s_x[2][row] + s_x[3][row]);
    float f, lse;
    if (it.partial) {
      f = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      lse = l > 0.f ? lse2_of(m, l) : l == 0.f ? kNegInf : l;
      if (wave == 0 && hq == 0) p.part_lse[pr + ro.r] = lse;
    } else {
      f = finish_row(p, ro.h, ro.t < it.nodes, m, l, lse);
      if (wave == 0 && hq == 0) p.lse[b * p.l_sb + ro.t * p.l_ss + ro.h * p.l_sh] = lse;
    }
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const f32x4 of = oacc[o][n] * f, x = f == 0.f ? f32x4{} : of;
      const int d = 64 * wave + 16 * o + 4 * hq;
      if (it.partial) {
        *reinterpret_cast<f32x4*>(p.part_o + (pr + ro.r) * C::kDv + d) = x;
      } else {
        const bf16x4 o4 = {(bf16)x[0], (bf16)x[1], (bf16)x[2], (bf16)x[3]};
        *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(p.out) + b * p.o_sb + ro.t * p.o_ss + ro.h * p.o_sh + d) = o4;
      }
    }
  }
}

// ---- joining the slots of a sequence -------------------------------------------
// WPR waves a row; LPR lanes hold the row (4 dims each), 64 / LPR slots at a time
// and wave.  A slot in which the row sees nothing has LSE -inf.
template <typename T, int LPR, int WPR>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void tree_combine_kernel(TreeParams p) {
  constexpr int RPB = WPR > 1 ? 1 : 4;  // rows a workgroup
  __shared__ f32x4 s_x[WPR > 1 ? WPR - 1 : 1][LPR];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % WPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + wave / WPR, per = (int64_t)p.T * p.Hq;
  if (row >= p.B * per) return;
  const int b = (int)(row / per), r = (int)(row % per), h = r % p.Hq, t = r / p.Hq;
  const int first = p.seq_slots[2 * b], ns = p.seq_slots[2 * b + 1];
  if (ns <= 1) return;
  const float* pl = p.part_lse + first * per + r;
  const float* po = p.part_o + (first * per + r) * p.Dv;
  const bool live = t < seq_lens(p, b).nodes;
  float m = kNegInf, nan = 0.f;
  for (int i = lane; i < ns; i += 64) {
    const float x = pl[i * per];
    nan += x != x ? x : 0.f;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  const float moff = m == kNegInf ? 0.f : m;
  float l = 0.f;
  for (int i = lane; i < ns; i += 64) l += exp2f(pl[i * per] - moff);
  l = wave_sum(l + nan);
  float lse;
  const float f = finish_row(p, h, live, m, l, lse);
  if (part == 0 && lane == 0) p.lse[b * p.l_sb + t * p.l_ss + h * p.l_sh] = lse;
  T* o = reinterpret_cast<T*>(p.out) + b * p.o_sb + t * p.o_ss + h * p.o_sh;
  constexpr int NP = 64 / LPR * WPR;  // slots at a time
  const int sub = lane / LPR;
  for (int d0 = 0; d0 < p.Dv; d0 += 4 * LPR) {
    const int d = d0 + 4 * (lane % LPR);
    f32x4 x = {};
    if (f != 0.f) {
#pragma unroll 4
      for (int i = part * (64 / LPR) + sub; i < ns; i += NP) {
        const float e = exp2f(pl[i * per] - moff);
        f32x4 v = {};
        const float* at = po + i * per * p.Dv + d;
        if (p.Dv % 4 == 0) {
          if (d < p.Dv) v = *reinterpret_cast<const f32x4*>(at);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = d + k < p.Dv ? at[k] : 0.f;
        }
        x += v * e;
      }
    }
#pragma unroll
    for (int s = LPR; s < 64; s <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] += __shfl_xor(x[k], s, 64);
    if constexpr (WPR > 1) {  // (one row a workgroup: all of it comes here)
      if (part > 0 && sub == 0) s_x[part - 1][lane] = x;
      __syncthreads();
      if (part == 0 && sub == 0)
#pragma unroll
        for (int w = 0; w < WPR - 1; ++w) x += s_x[w][lane];
      __syncthreads();
    }
    if (part == 0 && sub == 0)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < p.Dv) o[d + k] = from_f32<T>(f == 0.f ? 0.f : x[k] * f);
  }
}

template <typename T, int WPR>
void launch_combine(const TreeParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.B * p.T * p.Hq;
  const unsigned grid = (unsigned)(WPR > 1 ? rows : (rows + 3) / 4), threads = WPR > 1 ? 64 * WPR : 256;
  if (p.Dv <= 64) tree_combine_kernel<T, 16, WPR><<<grid, threads, 0, s>>>(p);
  else if (p.Dv <= 128) tree_combine_kernel<T, 32, WPR><<<grid, threads, 0, s>>>(p);
  else tree_combine_kernel<T, 64, WPR><<<grid, threads, 0, s>>>(p);
}
template <typename T>
void launch_combine(const TreeParams& p, hipStream_t s) {
  // Many slots of few rows are joined by eight waves a row (d = 128, 256 slots of
  // 256 rows: 13 us, 45 by one wave; 64 of 1024: 17 both ways; 32 of 2048: 17 and 13).
  if (p.want / p.B >= 32 && (int64_t)p.B * p.T * p.Hq <= 1024) launch_combine<T, 8>(p, s);
  else launch_combine<T, 1>(p, s);
}

// Kernels by query rows per (sequence, kv head): rows a workgroup, tile keys, threads.
enum { kGeneric = 0, kRows16, kRows32, kRows64, kRows128, kRows256, kMla };
struct KernelShape {
  int rows, tile, threads;
};
constexpr KernelShape kShapes[] = {{kGR, kGK, 256}, {16, 128, 256}, {32, 128, 256}, {64, 128, 256},
                                   {128, 64, 512},  {256, 32, 512}, {64, 64, 512}};
constexpr int kWorkgroups = 256;  // key ranges are cut until about so many workgroups (one a CU) are in flight

template <int D, int NG, int WR, int WK, int NS>
void launch_pipe(const TreeParams& p, unsigned grid, hipStream_t s) {
  // (a page's byte offsets fit the loads' 32 bits)
  const int64_t row = 2 * (p.k_ss > p.v_ss ? p.k_ss : p.v_ss);
  if (p.page_shift >= 5 && p.k_ss > 0 && p.v_ss > 0 && row < ((int64_t)1 << 25))
    tree_pipe_kernel<D, NG, WR, WK, NS, true><<<grid, 64 * WR * WK, 0, s>>>(p);
  else
    tree_pipe_kernel<D, NG, WR, WK, NS, false><<<grid, 64 * WR * WK, 0, s>>>(p);
}

template <int D>
void launch_mfma(const TreeParams& p, int kernel, unsigned grid, hipStream_t s) {
  switch (kernel) {
    case kRows16: tree_mfma_kernel<D, 1><<<grid, 256, 0, s>>>(p); break;
    case kRows32: tree_mfma_kernel<D, 2><<<grid, 256, 0, s>>>(p); break;
    case kRows64: tree_mfma_kernel<D, 4><<<grid, 256, 0, s>>>(p); break;
    case kRows128: launch_pipe<D, 2, 4, 2, 4>(p, grid, s); break;
    default: launch_pipe<D, 2, 8, 1, 5>(p, grid, s);
  }
}

}  // namespace

TreePlan tree_plan(const TreeParams& p, int dtype, bool vec) {
  TreePlan pl{};
  const int64_t R = (int64_t)p.T * p.G;
  // Few keys and heads: fewer rows a workgroup give more workgroups, whose key
  // rows meet in the L2 (kernel and join, 1 sequence, d = 128, us by rows a workgroup;
  // 128 query rows: 2K keys 17 with 16, 19 with 32, 23 with 128; 32K: 28, 26, 33; 1024
  // query rows: 4K 45 with 16, 28 with 32, 38 with 256; 16K 111, 49, 46).  By the
  // table's width, the lengths being on the device: 128 rows on 2K keys of a table of
  // 128K take 20 us a call for 18.  fit: workgroups of the shortest ranges, 256 keys.
  auto fit = [&](int rows) { return (int64_t)p.B * p.Hkv * ((R + rows - 1) / rows) * (((int64_t)p.cap + 255) / 256); };
  if (dtype == SFA_DTYPE_BF16 && vec && p.Dqk == p.Dv && (p.Dqk == 64 || p.Dqk == 128))
    pl.kernel = R <= 16 || fit(16) <= 2 * kWorkgroups ? kRows16 : R <= 32 || fit(32) <= 5 * kWorkgroups ? kRows32
              : R <= 64 ? kRows64 : R <= 128 ? kRows128 : kRows256;
  if (dtype == SFA_DTYPE_BF16 && vec && p.Dqk == 576 && p.Dv == 512 && p.v == p.k && p.v_sb == p.k_sb && p.v_ss == p.k_ss &&
      p.v_sh == p.k_sh)
    pl.kernel = kMla;
  pl.rows = kShapes[pl.kernel].rows;
  const int64_t nrb = (R + pl.rows - 1) / pl.rows, min_len = 2 * kShapes[pl.kernel].tile;
  // (the generic kernel's workgroups are four to a CU)
  int64_t want = (pl.kernel == kGeneric ? 4 : 1) * kWorkgroups / (p.Hkv * nrb);
  const int64_t most = ((int64_t)p.cap + min_len - 1) / min_len * p.B;
  if (want > most) want = most;
  pl.want = want > p.B ? (int)want : 0;
  pl.slots = p.B + pl.want;
  // (whole eights of items: the row blocks of one meet in the L2 of one XCD)
  if (nrb > 1 && (int64_t)pl.slots * p.Hkv > 4)
    while (pl.slots * p.Hkv % 8 != 0) ++pl.slots;
  pl.wgs = (int64_t)pl.slots * p.Hkv * nrb;
  pl.threads = kShapes[pl.kernel].threads;
  if (pl.want > 0) {
    const size_t rows = (size_t)pl.slots * p.T * p.Hq;
    pl.part_o_bytes = (rows * p.Dv * sizeof(float) + 255) / 256 * 256;
    pl.part_lse_bytes = (rows * sizeof(float) + 255) / 256 * 256;
    pl.seq_bytes = (size_t)2 * p.B * sizeof(int32_t);
  }
  return pl;
}

hipError_t launch_tree(const TreeParams& p0, const TreePlan& pl, int dtype, hipStream_t s) {
  TreeParams p = p0;
  p.want = pl.want;
  p.tile = kShapes[pl.kernel].tile;
  p.nrb = (p.T * p.G + pl.rows - 1) / pl.rows;
  const unsigned grid = (unsigned)pl.wgs;
  if (pl.kernel == kMla) {
    // (row offsets of a tile fit the loads' 32 bits)
    if (p.page_shift >= 6 && p.k_ss > 0 && p.k_ss < ((int64_t)1 << 24)) tree_mla_kernel<true><<<grid, 512, 0, s>>>(p);
    else tree_mla_kernel<false><<<grid, 512, 0, s>>>(p);
  } else if (pl.kernel != kGeneric) {
    if (p.Dqk == 64) launch_mfma<64>(p, pl.kernel, grid, s);
    else launch_mfma<128>(p, pl.kernel, grid, s);
  } else if (dtype == SFA_DTYPE_F32) {
    tree_generic_kernel<float><<<grid, 256, 0, s>>>(p);
  } else {
    tree_generic_kernel<bf16><<<grid, 256, 0, s>>>(p);
  }
  if (pl.want > 0) {
    if (dtype == SFA_DTYPE_F32) launch_combine<float>(p, s);
    else launch_combine<bf16>(p, s);
  }
  return hipGetLastError();
}

}  // namespace sfa

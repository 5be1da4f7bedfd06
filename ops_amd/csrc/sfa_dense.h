// Dense attention (no index rows): a chunk of new tokens over a paged cache, or
// a whole sequence, both through an optional window.  Shared by its kernels
// (sfa_dense_*.hip).
//
// Token t < n_b of sequence b stands at row pos = ctx_b + t and sees the rows j <=
// pos with j < first or pos - j < window.  The query rows of a (sequence, kv head)
// are r = t G + h, h < G = Hq / Hkv: its keys serve all G heads.
#pragma once

#include "sfa_lds.h"
#include "sfa_mfma.h"
#include "sfa_ops.h"

namespace sfa {

// Base-2 log-sum-exp of 2^m2 l (the logarithm of l's mantissa: its own whole
// part would round the sum once more), and the natural one.
__device__ __forceinline__ float dense_lse2(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return m2 + ((float)e + log2f(f));
}
__device__ __forceinline__ float dense_lse(float m2, float l) {
  int e;
  const float f = frexpf(l, &e);
  return fmaf(m2, kLn2, fmaf((float)e, kLn2, logf(f)));
}

struct DenseSeq {
  int ctx, n;  // rows before the first token, tokens
};
// A token past the table sees what its window leaves of it, so there only ctx - window counts:
// what a window of more than 2^30 has over that (p.over; without a window: more than any
// context) is taken off the context, down to the table's end, and from cap + 2^30 on no window
// reaches a row (p.cap <= 2^29).  Positions so stay below 2^31 - 1 (S <= 2^29).
constexpr int kFarCtx = (1 << 30) + (1 << 29) - 1;
__device__ __forceinline__ DenseSeq dense_seq(const DenseParams& p, int b) {
  DenseSeq s;
  s.ctx = 0;
  if (p.ctx_lens != nullptr) {
    const int c = max(p.ctx_lens[b], 0);
    s.ctx = max(min(c, p.cap), min(c - p.over, kFarCtx));
  }
  s.n = p.lens != nullptr ? min(max(p.lens[b], 0), p.S) : p.S;
  return s;
}

__device__ __forceinline__ bool dense_seen(const DenseParams& p, int j, int pos) {
  return j <= pos && (j < p.first || pos - j < p.window);
}

// The key tiles of 2^shift keys that some row of a block sees: the first ones,
// then those of the window; tile(v) is the v-th.
struct KeyTiles {
  int head, from, n;
  __device__ __forceinline__ int tile(int v) const { return v < head ? v : v - head + from; }
};
__device__ __forceinline__ KeyTiles key_tiles(const DenseParams& p, const DenseSeq& s, int row0, int rows, int shift) {
  KeyTiles k{0, 0, 0};
  const int t0 = row0 / p.G, t1 = min((row0 + rows - 1) / p.G, s.n - 1);
  if (t0 > t1) return k;
  const int hi = min(s.ctx + t1 + 1, p.cap), lo = max(0, s.ctx + t0 - p.window + 1), one = (1 << shift) - 1;
  const int end = (hi + one) >> shift;
  k.head = lo > 0 ? min((min(p.first, hi) + one) >> shift, end) : 0;
  k.from = max(min(lo >> shift, end), k.head);  // (lo: past all rows, where a context is past the table)
  k.n = k.head + max(end - k.from, 0);
  return k;
}

// Element offset of key j of sequence b, or -1: rows of unmapped pages and
// (contiguous) of none.
__device__ __forceinline__ int64_t dense_row(const DenseParams& p, int b, int j, int64_t sb, int64_t ss) {
  if (j >= p.cap) return -1;
  if (p.block_table == nullptr) return b * sb + j * ss;
  const int pg = p.block_table[b * p.bt_sb + (j >> p.page_shift)];
  if (pg < 0 || pg >= p.num_pages) return -1;
  return (int64_t)pg * sb + (int64_t)(j & ((1 << p.page_shift) - 1)) * ss;
}

// ---- key ranges of a launch ("slots") ---------------------------------------------
// A unit is a (sequence, row block).  p.fit workgroups of a kv head run at once.  With
// want > 0 (few units) the units' tiles are cut into ranges of up to one length, found
// on the device as the lengths are there: the shortest that gives p.fit ranges or
// fewer, or, where that leaves less work on the longest path, `want`, twice as many.  To
// write partial results and join them takes the time of p.join tiles.
// (Each unit has one at least.)
struct DenseSlot {
  int unit;       // or -1: none
  int v0, v1;     // its tiles, as KeyTiles counts them
  int first, n;   // the unit's first slot and how many it has
};
__device__ __forceinline__ int dense_lanes_sum(int x) {
  x += __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true);  // row_ror:8
  x += __builtin_amdgcn_mov_dpp(x, 0x124, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x122, 0xf, 0xf, true);
  x += __builtin_amdgcn_mov_dpp(x, 0x121, 0xf, 0xf, true);
  const auto a = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
  x = (int)(a[0] + a[1]);
  const auto c = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
  return (int)(c[0] + c[1]);
}
__device__ __forceinline__ int unit_tiles(const DenseParams& p, int u) {
  const int b = u / p.nrb, rb = u - b * p.nrb;
  return key_tiles(p, dense_seq(p, b), rb * p.rows, p.rows, p.tile_shift).n;
}
__device__ __forceinline__ DenseSlot dense_slot(const DenseParams& p, int slot) {
  const int units = p.B * p.nrb;
  if (p.want == 0) {
    if (slot >= units) return DenseSlot{-1, 0, 0, 0, 0};
    return DenseSlot{slot, 0, unit_tiles(p, slot), slot, 1};
  }
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int u) { return u < units ? unit_tiles(p, u) : 0; };
  int tiles[kDenseUnits / 64], sum = 0, most = 0;
#pragma unroll
  for (int i = 0; i < kDenseUnits / 64; ++i) {
    tiles[i] = 64 * i < units ? tiles_of(64 * i + lane) : 0;
    sum += tiles[i];
    most = max(most, tiles[i]);
  }
  sum = dense_lanes_sum(sum);
  most = wave_max_int(most);
  auto ranges = [&](int len) {  // of up to len tiles
    int n = 0;
#pragma unroll
    for (int i = 0; i < kDenseUnits / 64; ++i)
      if (64 * i < units) n += 64 * i + lane < units ? max(1, (tiles[i] + len - 1) / len) : 0;
    return dense_lanes_sum(n);
  };
  auto shortest = [&](int slots) {  // (a few steps come within a tile of the best)
    int len = max(p.min_len, (sum + slots - 1) / slots);
    for (int i = 0; i < 6 && len < most; ++i) {
      const int n = ranges(len);
      if (n <= slots) return len;
      len = max(len + 1, (int)((int64_t)len * n / slots));
    }
    return max(len, most);
  };
  int len = most;
  if (units <= p.fit) {
    const int l1 = shortest(p.fit);
    if (l1 + p.join < most) len = l1;
  }
  if (len > p.min_len) {
    const int l2 = shortest(p.want);
    // (rounds of p.fit ranges; more of them cost a tenth or so)
    const int rounds = units <= p.fit ? 1 : (units + p.fit - 1) / p.fit, r2 = (p.want + p.fit - 1) / p.fit;
    if (l2 < most && 11 * r2 * l2 + (len == most ? 10 * p.join : 0) < 10 * rounds * len) len = l2;
  }
  len = max(len, 1);
  int before = 0;
  for (int u0 = 0; u0 < units; u0 += 64) {
    const int u = u0 + lane;
    int t = tiles[0];
#pragma unroll
    for (int i = 1; i < kDenseUnits / 64; ++i) t = u0 == 64 * i ? tiles[i] : t;
    const int n = u < units ? max(1, (t + len - 1) / len) : 0;
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
      DenseSlot s;
      s.unit = u0 + w;
      s.first = __builtin_amdgcn_readlane(first, w);
      s.n = __builtin_amdgcn_readlane(n, w);
      const int mine = __builtin_amdgcn_readlane(t, w);
      // (even ranges: the unit's tiles over its own number of slots)
      const int i = slot - s.first;
      s.v0 = (int)((int64_t)mine * i / s.n);
      s.v1 = (int)((int64_t)mine * (i + 1) / s.n);
      return s;
    }
    before += __builtin_amdgcn_readlane(incl, 63);
  }
  return DenseSlot{-1, 0, 0, 0, 0};
}

// A workgroup's share of a launch.
struct DenseItem {
  int b, g, rb, row0;
  DenseSeq s;
  KeyTiles tiles;
  int v0, v1;
  int64_t part;   // row of the partial results of the block's first row
  bool partial;
};
__device__ __forceinline__ bool dense_item(const DenseParams& p, int slot, int g, DenseItem& it) {
  const DenseSlot sl = dense_slot(p, slot);
  if (sl.unit < 0) return false;
  const int unit = __builtin_amdgcn_readfirstlane(sl.unit);
  it.b = unit / p.nrb;
  it.rb = unit - it.b * p.nrb;
  it.g = g;
  it.row0 = it.rb * p.rows;
  it.s = dense_seq(p, it.b);
  it.tiles = key_tiles(p, it.s, it.row0, p.rows, p.tile_shift);
  it.v0 = __builtin_amdgcn_readfirstlane(sl.v0);
  it.v1 = __builtin_amdgcn_readfirstlane(sl.v1);
  it.part = ((int64_t)slot * p.Hkv + g) * p.rows;
  it.partial = sl.n > 1;
  if (p.want > 0 && slot == sl.first && g == 0 && threadIdx.x == 0) {
    p.unit_slots[2 * unit] = sl.first;
    p.unit_slots[2 * unit + 1] = sl.n;
  }
  return true;
}

// The factor and LSE of a finished row of head h with maximum m (base 2) and sum l.
__device__ __forceinline__ float dense_finish(const DenseParams& p, int h, bool live, float m, float l, float& lse) {
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
  lse = x > 0.f ? dense_lse(mm, x) : x == 0.f ? kNegInf : x;
  return x > 0.f ? f / x : x == 0.f ? 0.f : x;
}
// ... of a partial one: its own sum, base-2 LSE
__device__ __forceinline__ float dense_part(float m, float l, float& lse2) {
  lse2 = l > 0.f ? dense_lse2(m, l) : l == 0.f ? kNegInf : l;
  return l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
}

}  // namespace sfa

// Key tiles of the bf16 dense attention kernels in LDS: 64 rows of K and of V, from
// contiguous tensors, pages, or pages of e4m3 rows.
#pragma once

#include "sfa_dense.h"

namespace sfa {

constexpr int kWideKeys = 64;

// A tile is written 1024 bytes (4 rows of 128 dims, 8 of 64) at a time, with 16 bytes
// between, and chunk c (16 bytes) of row r goes to place c ^ at(r) of its row.  So
// lanes that read one chunk of 16 consecutive rows (K) meet all 16 bank groups, as
// do those that read four consecutive rows of an aligned group of four chunks (V,
// transposed), and rows 8 further lie at a constant distance.
template <int D>
struct Tile {
  static constexpr int CH = D / 8, RPI = 64 / CH, GROUP = 65;  // chunks a row, rows a group, chunks from group to group
  static constexpr int SLOTS = kWideKeys / RPI * GROUP;
  static __device__ __forceinline__ int at(int r) {
    if constexpr (D == 128) return (r & 3) << 2;
    else return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1);
  }
  static constexpr int rows(int n) { return n / RPI * GROUP * 16; }  // bytes to a row n further, n a multiple of 8
  static __device__ __forceinline__ int slot(int r, int c) { return r / RPI * GROUP + r % RPI * CH + (c ^ at(r)); }
};

// Lane l: 16 bytes from base + its offset to dst + 16 l; not seen by the compiler:
// the kernel waits for vmcnt itself.
__device__ __forceinline__ void dense_dma16(const void* lds, uint64_t base, uint32_t off) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(d), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dense_dma16(const void* lds, uint64_t addr) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(d), "v"(addr) : "memory", "m0");
}
// 4 bytes (1 byte, as 4) to dst + 4 l
__device__ __forceinline__ void dense_dma4(const void* lds, uint64_t addr) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" ::"s"(d), "v"(addr) : "memory", "m0");
}
__device__ __forceinline__ void dense_dma1(const void* lds, uint64_t addr) {
  const uint32_t d = (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(lds);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_ubyte %1, off" ::"s"(d), "v"(addr) : "memory", "m0");
}
__device__ __forceinline__ void dense_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Reads at an LDS address and a constant.
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(lds_void*)const_cast<void*>(p); }
__device__ __forceinline__ bf16x8 lds_b128_at(uint32_t a) {
  return *(const __attribute__((address_space(3))) bf16x8*)(uintptr_t)a;
}
__device__ __forceinline__ bf16x4 lds_tr16_at(uint32_t a) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)a);
}

// Whether the 2^shift rows of a tile have one base and stride (contiguous tensors, pages of
// so many rows or more), with 32-bit offsets.
inline bool dense_one_base(const DenseParams& p, int esize, int shift) {
  const int64_t row = esize * (p.k_ss > p.v_ss ? p.k_ss : p.v_ss);
  return (p.block_table == nullptr || p.page_shift >= shift) && p.k_ss >= 0 && p.v_ss >= 0 && row < (int64_t)1 << 25;
}

// Tiles of 64 keys for NW waves.  at(i): the first key of the workgroup's i-th tile.
// load(i, ..): that tile's rows go to LDS (e4m3: to registers, and from there by
// store()); returns the rows that are there.  on = false: zeros, so that the number
// of loads in flight does not depend on the range.  Calls of load come in order of i.
// Page ids are held ahead of use, as a wait for one is a wait for every load before
// it: ONE: those of 64 tiles by lane; else those of the next tile's rows.
template <int D, int NW, bool FP8, bool ONE>
struct TileSource {
  static constexpr int KT = kWideKeys, CH = D / 8, RPI = 64 / CH, NI = KT / RPI / NW;
  static_assert(NI >= 1 && KT / 8 == NW, "whole load instructions and eight rows a wave");
  uint64_t kbase, vbase;
  int64_t kpage, vpage, krow, vrow;
  const int32_t* trow;
  KeyTiles tiles;
  int v0, n;
  int cap, page_shift, num_pages, wave, lane;
  int pg, pgr;  // page ids: of tiles by lane, or of the next tile's key `lane`; of its row that the lane loads (e4m3)

  __device__ __forceinline__ TileSource(const DenseParams& p, const DenseItem& it, int wave_, int lane_)
      : tiles(it.tiles), v0(it.v0), n(it.v1 - it.v0), cap(p.cap), page_shift(p.page_shift), num_pages(p.num_pages), wave(wave_),
        lane(lane_) {
    const int64_t e = FP8 ? 1 : 2;
    kbase = (uint64_t)(uintptr_t)p.k + (uint64_t)(e * it.g * p.k_sh);
    vbase = (uint64_t)(uintptr_t)p.v + (uint64_t)(e * it.g * p.v_sh);
    kpage = e * p.k_sb;
    vpage = e * p.v_sb;
    krow = e * p.k_ss;
    vrow = e * p.v_ss;
    trow = nullptr;
    if (p.block_table != nullptr) {
      trow = p.block_table + it.b * p.bt_sb;
    } else {  // one page of all rows
      kbase += (uint64_t)(it.b * kpage);
      vbase += (uint64_t)(it.b * vpage);
      page_shift = 30;
      num_pages = 1;
    }
    if constexpr (FP8) {
      ksc = p.ks + it.g * p.ks_sh;
      vsc = p.vs + it.g * p.vs_sh;
      ks_sb = p.ks_sb; ks_ss = p.ks_ss; vs_sb = p.vs_sb; vs_ss = p.vs_ss;
    }
    ids(0);
  }
  // (past the range: its last tile)
  __device__ __forceinline__ int at(int i) const { return tiles.tile(v0 + max(min(i, n - 1), 0)) * KT; }
  __device__ __forceinline__ int entry(int j) const { return trow == nullptr ? 0 : trow[min(j, cap - 1) >> page_shift]; }
  __device__ __forceinline__ void ids(int i) {
    if constexpr (ONE) {
      pg = entry(at(i + lane));
    } else {
      pg = entry(at(i) + lane);
      if constexpr (FP8) pgr = entry(at(i) + wave * 8 + (lane >> 3));
    }
  }
  // at most N tiles of this wave in flight
  template <int N>
  __device__ __forceinline__ void wait() const {
    if constexpr (!FP8) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N * 2 * NI) : "memory");
  }

  __device__ __forceinline__ uint64_t load(int i, u32x4* kt, u32x4* vt) {
    const bool on = i < n;
    const int j0 = at(i), in_page = (1 << page_shift) - 1;
    const uint64_t zero = (uint64_t)(uintptr_t)kZeroRow;
    uint64_t mask;
    if constexpr (ONE) {
      const int in = j0 & in_page, rows = cap - j0, pgu = __builtin_amdgcn_readlane(pg, i & 63);
      const bool ok = on && pgu >= 0 && pgu < num_pages;
      const uint64_t kb = ok ? kbase + (uint64_t)(pgu * kpage + in * krow) : zero;
      const uint64_t vb = ok ? vbase + (uint64_t)(pgu * vpage + in * vrow) : zero;
      if constexpr (FP8) {
        const int row = wave * 8 + (lane >> 3);
        const bool there = ok && row < rows;
        const uint32_t piece = (uint32_t)((lane & 7) * (D / 8));
        raw(kb + (there ? (uint32_t)(row * (int)krow) : 0u) + piece, vb + (there ? (uint32_t)(row * (int)vrow) : 0u) + piece,
            there, pgu, in + row);
      } else {
        // (lane constants are formed per tile: held across the loop they spill)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int sub = ln / CH;
        const uint32_t c = 16u * (uint32_t)((ln % CH) ^ Tile<D>::at(sub));
        const uint32_t ko = (uint32_t)(sub * (int)krow) + c, vo = (uint32_t)(sub * (int)vrow) + c;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const int q = wave * NI + k, left = ok ? rows - q * RPI : 0;
          // (rows past the last one read some row's chunks: no row of the result sees them)
          const bool there = sub < left;
          const uint32_t step = left > 0 ? (uint32_t)(q * RPI) : 0;  // (times a stride: below 2^31)
          dense_dma16(kt + q * Tile<D>::GROUP, kb + step * (uint32_t)krow, there ? ko : c);
          dense_dma16(vt + q * Tile<D>::GROUP, vb + step * (uint32_t)vrow, there ? vo : c);
        }
      }
      mask = !ok ? 0 : rows >= KT ? ~0ull : (1ull << rows) - 1;
      if (((i + 1) & 63) == 0) ids(i + 1);
    } else {
      const int j = j0 + lane;
      const bool ok = on && j < cap && pg >= 0 && pg < num_pages;
      if constexpr (FP8) {
        const int jr = j0 + wave * 8 + (lane >> 3), in = jr & in_page;
        const bool there = on && jr < cap && pgr >= 0 && pgr < num_pages;
        const uint64_t piece = (uint64_t)((lane & 7) * (D / 8));
        raw((there ? kbase + (uint64_t)(pgr * kpage + in * krow) : zero) + piece,
            (there ? vbase + (uint64_t)(pgr * vpage + in * vrow) : zero) + piece, there, pgr, in);
      } else {
        const uint64_t ka = ok ? kbase + (uint64_t)(pg * kpage + (j & in_page) * krow) : zero;
        const uint64_t va = ok ? vbase + (uint64_t)(pg * vpage + (j & in_page) * vrow) : zero;
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const int q = wave * NI + k, row = q * RPI + lane / CH;
          const uint64_t c = (uint64_t)(16 * ((lane % CH) ^ Tile<D>::at(row)));
          dense_dma16(kt + q * Tile<D>::GROUP, from(ka, row) + c);
          dense_dma16(vt + q * Tile<D>::GROUP, from(va, row) + c);
        }
      }
      mask = __ballot(ok);
      ids(i + 1);
    }
    return mask;
  }
  __device__ __forceinline__ void store(u32x4* kt, u32x4* vt) const {
    if constexpr (FP8) {
      const int row = wave * 8 + (lane >> 3), c0 = (lane & 7) * (D / 64);
      const float sk = scale_of((uint8_t)kexp), sv = scale_of((uint8_t)vexp);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        kt[Tile<D>::slot(row, c0 + i)] = chunk(kraw, i, sk);
        vt[Tile<D>::slot(row, c0 + i)] = chunk(vraw, i, sv);
      }
    }
  }

  // dims d .. d + 3 of the V row of key j, which is there
  __device__ __forceinline__ void value4(int j, int d, float (&v)[4]) const {
    const int id = entry(j), in = j & ((1 << page_shift) - 1);
    const uint64_t a = vbase + (uint64_t)(id * vpage + in * vrow);
    if constexpr (FP8) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(a + d);
      const float s = scale_of(vsc[id * vs_sb + in * vs_ss]);
      v[0] = __builtin_amdgcn_cvt_f32_fp8((int)x, 0) * s;
      v[1] = __builtin_amdgcn_cvt_f32_fp8((int)x, 1) * s;
      v[2] = __builtin_amdgcn_cvt_f32_fp8((int)x, 2) * s;
      v[3] = __builtin_amdgcn_cvt_f32_fp8((int)x, 3) * s;
    } else {
      const bf16x4 x = *reinterpret_cast<const bf16x4*>(a + 2 * d);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = (float)x[q];
    }
  }

 private:
  typedef typename std::conditional<D == 128, u32x4, u32x2>::type raw_t;
  const uint8_t *ksc, *vsc;
  int64_t ks_sb, ks_ss, vs_sb, vs_ss;
  raw_t kraw, vraw;
  int kexp, vexp;
  // the lane's bytes of row `in` of page id, and their exponents
  __device__ __forceinline__ void raw(uint64_t ka, uint64_t va, bool there, int id, int in) {
    kraw = *reinterpret_cast<const raw_t*>(ka);
    vraw = *reinterpret_cast<const raw_t*>(va);
    kexp = there ? ksc[id * ks_sb + in * ks_ss] : 127;
    vexp = there ? vsc[id * vs_sb + in * vs_ss] : 127;
  }
  static __device__ __forceinline__ uint64_t from(uint64_t a, int lane) {
    return ((uint64_t)(uint32_t)__shfl((int)(a >> 32), lane, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)a, lane, 64);
  }
  // bytes 8 i .. 8 i + 7 as bf16 times a power of two (exact)
  static __device__ __forceinline__ u32x4 chunk(const raw_t& x, int i, float s) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      r[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + w], s, false));
      r[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + w], s, true));
    }
    return r;
  }
};

// The rows of the tile at key j0 that a token at pos (-1: none) sees, as bits.
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1; }
__device__ __forceinline__ uint64_t seen_of(const DenseParams& p, int pos, int j0) {
  return low_bits(pos + 1 - j0) & (~low_bits(pos + 1 - p.window - j0) | low_bits(p.first - j0));
}

// Infinities and NaN of a V tile whose rows not every query row sees: noted as bits
// (of s_bad, 0 before) and cleared in LDS, as 0 times them would reach the rows that
// do not see them; add_bad adds them to those that do.
__device__ __forceinline__ uint32_t bad16(uint32_t w) {  // halves of w that are no numbers: their masks
  return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
template <int D, int NW>
__device__ __forceinline__ uint64_t clear_bad(u32x4* vt, unsigned long long* s_bad, int wave, int lane) {
  constexpr int CH = D / 8, PER = kWideKeys * CH / 64 / NW;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int q = wave * PER + i, at = q * Tile<D>::GROUP + lane;
    const u32x4 w = vt[at];
    u32x4 m;
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = bad16(w[e]);
    if ((m[0] | m[1] | m[2] | m[3]) != 0) {
      vt[at] = w & ~m;
      atomicOr(s_bad, 1ull << (q * Tile<D>::RPI + lane / CH));
    }
  }
  dense_barrier();
  return *s_bad;
}

// Elements of 32 rows from `row` on that are no numbers, cleared, and a barrier.  The caller sees
// to it that all waves have read what they need of them as they were.
template <int D, int NW>
__device__ __forceinline__ void clear_rows(u32x4* t, int row, int wave, int lane) {
  constexpr int N = 32 / Tile<D>::RPI;  // groups of 64 chunks
#pragma unroll
  for (int i = 0; i < (N + NW - 1) / NW; ++i) {
    const int q = i * NW + wave;
    if (N % NW != 0 && q >= N) break;
    const int at = (row / Tile<D>::RPI + q) * Tile<D>::GROUP + lane;
    const u32x4 w = t[at];
    u32x4 m;
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = bad16(w[e]);
    if ((m[0] | m[1] | m[2] | m[3]) != 0) t[at] = w & ~m;
  }
  dense_barrier();
}

// A wave's results go to memory through LDS (its own part of it), whole rows at a time: as
// the lanes hold them a store would reach 32 rows with 16 bytes each (35 us of a 216 us
// forward pass, 8192 tokens, 32 heads).  Rows of CH 16-byte chunks, chunk c of row r at
// c ^ r % CH.
template <int CH>
struct RowsOut {
  u32x4* buf;
  __device__ __forceinline__ u32x4* slot(int row, int c) const { return buf + row * CH + (c ^ (row & (CH - 1))); }
  __device__ __forceinline__ void put(int row, int d, bf16x4 x) const {  // dims d .. d + 3
    *reinterpret_cast<bf16x4*>(reinterpret_cast<char*>(slot(row, d >> 3)) + 8 * ((d >> 2) & 1)) = x;
  }
  __device__ __forceinline__ void put(int row, int d, f32x4 x) const { *reinterpret_cast<f32x4*>(slot(row, d >> 2)) = x; }
  // its 32 rows to where lane r % 32 says (0: nowhere)
  __device__ __forceinline__ void store(uint64_t at, int lane) const {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int k = 0; k < 32 * CH / 64; ++k) {
      const int i = k * 64 + lane, row = i / CH;
      const uint64_t a = ((uint64_t)(uint32_t)__shfl((int)(at >> 32), row, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)at, row, 64);
      const u32x4 x = *slot(row, i % CH);
      if (a != 0) *reinterpret_cast<u32x4*>(a + (uint64_t)(16 * (i % CH))) = x;
    }
  }
};

// The kernel's arguments, loaded where they are used from here on: those that only the results
// need would be held across the loop (scalar registers spill to lanes of vector ones).  1 to 3% in
// the kernels that use it; the one over latent rows is 3% faster without.
__device__ __forceinline__ const DenseParams& late_params() {
  typedef const __attribute__((address_space(4))) DenseParams* args_t;
  uint64_t a = (uint64_t)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return *(const DenseParams*)(args_t)a;
}

// Where the workgroup's share of a launch is: the row blocks of a (sequence, kv head)
// on one XCD (workgroup i is on XCD i % 8), whose L2 their keys then stay in; the
// longest ones, which are a sequence's last, first.
__device__ __forceinline__ void dense_place(const DenseParams& p, int& slot, int& g) {
  int w = blockIdx.x;
  if (p.want > 0) {
    g = w % p.Hkv;
    slot = w / p.Hkv;
    return;
  }
  const int groups = p.B * p.Hkv, x = w & 7;
  int group, rb;
  if (groups % 8 == 0) {
    w >>= 3;
    group = x + 8 * (w / p.nrb);
    rb = w % p.nrb;
  } else if (8 % groups == 0 && p.nrb % (8 / groups) == 0) {  // 1, 2 or 4: each on several
    group = x % groups;
    rb = (w >> 3) * (8 / groups) + x / groups;
  } else {
    group = w % groups;
    rb = w / groups;
  }
  g = group % p.Hkv;
  slot = group / p.Hkv * p.nrb + (p.nrb - 1 - rb);
}

}  // namespace sfa

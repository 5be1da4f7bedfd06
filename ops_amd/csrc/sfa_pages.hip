// Pages of a paged cache: copying, forking, freeing, compacting, and the two
// that go with them, mapping pages for rows to come and keeping the accepted
// path of a drafted tree.
//
// State: block_table [B][max_pages] (page of each sequence's i-th run of
// page_size rows, -1: none) and ref_counts [num_pages], the number of table
// entries that map a page; a page is free iff its count is 0, and a page that
// is taken is the lowest free one, so a call's result does not depend on the
// order in which workgroups run.  Everything stays on the device: no count
// comes back to the host, so the calls can be captured.
//
// An operation that has to order its pages runs as a plan by one workgroup
// (prefix sums over the pairs and the counts, 16 counts a thread and step)
// and a kernel that copies.  The copies bound the large calls: 16 bytes a
// lane, a page of every cache split into segments that are taken by
// workgroups independently.  Small calls are bound by launches and by the
// plan's chain of dependent loads.

#include "sfa_ops.h"

namespace sfa {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kCountsPer = 16;     // ref counts per thread and step of a scan
constexpr int kSegBytes = 16384;   // of a page, per workgroup and item
constexpr int kWsHead = 16;

// Workspace: head, then three arrays of num_pages, then two of n.
__device__ __forceinline__ int32_t* ws_pages(const PagesParams& p, int i) { return p.ws + kWsHead + (int64_t)i * p.num_pages; }
__device__ __forceinline__ int32_t* ws_pairs(const PagesParams& p, int i, int n) {
  return p.ws + kWsHead + 3 * (int64_t)p.num_pages + (int64_t)i * n;
}

// Exclusive prefix sum of x over the workgroup; total: the sum.  s: 17 ints.
__device__ __forceinline__ int block_scan(int x, int* s, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int v = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();  // (the last use of s is over)
  if (lane == 63) s[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const int y = s[w];
    if (w < wave) before += y;
    all += y;
  }
  total = all;
  return before + v - x;
}

// 16 counts from refs[i0]; past the end: 1 (in use).
__device__ __forceinline__ void load_counts(const PagesParams& p, int i0, int (&c)[kCountsPer]) {
#pragma unroll
  for (int j = 0; j < kCountsPer; ++j) c[j] = i0 + j < p.num_pages ? p.refs[i0 + j] : 1;
}

// The lowest `want` free pages, ascending, into list; returns how many there are.
__device__ int find_free(const PagesParams& p, int want, int32_t* list, int* s) {
  int found = 0;
  for (int base = 0; base < p.num_pages && found < want; base += kPlanThreads * kCountsPer) {
    const int i0 = base + threadIdx.x * kCountsPer;
    int c[kCountsPer], n = 0, total;
    load_counts(p, i0, c);
#pragma unroll
    for (int j = 0; j < kCountsPer; ++j) n += c[j] == 0;
    int at = found + block_scan(n, s, total);
#pragma unroll
    for (int j = 0; j < kCountsPer; ++j)
      if (c[j] == 0) {
        if (at < want) list[at] = i0 + j;
        ++at;
      }
    found += total;
  }
  __threadfence_block();
  __syncthreads();
  return found < want ? found : want;
}

__device__ __forceinline__ bool page_ok(const PagesParams& p, int pg) { return pg >= 0 && pg < p.num_pages; }

__device__ __forceinline__ int clamp_len(const PagesParams& p, int len) {
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;
  return len < 0 ? 0 : (int64_t)len > cap ? (int)cap : len;
}

// bytes [off, off + n) of page src to page dst, by the whole workgroup.
// U: u32x4 (everything a multiple of 16 bytes) or uint8_t
template <typename U>
__device__ __forceinline__ void copy_span(char* d, const char* s, int64_t n) {
  const int64_t m = n / (int64_t)sizeof(U);
  U* dd = reinterpret_cast<U*>(d);
  const U* ss = reinterpret_cast<const U*>(s);
  int64_t i = threadIdx.x;
  for (; i + 3 * 256 < m; i += 4 * 256) {
    const U a = ss[i], b = ss[i + 256], c = ss[i + 512], e = ss[i + 768];
    dd[i] = a;
    dd[i + 256] = b;
    dd[i + 512] = c;
    dd[i + 768] = e;
  }
  for (; i < m; i += 256) dd[i] = ss[i];
}

// ---- copying ------------------------------------------------------------------
// Pairs take effect as if every source were read before any destination is
// written, as far as that needs no copy aside: a pair is left out if a page is
// outside the pool, if a later pair has its destination, or if its
// destination is the source of another pair.
__global__ __launch_bounds__(256) void copy_check_kernel(PagesParams p, const int32_t* src, const int32_t* dst, int n) {
  __shared__ int s_s[256], s_d[256];
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int a = i < n ? src[i] : -1, b = i < n ? dst[i] : -1;
  bool ok = i < n && page_ok(p, a) && page_ok(p, b) && a != b;
  for (int j0 = 0; j0 < n; j0 += 256) {
    __syncthreads();
    const int j = j0 + threadIdx.x;
    s_s[threadIdx.x] = j < n ? src[j] : -1;
    s_d[threadIdx.x] = j < n ? dst[j] : -1;
    __syncthreads();
    const int m = min(256, n - j0);
    for (int k = 0; k < m; ++k) {
      const bool real = s_s[k] >= 0 && s_s[k] < p.num_pages && s_d[k] >= 0 && s_d[k] < p.num_pages;
      if (real && ((s_d[k] == b && j0 + k > i) || (s_s[k] == b && j0 + k != i))) ok = false;
    }
  }
  if (i < n) ws_pairs(p, 0, n)[i] = ok;
}

template <typename U>
__global__ __launch_bounds__(256) void copy_kernel(PagesParams p, PoolList pools, const int32_t* src,
                                                   const int32_t* dst, int n) {
  const int k = blockIdx.y;
  const int64_t bytes = pools.page_bytes[k];
  const int segs = (int)((bytes + kSegBytes - 1) / kSegBytes);
  const int32_t* ok = ws_pairs(p, 0, n);
  for (int64_t it = blockIdx.x; it < (int64_t)n * segs; it += gridDim.x) {
    const int i = (int)(it / segs);
    if (!ok[i]) continue;
    const int64_t off = (it % segs) * (int64_t)kSegBytes;
    const int64_t len = bytes - off < kSegBytes ? bytes - off : kSegBytes;
    copy_span<U>(pools.base[k] + (int64_t)dst[i] * pools.page_stride[k] + off,
                 pools.base[k] + (int64_t)src[i] * pools.page_stride[k] + off, len);
  }
}

// ---- forking --------------------------------------------------------------------
// Pair i makes row children[i] of the table a fork of row parents[i]: whole
// pages shared, the last page, filled in part, copied to a free page.  Left
// out (ok[i] = 0, nothing written): rows outside the table, a child that is
// its own parent, that an earlier pair has, or that any pair has as parent,
// and pairs that find no free page.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(PagesParams p, const int32_t* parents,
                                                                 const int32_t* children, int n, int32_t* ok) {
  __shared__ int s_scan[kPlanWaves + 1];
  __shared__ int s_owner[kMaxSeqs];  // first pair that has the row as child
  __shared__ uint32_t s_par[kMaxSeqs / 32];
  const int tid = threadIdx.x;
  for (int r = tid; r < p.B; r += kPlanThreads) s_owner[r] = 0x7fffffff;
  for (int r = tid; r < (p.B + 31) / 32; r += kPlanThreads) s_par[r] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    const int a = parents[i], c = children[i];
    if (c >= 0 && c < p.B) atomicMin(&s_owner[c], i);
    if (a >= 0 && a < p.B) atomicOr(&s_par[a >> 5], 1u << (a & 31));
  }
  __syncthreads();
  // ws_pairs 0: the pair's new page (-1: none needed); -2 - rank until the pages are known
  int32_t* fresh = ws_pairs(p, 0, n);
  int want = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    bool valid = false, need = false;
    if (i < n) {
      const int a = parents[i], c = children[i];
      valid = a >= 0 && a < p.B && c >= 0 && c < p.B && s_owner[c] == i && !((s_par[c >> 5] >> (c & 31)) & 1u);
      if (valid) {
        const int len = clamp_len(p, p.kv_lens[a]), full = len >> p.page_shift;
        need = (len & ((1 << p.page_shift) - 1)) != 0 && page_ok(p, p.block_table[a * p.bt_sb + full]);
      }
    }
    int total;
    const int at = want + block_scan(need, s_scan, total);
    if (i < n) {
      ok[i] = valid;
      fresh[i] = need ? -2 - at : -1;
    }
    want += total;
  }
  int32_t* list = ws_pages(p, 0);
  const int found = find_free(p, want < p.num_pages ? want : p.num_pages, list, s_scan);
  for (int i = tid; i < n; i += kPlanThreads) {
    const int f = fresh[i];
    if (f > -2) continue;
    const int at = -2 - f;
    if (at < found) {
      fresh[i] = list[at];
      p.refs[list[at]] = 1;
    } else {
      fresh[i] = -1;
      ok[i] = 0;
    }
  }
}

// blockIdx.y = 0: tables, counts and lengths (first launch only); else pool y - 1
template <typename U>
__global__ __launch_bounds__(256) void fork_kernel(PagesParams p, PoolList pools, const int32_t* parents,
                                                   const int32_t* children, int n, const int32_t* ok, int tables) {
  const int32_t* fresh = ws_pairs(p, 0, n);
  if (blockIdx.y == 0) {
    if (!tables) return;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
      if (!ok[i]) continue;
      const int a = parents[i], c = children[i];
      const int len = clamp_len(p, p.kv_lens[a]), full = len >> p.page_shift, f = fresh[i];
      for (int e = threadIdx.x; e < p.max_pages; e += 256) {
        int pg = -1;
        if (e < full) {
          pg = p.block_table[a * p.bt_sb + e];
          if (page_ok(p, pg)) atomicAdd(&p.refs[pg], 1);
          else pg = -1;
        } else if (e == full) {
          pg = f;
        }
        p.block_table[c * p.bt_sb + e] = pg;
      }
      if (threadIdx.x == 0) p.kv_lens[c] = len;
    }
    return;
  }
  const int k = blockIdx.y - 1;
  const int64_t row = pools.page_bytes[k] >> p.page_shift;
  const int segs = (int)((pools.page_bytes[k] + kSegBytes - 1) / kSegBytes);
  for (int64_t it = blockIdx.x; it < (int64_t)n * segs; it += gridDim.x) {
    const int i = (int)(it / segs);
    if (!ok[i] || fresh[i] < 0) continue;
    const int a = parents[i], len = clamp_len(p, p.kv_lens[a]);
    const int64_t bytes = (len & ((1 << p.page_shift) - 1)) * row, off = (it % segs) * (int64_t)kSegBytes;
    if (off >= bytes) continue;
    const int pg = p.block_table[a * p.bt_sb + (len >> p.page_shift)];
    copy_span<U>(pools.base[k] + (int64_t)fresh[i] * pools.page_stride[k] + off,
                 pools.base[k] + (int64_t)pg * pools.page_stride[k] + off,
                 bytes - off < kSegBytes ? bytes - off : kSegBytes);
  }
}

// ---- freeing ----------------------------------------------------------------------
// The entries of rows[i] past its kept length become -1 and their pages lose
// a reference (an entry is taken once, so a row listed twice loses no more).
__global__ __launch_bounds__(256) void free_kernel(PagesParams p, const int32_t* rows, const int32_t* keep, int n) {
  const int i = blockIdx.y, r = rows[i];
  if (r < 0 || r >= p.B) return;
  int e = blockIdx.x * 256 + threadIdx.x;
  if (keep != nullptr) {
    const int64_t k = keep[i] < 0 ? 0 : keep[i];
    if (e < ((k + (1 << p.page_shift) - 1) >> p.page_shift)) return;
  }
  if (e >= p.max_pages) return;
  int32_t* at = &p.block_table[r * p.bt_sb + e];
  if (*at == -1) return;
  const int pg = atomicExch(at, -1);
  if (!page_ok(p, pg)) return;
  int c = p.refs[pg];
  while (c > 0) {
    const int was = atomicCAS(&p.refs[pg], c, c - 1);
    if (was == c) break;
    c = was;
  }
}

// ---- mapping pages for rows to come -------------------------------------------------
// Sequence b gets pages for rows kv_lens[b] .. new_lens[b] - 1 where it has
// none, all or none of them: in order of b, as long as free pages last (one
// that needs none has what it needs, also behind the last free page).
__global__ __launch_bounds__(kPlanThreads) void extend_kernel(PagesParams p, const int32_t* new_lens, int32_t* ok) {
  __shared__ int s_scan[kPlanWaves + 1];
  __shared__ int s_need[kMaxSeqs];
  const int tid = threadIdx.x, l = tid & 15;
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;
  const int ps1 = (1 << p.page_shift) - 1;
  auto range = [&](int b, int& e0, int& e1) {
    const int64_t want = new_lens[b] < 0 ? 0 : new_lens[b];
    e0 = clamp_len(p, p.kv_lens[b]) >> p.page_shift;
    e1 = want > cap ? -1 : (int)((want + ps1) >> p.page_shift);
    if (want > cap) e0 = 0;
  };
  // (16 lanes a sequence; -1: longer than the table)
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads / 16) {
    const int b = b0 + tid / 16;
    int need = 0, e0 = 0, e1 = 0;
    if (b < p.B) {
      range(b, e0, e1);
      for (int e = e0 + l; e < e1; e += 16) need += !page_ok(p, p.block_table[b * p.bt_sb + e]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) need += __shfl_xor(need, o, 64);
    if (b < p.B && l == 0) s_need[b] = e1 < 0 ? -1 : need;
  }
  __syncthreads();
  int want = 0;  // (at most the table's entries) s_need[b] becomes the rank of b's first page; ok[b]: its count for now
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + tid, need = b < p.B ? s_need[b] : 0;
    int total;
    const int at = block_scan(need > 0 ? need : 0, s_scan, total);
    if (b < p.B) {
      s_need[b] = want + at;
      ok[b] = need;
    }
    want += total;
  }
  int32_t* list = ws_pages(p, 0);
  const int found = find_free(p, want < p.num_pages ? want : p.num_pages, list, s_scan);
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads / 16) {
    const int b = b0 + tid / 16;
    if (b >= p.B) continue;  // (whole groups of 16 lanes)
    const int need = ok[b], first = s_need[b];
    const bool good = need == 0 || (need > 0 && (int64_t)first + need <= found);
    if (good && need > 0) {
      int e0, e1, at = first;
      range(b, e0, e1);
      for (int e = e0; e < e1; e += 16) {
        const bool miss = e + l < e1 && !page_ok(p, p.block_table[b * p.bt_sb + e + l]);
        const uint32_t m = (uint32_t)(__ballot(miss) >> ((tid & 63) & ~15)) & 0xffffu;
        if (miss) {
          const int pg = list[at + __popc(m & ((1u << l) - 1u))];
          p.block_table[b * p.bt_sb + e + l] = pg;
          p.refs[pg] = 1;
        }
        at += __popc(m);
      }
    }
    if (l == 0) s_need[b] = good;
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += kPlanThreads) ok[b] = s_need[b];
}

// ---- compacting -----------------------------------------------------------------------
// With `used` pages in use, those with ids >= used move, in order, to the free
// ids below (sources and destinations are disjoint).  ws_pages 0 / 1: source
// and destination of the k-th move, 2: the move of a page >= used, or -1;
// ws[0]: moves, ws[1]: used.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(PagesParams p, int32_t* used_out) {
  __shared__ int s_scan[kPlanWaves + 1];
  const int tid = threadIdx.x;
  int mine = 0, used;
  for (int base = 0; base < p.num_pages; base += kPlanThreads * kCountsPer) {
    int c[kCountsPer];
    load_counts(p, base + tid * kCountsPer, c);
#pragma unroll
    for (int j = 0; j < kCountsPer; ++j) mine += c[j] > 0 && base + tid * kCountsPer + j < p.num_pages;
  }
  block_scan(mine, s_scan, used);
  int32_t *src = ws_pages(p, 0), *dst = ws_pages(p, 1), *move = ws_pages(p, 2);
  int nsrc = 0, ndst = 0;
  for (int base = 0; base < p.num_pages; base += kPlanThreads * kCountsPer) {
    const int i0 = base + tid * kCountsPer;
    int c[kCountsPer], n = 0, total;  // n: moves << 16 | holes of this thread (16384 counts a step)
    load_counts(p, i0, c);
#pragma unroll
    for (int j = 0; j < kCountsPer; ++j) {
      if (i0 + j >= p.num_pages) continue;
      if (i0 + j >= used) n += c[j] > 0 ? 1 << 16 : 0;
      else n += c[j] <= 0;
    }
    const int at = block_scan(n, s_scan, total);
    int a = nsrc + (at >> 16), h = ndst + (at & 0xffff);
#pragma unroll
    for (int j = 0; j < kCountsPer; ++j) {
      const int i = i0 + j;
      if (i >= p.num_pages) continue;
      if (i >= used) {
        move[i] = c[j] > 0 ? a : -1;
        if (c[j] > 0) src[a++] = i;
      } else if (c[j] <= 0) {
        dst[h++] = i;
      }
    }
    nsrc += total >> 16;
    ndst += total & 0xffff;
  }
  __threadfence_block();
  __syncthreads();
  for (int k = tid; k < nsrc; k += kPlanThreads) {
    p.refs[dst[k]] = p.refs[src[k]];
    p.refs[src[k]] = 0;
  }
  if (tid == 0) {
    p.ws[0] = nsrc;
    p.ws[1] = used;
    used_out[0] = used;
  }
}

template <typename U>
__global__ __launch_bounds__(256) void compact_kernel(PagesParams p, PoolList pools, int tables) {
  const int32_t *src = ws_pages(p, 0), *dst = ws_pages(p, 1), *move = ws_pages(p, 2);
  const int m = p.ws[0], used = p.ws[1];
  if (blockIdx.y == 0) {
    if (!tables) return;
    const int64_t n = (int64_t)p.B * p.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
      int32_t* at = &p.block_table[(i / p.max_pages) * p.bt_sb + i % p.max_pages];
      const int pg = *at;
      if (pg >= used && pg < p.num_pages) *at = move[pg] >= 0 ? dst[move[pg]] : -1;
    }
    return;
  }
  const int k = blockIdx.y - 1;
  const int64_t bytes = pools.page_bytes[k];
  const int segs = (int)((bytes + kSegBytes - 1) / kSegBytes);
  for (int64_t it = blockIdx.x; it < (int64_t)m * segs; it += gridDim.x) {
    const int i = (int)(it / segs);
    const int64_t off = (it % segs) * (int64_t)kSegBytes;
    copy_span<U>(pools.base[k] + (int64_t)dst[i] * pools.page_stride[k] + off,
                 pools.base[k] + (int64_t)src[i] * pools.page_stride[k] + off,
                 bytes - off < kSegBytes ? bytes - off : kSegBytes);
  }
}

// ---- keeping the accepted path ------------------------------------------------------------
// Row ctx + i of sequence b becomes what row ctx + path[b][i] was; entries < 0
// leave their row.  A workgroup holds the path's rows of `kCols` units in LDS
// between reading all and writing any, so paths in any order are right.
constexpr int kCols = 32;
template <typename U>
__global__ __launch_bounds__(256) void keep_kernel(PagesParams p, PoolList pools, const int32_t* ctx_lens,
                                                   const int32_t* path, int64_t path_sb, int plen) {
  __shared__ U s_row[kMaxPathLen * kCols];
  const int k = blockIdx.y, b = blockIdx.z, ctx = ctx_lens[b];
  if (ctx < 0) return;
  const int64_t cap = (int64_t)p.max_pages << p.page_shift;
  const int64_t row_bytes = pools.page_bytes[k] >> p.page_shift, units = row_bytes / (int64_t)sizeof(U);
  const int64_t c0 = (int64_t)blockIdx.x * kCols + (threadIdx.x & (kCols - 1));
  auto row_at = [&](int64_t slot) -> char* {
    if (slot < 0 || slot >= cap) return nullptr;
    const int pg = p.block_table[b * p.bt_sb + (slot >> p.page_shift)];
    if (!page_ok(p, pg)) return nullptr;
    return pools.base[k] + (int64_t)pg * pools.page_stride[k] + (slot & ((1 << p.page_shift) - 1)) * row_bytes;
  };
  for (int i = threadIdx.x / kCols; i < plen; i += 256 / kCols) {
    const int n = path[b * path_sb + i];
    const char* s = n >= 0 && n != i ? row_at((int64_t)ctx + n) : nullptr;
    if (s != nullptr && c0 < units) s_row[i * kCols + (threadIdx.x & (kCols - 1))] = reinterpret_cast<const U*>(s)[c0];
  }
  __syncthreads();
  for (int i = threadIdx.x / kCols; i < plen; i += 256 / kCols) {
    const int n = path[b * path_sb + i];
    if (n < 0 || n == i || row_at((int64_t)ctx + n) == nullptr) continue;
    char* d = row_at((int64_t)ctx + i);
    if (d != nullptr && c0 < units) reinterpret_cast<U*>(d)[c0] = s_row[i * kCols + (threadIdx.x & (kCols - 1))];
  }
}

int64_t max_page_bytes(const PoolList& l) {
  int64_t m = 0;
  for (int k = 0; k < l.n; ++k) m = l.page_bytes[k] > m ? l.page_bytes[k] : m;
  return m;
}

// Workgroups for `items` segments, at most what fills the card several times.
unsigned copy_grid(int64_t items) { return (unsigned)(items < 1 ? 1 : items > 4096 ? 4096 : items); }

}  // namespace

size_t pages_workspace_ints(int num_pages, int n) { return (size_t)kWsHead + 3 * (size_t)num_pages + 2 * (size_t)n; }

hipError_t launch_pages_copy(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* src,
                             const int32_t* dst, int n, bool vec, hipStream_t s) {
  copy_check_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p, src, dst, n);
  for (int l = 0; l < nlists; ++l) {
    const int64_t segs = (max_page_bytes(pools[l]) + kSegBytes - 1) / kSegBytes;
    const dim3 grid(copy_grid(n * segs), (unsigned)pools[l].n);
    if (vec) copy_kernel<u32x4><<<grid, 256, 0, s>>>(p, pools[l], src, dst, n);
    else copy_kernel<uint8_t><<<grid, 256, 0, s>>>(p, pools[l], src, dst, n);
  }
  return hipGetLastError();
}

hipError_t launch_pages_fork(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* parents,
                             const int32_t* children, int n, int32_t* ok, bool vec, hipStream_t s) {
  fork_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, parents, children, n, ok);
  for (int l = 0; l < nlists; ++l) {
    const int64_t segs = (max_page_bytes(pools[l]) + kSegBytes - 1) / kSegBytes;
    const dim3 grid(copy_grid(n * (segs > 0 ? segs : 1)), (unsigned)pools[l].n + 1);
    if (vec) fork_kernel<u32x4><<<grid, 256, 0, s>>>(p, pools[l], parents, children, n, ok, l == 0);
    else fork_kernel<uint8_t><<<grid, 256, 0, s>>>(p, pools[l], parents, children, n, ok, l == 0);
  }
  return hipGetLastError();
}

hipError_t launch_pages_free(const PagesParams& p, const int32_t* rows, const int32_t* keep_lens, int n, hipStream_t s) {
  free_kernel<<<dim3((unsigned)((p.max_pages + 255) / 256), (unsigned)n), 256, 0, s>>>(p, rows, keep_lens, n);
  return hipGetLastError();
}

hipError_t launch_pages_extend(const PagesParams& p, const int32_t* new_lens, int32_t* ok, hipStream_t s) {
  extend_kernel<<<1, kPlanThreads, 0, s>>>(p, new_lens, ok);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesParams& p, const PoolList* pools, int nlists, int32_t* used, bool vec,
                                hipStream_t s) {
  compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(p, used);
  for (int l = 0; l < nlists; ++l) {
    // (at most half of the pages move)
    const int64_t segs = (max_page_bytes(pools[l]) + kSegBytes - 1) / kSegBytes;
    const int64_t items = (int64_t)p.num_pages / 2 * (segs > 0 ? segs : 1), tab = ((int64_t)p.B * p.max_pages + 255) / 256;
    const dim3 grid(copy_grid(items > tab ? items : tab), (unsigned)pools[l].n + 1);
    if (vec) compact_kernel<u32x4><<<grid, 256, 0, s>>>(p, pools[l], l == 0);
    else compact_kernel<uint8_t><<<grid, 256, 0, s>>>(p, pools[l], l == 0);
  }
  return hipGetLastError();
}

hipError_t launch_pages_keep(const PagesParams& p, const PoolList* pools, int nlists, const int32_t* ctx_lens,
                             const int32_t* path, int64_t path_sb, int plen, bool vec, hipStream_t s) {
  for (int l = 0; l < nlists; ++l) {
    const int64_t row = max_page_bytes(pools[l]) >> p.page_shift, units = vec ? row / 16 : row;
    const dim3 grid((unsigned)((units + kCols - 1) / kCols), (unsigned)pools[l].n, (unsigned)p.B);
    if (vec) keep_kernel<u32x4><<<grid, 256, 0, s>>>(p, pools[l], ctx_lens, path, path_sb, plen);
    else keep_kernel<uint8_t><<<grid, 256, 0, s>>>(p, pools[l], ctx_lens, path, path_sb, plen);
  }
  return hipGetLastError();
}

}  // namespace sfa

// Pages of a cache that sequences share, on the device: taken, shared, copied, packed and given back without the host, so that a step which forks its
// sequences runs inside a CUDA graph.
//
// A pool is a table of pages per slot, the positions each slot holds, and per page the number of table entries that name it. Which page a call takes is part of what
// it computes: always the lowest free one, in the order of the call's list, so that the same calls give the same table. Counts change by integer atomics, whose
// order changes nothing, and the free pages are a bit each that every change from or to a count of 0 turns over: whatever the order of the changes, the bits are
// right behind them. A bit a page keeps the search for free pages short: one CTA reads them all at once.
//
//   extend     one CTA: pages that each slot of the list lacks, free bits counted per thread, all of them handed out by rank
//   fork       rows of the table as they were go to a workspace while counts follow (a CTA a parent and piece of its row, which changes a page's count once for all its
//              children); the last CTA to finish takes the pages for partly filled ones. Behind it, copies of those pages in all caches, and the rows into the table;
//              or, where pages lack, the counts back.
//   free       a thread has an entry of eight slots and changes a page's count once for those of them next to one another that name it: forks do
//   compact    one CTA ranks holes below and pages above the number of live pages; then copies and every entry of the table
//   copy       a CTA copies a page of a cache
// Bound by the bytes that are copied; launches otherwise. Measured: two sequences of 4090 positions, 12 layers of 512 columns, copied out, given back, packed and taken up again 223 us (1.15 GB,
// 175 us at the copy rate); of 200 positions 79, which is what the ten calls take (5 - 6 us each, a fork 9). A turn of fork, extend, fork, free: 4 children of 300 positions 46 - 48 us (the
// calls), 64 children of 30011 65 (device time: forks 16 - 20 and 7, extend 8, free 8).
#include <algorithm>

#include "common.cuh"
#include "ifab_kernels.h"
#include "tc_common.cuh"

using namespace ifab;

namespace {

constexpr int PLAN = 1024;              // threads of a planning CTA
constexpr int MAX_SLOTS = 8192;

struct Pool {
  IfabPagePool p;
  // the workspace: control words, list of copies (from, to, rows in use), pages' new places, staged rows
  __device__ __forceinline__ int32_t* control() const { return p.work; }
  __device__ __forceinline__ int32_t* from() const { return p.work + 8; }
  __device__ __forceinline__ int32_t* to() const { return from() + max(p.set.pages, p.slots); }
  __device__ __forceinline__ int32_t* place() const { return to() + max(p.set.pages, p.slots); }
  __device__ __forceinline__ int32_t* used() const { return place() + max(p.set.pages, p.slots); }
  __device__ __forceinline__ int32_t* staged() const { return used() + p.slots; }
};
enum Control { COUNT, TICKET, GO, LIVE };
uint64_t work_words(int slots, int max_pages, int pages) { return 8 + 3ull * std::max(pages, slots) + slots + (uint64_t)slots * max_pages; }

__device__ __forceinline__ void turn(const IfabPagePool& p, int page) { atomicXor(p.free_bits + (page >> 5), 1u << (page & 31)); }
__device__ __forceinline__ void take(const IfabPagePool& p, int page, int times = 1) {
  if (page >= 0 && page < p.set.pages && atomicAdd(p.refs + page, times) == 0) turn(p, page);
}
__device__ __forceinline__ void give(const IfabPagePool& p, int page, int times = 1) {
  if (page >= 0 && page < p.set.pages && atomicSub(p.refs + page, times) == times) turn(p, page);
}
__device__ __forceinline__ void report(uint32_t* status, uint32_t bit) {
  if (status) atomicOr(status, bit);
}

// sums of all threads of the CTA ahead of this one's; `total`: of all. `warps`: 33 ints of shared memory
__device__ __forceinline__ int scan(int v, int* warps, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int w = lane < n ? warps[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    if (lane < n) warps[lane] = w;
  }
  __syncthreads();
  *total = warps[n - 1];
  return s - v + (warp ? warps[warp - 1] : 0);
}
// whether the list names slots of the pool, each once; all threads. `seen`: MAX_SLOTS bits of shared memory
__device__ __forceinline__ bool distinct(const int32_t* list, int n, int slots, uint32_t* seen) {
  for (int i = threadIdx.x; i < (slots + 31) / 32; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  bool good = true;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = list[i];
    good = good && s >= 0 && s < slots && !(atomicOr(seen + (s >> 5), 1u << (s & 31)) >> (s & 31) & 1);
  }
  return __syncthreads_and(good);
}
// `take_page(rank, page)` for the lowest `want` free pages (there are as many), threads of one CTA that `ahead` free pages of lie below this one's; their bits are cleared.
// Words of the bits are spread over the threads in order, pages over all threads by way of `list` (TAKEN ints of shared memory).
constexpr int TAKEN = 2048;
template <class F>
__device__ __forceinline__ void lowest_free(const IfabPagePool& p, int want, int ahead, int* list, F&& take_page) {
  const int words = (p.set.pages + 31) / 32, per = (words + blockDim.x - 1) / blockDim.x;
  int w = threadIdx.x * per;
  const int end = min(w + per, words);
  uint32_t bits = w < end ? *(volatile uint32_t*)(p.free_bits + w) : 0;
  bool changed = false;
  for (int t0 = 0; t0 < want; t0 += TAKEN) {
    const int t1 = min(t0 + TAKEN, want);
    while (w < end && ahead < t1) {
      if (!bits) {
        if (changed) p.free_bits[w] = 0;
        changed = false;
        if (++w < end) bits = *(volatile uint32_t*)(p.free_bits + w);
        continue;
      }
      list[ahead++ - t0] = w * 32 + __ffs(bits) - 1;
      bits &= bits - 1;
      changed = true;
    }
    __syncthreads();
    for (int i = t0 + threadIdx.x; i < t1; i += blockDim.x) take_page(i, list[i - t0]);
    __syncthreads();
  }
  if (changed) p.free_bits[w] = bits;
}
__device__ __forceinline__ int my_free(const IfabPagePool& p) {
  const int words = (p.set.pages + 31) / 32, per = (words + blockDim.x - 1) / blockDim.x;
  int n = 0;
  for (int i = 0; i < per; ++i) {
    const int w = threadIdx.x * per + i;
    if (w < words) n += __popc(*(volatile uint32_t*)(p.free_bits + w));
  }
  return n;
}

// the first `bytes` of a page, a multiple of 16; the threads of a CTA
__device__ __forceinline__ void copy_page(unsigned char* to, const unsigned char* from, long bytes) {
  const long n = bytes / 16;
  uint4* d = reinterpret_cast<uint4*>(to);
  const uint4* s = reinterpret_cast<const uint4*>(from);
  long i = threadIdx.x;
  for (; i + 3 * (long)blockDim.x < n; i += 4 * (long)blockDim.x) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = s[i + u * (long)blockDim.x];
#pragma unroll
    for (int u = 0; u < 4; ++u) d[i + u * (long)blockDim.x] = v[u];
  }
  for (; i < n; i += blockDim.x) d[i] = s[i];
}

__global__ void __launch_bounds__(256) copy_kernel(IfabPageSet src, IfabPageSet dst, const int32_t* src_ids, const int32_t* dst_ids, const int32_t* rows, int n, uint32_t* status) {
  grid_dep_launch();
  grid_dep_wait();
  for (long i = blockIdx.x; i < (long)n * src.caches; i += gridDim.x) {
    const int e = (int)(i / src.caches), l = (int)(i - (long)e * src.caches), a = src_ids[e], b = dst_ids[e], r = rows ? rows[e] : src.page_tokens;
    if (a < 0 || a >= src.pages || b < 0 || b >= dst.pages || r < 0 || r > src.page_tokens) {
      if (threadIdx.x == 0) report(status, IFAB_STATUS_BAD_INDEX);
      continue;
    }
    const long row = src.row_bytes[l], page = row * src.page_tokens;
    copy_page((unsigned char*)dst.ptrs[l] + b * page, (const unsigned char*)src.ptrs[l] + a * page, r * row);
  }
}

__global__ void __launch_bounds__(PLAN) extend_kernel(Pool q, const int32_t* slots, const int32_t* tokens, int n) {
  __shared__ uint32_t seen[MAX_SLOTS / 32];
  __shared__ int warps[33];
  __shared__ int ahead[MAX_SLOTS + 1], list[TAKEN];           // ahead: pages that the slots of the list ahead of each lack
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int pt = p.set.page_tokens;
  bool good = distinct(slots, n, p.slots, seen);
  int base = 0;
  if (good) {
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
      const int i = i0 + threadIdx.x;
      int lack = 0;
      if (i < n) {
        const int have = p.lengths[slots[i]], want = tokens[i];
        if (want < 0 || want > (long)p.max_pages * pt) good = false;
        else lack = max(0, (want + pt - 1) / pt - (have + pt - 1) / pt);
      }
      int total;
      const int before = scan(lack, warps, &total);
      if (i < n) ahead[i] = base + before;
      base += total;
    }
    if (threadIdx.x == 0) ahead[n] = base;
    good = __syncthreads_and(good);
  }
  int free_pages;
  const int mine = scan(my_free(p), warps, &free_pages);
  if (!good || free_pages < base) {
    if (threadIdx.x == 0) report(p.status, good ? IFAB_STATUS_NO_PAGES : IFAB_STATUS_BAD_INDEX);
    return;
  }
  lowest_free(p, base, mine, list, [&](int rank, int page) {
    int lo = 0, hi = n - 1;                      // the last slot of the list with ahead <= rank
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ahead[mid] <= rank) lo = mid;
      else hi = mid - 1;
    }
    const int s = slots[lo];
    p.table[(long)s * p.max_pages + (p.lengths[s] + pt - 1) / pt + rank - ahead[lo]] = page;
    p.refs[page] = 1;
  });
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) p.lengths[slots[i]] = max(p.lengths[slots[i]], tokens[i]);
}

// grid (entries of the list, pieces of a row): the CTAs of the first entry that names a parent have all of its children
__global__ void __launch_bounds__(256) fork_kernel(Pool q, const int32_t* src, const int32_t* dst, int n) {
  __shared__ uint32_t seen[MAX_SLOTS / 32], named[MAX_SLOTS / 32];
  __shared__ int warps[33], list[TAKEN], children, parents;
  __shared__ uint32_t child[MAX_SLOTS];          // entry of the list, slot above
  __shared__ bool last;
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int parent = src[blockIdx.x];
  if (threadIdx.x == 0) children = parents = 0;
  for (int i = threadIdx.x; i < (p.slots + 31) / 32; i += blockDim.x) named[i] = 0;
  bool good = distinct(dst, n, p.slots, seen), earlier = false;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int a = src[i];
    good = good && a >= 0 && a < p.slots;
    earlier = earlier || (a == parent && i < (int)blockIdx.x);
    if (a == parent) child[atomicAdd(&children, 1)] = (uint32_t)i | (uint32_t)dst[i] << 16;
    if (good && !(atomicOr(named + (a >> 5), 1u << (a & 31)) >> (a & 31) & 1)) atomicAdd(&parents, 1);
  }
  good = __syncthreads_and(good);
  earlier = __syncthreads_or(earlier);
  if (!good && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    report(p.status, IFAB_STATUS_BAD_INDEX);
    q.control()[COUNT] = 0;
    q.control()[GO] = -1;
  }
  if (!good || earlier) return;                  // the others have no part in the ticket: of 1152 CTAs for 64 children, 18 draw one (5 us of a turn's 70)
  // 64 entries side by side, every fourth child a thread
  const int32_t* row = p.table + (long)parent * p.max_pages;
  for (int j = blockIdx.y * 64 + (threadIdx.x & 63); j < p.max_pages; j += gridDim.y * 64) {
    const int then = row[j];
    int times = 0;
    for (int c0 = threadIdx.x >> 6; c0 < children; c0 += 32) {
      int now[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c0 + 4 * c < children) now[c] = p.table[(long)(child[c0 + 4 * c] >> 16) * p.max_pages + j];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c0 + 4 * c < children) {
          q.staged()[(long)(child[c0 + 4 * c] & 0xffff) * p.max_pages + j] = then;
          if (now[c] != then) {
            ++times;
            give(p, now[c]);
          }
        }
    }
    if (times) take(p, then, times);
  }
  if (blockIdx.y == 0)
    for (int c = threadIdx.x; c < children; c += blockDim.x) q.used()[child[c] & 0xffff] = p.lengths[parent];
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(q.control() + TICKET, 1) == parents * (int)gridDim.y - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // Every count has been changed. Children that need a page of their own for a partly filled one: all but the first of a parent that is itself replaced.
  int32_t* control = q.control();
  int count = 0;
  for (int i0 = 0; i0 < n; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    bool copies = false;
    int page = -1, used = 0;
    if (i < n) {
      const int a = src[i], length = ((volatile int32_t*)q.used())[i];
      used = length % p.set.page_tokens;
      if (used) page = ((volatile int32_t*)q.staged())[(long)i * p.max_pages + length / p.set.page_tokens];
      copies = page >= 0 && page < p.set.pages;
      if (copies && (seen[a >> 5] >> (a & 31) & 1)) {
        copies = false;                          // unless an earlier child has it
        for (int k = 0; k < i && !copies; ++k) copies = src[k] == a;
      }
    }
    int total;
    const int at = scan(copies, warps, &total) + count;
    if (copies) {
      q.from()[at] = page;
      q.place()[at] = i;
    }
    count += total;
  }
  int free_pages;
  const int mine = scan(my_free(p), warps, &free_pages);
  __syncthreads();
  const bool enough = free_pages >= count;
  if (enough)
    lowest_free(p, count, mine, list, [&](int rank, int page) {
      const int i = ((volatile int32_t*)q.place())[rank], length = ((volatile int32_t*)q.used())[i];
      q.to()[rank] = page;
      q.staged()[(long)i * p.max_pages + length / p.set.page_tokens] = page;
      atomicSub(p.refs + ((volatile int32_t*)q.from())[rank], 1);      // its first owner keeps it
      p.refs[page] = 1;
    });
  if (threadIdx.x == 0) {
    if (!enough) report(p.status, IFAB_STATUS_NO_PAGES);
    control[TICKET] = 0;
    control[COUNT] = enough ? count : 0;
    control[GO] = enough;
  }
}

// copies of partly filled pages, and rows into the table; counts back where pages lacked
__global__ void __launch_bounds__(256) fork_rows_kernel(Pool q, const int32_t* src, const int32_t* dst, int n) {
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int go = q.control()[GO];
  if (go < 0) return;
  const int pt = p.set.page_tokens, step = gridDim.x * blockDim.x, copies = q.control()[COUNT];
  for (long e = blockIdx.x * blockDim.x + threadIdx.x; e < (long)n * p.max_pages; e += step) {
    const int i = (int)(e / p.max_pages), j = (int)(e - (long)i * p.max_pages);
    const int then = q.staged()[e];
    int32_t* entry = p.table + (long)dst[i] * p.max_pages + j;
    if (go) {
      if (*entry != then) *entry = then;
      if (j == 0) p.lengths[dst[i]] = q.used()[i];
    } else if (*entry != then) {
      take(p, *entry);
      give(p, then);
    }
  }
  for (long i = blockIdx.x; i < (long)copies * p.set.caches; i += gridDim.x) {
    const int e = (int)(i / p.set.caches), l = (int)(i - (long)e * p.set.caches);
    const long row = p.set.row_bytes[l], page = row * pt;
    unsigned char* base = (unsigned char*)p.set.ptrs[l];
    copy_page(base + q.to()[e] * page, base + q.from()[e] * page, q.used()[q.place()[e]] % pt * row);
  }
}

// grid (eight entries of the list, pieces of a row)
constexpr int TOGETHER = 8;
__global__ void __launch_bounds__(256) free_kernel(Pool q, const int32_t* slots, const int32_t* below, int n) {
  __shared__ int slot[TOGETHER], end[TOGETHER];
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int first = blockIdx.x * TOGETHER, count = min(TOGETHER, n - first), step = gridDim.y * blockDim.x;
  bool good = true;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int s = slots[i], b = below ? below[i] : 0, c = i - first;
    const bool mine = s >= 0 && s < p.slots && b >= 0;
    good = good && mine;
    if (c < 0 || c >= count || !mine) continue;
    slot[c] = s;
    // a page that is partly filled stays with its sequence
    end[c] = below ? min(b, p.lengths[s]) / p.set.page_tokens : p.max_pages;
  }
  // a list with a bad entry is refused as a whole, and so every slot that is compared and looked up below is one of the pool's
  if (!__syncthreads_and(good)) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) report(p.status, IFAB_STATUS_BAD_INDEX);
    return;
  }
  if (!below && blockIdx.y == 0 && threadIdx.x < count) p.lengths[slots[first + threadIdx.x]] = 0;
  // a slot that is named more than once: the first entry does it, as far as the furthest of them goes
  for (int e = threadIdx.x; e < count * n; e += blockDim.x) {
    const int c = e / n, k = e - c * n;
    if (k == first + c || slots[k] != slots[first + c]) continue;
    if (k < first + c) atomicExch(&slot[c], -1);
    else if (below) atomicMax(&end[c], min(below[k], p.lengths[slots[k]]) / p.set.page_tokens);
  }
  __syncthreads();
  for (int j = blockIdx.y * blockDim.x + threadIdx.x; j < p.max_pages; j += step) {
    int page = -1, times = 0;
    int had[TOGETHER];
#pragma unroll
    for (int c = 0; c < TOGETHER; ++c) {
      const bool mine = c < count && slot[c] >= 0 && j < end[c];
      had[c] = mine ? p.table[(long)slot[c] * p.max_pages + j] : -1;
    }
#pragma unroll
    for (int c = 0; c < TOGETHER; ++c)
      if (had[c] >= 0) p.table[(long)slot[c] * p.max_pages + j] = -1;
#pragma unroll
    for (int c = 0; c < TOGETHER; ++c) {
      if (had[c] < 0) continue;
      if (had[c] != page) {
        if (times) give(p, page, times);
        page = had[c];
        times = 0;
      }
      ++times;
    }
    if (times) give(p, page, times);
  }
}

__global__ void __launch_bounds__(PLAN) compact_plan_kernel(Pool q, int32_t* live_out) {
  __shared__ int warps[33];
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int pages = p.set.pages, words = (pages + 31) / 32, per = (words + blockDim.x - 1) / blockDim.x;
  int free_pages, total;
  scan(my_free(p), warps, &free_pages);
  const int live = pages - free_pages;
  // of word w: holes below `live`, pages at or above it
  auto parts = [&](int w, uint32_t* holes, uint32_t* above) {
    const int left = pages - w * 32, low = min(max(live - w * 32, 0), 32);
    const uint32_t all = left >= 32 ? 0xffffffffu : (1u << left) - 1, below = low == 32 ? 0xffffffffu : (1u << low) - 1, bits = p.free_bits[w] & all;
    *holes = bits & below;
    *above = ~bits & all & ~below;
  };
  int holes = 0, above = 0;
  for (int i = 0; i < per; ++i) {
    const int w = threadIdx.x * per + i;
    if (w >= words) break;
    uint32_t h, a;
    parts(w, &h, &a);
    holes += __popc(h);
    above += __popc(a);
  }
  int h0 = scan(holes, warps, &total);
  int a0 = scan(above, warps, &total);
  for (int i = 0; i < per; ++i) {
    const int w = threadIdx.x * per + i;
    if (w >= words) break;
    uint32_t h, a;
    parts(w, &h, &a);
    for (; h; h &= h - 1) q.to()[h0++] = w * 32 + __ffs(h) - 1;
    for (; a; a &= a - 1) q.from()[a0++] = w * 32 + __ffs(a) - 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += blockDim.x) q.place()[q.from()[i]] = q.to()[i];
  if (threadIdx.x == 0) {
    q.control()[COUNT] = total;
    q.control()[LIVE] = live;
    if (live_out) *live_out = live;
  }
}

__global__ void __launch_bounds__(256) compact_kernel(Pool q) {
  grid_dep_launch();
  grid_dep_wait();
  const IfabPagePool& p = q.p;
  const int count = q.control()[COUNT], live = q.control()[LIVE], step = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + threadIdx.x;
  if (count) {
    for (long e = first; e < (long)p.slots * p.max_pages; e += step) {
      const int page = p.table[e];
      if (page >= live && page < p.set.pages) p.table[e] = q.place()[page];
    }
    for (int i = first; i < count; i += step) {
      p.refs[q.to()[i]] = p.refs[q.from()[i]];
      p.refs[q.from()[i]] = 0;
    }
    for (int w = first; w < (p.set.pages + 31) / 32; w += step) {
      const int left = p.set.pages - w * 32, low = min(max(live - w * 32, 0), 32);
      p.free_bits[w] = (left >= 32 ? 0xffffffffu : (1u << left) - 1) & ~(low == 32 ? 0xffffffffu : (1u << low) - 1);
    }
  }
  for (long i = blockIdx.x; i < (long)count * p.set.caches; i += gridDim.x) {
    const int e = (int)(i / p.set.caches), l = (int)(i - (long)e * p.set.caches);
    const long page = p.set.row_bytes[l] * p.set.page_tokens;
    unsigned char* base = (unsigned char*)p.set.ptrs[l];
    copy_page(base + q.to()[e] * page, base + q.from()[e] * page, page);
  }
}

bool good_set(const IfabPageSet* s) { return s && s->ptrs && s->row_bytes && s->caches > 0 && s->pages > 0 && s->page_tokens > 0; }
bool good_pool(const IfabPagePool* p) {
  return p && good_set(&p->set) && p->table && p->lengths && p->refs && p->free_bits && p->work && p->slots > 0 && p->slots <= MAX_SLOTS && p->max_pages > 0 &&
         (p->max_pages + 1l) * p->set.page_tokens < 1l << 31 && (long)p->slots * p->max_pages < 1l << 31;      // positions and entries are counted in 32 bits
}
int grid_of(long items) { return (int)std::min<long>(std::max<long>(items, 1), 8l * tc::device_sms()); }
// CTAs that share a row by `entries` entries each, as long as they all run at once
int pieces_of(int rows, int max_pages, int entries) { return std::max(1, std::min((max_pages + entries - 1) / entries, 8 * tc::device_sms() / std::max(rows, 1))); }

}  // namespace

extern "C" uint64_t ifab_pages_work_words(int slots, int max_pages, int pages) { return work_words(slots, max_pages, pages); }

// the first rows[e] rows (all without `rows`) of page src_ids[e] into page dst_ids[e] of every cache of the sets, which are alike
extern "C" int ifab_pages_copy(const IfabPageSet* src, const IfabPageSet* dst, const int32_t* src_ids, const int32_t* dst_ids, const int32_t* rows, int n, uint32_t* status,
                               void* stream) {
  if (!good_set(src) || !good_set(dst) || src->caches != dst->caches || src->page_tokens != dst->page_tokens || src->max_row_bytes != dst->max_row_bytes || n < 0) return -1;
  if (n == 0) return 0;
  return launch_chain(copy_kernel, dim3(grid_of((long)n * src->caches)), dim3(256), 0, (cudaStream_t)stream, *src, *dst, src_ids, dst_ids, rows, n, status);
}
// pages for positions below tokens[i] of slots[i]
extern "C" int ifab_pages_extend(const IfabPagePool* p, const int32_t* slots, const int32_t* tokens, int n, void* stream) {
  if (!good_pool(p) || n < 0 || n > p->slots) return -1;
  if (n == 0) return 0;
  return launch_chain(extend_kernel, dim3(1), dim3(PLAN), 0, (cudaStream_t)stream, Pool{*p}, slots, tokens, n);
}
// slot dst[i] becomes what slot src[i] was
extern "C" int ifab_pages_fork(const IfabPagePool* p, const int32_t* src, const int32_t* dst, int n, void* stream) {
  if (!good_pool(p) || n < 0 || n > p->slots) return -1;
  if (n == 0) return 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (int rc = launch_chain(fork_kernel, dim3(n, pieces_of(n, p->max_pages, 64)), dim3(256), 0, s, Pool{*p}, src, dst, n)) return rc;
  return launch_chain(fork_rows_kernel, dim3(grid_of((long)n * p->set.caches)), dim3(256), 0, s, Pool{*p}, src, dst, n);
}
// all pages of slots[i], or those whose positions all lie below below[i]
extern "C" int ifab_pages_free(const IfabPagePool* p, const int32_t* slots, const int32_t* below, int n, void* stream) {
  if (!good_pool(p) || n < 0) return -1;
  if (n == 0) return 0;
  const int groups = (n + TOGETHER - 1) / TOGETHER;
  return launch_chain(free_kernel, dim3(groups, pieces_of(groups, p->max_pages, 256)), dim3(256), 0, (cudaStream_t)stream, Pool{*p}, slots, below, n);
}
// live pages into the lowest places; their number into *live (may be null)
extern "C" int ifab_pages_compact(const IfabPagePool* p, int32_t* live, void* stream) {
  if (!good_pool(p)) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  if (int rc = launch_chain(compact_plan_kernel, dim3(1), dim3(PLAN), 0, s, Pool{*p}, live)) return rc;
  return launch_chain(compact_kernel, dim3(8 * tc::device_sms()), dim3(256), 0, s, Pool{*p});
}

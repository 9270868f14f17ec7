// Rows, groups and parts of the attention over shared prefixes, as its kernels see them.
#pragma once
#include "common.cuh"
#include "ifab_kernels.h"

namespace ifab {

// rows first .. first + rows - 1 see the positions below `shared` through the pages of `slot`
struct PrefixGroup {
  int first, rows, shared, slot;
};
// positions [begin, end) that a row sees by itself, through the pages of `slot`
struct PrefixOwn {
  int begin, end, slot;
};

struct PrefixParams {
  const bf16* q;
  long ldq;
  const bf16 *k_cache, *v_cache;
  const int32_t *positions, *slots, *page_table, *group_list;
  int num_slots, max_pages, page_tokens, num_pages, groups;
  float scale_log2;                              // of a score in powers of two
  int T, Hq, Hkv, G;
  // stretches that a group's prefix (by the parts kernel; by the tiles kernel, which leaves two parts of each) and a row's own positions are shared out to at most
  int part_splits, tile_splits, own_splits;
  int tile_share, tile_shares;                   // a stretch of the tiles kernel's but the last one is so large a share of the prefix, where last ones come by `tile_share` turns
  int prefix_parts;                              // parts that a row and head has room for ahead of those of its own positions
  long tiles_from;                               // length of the longest prefix from which on the tiles kernel has all of them
  float* parts;                                  // [T, Hq, prefix_parts + own_splits, head_dim]: sums of values
  float2* sums;                                  // [T, Hq, prefix_parts + own_splits]: maximum (in powers of two), sum of weights
  uint32_t* status;
  // A word of the scratch and what the tiles kernel writes there, another number in every call that launches it; 0: this call does not
  unsigned long long *word, number;

  // The kernel behind the tiles kernel does its work ahead of that one's end. What kernels before both wrote is visible to a grid that waits for them: the tiles kernel has, and by this word hands it on.
  // A CTA that does not find it waits itself, so no more than time hangs on it. What the two kernels write are places of their own. 64 rows behind 30011 positions 93 us without, 88 with it, 27 in three
  // groups 41.6 and 39.6
  __device__ __forceinline__ void hand_on() const { asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(word), "l"(number) : "memory"); }        // by a thread, behind the wait
  __device__ __forceinline__ void take_over() const {                   // by all CTAs
    unsigned long long found = 0;
    if (number && threadIdx.x == 0) asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(found) : "l"(word) : "memory");
    if (!__syncthreads_or(number && found == number)) grid_dep_wait();
    // taken back by the one that starts last: a graph that is replayed has the same number
    if (number && threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(word), "l"(0ull) : "memory");
  }

  // row of the caches; -1: there is none
  __device__ __forceinline__ int row_of(int pos, int slot) const {
    const int lp = pos / page_tokens;
    if (slot < 0 || slot >= num_slots || lp >= max_pages) return -1;
    const int page = page_table[(long)slot * max_pages + lp];
    return page < 0 || page >= num_pages ? -1 : page * page_tokens + (pos - lp * page_tokens);
  }
  // Group i of a pass over all of them; `end`: where the rows of those before it end. One that cannot be - rows that are none or another group's, positions that no slot holds - is one
  // without rows
  __device__ __forceinline__ PrefixGroup group(int i, int* end) const {
    const int4 g = *reinterpret_cast<const int4*>(group_list + 4 * i);
    const bool ok = g.x >= *end && g.y >= 1 && g.x <= T - g.y && g.z >= 0 && g.z <= max_pages * page_tokens && g.w >= 0 && g.w < num_slots;
    if (!ok && g.y && status) atomicOr(status, IFAB_STATUS_BAD_INDEX);
    if (!ok) return {0, 0, 0, 0};
    *end = g.x + g.y;
    return {g.x, g.y, g.z, g.w};
  }
  __device__ __forceinline__ PrefixGroup naming(int t) const {          // the group that names row t; without rows: none does
    int end = 0;
    for (int i = 0; i < groups; ++i) {
      const PrefixGroup g = group(i, &end);
      if (t >= g.first && t < g.first + g.rows) return g;
    }
    return {0, 0, 0, 0};
  }
  __device__ __forceinline__ bool by_tiles() const {
    int longest = 0, end = 0;
    for (int i = 0; i < groups; ++i) longest = max(longest, group(i, &end).shared);
    return longest >= tiles_from;
  }
  // whether a row of a group sees its prefix as a whole
  __device__ __forceinline__ bool sees(const PrefixGroup& g, int t) const { return g.rows && positions[t] >= 0 && positions[t] >= g.shared - 1; }
  __device__ __forceinline__ PrefixOwn own(int t, const PrefixGroup& g) const {
    const int pos = positions[t], most = max_pages * page_tokens;
    if (pos < 0) return {0, 0, 0};
    if (pos >= most && status) atomicOr(status, IFAB_STATUS_BAD_INDEX);
    const int end = pos < most ? pos + 1 : most;
    if (!g.rows) return {0, end, slots[t]};
    return end >= g.shared ? PrefixOwn{g.shared, end, slots[t]} : PrefixOwn{0, end, g.slot};       // a position within the prefix
  }
  // keys of a stretch: whole tiles of the kernels'
  __device__ __forceinline__ int per_split(int n, int splits) const { return max(128, ((n + splits - 1) / splits + 127) / 128 * 128); }
  // (a stretch's start and end take as long as 256 keys)
  __device__ __forceinline__ int per_tile_split(int n) const { return max(128, (int)(((long)n * tile_share + (tile_share - 1) * 256 + tile_shares - 1) / tile_shares + 127) / 128 * 128); }
  __device__ __forceinline__ long part_of(int t, int h, int i) const { return ((long)t * Hq + h) * (prefix_parts + own_splits) + i; }
};

// Weights of a softmax, powers of two, as two bf16 terms: both are cut off below the value, so that none is 0 or negative and an infinite value of a key stays infinite (as in
// mma16816.cuh), which leaves an error of 2^-15 of a weight at most - one bf16 term would leave 2^-8, as much as the result's own rounding. For that a weight is at least 2^-89, and one of a
// key that is not there, whose values are read as zeros, just that.
constexpr float PREFIX_LEAST_WEIGHT = 1.6155871e-27f;
__device__ __forceinline__ float prefix_weight(float x) {       // 2^x; NaN stays NaN
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-89.f));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
// what a part leaves beside its sums of values: a NaN counts wherever its maximum lies
__device__ __forceinline__ float2 prefix_sums(float m, float l) { return make_float2(l != l ? INFINITY : m, l); }
template <bool NONE>                             // whether there are weights of 0: both their terms are 0
__device__ __forceinline__ void two_terms(float a, float b, uint32_t* hi, uint32_t* lo) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  const float a0 = __uint_as_float((x - (NONE ? min(x, 1u) : 1u)) & 0xffff0000u), b0 = __uint_as_float((y - (NONE ? min(y, 1u) : 1u)) & 0xffff0000u);
  *hi = __byte_perm(__float_as_uint(a0), __float_as_uint(b0), 0x7632);
  *lo = __byte_perm(__float_as_uint(a - a0), __float_as_uint(b - b0), 0x7632);
}

// shared_prefix_tiles.cu: `items` = tiles of 256 pairs, however the rows are shared out, by kv heads
int launch_prefix_tiles(const PrefixParams& p, int head_dim, long items, cudaStream_t s);

}  // namespace ifab

// A token for every row of logits, drawn from the whole vocabulary with a random number that the caller gives.
//
//   z_i = logit_i / temperature; order: logits falling, ids rising
//   kept: the first top_k; of them those with exp(z_i - z_max) >= min_p; of them the shortest run whose mass reaches top_p of theirs; at least one
//   drawn: the first kept id, ids rising, at which the sum of exp(z - z_max) exceeds u times that of all kept
//
// A row is a cluster of CTAs that keep the row's logits in shared memory where they fit: they are read from memory once. What the cuts ask for is a place in the order (the k-th token, the token at
// which the mass passes a share), which is found without a sort: a histogram over the row, equal stretches of the values, says in which of 1024 bins the place lies; the bin's tokens - a
// few - are gathered and put in order by counting. A bin with more tokens than the list takes (ties, values far apart) is split again by the bits of (value, id), 10 at a time.
//
// What bounds it: for one row dependent steps - loads, a handful of barriers of the cluster, searches by a warp - of 11 to 18 us; for many, instructions, of which a token takes 6 to 7 for
// the largest value, 47 for a weight that is summed without an error, 41 to 52 more where a share of the mass is looked for (counted: 54 and 60 without a cut, 94 and 112 with a share, bf16 and f32).
// 64 rows of 151936 f32 without a cut 44 us, 256 rows of 128000 bf16 with a share 214 us (0.9 and 0.3 TB/s): instructions in 52 and 64 % of the issue slots of SMs that are at work, and SMs are that two
// thirds of the time, as 256 CTAs lie two on 108 of them and one on 40.
//
// Weights are summed as integers of 2^-44: the sums decide between tokens, so they must not depend on an order of additions, and a weight below 2^-45 of the
// largest is nothing. 2^18 weights of at most 1 are 2^62 at most.
#include <climits>
#include <utility>

#include <cooperative_groups.h>

#include "common.cuh"
#include "ifab_kernels.h"

using namespace ifab;
namespace cg = cooperative_groups;

namespace {

constexpr int NT = 512, WARPS = NT / 32, BINS = 1024, LIST = 1024, MAX_CLUSTER = 8, ID_BITS = 20, PARTS = 128;
constexpr int MAX_VOCAB = 1 << 18, PART_EIGHTS = 1 << 12;
typedef unsigned long long u64;

struct DrawParams {
  const void* logits;
  long ld;
  int T, V, slice;                  // slice: tokens a CTA holds, a multiple of 8
  bool wide;                        // rows lie on 16 bytes
  const float *inv_temperature, *top_p, *min_p, *uniforms;
  const int32_t* top_k;
  int32_t* out_ids;
  float* out_probs;
};

// what is kept: values above x, and those equal to it with ids up to i
struct Cut {
  float x;
  int i;
  __device__ __forceinline__ bool has(float v, int id) const { return (v > x) | ((v == x) & (id <= i)); }      // (no branches in the loops over a row)
};

struct __align__(16) Entry {
  u64 place, mass;
};
struct Shared {
  union {
    uint32_t part[3][BINS];                    // tokens by bin: their number, or their mass in three words, 17 bits of a token in each, which 2^15 tokens cannot overflow
    Entry list[LIST];                          // (when the bins have been added up)
  };
  u64 mine[BINS], total[BINS];                 // this CTA's, the row's
  u64 parts[PARTS];                            // 2^(62 - i / 128) + 2^31
  uint32_t listed[2];                          // by turns
  u64 from[MAX_CLUSTER], ahead[MAX_CLUSTER], all[MAX_CLUSTER];           // values of each CTA
  u64 kept[WARPS];                             // masses of the kept tokens of the warps' stretches
  float most[MAX_CLUSTER];
  int best[MAX_CLUSTER];
  u64 warp_sum[WARPS];
  float warp_a[WARPS];
  int warp_i[WARPS];
  int bin;
  u64 above;
  int first_bin, found;
  Cut cut;
};
static_assert(8 * PART_EIGHTS <= 1 << 15, "17 bits of each token's mass in 32");

// of values that are no NaN: unsigned integers in their order
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// (value, id) in the order of the tokens
__device__ __forceinline__ u64 place_of(float v, int id) { return (u64)key_of(v) << ID_BITS | (u64)((1 << ID_BITS) - 1 - id); }

// the cut whose last token lies there
__device__ __forceinline__ Cut cut_at(u64 place) { return {value_of((uint32_t)(place >> ID_BITS)), (1 << ID_BITS) - 1 - (int)(place & ((1 << ID_BITS) - 1))}; }

// Weights e^((v - most) it) in units of 2^-44, rounded. With c = it log2 e as two floats,
//   v c = n / 128 + r: n / 128 by an addition of 1.5 2^16, whose floats lie 1 / 128 apart, and r (at most 1 / 256) by a product that is rounded only then, so both without loss
//   weight = 2^-((n_most - n) / 128) (1 + q), q = 2^(r - r_most) - 1 by Taylor's series: of at most 0.0055, it is off by 2^-31 as a float
// The first factor is a table's (62 bits) and a shift, the product's upper word is taken: the largest value's weight is 1 exactly, another one's is off by 2^-28 of itself and 2^-45 at most. In units of
// 2^-30 of a weight: r less r_most, sums below 2^-6.8 in floats, 0.9; the cubic's coefficients and roundings 0.8, what it leaves out 0.1; 24 bits of the table under q 0.8; the product's last bit 1.0; where
// the weight lies below 2^-15, its rounding to units of 2^-44 beside. What a row costs is instructions, and that is half of them in 64-bit arithmetic. Factors that floats hold badly, and values whose v c
// the addition does not take, go the 64-bit way.
struct Weights {
  float most, floor;           // below `floor` a weight is less than 2^-45
  double it, z_most;
  const u64* parts;            // 2^(62 - i / 128) + 2^31: the upper word is rounded
  float ch, cl, r_most;
  int n_most;
  bool fast;
  static constexpr float MAGIC = 98304.f, C1 = 0.69314718f * 0x1p38f, C2 = 0.24022651f * 0x1p38f, C3 = 0.055504109f * 0x1p38f;
  __device__ __forceinline__ Weights(float most, float it_, const u64* parts) : most(most), it((double)it_), z_most((double)most * (double)it_), parts(parts) {
    const double lowest = (z_most - 32.0) / it, c = it * 1.4426950408889634;          // e^-32 < 2^-46
    floor = most == INFINITY ? INFINITY : lowest > -3.4e38 ? __double2float_rd(lowest) : -3.4028234664e38f;
    fast = c < 0x1p90 && c > 0x1p-90 && fabs(most * c) < 8192.0;
    ch = (float)c;
    cl = (float)(c - (double)ch);
    const float y = __fmaf_rn(most, ch, MAGIC);
    n_most = __float_as_int(y);
    r_most = __fmaf_rn(most, cl, __fmaf_rn(most, ch, MAGIC - y));
  }
  // of `most` itself 1, an infinite one among them; a product of two floats is exact
  __device__ __forceinline__ double real(float v) const { return v == most ? 1.0 : exp((double)v * it - z_most); }
  __device__ __forceinline__ u64 slow(float v) const {
    const u64 m = (u64)__double_as_longlong(real(v) + 256.0) & ((1ull << 52) - 1);       // 256 + w has its last bit at 2^-44
    return v == most ? 1ull << 44 : v >= floor ? m : 0;
  }
  // The weights of v (a NaN's is 0): those up to 2^-15 by `small(i, 32 bits)`, which the others get as 0, the others by `large(i, 64 bits)` beside that
  template <int N, typename Small, typename Large>
  __device__ __forceinline__ void of(const float (&v)[N], Small small, Large large) const {
    if (!fast) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        small(i, 0u);
        large(i, slow(v[i]));
      }
      return;
    }
    uint32_t top[N];                                       // 30 bits of a weight
    int by[N];                                             // 0 or more: what they are shifted by before their last bit is rounded away
#pragma unroll
    for (int i = 0; i < N; ++i) {                          // (all of them ahead of what is done with them: chains that run side by side)
      const float y = __fmaf_rn(v[i], ch, MAGIC), r = __fmaf_rn(v[i], cl, __fmaf_rn(v[i], ch, MAGIC - y)) - r_most;
      const float q = __fmaf_rn(__fmaf_rn(r, C3, C2), r, C1) * r;
      const int n = n_most - __float_as_int(y);
      const u64 t = parts[n & 127];
      u64 part;
      asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(part) : "r"((int)(t >> 38)), "r"(__float2int_rn(q)), "l"(t));
      top[i] = v[i] >= floor ? (uint32_t)(part >> 32) : 0u;                      // what lies below, or is none, has been anything
      by[i] = (n >> 7) - 15;
    }
    int least = by[0];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t m;
      asm("shr.u32 %0, %1, %2;" : "=r"(m) : "r"(top[i]), "r"(by[i]));            // (32 and more, and less than 0, leave 0)
      small(i, (m + 1) >> 1);
      least = min(least, by[i]);
    }
    if (least < 0)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (by[i] < 0 && top[i]) large(i, (u64)top[i] << (-1 - by[i]));
  }
  __device__ __forceinline__ u64 fixed(float v) const {
    const float a[1] = {v};
    u64 w = 0;
    of(a, [&](int, uint32_t m) { w = m; }, [&](int, u64 m) { w = m; });
    return w;
  }
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int by) { return __shfl_up_sync(0xffffffffu, v, by); }
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The lowest value of those up to `most` for which `enough`, which is so for no value and all above it, holds, by a warp: near `guess`, or 32 places at a time, 32 times finer every round
template <typename F>
__device__ float lowest(F enough, float guess, float most, int lane) {
  const uint32_t end = key_of(most), least = key_of(-INFINITY);
  const uint32_t near = key_of(guess) > least + 16 ? key_of(guess) - 16 : least;
  uint32_t vote = __ballot_sync(0xffffffffu, near + lane < end && enough(value_of(near + lane)));
  if (vote && !(vote & 1) && near + 31 < end) return value_of(near + __ffs(vote) - 1);
  uint32_t at = least, step = 1u << 27;          // it lies in (at, at + 32 steps], or is `most` itself
  for (int round = 0; round < 7; ++round) {
    const u64 mine = (u64)at + (u64)(lane + 1) * step;
    vote = __ballot_sync(0xffffffffu, mine >= end || enough(value_of((uint32_t)mine)));
    at += (uint32_t)(vote ? __ffs(vote) - 1 : 32) * step;
    step = step >= 32 ? step / 32 : 1;
  }
  const u64 key = (u64)at + 1;
  return key >= end ? most : value_of((uint32_t)key);
}

__device__ __forceinline__ float clean(float v) { return v + 0.f; }      // -0 is 0; a NaN is above nothing, so it is nowhere

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float4 load_four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load_four(const bf16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}

// A CTA's tokens by eights, in shared memory (HELD) or where they come from; those behind the last one are -inf, with ids that no place reaches
template <typename In, bool HELD>
struct Row {
  float4* own;                 // HELD: the tokens. Otherwise a ring of each thread, through which what it reads comes AHEAD eights ahead of its use (one ahead in registers: 1260 cycles a four)
  const In* src;
  int n, full;                 // tokens; eights that can be read as such
  static constexpr int AHEAD = 4, SLOT = 8 * sizeof(In);
  __device__ __forceinline__ float at(int i) const { return HELD ? reinterpret_cast<const float*>(own)[i] : load_one(src + i); }
  __device__ __forceinline__ float4 slow(int i) const { return make_float4(i < n ? at(i) : -INFINITY, i + 1 < n ? at(i + 1) : -INFINITY, i + 2 < n ? at(i + 2) : -INFINITY, i + 3 < n ? at(i + 3) : -INFINITY); }
  __device__ __forceinline__ static void eight(const In* p, float4& a, float4& b) {
    a = load_four(p);
    b = load_four(p + 4);
  }
  __device__ __forceinline__ static void request(uint32_t to, const In* from) {
#pragma unroll
    for (int i = 0; i < SLOT; i += 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i), "l"((const char*)from + i) : "memory");
  }
  // f(first token, four of them) for the eights first, first + step, ... below last
  template <typename F>
  __device__ __forceinline__ void each(int first, int last, int step, F f) const {
    if constexpr (HELD) {
      for (int o = first; o < last; o += step) {
        const float4 a = own[2 * o], b = own[2 * o + 1];
        f(8 * o, a);
        f(8 * o + 4, b);
      }
    } else {
      const int whole = min(last, full);
      const In* next = src + 8 * first;
      const uint32_t ring = (uint32_t)__cvta_generic_to_shared(own) + threadIdx.x * SLOT;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (first + k * step < whole) request(ring + k * NT * SLOT, next);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += 8 * step;
      }
      uint32_t slot = 0;
      int o = first;
      for (; o < whole; o += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
        float4 a, b;
        eight(reinterpret_cast<const In*>(reinterpret_cast<const char*>(own) + threadIdx.x * SLOT + slot), a, b);
        f(8 * o, a);
        f(8 * o + 4, b);
        if (o + AHEAD * step < whole) request(ring + slot, next);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += 8 * step;
        slot = slot == (AHEAD - 1) * NT * SLOT ? 0 : slot + NT * SLOT;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      for (; o < last; o += step) {
        f(8 * o, slow(8 * o));
        f(8 * o + 4, slow(8 * o + 4));
      }
    }
  }
};

// The place in the order at which what lies ahead reaches a number of tokens, or a share of their mass. Tokens of -inf and NaN are not among them
template <bool MASS, typename R>
struct Search {
  Shared* s;
  R row;
  int eights, base, tid, rank, ranks;          // eights: of tokens in this CTA
  uint32_t* turn;
  Cut cut;
  Weights w;
  float top, scale;            // bins of equal stretches below `top`; scale 0: one for all
  float from, below;           // values of the bin that was found: from <= v, not below <= v
  u64 lo, hi;                  // places within it, once it is split
  bool split;
  static constexpr float MAGIC = 12582912.f;

  // 1.5 2^23 + bin: whole numbers are what floats hold there. The bin rises as v falls
  __device__ __forceinline__ float stretch(float v) const { return fminf(__fmaf_rn(top - v, scale, MAGIC), scale > 0.f ? MAGIC + (BINS - 1) : MAGIC); }
  __device__ __forceinline__ bool near(float v) const { return (v >= from) & !(v >= below); }
  __device__ __forceinline__ bool member(float v, int id) const {
    const u64 at = place_of(clean(v), id);
    return near(v) && cut.has(v, id) && (!split || (at >= lo && at <= hi));
  }

  template <typename Bin>
  __device__ void count(Bin bin) {
    const bool whole = cut.x == -INFINITY;
    for (int b = tid; b < BINS; b += NT) s->mine[b] = 0;
    for (int first = 0; first < eights || first == 0; first += PART_EIGHTS) {
      for (int b = tid; b < BINS * (MASS ? 3 : 1); b += NT) s->part[0][b] = 0;
      __syncthreads();
      row.each(first + tid, min(eights, first + PART_EIGHTS), NT, [&](int i, const float4& q) {
        const float v[4] = {q.x, q.y, q.z, q.w};
        if (!whole && !__any_sync(__activemask(), (v[0] >= cut.x) | (v[1] >= cut.x) | (v[2] >= cut.x) | (v[3] >= cut.x))) return;
        int b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int id = base + i + j;
          b[j] = whole || cut.has(v[j], id) ? bin(v[j], id) : -1;
          if (!MASS && b[j] >= 0 && v[j] > -INFINITY) atomicAdd(&s->part[0][b[j]], 1u);
        }
        constexpr uint32_t low = (1u << 17) - 1;
        if (MASS)
          w.of(
              v,
              [&](int j, uint32_t m) {
                if (b[j] < 0) return;
                atomicAdd(&s->part[0][b[j]], m & low);               // (additions of 0 cost less than branches)
                atomicAdd(&s->part[1][b[j]], m >> 17);
              },
              [&](int j, u64 m) {
                if (b[j] < 0) return;
                atomicAdd(&s->part[0][b[j]], (uint32_t)m & low);
                atomicAdd(&s->part[1][b[j]], (uint32_t)(m >> 17) & low);
                atomicAdd(&s->part[2][b[j]], (uint32_t)(m >> 34));
              });
      });
      __syncthreads();
      for (int b = tid; b < BINS; b += NT) s->mine[b] += MASS ? s->part[0][b] + ((u64)s->part[1][b] << 17) + ((u64)s->part[2][b] << 34) : s->part[0][b];
      __syncthreads();
    }
  }
  // The bins' sums over the cluster
  __device__ void add_up(cg::cluster_group& cluster) {
    cluster.sync();
    // each CTA adds up its share of the bins, four threads a bin
    const int four = tid & 3;
    for (int b = rank * (BINS / ranks) + (tid >> 2); b < (rank + 1) * (BINS / ranks); b += NT / 4) {
      u64 m = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = four + 4 * h;
        if (r < ranks) m += cluster.map_shared_rank(s, r)->mine[b];
      }
      m += __shfl_xor_sync(0xffffffffu, m, 1);
      m += __shfl_xor_sync(0xffffffffu, m, 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (four + 4 * h < ranks) cluster.map_shared_rank(s, four + 4 * h)->total[b] = m;
    }
    cluster.sync();
  }
  // Two values a thread: what the threads before have (`before`) and what all have
  __device__ void scan(u64 sum, u64* before, u64* all) {
    const int lane = tid & 31, warp = tid >> 5;
    u64 incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = shfl_up64(incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) s->warp_sum[warp] = incl;
    __syncthreads();
    *before = incl - sum;
    *all = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const u64 x = s->warp_sum[i];
      if (i < warp) *before += x;
      *all += x;
    }
  }
  static __device__ u64 share_of(float share, u64 all) {                 // a token is kept while the mass ahead of it is below share * all
    const double t = ceil((double)share * (double)all);
    return t < 1.0 ? 1 : t < (double)all ? (u64)t : all;
  }
  // Sums over the cluster, then the bin at which the order passes the place `want`; `above` counts on from `ahead`. Returns all that there is. fresh: `want` follows from `share` and the total
  __device__ u64 find(cg::cluster_group& cluster, u64 ahead, bool fresh, u64* want, float share) {
    add_up(cluster);
    static_assert(BINS == 2 * NT, "two bins a thread");
    const u64 a = s->total[2 * tid], b = s->total[2 * tid + 1];
    u64 excl, all;
    scan(a + b, &excl, &all);
    if (MASS && fresh) *want = share_of(share, all);
    excl += ahead;
    const u64 mid = excl + a, incl = mid + b;
    if (excl < *want && *want <= incl) {
      const bool second = mid < *want;
      s->bin = 2 * tid + second;
      s->above = second ? mid : excl;
    }
    __syncthreads();
    return ahead + all;
  }
  // the members into every CTA's list; their number (of which the list holds LIST at most)
  __device__ uint32_t gather(cg::cluster_group& cluster) {
    uint32_t* counter = &cluster.map_shared_rank(s, 0)->listed[*turn & 1];
    if (rank == 0 && tid == 0) s->listed[(*turn + 1) & 1] = 0;        // the next turn's; the turn before has been read ahead of a barrier of the cluster
    *turn += 1;
    row.each(tid, eights, NT, [&](int i, const float4& q) {
      const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int id = base + i + j;
        if (!near(v[j]) || !member(v[j], id)) continue;
        const uint32_t at = atomicAdd(counter, 1u);
        if (at < LIST) {
          const Entry e{place_of(clean(v[j]), id), MASS ? w.fixed(v[j]) : 1};
          for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(s, r)->list[at] = e;
        }
      }
    });
    cluster.sync();
    return *counter;
  }

  // the cut at the member of the list at which what lies ahead of it and `above` reaches `want`; whether there is one
  __device__ bool resolve(uint32_t m, u64 above, u64 want) {
    if (tid == 0) s->found = 0;
    __syncthreads();
    auto cut_here = [&](u64 place) {
      s->cut = cut_at(place);
      s->found = 1;
    };
    if (m <= 128) {                              // in order by counting: a pair of them costs 7 instructions
      if (tid < m) {
        const Entry mine = s->list[tid];
        u64 ahead = above;
#pragma unroll 8
        for (uint32_t j = 0; j < m; ++j) {
          const Entry e = s->list[j];
          ahead += e.place > mine.place ? e.mass : 0;
        }
        if (ahead < want && want <= ahead + mine.mass) cut_here(mine.place);
      }
    } else {                                     // a bitonic sort, then their sums: 1000 tokens by counting took as long as a pass over the row
      uint32_t size = 256;
      while (size < m) size *= 2;
      for (uint32_t i = m + tid; i < size; i += NT) s->list[i] = Entry{0, 0};
      static_assert(LIST <= 2 * NT, "a pair a thread");
      for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
          __syncthreads();
          if (tid < size / 2) {
            const uint32_t at = 2 * tid - (tid & (j - 1));
            const Entry x = s->list[at], y = s->list[at + j];
            if ((x.place < y.place) == ((at & k) == 0)) {
              s->list[at] = y;
              s->list[at + j] = x;
            }
          }
        }
      __syncthreads();
      const bool mine = 2 * tid < size;
      const Entry x = mine ? s->list[2 * tid] : Entry{0, 0}, y = mine ? s->list[2 * tid + 1] : Entry{0, 0};
      u64 sum = x.mass + y.mass;
      const int warp = tid >> 5, lane = tid & 31;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 z = shfl_up64(sum, o);
        if (lane >= o) sum += z;
      }
      if (lane == 31) s->warp_sum[warp] = sum;
      __syncthreads();
      u64 ahead = above + sum - x.mass - y.mass;
      for (int i = 0; i < warp; ++i) ahead += s->warp_sum[i];
      if (ahead < want && want <= ahead + x.mass) cut_here(x.place);
      ahead += x.mass;
      if (ahead < want && want <= ahead + y.mass) cut_here(y.place);
    }
    __syncthreads();
    return s->found;
  }
  // f(value, &amount): a token's bin and what it adds to it, 17 bits; less than 0: none. Leaves the sums over the cluster
  template <typename F>
  __device__ void tally(cg::cluster_group& cluster, F f) {
    const bool whole = cut.x == -INFINITY;
    for (int b = tid; b < BINS; b += NT) s->mine[b] = 0;
    for (int at = 0; at < eights || at == 0; at += PART_EIGHTS) {
      for (int b = tid; b < BINS; b += NT) s->part[0][b] = 0;
      __syncthreads();
      row.each(at + tid, min(eights, at + PART_EIGHTS), NT, [&](int i, const float4& q) {
        const float v[4] = {q.x, q.y, q.z, q.w};
        if (!whole && !__any_sync(__activemask(), (v[0] >= cut.x) | (v[1] >= cut.x) | (v[2] >= cut.x) | (v[3] >= cut.x))) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t amount;
          const int bin = f(v[j], &amount);
          if (bin >= 0 && (whole || cut.has(v[j], base + i + j))) atomicAdd(&s->part[0][bin], amount);
        }
      });
      __syncthreads();
      for (int b = tid; b < BINS; b += NT) s->mine[b] += s->part[0][b];
      __syncthreads();
    }
    add_up(cluster);
  }
  // The first and the last bin that masses between `least` and `most` reach to, where those ahead of the bins have `ahead` and bin b has mass(b); into s->first_bin and s->bin, -1: none; what lies ahead of the first
  // one into s->above
  template <typename F, typename G>
  __device__ void locate(u64 ahead, F mass, G bounds) {
    u64 bins[2], excl, all, least, most;
#pragma unroll
    for (int h = 0; h < 2; ++h) bins[h] = mass(2 * tid + h);
    if (tid == 0) s->first_bin = s->bin = -1;
    scan(bins[0] + bins[1], &excl, &all);        // (a barrier of the CTA)
    bounds(all, &least, &most);
    excl += ahead;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (excl <= least && least < excl + bins[h]) {
        s->first_bin = 2 * tid + h;
        s->above = excl;
      }
      if (excl <= most && most < excl + bins[h]) s->bin = 2 * tid + h;
      excl += bins[h];
    }
    __syncthreads();
  }
  // The mass' share in two passes, where the bins' masses, to 2^-15 of all, say well enough between which tokens the place lies; leaves the kept masses of the warps' stretches. In a bin, a weight is
  // that of the bin's middle times 1 - x + x^2 / 2, which is summed in 17 bits and off by x^3 / 6 < 2^-21: one addition in shared memory a token, and a part of the instructions, where weights of 2^-44
  // take two. The last pass takes those, of all tokens, and has the list. (What is less than e^-24 counts as that in the last bin: 2^-16 of the largest weight, if all tokens lie there.) Where the bin has
  // more tokens than the list takes, one more pass, which counts only, has it in 1024 stretches. 256 rows of 128000 bf16 291 to 212 us, 27 of 151936 with cuts of their own 49 to 40 us.
  // False: the place is among the smallest weights, or too many tokens are nearly equal
  __device__ bool quick(cg::cluster_group& cluster, float share, int first, int last, int each) {
    constexpr float WIDTH = 24.f / (BINS - 1);
    if (!(scale > 0.f) || scale >= 1e30f) return false;
    const bool whole = cut.x == -INFINITY;
    const int lane = tid & 31, warp = tid >> 5;
    tally(cluster, [&](float v, uint32_t* amount) {
      const float y = stretch(v), x = fminf(__fmaf_rn(top - v, scale, MAGIC - y), 0.5f);
      *amount = (uint32_t)__float2int_rn(__fmaf_rn(__fmaf_rn(x, 0x1p15f * WIDTH * WIDTH, -0x1p16f * WIDTH), x, 0x1p16f));
      return __float_as_int(y) & (BINS - 1);
    });
    u64 least, most;
    locate(
        0, [&](int b) { return __float2ull_rn((float)s->total[b] * expf(-WIDTH * b) * 0x1p16f); },
        [&](u64 all, u64* l, u64* m) {
          const float goal = share * (float)all, room = (float)all * 0x1p-15f;
          least = *l = goal > room ? (u64)(goal - room) : 0;
          most = *m = goal > -room ? (u64)(goal + room) : 0;
        });
    const int b0 = s->first_bin, b1 = s->bin;
    if (b0 < 0 || b1 < b0 || b1 == BINS - 1) return false;
    from = fmaxf(lowest([&](float v) { return stretch(v) <= MAGIC + b1; }, top - (b1 + 0.5f) / scale, top, lane), -3.4028234664e38f);
    below = b0 ? lowest([&](float v) { return stretch(v) < MAGIC + b0; }, top - (b0 - 0.5f) / scale, top, lane) : NAN;
    split = false;
    u64 members = 0;
    for (int b = b0; b <= b1; ++b) members += s->total[b] >> 16;
    // A pass more or a longer list, which every CTA of a cluster writes to every other's: 27 rows of 151936 over eight CTAs each 51.9 us with lists of up to 960, 42.5 of 384, 41.0 of 128; 256 rows of
    // 128000, a CTA each, 210, 214 and 220
    if (members > (ranks > 1 ? 256 : LIST * 15 / 16)) {
      const float finer = (float)BINS / (b1 - b0 + 1), start = -(b0 - 0.5f) * finer - 0.5f, scale2 = scale * finer, width = WIDTH / finer;
      const u64 ahead = s->above;
      auto place = [&](float v) { return fminf(fmaxf(__fmaf_rn(top - v, scale2, start), 0.f), BINS - 1) + MAGIC; };
      tally(cluster, [&](float v, uint32_t* amount) {
        *amount = 1;
        return near(v) ? __float_as_int(place(v)) & (BINS - 1) : -1;
      });
      locate(
          ahead, [&](int b) { return __float2ull_rn((float)s->total[b] * expf(-WIDTH * (b0 - 0.5f) - width * (b + 0.5f)) * 0x1p32f); },
          [&](u64, u64* l, u64* m) {
            *l = least;
            *m = most;
          });
      const int c0 = s->first_bin, c1 = s->bin;
      if (c1 >= 0 && c1 < BINS - 1)              // (the ends of the bin stay where the stretches do not say)
        from = fmaxf(from, lowest([&](float v) { return place(v) <= MAGIC + c1; }, top - (c1 + 0.5f - start) / scale2, top, lane));
      if (c0 > 0) {
        const float edge = lowest([&](float v) { return place(v) < MAGIC + c0; }, top - (c0 - 0.5f - start) / scale2, top, lane);
        if (!(edge >= below)) below = edge;
      }
    }

    uint32_t* counter = &cluster.map_shared_rank(s, 0)->listed[*turn & 1];
    if (rank == 0 && tid == 0) s->listed[(*turn + 1) & 1] = 0;        // as in gather
    *turn += 1;
    u64 ahead = 0, sum = 0;
    row.each(first + lane, last, 32, [&](int i, const float4& q) {
      const float v[4] = {q.x, q.y, q.z, q.w};
      if (!whole && !__any_sync(__activemask(), (v[0] >= cut.x) | (v[1] >= cut.x) | (v[2] >= cut.x) | (v[3] >= cut.x))) return;
      u64 m[4];
      w.of(v, [&](int j, uint32_t x) { m[j] = x; }, [&](int j, u64 x) { m[j] = x; });
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int id = base + i + j;
        if (!whole && !cut.has(v[j], id)) continue;
        sum += m[j];
        ahead += v[j] >= below ? m[j] : 0;
        if (!near(v[j])) continue;
        const uint32_t at = atomicAdd(counter, 1u);
        if (at < LIST) {
          const Entry e{place_of(clean(v[j]), id), m[j]};
          for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(s, r)->list[at] = e;
        }
      }
    });
    ahead = warp_total(ahead);
    sum = warp_total(sum);
    if (lane == 0) {
      s->kept[warp] = ahead;
      s->warp_sum[warp] = sum;
    }
    __syncthreads();
    if (tid < ranks) {
      u64 mine = 0, its = 0;
      for (int i = 0; i < WARPS; ++i) {
        mine += s->kept[i];
        its += s->warp_sum[i];
      }
      cluster.map_shared_rank(s, tid)->ahead[rank] = mine;
      cluster.map_shared_rank(s, tid)->all[rank] = its;
    }
    cluster.sync();
    const uint32_t m = *counter;
    ahead = sum = 0;
    for (int r = 0; r < ranks; ++r) {
      ahead += s->ahead[r];
      sum += s->all[r];
    }
    if (m > LIST || !resolve(m, ahead, share_of(share, sum))) return false;
    const u64 cut_place = place_of(s->cut.x, s->cut.i);
    for (uint32_t i = tid; i < m; i += NT) {
      const Entry e = s->list[i];
      const int id = (1 << ID_BITS) - 1 - (int)(e.place & ((1 << ID_BITS) - 1)) - base;
      if (e.place >= cut_place && id >= 0 && id < 8 * eights) atomicAdd(&s->kept[id / 8 / each], e.mass);
    }
    __syncthreads();
    return true;
  }

  __device__ Cut run(cg::cluster_group& cluster, u64 want, float share) {
    count([&](float v, int) { return __float_as_int(stretch(v)) & (BINS - 1); });
    if (find(cluster, 0, true, &want, share) < want) return Cut{-INFINITY, INT_MAX};          // fewer tokens than that
    u64 above = s->above;
    const float bin = MAGIC + s->bin;
    const int lane = tid & 31;
    from = fmaxf(lowest([&](float v) { return stretch(v) <= bin; }, scale > 0.f ? top - (s->bin + 0.5f) / scale : 0.f, top, lane), -3.4028234664e38f);
    below = s->bin ? lowest([&](float v) { return stretch(v) < bin; }, top - (s->bin - 0.5f) / scale, top, lane) : NAN;
    split = false;
    lo = 0;
    hi = (1ull << (32 + ID_BITS)) - 1;
    uint32_t m = gather(cluster);
    for (int shift = 32 + ID_BITS - 10; m > LIST; shift = max(0, shift - 10)) {
      split = true;
      count([&](float v, int id) { return near(v) && member(v, id) ? (int)((hi - place_of(clean(v), id)) >> shift) : -1; });
      find(cluster, above, false, &want, share);
      above = s->above;
      hi -= (u64)s->bin << shift;
      lo = hi - ((1ull << shift) - 1);
      m = gather(cluster);
    }
    resolve(m, above, want);
    return s->cut;
  }
};

template <typename In, bool HELD>
__global__ void __launch_bounds__(NT, 2) draw_kernel(DrawParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared* s = reinterpret_cast<Shared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = rank * p.slice, n = max(0, min(p.slice, p.V - base)), eights = (n + 7) / 8;
  using R = Row<In, HELD>;
  const R tokens{reinterpret_cast<float4*>(raw + (sizeof(Shared) + 15) / 16 * 16), reinterpret_cast<const In*>(p.logits) + (long)row * p.ld + base, n, p.wide ? n / 8 : 0};
  grid_dep_launch();
  if (tid < 2) s->listed[tid] = 0;
  if (tid < PARTS) s->parts[tid] = (u64)(exp2(-(double)tid / PARTS) * 0x1p62) + (1ull << 31);
  auto here = cluster.barrier_arrive();          // the others' memory is written to once they run
  grid_dep_wait();
  float most = -INFINITY;
  auto take = [&](int i, const float4& q) {
    most = fmaxf(fmaxf(most, fmaxf(q.x, q.y)), fmaxf(q.z, q.w));         // (passes over NaN)
    if (HELD) tokens.own[i / 4] = q;
  };
  if constexpr (HELD) {
    constexpr int AT_ONCE = 5;                   // (a row of 160000 over eight CTAs at one go)
    for (int o0 = tid; o0 < tokens.full; o0 += AT_ONCE * NT) {
      float4 a[AT_ONCE], b[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (o0 + k * NT < tokens.full) R::eight(tokens.src + 8 * (o0 + k * NT), a[k], b[k]);
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (o0 + k * NT < tokens.full) {
          take(8 * (o0 + k * NT), a[k]);
          take(8 * (o0 + k * NT) + 4, b[k]);
        }
    }
    for (int i = 8 * tokens.full + tid; i < 8 * eights; i += NT) {
      const float v = i < n ? load_one(tokens.src + i) : -INFINITY;
      reinterpret_cast<float*>(tokens.own)[i] = v;
      most = fmaxf(most, v);
    }
  } else {
    tokens.each(tid, eights, NT, take);
  }
  most = warp_max(most);
  if (lane == 0) s->warp_a[warp] = most;
  __syncthreads();
  most = warp_max(s->warp_a[lane % WARPS]);
  cluster.barrier_wait(std::move(here));
  if (tid < ranks) cluster.map_shared_rank(s, tid)->most[rank] = most;
  cluster.sync();
  for (int r = 0; r < ranks; ++r) most = fmaxf(most, s->most[r]);
  const float it = p.inv_temperature ? p.inv_temperature[row] : 1.f;
  const bool greedy = !(it > 0.f) || it == INFINITY;
  if (greedy || most == -INFINITY) {              // the first of the largest; nothing where everything is masked
    int id = INT_MAX;
    tokens.each(tid, eights, NT, [&](int i, const float4& q) {
      const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v[j] == most && id == INT_MAX) id = base + i + j;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) id = min(id, __shfl_xor_sync(0xffffffffu, id, o));
    if (lane == 0) s->warp_i[warp] = id;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < WARPS; ++i) id = min(id, s->warp_i[i]);
      cluster.map_shared_rank(s, 0)->best[rank] = id;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int r = 1; r < ranks; ++r) id = min(id, s->best[r]);
      const bool none = most == -INFINITY;
      p.out_ids[row] = none ? -1 : id;
      if (p.out_probs) p.out_probs[row] = none ? 0.f : 1.f;
    }
    return;
  }

  const Cut all{-INFINITY, INT_MAX};
  Cut cut = all;
  const Weights w(most, it, s->parts);
  const float scale = most < INFINITY ? fminf(it * ((BINS - 1) / 24.f), 1e30f) : 0.f;         // the bins reach down to weights of e^-24; what lies below is in the last one
  uint32_t turn = 0;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float least_share = p.min_p ? p.min_p[row] : 0.f, share = p.top_p ? p.top_p[row] : 1.f;
  // of a weight limit above 1 the first token is left
  const int count = least_share > 1.f ? 1 : k;
  if (count >= 1 && count < p.V) {
    Search<false, R> f{s, tokens, eights, base, tid, rank, ranks, &turn, all, w, most, scale};
    cut = f.run(cluster, count, 0.f);
  }
  if (least_share > 0.f && least_share <= 1.f) {
    const float v = lowest([&](float x) { return w.real(x) >= (double)least_share; }, (float)((w.z_most + log((double)least_share)) / w.it), most, lane);
    if (v > cut.x) cut = Cut{v, INT_MAX};
  }
  // the kept tokens' masses: a warp's stretch of ids each, so that sums by rising ids need no more than the stretches' sums
  const int each = max(1, (eights + WARPS - 1) / WARPS), first = min(eights, warp * each), last = min(eights, first + each);
  bool summed = false;
  if (share < 1.f) {
    Search<true, R> f{s, tokens, eights, base, tid, rank, ranks, &turn, cut, w, most, scale};
    summed = f.quick(cluster, share, first, last, each);
    cut = summed ? s->cut : f.run(cluster, 0, share);
  }
  const bool everyone = cut.x == -INFINITY;
  // m(j, weight) for the kept ones of a four, maybe in two calls
  auto kept = [&](int i, const float4& q, auto m) {
    const float v[4] = {q.x, q.y, q.z, q.w};
    if (!everyone && !__any_sync(__activemask(), (v[0] >= cut.x) | (v[1] >= cut.x) | (v[2] >= cut.x) | (v[3] >= cut.x))) return;
    bool has[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) has[j] = everyone || cut.has(v[j], base + i + j);
    w.of(v, [&](int j, uint32_t x) { m(j, (u64)(has[j] ? x : 0u)); }, [&](int j, u64 x) { if (has[j]) m(j, x); });
  };
  u64 sum = 0;
  if (!summed) tokens.each(first + lane, last, 32, [&](int i, const float4& q) { kept(i, q, [&](int, u64 x) { sum += x; }); });
  sum = warp_total(sum);
  if (lane == 0) s->warp_sum[warp] = summed ? s->kept[warp] : sum;
  __syncthreads();
  if (tid < ranks) {
    u64 mine = 0;
    for (int i = 0; i < WARPS; ++i) mine += s->warp_sum[i];
    cluster.map_shared_rank(s, tid)->from[rank] = mine;
  }
  const float u = p.uniforms[row];               // ahead of the barrier, as all that is read of the row's: results may lie in its place
  cluster.sync();
  u64 before = 0, total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += s->from[r];
    total += s->from[r];
  }
  const double t = (double)u * (double)total;
  const u64 target = t > 0.0 ? (t < (double)(total - 1) ? (u64)t : total - 1) : 0;      // drawn is the first sum above it
  if (target < before || target >= before + s->from[rank]) return;
  for (int i = 0; i < warp; ++i) before += s->warp_sum[i];
  if (target < before || target >= before + s->warp_sum[warp]) return;
  for (int i0 = 8 * first; i0 < 8 * last && target >= before; i0 += 128) {
    const int i = i0 + 4 * lane;
    u64 m[4] = {0, 0, 0, 0};
    if (i < 8 * last) kept(i, tokens.slow(i), [&](int j, u64 x) { m[j] += x; });
    const u64 mine = (m[0] + m[1]) + (m[2] + m[3]);
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = shfl_up64(incl, o);
      if (lane >= o) incl += x;
    }
    incl += before;
    if (target < incl && target >= incl - mine) {
      u64 run = incl - mine;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (target >= run && target < run + m[j]) {
          p.out_ids[row] = base + i + j;
          if (p.out_probs) p.out_probs[row] = (float)(w.real(tokens.at(i + j)) / ((double)total * 0x1p-44));
        }
        run += m[j];
      }
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
  }
}

template <typename In, bool HELD>
int launch(const DrawParams& p, int ranks, size_t smem, cudaStream_t s) {
  if (int rc = opt_in_smem_once<draw_kernel<In, HELD>>(200 * 1024)) return rc;
  return launch_clusters(true, draw_kernel<In, HELD>, dim3((unsigned)(p.T * ranks)), dim3(NT), (unsigned)ranks, smem, s, p);
}

}  // namespace

extern "C" int ifab_draw(const void* logits, long ld, int f32, int T, int V, const float* inv_temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         const float* uniforms, int32_t* out_ids, float* out_probs, void* stream) {
  if (!logits || !uniforms || !out_ids || T < 1 || T > 1 << 20 || V < 1 || V > MAX_VOCAB || (T > 1 && ld < V)) return -1;
  // As many CTAs a row as run at once, two an SM. Few rows are held in shared memory; of many, a CTA's share does not fit, and is read again from the L2 cache by each pass
  int ranks = MAX_CLUSTER;
  while (ranks > 1 && (V < 1024 * ranks || (long)T * ranks > 296)) ranks /= 2;
  const int slice = ((V + ranks - 1) / ranks + 7) / 8 * 8, size = f32 ? 4 : 2;
  const size_t fixed = (sizeof(Shared) + 15) / 16 * 16, held = fixed + (size_t)slice * sizeof(float), rings = fixed + (size_t)Row<float, false>::AHEAD * NT * 8 * size;
  const bool holds = held <= ((long)T * ranks <= 148 ? 200 : 112) * 1024;
  const bool wide = (uintptr_t)logits % 16 == 0 && (T == 1 || ld * size % 16 == 0);
  const DrawParams p{logits, ld, T, V, slice, wide, inv_temperature, top_p, min_p, uniforms, top_k, out_ids, out_probs};
  cudaStream_t s = (cudaStream_t)stream;
  if (holds) return f32 ? launch<float, true>(p, ranks, held, s) : launch<bf16, true>(p, ranks, held, s);
  return f32 ? launch<float, false>(p, ranks, rings, s) : launch<bf16, false>(p, ranks, rings, s);
}

// A token for every row of logits, drawn from the whole vocabulary with a random number that the caller gives.
//
//   z_i = logit_i / temperature; order: logits falling, ids rising
//   kept: the first top_k; of them those with exp(z_i - z_max) >= min_p; of them the shortest run whose mass reaches top_p of theirs; at least one
//   drawn: the first kept id, ids rising, at which the sum of exp(z - z_max) exceeds u times that of all kept
//
// A row is a cluster of CTAs that keep the row's logits in shared memory: they are read from memory once. What the cuts ask for is a place in the order (the k-th token, the token at
// which the mass passes a share), which is found without a sort: a histogram over the row, equal stretches of the values, says in which of 1024 bins the place lies; the bin's tokens - a
// few - are gathered and put in order by counting. A bin with more tokens than the list takes (ties, values far apart) is split again by the bits of (value, id), 10 at a time.
//
// Weights are e^(z - z_max) in double, summed as integers of 2^-44: the sums decide between tokens, so they must not depend on an order of additions, and a weight below 2^-45 of the
// largest is nothing. 2^18 weights of at most 1 stay below 2^62.
#include <climits>
#include <utility>

#include <cooperative_groups.h>

#include "common.cuh"
#include "ifab_kernels.h"

using namespace ifab;
namespace cg = cooperative_groups;

namespace {

constexpr int NT = 512, WARPS = NT / 32, BINS = 1024, LIST = 1024, MAX_CLUSTER = 8, ID_BITS = 20, PARTS = 32;
constexpr int MAX_VOCAB = 1 << 18, MAX_SLICE = MAX_VOCAB / MAX_CLUSTER;
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
  uint32_t part[3][BINS];                      // this CTA's tokens by bin: their number, or their mass in three words (which its tokens cannot overflow: 17 bits of each, 2^15 tokens)
  Entry list[LIST];
  u64 total[BINS];                             // the row's
  double parts[PARTS];                         // 2^(i / 32)
  uint32_t listed[2];                          // by turns
  u64 from[MAX_CLUSTER];                       // a value of each CTA
  float most[MAX_CLUSTER], least[MAX_CLUSTER];
  int best[MAX_CLUSTER];
  u64 warp_sum[WARPS];
  float warp_a[WARPS], warp_b[WARPS];
  int warp_i[WARPS];
  int bin;
  u64 above;
  Cut cut;
};
static_assert(MAX_SLICE <= 1 << 15, "17 bits of each token's mass in 32");

// of values that are no NaN: unsigned integers in their order
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// (value, id) in the order of the tokens
__device__ __forceinline__ u64 place_of(float v, int id) { return (u64)key_of(v) << ID_BITS | (u64)((1 << ID_BITS) - 1 - id); }

struct Weights {
  float most, floor;           // below `floor` a weight is less than 2^-45
  double it, z_most;
  const double* parts;
  __device__ __forceinline__ Weights(float most, float it_, const double* parts) : most(most), it((double)it_), z_most((double)most * (double)it_), parts(parts) {
    const double lowest = (z_most - 32.0) / it;          // e^-32 < 2^-46
    floor = most == INFINITY ? INFINITY : lowest > -3.4e38 ? __double2float_rd(lowest) : -3.4028234664e38f;
  }
  // of `most` itself 1, an infinite one among them; a product of two floats is exact
  __device__ __forceinline__ double real(float v) const { return v == most ? 1.0 : exp((double)v * it - z_most); }
  // In units of 2^-44, rounded. e^d = 2^(n / 32) e^r, r = d - n ln 2 / 32 of at most 0.011 by Taylor's series up to r^5 / 120 (what it leaves is below 2^-48), without a branch, so that
  // several tokens' chains run side by side: exp() took 25 cycles a token of each lane with 16 warps.
  __device__ __forceinline__ u64 fixed(float v) const {
    const double d = (double)fmaxf(v, floor) * it - z_most;
    const double turn = fma(d, 32 * 1.4426950408889634, 6755399441055744.0);          // 1.5 2^52: the last bits are n
    const int n = (int)__double_as_longlong(turn);
    const double r = fma(turn - 6755399441055744.0, -0.6931471805599453 / 32, d);
    const double e = fma(fma(fma(fma(fma(r, 1.0 / 120, 1.0 / 24), r, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0) * parts[n & (PARTS - 1)];
    const double scaled = __longlong_as_double(__double_as_longlong(e) + ((u64)(long long)(n >> 5) << 52));
    const u64 m = (u64)__double_as_longlong(scaled + 256.0) & ((1ull << 52) - 1);       // 256 + w has its last bit at 2^-44
    return v == most ? 1ull << 44 : v < floor ? 0 : m;
  }
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int by) { return __shfl_up_sync(0xffffffffu, v, by); }
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v + 0.f; }      // a NaN is never drawn; -0 is 0

// The place in the order at which what lies ahead reaches a number of tokens, or a share of their mass
template <bool MASS>
struct Search {
  Shared* s;
  const float4* vals;
  int quads, base, tid, rank, ranks;           // quads: fours of tokens in this CTA; those behind the last one are -inf, with ids that no place reaches
  uint32_t* turn;
  Cut cut;
  Weights w;
  float top, scale;            // bins of equal stretches below `top`
  float first_bin;
  u64 lo, hi;                  // places within first_bin, once it is split
  bool split;

  __device__ __forceinline__ float stretch(float v) const { return scale > 0.f ? fminf((top - v) * scale, (float)(BINS - 1)) : 0.f; }
  __device__ __forceinline__ bool member(float v, int id) const {
    const float at = stretch(v);
    bool in = (at >= first_bin) & (at < first_bin + 1.f) & cut.has(v, id);
    if (split) in = in & (place_of(v, id) >= lo) & (place_of(v, id) <= hi);
    return in;
  }

  template <typename Bin>
  __device__ void count(Bin bin) {
    for (int b = tid; b < BINS * (MASS ? 3 : 1); b += NT) s->part[0][b] = 0;
    __syncthreads();
    for (int c = tid; c < quads; c += NT) {
      const float4 q = vals[c];
      const float v[4] = {q.x, q.y, q.z, q.w};
      u64 m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = MASS ? w.fixed(v[j]) : 1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int id = base + 4 * c + j;
        if (!cut.has(v[j], id)) continue;
        const int b = bin(v[j], id);
        if (b < 0) continue;
        if (!MASS) {
          atomicAdd(&s->part[0][b], 1u);
          continue;
        }
        constexpr uint32_t low = (1u << 17) - 1;
        const uint32_t a0 = (uint32_t)m[j] & low, a1 = (uint32_t)(m[j] >> 17) & low, a2 = (uint32_t)(m[j] >> 34);
        if (a0) atomicAdd(&s->part[0][b], a0);
        if (a1) atomicAdd(&s->part[1][b], a1);
        if (a2) atomicAdd(&s->part[2][b], a2);
      }
    }
  }
  // Sums over the cluster, then the bin at which the order passes the place `want`; `above` counts on from `from`. fresh: `want` follows from `share` and the total
  __device__ void find(cg::cluster_group& cluster, u64 from, bool fresh, u64* want, float share) {
    cluster.sync();
    // each CTA adds up its share of the bins, four threads a bin
    const int lane = tid & 31, warp = tid >> 5, four = tid & 3;
    for (int b = rank * (BINS / ranks) + (tid >> 2); b < (rank + 1) * (BINS / ranks); b += NT / 4) {
      u64 m = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = four + 4 * h;
        if (r < ranks) {
          const Shared* o = cluster.map_shared_rank(s, r);
          m += o->part[0][b];
          if (MASS) m += ((u64)o->part[1][b] << 17) + ((u64)o->part[2][b] << 34);
        }
      }
      m += __shfl_xor_sync(0xffffffffu, m, 1);
      m += __shfl_xor_sync(0xffffffffu, m, 2);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (four + 4 * h < ranks) cluster.map_shared_rank(s, four + 4 * h)->total[b] = m;
    }
    cluster.sync();
    // scan of two bins a thread
    static_assert(BINS == 2 * NT, "two bins a thread");
    const u64 a = s->total[2 * tid], b = s->total[2 * tid + 1];
    u64 sum = a + b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = shfl_up64(sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s->warp_sum[warp] = sum;
    __syncthreads();
    u64 before = from, all = from;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const u64 x = s->warp_sum[i];
      if (i < warp) before += x;
      all += x;
    }
    if (MASS && fresh) {                         // a token is kept while the mass ahead of it is below share * all
      const double t = ceil((double)share * (double)all);
      *want = t < 1.0 ? 1 : t < (double)all ? (u64)t : all;
    }
    const u64 incl = before + sum, mid = incl - b, excl = mid - a;
    if (excl < *want && *want <= incl) {
      const bool second = mid < *want;
      s->bin = 2 * tid + second;
      s->above = second ? mid : excl;
    }
    __syncthreads();
  }
  // the members into every CTA's list; their number (of which the list holds LIST at most)
  __device__ uint32_t gather(cg::cluster_group& cluster) {
    uint32_t* counter = &cluster.map_shared_rank(s, 0)->listed[*turn & 1];
    if (rank == 0 && tid == 0) s->listed[(*turn + 1) & 1] = 0;        // the next turn's; the turn before has been read ahead of a barrier of the cluster
    *turn += 1;
    for (int c = tid; c < quads; c += NT) {
      const float4 q = vals[c];
      const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int id = base + 4 * c + j;
        if (!member(v[j], id)) continue;
        const uint32_t at = atomicAdd(counter, 1u);
        if (at < LIST) {
          const Entry e{place_of(v[j], id), MASS ? w.fixed(v[j]) : 1};
          for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(s, r)->list[at] = e;
        }
      }
    }
    cluster.sync();
    return *counter;
  }

  __device__ Cut run(cg::cluster_group& cluster, u64 want, float share) {
    count([&](float v, int) { return (int)stretch(v); });
    find(cluster, 0, true, &want, share);
    first_bin = (float)s->bin;
    u64 above = s->above;
    split = false;
    lo = 0;
    hi = (1ull << (32 + ID_BITS)) - 1;
    uint32_t m = gather(cluster);
    for (int shift = 32 + ID_BITS - 10; m > LIST; shift = max(0, shift - 10)) {
      split = true;
      count([&](float v, int id) { return member(v, id) ? (int)((hi - place_of(v, id)) >> shift) : -1; });
      find(cluster, above, false, &want, share);
      above = s->above;
      hi -= (u64)s->bin << shift;
      lo = hi - ((1ull << shift) - 1);
      m = gather(cluster);
    }
    for (uint32_t i = tid; i < m; i += NT) {
      const Entry mine = s->list[i];
      u64 ahead = above;
#pragma unroll 8
      for (uint32_t j = 0; j < m; ++j) {
        const Entry e = s->list[j];
        ahead += e.place > mine.place ? e.mass : 0;
      }
      if (ahead < want && want <= ahead + mine.mass) s->cut = Cut{value_of((uint32_t)(mine.place >> ID_BITS)), (1 << ID_BITS) - 1 - (int)(mine.place & ((1 << ID_BITS) - 1))};
    }
    __syncthreads();
    return s->cut;
  }
};

__device__ __forceinline__ float load_one(const float* p) { return __ldcs(p); }
__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void load_eight(const float* p, float (&f)[8]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load_eight(const bf16* p, float (&f)[8]) { unpack8(__ldcs(reinterpret_cast<const uint4*>(p)), f); }

template <typename In>
__global__ void __launch_bounds__(NT, 2) draw_kernel(DrawParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared* s = reinterpret_cast<Shared*>(raw);
  float* vals = reinterpret_cast<float*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  float4* quad = reinterpret_cast<float4*>(vals);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = rank * p.slice, n = max(0, min(p.slice, p.V - base)), quads = (n + 3) / 4;
  grid_dep_launch();
  if (tid < 2) s->listed[tid] = 0;
  if (tid < PARTS) s->parts[tid] = exp2((double)tid / PARTS);
  auto here = cluster.barrier_arrive();          // the others' memory is written to once they run
  grid_dep_wait();
  const In* src = reinterpret_cast<const In*>(p.logits) + (long)row * p.ld + base;
  float most = -INFINITY, least = INFINITY;
  const int whole = p.wide ? n / 8 : 0;
  constexpr int AT_ONCE = 4;
  for (int c0 = tid; c0 < whole; c0 += AT_ONCE * NT) {
    float f[AT_ONCE][8];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (c0 + k * NT < whole) load_eight(src + 8 * (c0 + k * NT), f[k]);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int c = c0 + k * NT;
      if (c >= whole) break;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[k][j] = clean(f[k][j]);
        most = fmaxf(most, f[k][j]);
        if (f[k][j] != -INFINITY) least = fminf(least, f[k][j]);
      }
      quad[2 * c] = make_float4(f[k][0], f[k][1], f[k][2], f[k][3]);
      quad[2 * c + 1] = make_float4(f[k][4], f[k][5], f[k][6], f[k][7]);
    }
  }
  for (int i = 8 * whole + tid; i < 4 * quads; i += NT) {
    const float v = i < n ? clean(load_one(src + i)) : -INFINITY;
    vals[i] = v;
    most = fmaxf(most, v);
    if (v != -INFINITY) least = fminf(least, v);
  }
  most = warp_max(most);
  least = -warp_max(-least);
  if (lane == 0) {
    s->warp_a[warp] = most;
    s->warp_b[warp] = least;
  }
  __syncthreads();
  for (int i = 0; i < WARPS; ++i) {
    most = fmaxf(most, s->warp_a[i]);
    least = fminf(least, s->warp_b[i]);
  }
  cluster.barrier_wait(std::move(here));
  if (tid < ranks) {
    Shared* o = cluster.map_shared_rank(s, tid);
    o->most[rank] = most;
    o->least[rank] = least;
  }
  cluster.sync();
  for (int r = 0; r < ranks; ++r) {
    most = fmaxf(most, s->most[r]);
    least = fminf(least, s->least[r]);
  }
  const float it = p.inv_temperature ? p.inv_temperature[row] : 1.f;
  const bool greedy = !(it > 0.f) || it == INFINITY;
  if (greedy || most == -INFINITY) {              // the first of the largest; nothing where everything is masked
    int id = INT_MAX;
    for (int i = tid; i < n; i += NT)
      if (vals[i] == most) { id = base + i; break; }
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
  const float span = fminf(most, 3.0e38f) - least;
  const float scale = span > 0.f && span < 3.0e38f && most < INFINITY ? (float)(BINS - 1) / span : 0.f;
  uint32_t turn = 0;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float least_share = p.min_p ? p.min_p[row] : 0.f, share = p.top_p ? p.top_p[row] : 1.f;
  // of a weight limit above 1 the first token is left
  const int count = least_share > 1.f ? 1 : k;
  if (count >= 1 && count < p.V) {
    Search<false> f{s, quad, quads, base, tid, rank, ranks, &turn, all, w, most, scale};
    cut = f.run(cluster, count, 0.f);
  }
  if (least_share > 0.f && least_share <= 1.f) {
    // the lowest value whose weight is enough: the predicate is monotone in the value's key, so each lane tries one of 32 places, 32 times finer every round
    uint32_t at = key_of(-INFINITY), step = 1u << 27;         // the value lies in (at, at + 32 steps], or is the largest itself
    const uint32_t end = key_of(most);
    for (int round = 0; round < 7; ++round) {
      const u64 mine = (u64)at + (u64)(lane + 1) * step;
      const bool enough = mine >= end || w.real(value_of((uint32_t)mine)) >= (double)least_share;
      const uint32_t vote = __ballot_sync(0xffffffffu, enough);
      const int first = vote ? __ffs(vote) - 1 : 32;
      at += (uint32_t)first * step;
      step = step >= 32 ? step / 32 : 1;
    }
    const u64 key = (u64)at + 1;
    const float v = key >= end ? most : value_of((uint32_t)key);
    if (v > cut.x) cut = Cut{v, INT_MAX};
  }
  if (share < 1.f) {
    Search<true> f{s, quad, quads, base, tid, rank, ranks, &turn, cut, w, most, scale};
    cut = f.run(cluster, 0, share);
  }

  // the kept tokens' masses: a warp's stretch of ids each, so that sums by rising ids need no more than the stretches' sums
  const int each = (quads + WARPS - 1) / WARPS, first = min(quads, warp * each), last = min(quads, first + each);
  auto kept = [&](int c, u64 (&m)[4]) {
    const float4 q = quad[c];
    const float v[4] = {q.x, q.y, q.z, q.w};
    bool has[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) has[j] = cut.has(v[j], base + 4 * c + j);
    if (__any_sync(__activemask(), has[0] || has[1] || has[2] || has[3])) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[j] = w.fixed(v[j]);
        if (!has[j]) m[j] = 0;
      }
    } else {
      m[0] = m[1] = m[2] = m[3] = 0;
    }
  };
  u64 sum = 0;
  for (int c = first + lane; c < last; c += 32) {
    u64 m[4];
    kept(c, m);
    sum += (m[0] + m[1]) + (m[2] + m[3]);
  }
  sum = warp_total(sum);
  if (lane == 0) s->warp_sum[warp] = sum;
  __syncthreads();
  if (tid < ranks) {
    u64 mine = 0;
    for (int i = 0; i < WARPS; ++i) mine += s->warp_sum[i];
    cluster.map_shared_rank(s, tid)->from[rank] = mine;
  }
  cluster.sync();
  u64 before = 0, total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r < rank) before += s->from[r];
    total += s->from[r];
  }
  const float u = p.uniforms[row];
  const double t = (double)u * (double)total;
  const u64 target = t > 0.0 ? (t < (double)(total - 1) ? (u64)t : total - 1) : 0;      // drawn is the first sum above it
  if (target < before || target >= before + s->from[rank]) return;
  for (int i = 0; i < warp; ++i) before += s->warp_sum[i];
  if (target < before || target >= before + s->warp_sum[warp]) return;
  for (int c0 = first; c0 < last && target >= before; c0 += 32) {
    const int c = c0 + lane;
    u64 m[4] = {0, 0, 0, 0};
    if (c < last) kept(c, m);
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
          p.out_ids[row] = base + 4 * c + j;
          if (p.out_probs) p.out_probs[row] = (float)(w.real(vals[4 * c + j]) / ((double)total * 0x1p-44));
        }
        run += m[j];
      }
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
  }
}

template <typename In>
int launch(const DrawParams& p, int ranks, cudaStream_t s) {
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)p.slice * sizeof(float);
  auto k = draw_kernel<In>;
  if (int rc = opt_in_smem_once<draw_kernel<In>>((sizeof(Shared) + 15) / 16 * 16 + MAX_SLICE * sizeof(float))) return rc;
  return launch_chain_cluster(k, dim3((unsigned)(p.T * ranks)), dim3(NT), (unsigned)ranks, smem, s, p);
}

}  // namespace

extern "C" int ifab_draw(const void* logits, long ld, int f32, int T, int V, const float* inv_temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         const float* uniforms, int32_t* out_ids, float* out_probs, void* stream) {
  if (!logits || !uniforms || !out_ids || T < 1 || T > 1 << 20 || V < 1 || V > MAX_VOCAB || (T > 1 && ld < V)) return -1;
  int ranks = MAX_CLUSTER;
  while (ranks > 1 && V < 1024 * ranks) ranks /= 2;
  const int slice = ((V + ranks - 1) / ranks + 7) / 8 * 8;
  const int size = f32 ? 4 : 2;
  const bool wide = (uintptr_t)logits % 16 == 0 && (T == 1 || ld * size % 16 == 0);
  const DrawParams p{logits, ld, T, V, slice, wide, inv_temperature, top_p, min_p, uniforms, top_k, out_ids, out_probs};
  return f32 ? launch<float>(p, ranks, (cudaStream_t)stream) : launch<bf16>(p, ranks, (cudaStream_t)stream);
}

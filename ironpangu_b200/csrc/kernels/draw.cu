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

constexpr int NT = 512, WARPS = NT / 32, BINS = 1024, LIST = 1024, MAX_CLUSTER = 8, ID_BITS = 20;
constexpr int MAX_VOCAB = 1 << 18;
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
  __device__ __forceinline__ bool has(float v, int id) const { return v > x || (v == x && id <= i); }
};

struct Shared {
  uint32_t cnt[BINS], lo[BINS], hi[BINS];      // this CTA's tokens and their mass (two words)
  uint32_t total_cnt[BINS];                    // the row's
  u64 total[BINS];
  float list_v[LIST];
  int list_id[LIST];
  uint32_t listed;
  u64 from[MAX_CLUSTER];                       // a value of each CTA
  float most[MAX_CLUSTER], least[MAX_CLUSTER];
  int best[MAX_CLUSTER];
  u64 warp_sum[WARPS];
  float warp_a[WARPS], warp_b[WARPS];
  int warp_i[WARPS];
  int bin;
  uint32_t members;
  u64 above;
  Cut cut;
};

// of values that are no NaN: unsigned integers in their order
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// (value, id) in the order of the tokens
__device__ __forceinline__ u64 place_of(float v, int id) { return (u64)key_of(v) << ID_BITS | (u64)((1 << ID_BITS) - 1 - id); }

struct Weights {
  float most;
  double it, z_most;
  // of `most` itself 1, an infinite one among them; a product of two floats is exact
  __device__ __forceinline__ double real(float v) const { return v == most ? 1.0 : exp((double)v * it - z_most); }
  // in units of 2^-44, rounded: 256 + w has its last bit there
  __device__ __forceinline__ u64 fixed(float v) const { return (u64)__double_as_longlong(real(v) + 256.0) & ((1ull << 52) - 1); }
};

__device__ __forceinline__ u64 shfl_up64(u64 v, int by) { return __shfl_up_sync(0xffffffffu, v, by); }
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v + 0.f; }      // a NaN is never drawn; -0 is 0

// Where the row's bins, lowest place first, pass `want(total)`: bin, what lies above it, its tokens
struct Level {
  int bin;
  u64 above;
  uint32_t members;
};

template <bool MASS>
struct Search {
  Shared* s;
  const float* vals;
  int n, base, tid, rank, ranks;
  Cut cut;
  Weights w;
  float top, scale;            // bins of equal stretches below `top`
  int first_bin;
  u64 lo, hi;                  // places within first_bin, once it is split

  __device__ __forceinline__ int stretch(float v) const { return scale > 0.f ? (int)fminf((top - v) * scale, (float)(BINS - 1)) : 0; }

  template <typename Bin>
  __device__ void count(Bin bin) {
    for (int b = tid; b < BINS; b += NT) s->cnt[b] = s->lo[b] = s->hi[b] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const float v = vals[i];
      if (!cut.has(v, base + i)) continue;
      const int b = bin(v, base + i);
      if (b < 0) continue;
      atomicAdd(&s->cnt[b], 1u);
      if (MASS) {
        const u64 m = w.fixed(v);
        const uint32_t part = (uint32_t)m, was = part ? atomicAdd(&s->lo[b], part) : 0u;
        const uint32_t up = (uint32_t)(m >> 32) + (part && was + part < was);
        if (up) atomicAdd(&s->hi[b], up);
      }
    }
  }
  // sums over the cluster, then the bin at which the order passes the place: count `k` (COUNT), or `share` of the mass (MASS). `above` counts on from `from`.
  __device__ Level find(cg::cluster_group& cluster, u64 from, bool fresh, u64* want, float share) {
    cluster.sync();
    const int mine = BINS / ranks;
    for (int j = tid; j < mine; j += NT) {
      const int b = rank * mine + j;
      uint32_t c = 0;
      u64 m = 0;
      for (int r = 0; r < ranks; ++r) {
        const Shared* o = cluster.map_shared_rank(s, r);
        c += o->cnt[b];
        if (MASS) m += ((u64)o->hi[b] << 32) + o->lo[b];
      }
      for (int r = 0; r < ranks; ++r) {
        Shared* o = cluster.map_shared_rank(s, r);
        o->total_cnt[b] = c;
        o->total[b] = MASS ? m : c;
      }
    }
    cluster.sync();
    // scan of two bins a thread
    static_assert(BINS == 2 * NT, "two bins a thread");
    const u64 a = s->total[2 * tid], b = s->total[2 * tid + 1];
    u64 sum = a + b;
    const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = shfl_up64(sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) s->warp_sum[warp] = sum;
    __syncthreads();
    u64 before = from, all = from;
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) before += s->warp_sum[i];
      all += s->warp_sum[i];
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
      s->members = s->total_cnt[2 * tid + second];
    }
    __syncthreads();
    const Level l{s->bin, s->above, s->members};
    return l;
  }
  __device__ __forceinline__ bool member(float v, int id) const {
    const u64 at = place_of(v, id);
    return cut.has(v, id) && stretch(v) == first_bin && at >= lo && at <= hi;
  }

  __device__ Cut run(cg::cluster_group& cluster, u64 want, float share) {
    count([&](float v, int) { return stretch(v); });
    Level l = find(cluster, 0, true, &want, share);
    first_bin = l.bin;
    lo = 0;
    hi = (1ull << (32 + ID_BITS)) - 1;
    for (int shift = 32 + ID_BITS - 10; l.members > LIST; shift = max(0, shift - 10)) {
      __syncthreads();
      count([&](float v, int id) { return member(v, id) ? (int)((hi - place_of(v, id)) >> shift) : -1; });
      l = find(cluster, l.above, false, &want, share);
      hi -= (u64)l.bin << shift;
      lo = hi - ((1ull << shift) - 1);
    }
    uint32_t* counter = &cluster.map_shared_rank(s, 0)->listed;
    for (int i = tid; i < n; i += NT) {
      const float v = vals[i];
      if (!member(v, base + i)) continue;
      const uint32_t at = atomicAdd(counter, 1u);
      if (at < LIST)
        for (int r = 0; r < ranks; ++r) {
          Shared* o = cluster.map_shared_rank(s, r);
          o->list_v[at] = v;
          o->list_id[at] = base + i;
        }
    }
    cluster.sync();
    if (tid == 0) s->listed = 0;                 // (appended to again two cluster barriers from here at the earliest)
    const int m = l.members;
    u64* mass = s->total;                        // LIST <= BINS
    for (int i = tid; i < m; i += NT) mass[i] = MASS ? w.fixed(s->list_v[i]) : 1;
    __syncthreads();
    for (int i = tid; i < m; i += NT) {
      const float v = s->list_v[i];
      const int id = s->list_id[i];
      u64 ahead = l.above;
      for (int j = 0; j < m; ++j)
        if (s->list_v[j] > v || (s->list_v[j] == v && s->list_id[j] < id)) ahead += mass[j];
      if (ahead < want && want <= ahead + mass[i]) s->cut = Cut{v, id};
    }
    __syncthreads();
    return s->cut;
  }
};
static_assert(LIST <= BINS, "the list's masses lie in the bins' place");

__device__ __forceinline__ float load_one(const float* p) { return __ldcs(p); }
__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void load_eight(const float* p, float (&f)[8]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void load_eight(const bf16* p, float (&f)[8]) { unpack8(__ldcs(reinterpret_cast<const uint4*>(p)), f); }

template <typename In>
__global__ void __launch_bounds__(NT) draw_kernel(DrawParams p) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared* s = reinterpret_cast<Shared*>(raw);
  float* vals = reinterpret_cast<float*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int base = rank * p.slice, n = max(0, min(p.slice, p.V - base));
  grid_dep_launch();
  if (tid == 0) s->listed = 0;
  auto here = cluster.barrier_arrive();          // the others' memory is written to once they run
  grid_dep_wait();
  const In* src = reinterpret_cast<const In*>(p.logits) + (long)row * p.ld + base;
  float most = -INFINITY, least = INFINITY;
  const int whole = p.wide ? n / 8 : 0;
  for (int c = tid; c < whole; c += NT) {
    float f[8];
    load_eight(src + 8 * c, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = clean(f[j]);
      most = fmaxf(most, f[j]);
      if (f[j] != -INFINITY) least = fminf(least, f[j]);
    }
    reinterpret_cast<float4*>(vals)[2 * c] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(vals)[2 * c + 1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  for (int i = 8 * whole + tid; i < n; i += NT) {
    const float v = clean(load_one(src + i));
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

  Cut cut{-INFINITY, INT_MAX};
  Weights w{most, (double)it, (double)most * (double)it};
  const float span = fminf(most, 3.0e38f) - least;
  const float scale = span > 0.f && span < 3.0e38f && most < INFINITY ? (float)(BINS - 1) / span : 0.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k >= 1 && k < p.V) {
    Search<false> f{s, vals, n, base, tid, rank, ranks, cut, w, most, scale};
    cut = f.run(cluster, k, 0.f);
  }
  const float least_share = p.min_p ? p.min_p[row] : 0.f;
  if (least_share > 0.f) {
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
    // of a weight limit above 1 the first token is left
    if (1.0 < (double)least_share) cut = Cut{most, -1};
  }
  const float share = p.top_p ? p.top_p[row] : 1.f;
  if (cut.i == -1) {
    Search<false> f{s, vals, n, base, tid, rank, ranks, Cut{-INFINITY, INT_MAX}, w, most, scale};
    cut = f.run(cluster, 1, 0.f);
  } else if (share < 1.f) {
    Search<true> f{s, vals, n, base, tid, rank, ranks, cut, w, most, scale};
    cut = f.run(cluster, 0, share);
  }

  // the kept tokens' masses: a warp's stretch of ids each, so that sums by rising ids need no more than the stretches' sums
  const int stretch = (n + WARPS - 1) / WARPS, first = min(n, warp * stretch), last = min(n, first + stretch);
  u64 sum = 0;
  for (int i = first + lane; i < last; i += 32) {
    const float v = vals[i];
    if (cut.has(v, base + i)) sum += w.fixed(v);
  }
  sum = warp_total(sum);
  if (lane == 0) s->warp_sum[warp] = sum;
  __syncthreads();
  if (tid < ranks) {
    u64 all = 0;
    for (int i = 0; i < WARPS; ++i) all += s->warp_sum[i];
    cluster.map_shared_rank(s, tid)->from[rank] = all;
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
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane;
    const float v = i < last ? vals[i] : -INFINITY;
    const u64 mine = i < last && cut.has(v, base + i) ? w.fixed(v) : 0;
    u64 incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = shfl_up64(incl, o);
      if (lane >= o) incl += x;
    }
    incl += before;
    if (target < incl && target >= incl - mine) {
      p.out_ids[row] = base + i;
      if (p.out_probs) p.out_probs[row] = (float)(w.real(v) / ((double)total * 0x1p-44));
    }
    before = __shfl_sync(0xffffffffu, incl, 31);
    if (target < before) break;
  }
}

template <typename In>
int launch(const DrawParams& p, int ranks, cudaStream_t s) {
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)p.slice * sizeof(float);
  auto k = draw_kernel<In>;
  if (int rc = opt_in_smem(k, smem)) return rc;
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

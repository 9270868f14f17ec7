// Attention of query rows that share a long prefix: the prefix's keys and values are read once for all rows of a group, each row's own ones behind it as usual.
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G],  j = 0 .. pos_t
//   positions j < n of a group's rows lie in the pages of the group's slot, j >= n in those of the row's own slot
//
// A softmax over two parts is put together from their maxima, sums and sums of values, so the parts are worked on by CTAs of their own, as are stretches of a long part; each leaves m, l and O of
// its rows and heads in the scratch.
//
//   tiles kernel     the prefix of a group with much work, on tcgen05 (shared_prefix_tiles.cu)
//   parts kernel     the prefix of the others and the rows' own positions: one CTA per (tile of 16 WM pairs of a group's rows and heads, kv head, stretch of the prefix) and per (row, kv head, stretch
//                    of its own keys): products on the tensor cores as m16n8k16, running maximum and sum in 32 bits, tiles of 64 keys through a ring in shared memory
//   merge kernel     four warps per (row, head): the parts, weighted by e^(m - largest m), over the sum
//   own kernel       where rows fill the chip, in place of the two before it: one CTA, with very many rows one warp, per (row, kv head): its own keys, then the prefix's parts and the result.
//                    Four rows of a question read their keys together: eight questions of 128 rows behind 16384 positions 426 us, without that 450
//
// Behind the tiles kernel the two others start where an SM is free, ahead of its end (PrefixParams::take_over).
//
// How long a prefix is is known on the device only, so both of the first two kernels start where a group might be either's, and one of them has nothing to do. us with the parts kernel and with the
// tiles kernel, rows of 4 heads over each of 8 kv heads, behind 500 / 4000 / 30000 positions: 8 rows 11.7 / 16.3 / 60.8 and 23.5 / 29 / 50, 16 rows 15.6 / 23.1 / 90.5 and 25.0 / 33.2 / 56.4; over 4 kv
// heads 16 rows 15.5 / 18.7 / 51.6 and 24.9 / 29.3 / 37.9. Three groups of 27 rows behind up to 5000 / 9000 / 15000 positions 36 / 51 / 80 and 39 / 41 / 47.
#include <algorithm>
#include <atomic>
#include <chrono>

#include "mma16816.cuh"
#include "shared_prefix.cuh"

using namespace ifab;

namespace {

constexpr int NT = 128, OWN_STAGES = 2, OWN_CTAS = 3;

// What a unit of W warps (a CTA of four, or a warp by itself) has in shared memory: its ring of tiles of 16 W keys, where they lie, and where its pairs' queries and results lie (-1: nobody's)
template <int HD, int W, int PAIRS, int STAGES_>
struct alignas(128) Unit {
  static constexpr int STAGES = STAGES_, KEYS = 16 * W, ROW = HD * 2, CH = HD / 8, STAGE = 2 * KEYS * ROW, RING = STAGES * STAGE;
  unsigned char ring[RING];
  int rows[STAGES + 1][KEYS];
  int whole[STAGES + 1][2];
  float2 ml[W * 16];
  long query[PAIRS], part[PAIRS];
  static_assert(W * 16 * HD * 4 <= RING, "the warps' results take the ring's place");
};

// One stretch of keys [begin, end) of the pages of `slot` against 16 WM pairs. WM warps side by side have 16 pairs each, the others other keys of a tile.
// `pair(i, &t, &h)`: pair i's row and head; false: nobody's. `finish(i, M, L, v)`, by a warp: maxima, sums and sums of values of the pairs from i on, AT_ONCE of them, HD / 32 columns a lane.
// `last(i)`, with EACH: where the keys of pair i end, `least` the first of these ends; keys behind it weigh nothing then. False: so that a value that is not finite must not count, nothing was finished
// The tensor core cuts off what does not fit a sum, 1.1e-8 of it a key (shared_prefix_tiles.cu). FAR: so a tile's sums of values start from 0 and are then added, rounded to nearest, to those of the tiles
// before
template <int HD, int W, int WM, int STAGES, int AT_ONCE, bool EACH, bool FAR, typename Pair, typename Last, typename Finish>
__device__ __forceinline__ bool attend(const PrefixParams& p, Unit<HD, W, 16 * WM, STAGES>& u, int begin, int end, int slot, int kvh, int part, int least, Pair pair, Last last, Finish finish) {
  using U = Unit<HD, W, 16 * WM, STAGES>;
  constexpr int WK = W / WM, KEYS = U::KEYS, KW = KEYS / WK, N = 32 * W, E = HD / 32;      // warps of other keys, keys of a warp, threads of the unit
  const int tid = threadIdx.x % N, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c2 = (lane & 3) * 2;
  const int wm = warp % WM, wk = warp / WM;
  const uint32_t ring = smem_addr(u.ring);
  const long kv_elems = (long)p.Hkv * HD;
  const int tiles = (end - begin + KEYS - 1) / KEYS;
  auto sync = [] {
    if (W == 1) __syncwarp();
    else __syncthreads();
  };
  // Where the keys of tile i lie, a thread a key; -1: nowhere. Asked for at a tile's start and noted at its end: the page table's answer takes as long as the tile
  auto ask = [&](int i) {
    const int key = begin + i * KEYS + tid;
    return tid < KEYS && i < tiles && key < end ? p.row_of(key, slot) : -1;
  };
  auto note = [&](int i, int r) {
    if (warp < (KEYS + 31) / 32 && i < tiles) {
      if (tid < KEYS) u.rows[i % (STAGES + 1)][tid] = r;
      if (tid < KEYS && begin + i * KEYS + tid < end && r < 0 && p.status) atomicOr(p.status, IFAB_STATUS_BAD_INDEX);
      const bool all = __all_sync(0xffffffffu, r >= 0 || tid >= KEYS);
      if (lane == 0) u.whole[i % (STAGES + 1)][warp] = all;
    }
  };
  auto load = [&](int i) {
    if (i < tiles) {
      const uint32_t dst0 = ring + (i % STAGES) * U::STAGE;
      const int ch = tid % U::CH;
#pragma unroll
      for (int j = 0; j < KEYS * U::CH / N; ++j) {
        const int key = tid / U::CH + j * (N / U::CH);
        const int r = u.rows[i % (STAGES + 1)][key];
        const long at = r < 0 ? 0 : r * kv_elems + (long)kvh * HD + ch * 8;
        const uint32_t dst = dst0 + key * U::ROW + ((ch ^ (key & 7)) << 4);
        copy16(dst, p.k_cache + at, r >= 0);
        copy16(dst + KEYS * U::ROW, p.v_cache + at, r >= 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  {
    int r[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES; ++i) r[i] = ask(i);
#pragma unroll
    for (int i = 0; i < STAGES; ++i) note(i, r[i]);
  }
  if (tid >= N - 16 * WM) {
    const int i = tid - (N - 16 * WM);
    int t, h;
    const bool live = pair(i, &t, &h);
    u.query[i] = live ? (long)t * p.ldq + (long)h * HD : -1;
    u.part[i] = live ? p.part_of(t, h, part) : -1;
  }
  sync();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i);

  uint32_t q[HD / 16][4];
  {
    const bf16* src[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const long at = u.query[wm * 16 + g + 8 * e];
      src[e] = at >= 0 ? p.q + at + c2 : nullptr;
    }
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[i][j] = src[j & 1] ? *reinterpret_cast<const uint32_t*>(src[j & 1] + 16 * i + 8 * (j >> 1)) : 0u;
  }
  float acc[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};       // of pairs g and g + 8; maxima in powers of two
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

  int ends[2];                                   // of pairs g and g + 8, from this thread's first key on
#pragma unroll
  for (int e = 0; e < 2; ++e) ends[e] = EACH ? last(wm * 16 + g + 8 * e) - begin - wk * KW - c2 : 0;

  for (int i = 0; i < tiles; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    sync();                                      // tile i has landed for all threads, tile i - 1 is read
    const int ahead = ask(i + STAGES);
    load(i + STAGES - 1);
    const uint32_t kb = ring + (i % STAGES) * U::STAGE + wk * KW * U::ROW, vb = kb + KEYS * U::ROW;
    float s[KW / 8][4];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        uint32_t b[4];
        const int key = n * 16 + (lane >> 4) * 8 + (lane & 7), ch = 2 * kk + ((lane >> 3) & 1);
        ldsm4(kb + key * U::ROW + ((ch ^ (key & 7)) << 4), b);
        mma16816(s[2 * n], q[kk][0], q[kk][1], q[kk][2], q[kk][3], b[0], b[1]);
        mma16816(s[2 * n + 1], q[kk][0], q[kk][1], q[kk][2], q[kk][3], b[2], b[3]);
      }
    const bool all = u.whole[i % (STAGES + 1)][0] && (KEYS <= 32 || u.whole[i % (STAGES + 1)][1]) && (!EACH || begin + (i + 1) * KEYS <= least);
    float mn[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= p.scale_log2;
        if (!all && (u.rows[i % (STAGES + 1)][wk * KW + 8 * n + c2 + (e & 1)] < 0 || (EACH && i * KEYS + 8 * n + (e & 1) >= ends[e >> 1]))) s[n][e] = -INFINITY;
        mn[e >> 1] = fmaxf(mn[e >> 1], s[n][e]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mn[e] = fmaxf(mn[e], __shfl_xor_sync(0xffffffffu, mn[e], 1));
      mn[e] = fmaxf(mn[e], __shfl_xor_sync(0xffffffffu, mn[e], 2));
    }
    if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float corr = mn[e] > m[e] ? exp2f(m[e] - mn[e]) : 1.f;
        l[e] *= corr;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
          acc[j][2 * e] *= corr;
          acc[j][2 * e + 1] *= corr;
        }
        m[e] = mn[e];
      }
    }
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = s[n][e] == -INFINITY ? (EACH ? 0.f : PREFIX_LEAST_WEIGHT) : prefix_weight(s[n][e] - m[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    auto terms = [&](int kk, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) two_terms<EACH>(s[2 * kk + (j >> 1)][2 * (j & 1)], s[2 * kk + (j >> 1)][2 * (j & 1) + 1], &hi[j], &lo[j]);
    };
    auto products = [&](int kk, int j, const uint32_t (&hi)[4], const uint32_t (&lo)[4], float (&even)[4], float (&odd)[4]) {
      uint32_t b[4];
      const int key = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), ch = 2 * j + (lane >> 4);
      ldsm4t(vb + key * U::ROW + ((ch ^ (key & 7)) << 4), b);
      mma16816(even, hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
      mma16816(odd, hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
      mma16816(even, lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
      mma16816(odd, lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
    };
    if constexpr (!FAR) {
#pragma unroll
      for (int kk = 0; kk < KW / 16; ++kk) {
        uint32_t hi[4], lo[4];
        terms(kk, hi, lo);
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) products(kk, j, hi, lo, acc[2 * j], acc[2 * j + 1]);
      }
    } else {
      uint32_t hi[KW / 16][4], lo[KW / 16][4];
#pragma unroll
      for (int kk = 0; kk < KW / 16; ++kk) terms(kk, hi[kk], lo[kk]);
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        float even[4] = {}, odd[4] = {};
#pragma unroll
        for (int kk = 0; kk < KW / 16; ++kk) products(kk, j, hi[kk], lo[kk], even, odd);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[2 * j][e] += even[e];
          acc[2 * j + 1][e] += odd[e];
        }
      }
    }
    __syncwarp();
    note(i + STAGES, ahead);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  // by pairs, over the ring: warps of the same pairs and other keys are added up
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (EACH) {
    float finite = 0.f;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) finite = fmaf(acc[j][e], 0.f, finite);
    if (__syncthreads_or(finite != 0.f)) return false;
  } else {
    sync();
  }
  float* all_acc = reinterpret_cast<float*>(u.ring);
  float* my_acc = all_acc + warp * 16 * HD;
  if ((lane & 3) == 0) {
    u.ml[warp * 16 + g] = prefix_sums(m[0], l[0]);
    u.ml[warp * 16 + g + 8] = prefix_sums(m[1], l[1]);
  }
#pragma unroll
  for (int j = 0; j < HD / 8; ++j) {
    *reinterpret_cast<float2*>(my_acc + g * HD + 8 * j + c2) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2*>(my_acc + (g + 8) * HD + 8 * j + c2) = make_float2(acc[j][2], acc[j][3]);
  }
  sync();
  for (int i0 = warp * AT_ONCE; i0 < 16 * WM; i0 += W * AT_ONCE) {
    bool any = false;
#pragma unroll
    for (int n = 0; n < AT_ONCE; ++n) any = any || u.part[i0 + n] >= 0;
    if (!any) continue;
    float M[AT_ONCE], L[AT_ONCE], v[AT_ONCE][E];
#pragma unroll
    for (int n = 0; n < AT_ONCE; ++n) {
      const int i = i0 + n;
      float w[WK];
      M[n] = -INFINITY;
      L[n] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[n][e] = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) M[n] = fmaxf(M[n], w[k] = u.ml[(k * WM + i / 16) * 16 + i % 16].x);
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        const int at = (k * WM + i / 16) * 16 + i % 16;
        w[k] = w[k] == -INFINITY ? 0.f : exp2f(w[k] - M[n]);
        if (w[k] == 0.f) continue;               // nothing, or an infinite value that weighs nothing
        L[n] += w[k] * u.ml[at].y;
#pragma unroll
        for (int e = 0; e < E; ++e) v[n][e] += w[k] * all_acc[at * HD + lane * E + e];
      }
    }
    finish(i0, M, L, v);
  }
  return true;
}
struct NoLast {
  __device__ int operator()(int) const { return 0; }
};

template <int E>
__device__ __forceinline__ void store_part(const PrefixParams& p, long at, float M, float L, const float (&v)[E], int lane) {
  if (E == 4) *reinterpret_cast<float4*>(p.parts + at * (32 * E) + lane * E) = make_float4(v[0], v[1], v[E - 2], v[E - 1]);
  else *reinterpret_cast<float2*>(p.parts + at * (32 * E) + lane * E) = make_float2(v[0], v[1]);
  if (lane == 0) p.sums[at] = make_float2(M, L);
}
__device__ __forceinline__ float largest(const PrefixParams& p, long base, int n, int lane) {
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, p.sums[base + i].x);
  return warp_max(M);
}
// Adds parts [first, last) of P pairs, each of them from `base` on (negative: nobody's), to the L and v of a warp, relative to M, which is not below their maxima: S parts of each pair are requested
// together. Parts that weigh nothing count as nothing, whatever they hold
template <int E, int P, int S>
__device__ __forceinline__ void add_parts(const PrefixParams& p, const long (&base)[P], int first, int last, const float (&M)[P], float (&L)[P], float (&v)[P][E], int lane) {
  for (int i0 = first; i0 < last; i0 += 32) {
    float w[P];
    uint32_t left = 0;
#pragma unroll
    for (int n = 0; n < P; ++n) {
      const float2 ml = base[n] >= 0 && i0 + lane < last ? p.sums[base[n] + i0 + lane] : make_float2(-INFINITY, 0.f);
      w[n] = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M[n]);
      const float l = w[n] != 0.f ? w[n] * ml.y : 0.f;
      L[n] += warp_sum(l);
      left |= __ballot_sync(0xffffffffu, w[n] != 0.f);
    }
    const int some = left ? __ffs(left) - 1 : 0;         // what a place without a part reads, to no effect: loads that depend on nothing stay together
    while (left) {
      float a[P][S][E], by[P][S];
#pragma unroll
      for (int k = 0; k < S; ++k) {
        const int j = left ? __ffs(left) - 1 : some;
#pragma unroll
        for (int n = 0; n < P; ++n) {
          by[n][k] = __shfl_sync(0xffffffffu, w[n], j);
          if (!left) by[n][k] = 0.f;
          const float* src = p.parts + (max(base[n], 0l) + i0 + j) * (32 * E) + lane * E;
          if (E == 4) *reinterpret_cast<float4*>(a[n][k]) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(a[n][k]) = *reinterpret_cast<const float2*>(src);
        }
        left &= left - 1;
      }
#pragma unroll
      for (int n = 0; n < P; ++n)
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) v[n][e] = by[n][k] != 0.f ? fmaf(by[n][k], a[n][k][e], v[n][e]) : v[n][e];
    }
  }
}
template <int E>
__device__ __forceinline__ void store_result(bf16* dst, float L, const float (&v)[E], int lane) {
  const float inv = L != 0.f ? 1.f / L : 0.f;      // (a NaN among the scores stays one)
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<__nv_bfloat162*>(dst + lane * E + e) = __floats2bfloat162_rn(v[e] * inv, v[e + 1] * inv);
}

// Items: those of prefixes (stretch fastest, then kv head, then tile), then own ones (stretch, kv head, row). Every part of a row that is somebody's gets its sums, if only to say that it is nothing,
// so that the merge need not know about groups
template <int HD, int WM, bool FAR>
__device__ __forceinline__ void part_item(const PrefixParams& p, int item, int prefix_items, unsigned char* smem) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const float2 nothing = make_float2(-INFINITY, 0.f);
  if (item < prefix_items) {
    const int split = item % p.part_splits, kvh = item / p.part_splits % p.Hkv;
    int tile = item / p.part_splits / p.Hkv, end = 0;
    PrefixGroup gr;
    for (int i = 0;; ++i) {
      if (i == p.groups) return;
      gr = p.group(i, &end);
      const int tiles = (gr.rows * p.G + 16 * WM - 1) / (16 * WM);
      if (tile < tiles) break;
      tile -= tiles;
    }
    if (p.by_tiles()) return;
    const int per = p.per_split(gr.shared, p.part_splits), begin = split * per, x0 = tile * 16 * WM;
    for (int x = x0 + threadIdx.x; x < min(x0 + 16 * WM, gr.rows * p.G); x += NT) {
      const int t = gr.first + x / p.G;
      const long at = p.part_of(t, kvh * p.G + x % p.G, split);
      if (begin >= gr.shared || !p.sees(gr, t)) p.sums[at] = nothing;
      if (split == 0)
        for (int i = p.part_splits; i < p.prefix_parts; ++i) p.sums[at + i] = nothing;
    }
    if (begin >= gr.shared) return;
    auto& u = *reinterpret_cast<Unit<HD, 4, 16 * WM, 3>*>(smem);
    attend<HD, 4, WM, 3, 1, false, FAR>(
        p, u, begin, begin + min(per, gr.shared - begin), gr.slot, kvh, split, 0,
        [&](int i, int* t, int* h) {
          const int x = x0 + i;
          if (x >= gr.rows * p.G) return false;
          *t = gr.first + x / p.G;
          *h = kvh * p.G + x % p.G;
          return p.sees(gr, *t);
        },
        NoLast{},
        [&](int i, const float (&M)[1], const float (&L)[1], const float (&v)[1][E]) { store_part<E>(p, u.part[i], M[0], L[0], v[0], lane); });
  } else {
    item -= prefix_items;
    const int split = item % p.own_splits, kvh = item / p.own_splits % p.Hkv, t0 = item / p.own_splits / p.Hkv;
    const PrefixGroup gr = p.naming(t0);
    const PrefixOwn own = p.own(t0, gr);
    const int per = p.per_split(own.end - own.begin, p.own_splits), begin = own.begin + split * per;
    if (p.positions[t0] < 0) return;
    if (!gr.rows && split == 0)
      for (int i = threadIdx.x; i < p.G * p.prefix_parts; i += NT) p.sums[p.part_of(t0, kvh * p.G + i / p.prefix_parts, i % p.prefix_parts)] = nothing;
    if (begin >= own.end) {
      for (int i = threadIdx.x; i < p.G; i += NT) p.sums[p.part_of(t0, kvh * p.G + i, p.prefix_parts + split)] = nothing;
      return;
    }
    auto& u = *reinterpret_cast<Unit<HD, 4, 16, 3>*>(smem);
    attend<HD, 4, 1, 3, 1, false, FAR>(
        p, u, begin, begin + min(per, own.end - begin), own.slot, kvh, p.prefix_parts + split, 0,
        [&](int i, int* t, int* h) {
          *t = t0;
          *h = kvh * p.G + i;
          return i < p.G;
        },
        NoLast{},
        [&](int i, const float (&M)[1], const float (&L)[1], const float (&v)[1][E]) { store_part<E>(p, u.part[i], M[0], L[0], v[0], lane); });
  }
}

template <int HD, int WM, bool FAR>
__global__ void __launch_bounds__(NT, 2) prefix_parts_kernel(PrefixParams p, int prefix_items) {
  extern __shared__ __align__(16) unsigned char smem[];
  grid_dep_launch();
  p.take_over();                                   // (the parts of the tiles kernel are of other places)
  part_item<HD, WM, FAR>(p, blockIdx.x, prefix_items, smem);
  grid_dep_wait();                               // that this kernel has ended says that the one ahead has
}

// four warps per (row, head), a stretch of its parts each
template <int HD>
__global__ void __launch_bounds__(NT) prefix_merge_kernel(PrefixParams p, bf16* out, long ldo) {
  constexpr int E = HD / 32, W = NT / 32;
  __shared__ float sm[W][HD], sm_l[W];
  grid_dep_launch();
  grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq;
  const long base = p.part_of(t, h, 0);
  const int n = p.prefix_parts + p.own_splits, each = (n + W - 1) / W;
  const float M[1] = {largest(p, base, n, lane)};
  const long bases[1] = {base};
  if (p.positions[t] < 0) return;
  float part[1][E] = {}, sum[1] = {0.f};
  add_parts<E, 1, 8>(p, bases, min(n, warp * each), min(n, (warp + 1) * each), M, sum, part, lane);
  float L = sum[0];
  float(&v)[E] = part[0];
#pragma unroll
  for (int e = 0; e < E; ++e) sm[warp][lane * E + e] = v[e];
  if (lane == 0) sm_l[warp] = L;
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int k = 1; k < W; ++k) {
    L += sm_l[k];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += sm[k][lane * E + e];
  }
  store_result<E>(out + (long)t * ldo + (long)h * HD, L, v, lane);
}

// Results of P pairs over kv head `kvh` from pair j of the rows from t0 on: their own sums M, L and `mine`, and `parts` that the prefix's kernel left of each from bases[n] on (negative: nobody's)
template <int E, int P, int S>
__device__ __forceinline__ void finish_pairs(const PrefixParams& p, bf16* out, long ldo, long t0, int kvh, int j, const long* bases, int parts, const float (&M)[P], const float (&L)[P],
                                             const float (&mine)[P][E], int lane) {
  long base[P];
  float top[P], sum[P], v[P][E];
  grid_dep_wait();
#pragma unroll
  for (int n = 0; n < P; ++n) base[n] = bases[n];
#pragma unroll
  for (int n = 0; n < P; ++n) top[n] = base[n] >= 0 ? fmaxf(M[n], largest(p, base[n], parts, lane)) : 0.f;
#pragma unroll
  for (int n = 0; n < P; ++n) {
    const float w = M[n] == -INFINITY ? 0.f : exp2f(M[n] - top[n]);
    sum[n] = w != 0.f ? w * L[n] : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[n][e] = w != 0.f ? w * mine[n][e] : 0.f;
  }
  add_parts<E, P, S>(p, base, 0, parts, top, sum, v, lane);
#pragma unroll
  for (int n = 0; n < P; ++n)
    if (base[n] >= 0) store_result<E>(out + (t0 + (j + n) / p.G) * ldo + (long)(kvh * p.G + (j + n) % p.G) * (32 * E), sum[n], v[n], lane);
}

// The row's own keys, what the prefix's kernel left, the result: four warps per (row, kv head), or (W = 1) a warp. With W = 1 a CTA has a kv head of four rows where these are of one sequence, as a
// question's are: they read its keys together, as 16 WM pairs that each see their own positions. Else it has four kv heads of one row, or as near to that as their number allows: warps of one length
template <int HD, int W, int WM, bool FAR>
__global__ void __launch_bounds__(NT, OWN_CTAS) prefix_own_kernel(PrefixParams p, bf16* out, long ldo) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int E = HD / 32, ROWS = 4 / W, P = W == 1 ? 4 : 1, S = W == 1 ? 2 : 8;
  // The tiles kernel's parts are read, and results written, behind the wait
  grid_dep_launch();
  p.take_over();
  const int lane = threadIdx.x & 31, unit = threadIdx.x / (32 * W), c = blockIdx.x % p.Hkv;
  const long t0 = (long)(blockIdx.x / p.Hkv) * ROWS;
  int r = (c * ROWS + unit) / p.Hkv, kvh = (c * ROWS + unit) % p.Hkv;
  PrefixOwn own{0, 0, -1};                       // of row r, with W = 1 of row lane % 4 to begin with
  int parts = -1;                                // that the prefix's kernel left of it; -1: nobody's row
  const long t = t0 + (W == 1 ? lane % ROWS : 0);
  if (t < p.T && p.positions[t] >= 0) {
    const PrefixGroup gr = p.naming((int)t);
    const int per = p.per_tile_split(gr.shared);
    own = p.own((int)t, gr);
    parts = p.sees(gr, (int)t) ? (gr.shared + per - 1) / per * 2 : 0;
  }
  if constexpr (W == 1) {
    constexpr uint32_t ALL = 0xffffffffu;
    const uint32_t live = __ballot_sync(ALL, parts >= 0);
    if (!live) {
      grid_dep_wait();                           // (as every path does: that this kernel has ended says that the one ahead has)
      return;
    }
    const int leader = __ffs(live) - 1, begin = __shfl_sync(ALL, own.begin, leader), slot = __shfl_sync(ALL, own.slot, leader), left = __shfl_sync(ALL, parts, leader);
    if (__all_sync(ALL, parts < 0 || (own.begin == begin && own.slot == slot && parts == left)) && (live & 15) > (live & -live)) {
      auto& u = *reinterpret_cast<Unit<HD, 4, 16 * WM, OWN_STAGES>*>(smem);
      if (attend<HD, 4, WM, OWN_STAGES, P, true, FAR>(
              p, u, begin, __reduce_max_sync(ALL, own.end), slot, c, 0, __reduce_min_sync(ALL, parts >= 0 ? own.end : 0x7fffffff),
              [&](int i, int* t, int* h) {
                *t = (int)t0 + i / p.G;
                *h = c * p.G + i % p.G;
                return i < ROWS * p.G && (live >> i / p.G & 1);
              },
              [&](int i) { return __shfl_sync(ALL, own.end, i / p.G % ROWS); },          // (of nobody's pairs: anything)
              [&](int i, const float (&M)[P], const float (&L)[P], const float (&v)[P][E]) {
                finish_pairs<E, P, S>(p, out, ldo, t0, c, i, u.part + i, left, M, L, v, lane);
              }))
        return;
      r = unit;
      kvh = c;
    }
    own = PrefixOwn{__shfl_sync(ALL, own.begin, r), __shfl_sync(ALL, own.end, r), __shfl_sync(ALL, own.slot, r)};
    parts = __shfl_sync(ALL, parts, r);
  }
  if (parts < 0) {
    grid_dep_wait();
    return;
  }
  auto& u = reinterpret_cast<Unit<HD, W, 16, OWN_STAGES>*>(smem)[unit];
  attend<HD, W, 1, OWN_STAGES, P, false, FAR>(
      p, u, own.begin, own.end, own.slot, kvh, 0, 0,
      [&](int i, int* t, int* h) {
        *t = (int)t0 + r;
        *h = kvh * p.G + i;
        return i < p.G;
      },
      NoLast{},
      [&](int i, const float (&M)[P], const float (&L)[P], const float (&mine)[P][E]) {
        finish_pairs<E, P, S>(p, out, ldo, t0, kvh, r * p.G + i, u.part + i, parts, M, L, mine, lane);
      });
}

// how a call is shared out
struct Plan {
  int wm;                                // tiles of 16 wm pairs by the parts kernel; 0: none of a prefix
  bool tiles;                            // by the tiles kernel
  int own_warps;                         // of the own kernel's units; 0: own parts by the parts kernel, and a merge
  int part_tiles, part_splits, tile_tiles, tile_splits, tile_share, tile_shares, own_splits;
  long tiles_from;
  bool far;                              // a warp may have more keys than it adds up in one sum
  int prefix_parts() const { return std::max(part_splits, 2 * tile_splits); }
};
// `most`: positions that a slot has room for
Plan plan_of(int T, int Hkv, int G, int head_dim, int groups, bool tcgen05, long most) {
  Plan a{};
  auto splits = [](long items, long ctas, int most) { return (int)std::max(1l, std::min((long)most, ctas / std::max(1l, items))); };
  auto tiles = [&](int pairs) { return groups ? (int)std::max((long)groups, ((long)T * G - groups) / pairs + groups) : 0; };          // at most, however the rows are shared out
  const long items = (long)T * Hkv;
  const int rows = groups ? (T + groups - 1) / groups * G : 1;
  const bool full = items >= 400;
  a.wm = !groups || (tcgen05 && full) ? 0 : rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  // One wave: 148 CTAs of the prefix and as many of the rows' own positions side by side, two an SM; the tiles kernel's have an SM each
  if (a.wm) {
    a.part_tiles = tiles(16 * a.wm);
    a.part_splits = splits((long)a.part_tiles * Hkv, 148, 148);
  }
  // The parts kernel takes as long as the longest prefix is, times the tiles that there may be, and is as fast as the tiles kernel at 3.1 to 5.5 million pairs by positions of 128 columns
  const long pairs = 16l * a.wm * a.part_tiles * Hkv;
  a.tiles_from = !tcgen05 ? 1l << 62 : full ? 0 : 3500000l * 128 / head_dim / std::max(1l, pairs);
  a.tiles = groups && most >= a.tiles_from;
  if (a.tiles) {
    a.tile_tiles = tiles(256);
    // Stretches for whole waves of 148 CTAs. SMs that a wave leaves over have short stretches, by up to four turns: us behind 16384 positions with and without them, rows of
    // 16 heads over 4, two turns (56 items) 190 and 216, three (100) 335 and 404, four (116) 371 and 413, (64) 222 and 220; of 32 over 8 by seven turns (128) 442 and 426. Behind 5000 positions 104 and 103,
    // 180 and 173, 200 and 182, 123 and 107: how long a prefix is is known on the device only, and here it is taken for long. 400 rows of 128 heads over 8 (200 items) in two stretches 623, in one 770.
    // Groups have half a tile less than they may have each, on the average
    const long items = (long)a.tile_tiles * Hkv, likely = std::max(1l, (long)(a.tile_tiles - groups / 2) * Hkv);
    a.tile_share = a.tile_shares = a.tile_splits = 1;
    if (items <= 148) {
      const int n = (int)(148 / items), left = (int)(148 - n * items), turns = left ? (int)((items + left - 1) / left) : 0;
      const bool more = turns && turns <= 4 && n * turns < 12;
      a.tile_splits = n + more;
      a.tile_share = more ? turns : 1;
      a.tile_shares = more ? n * turns + 1 : n;
    } else {
      float best = 1e30f;
      for (int n = 1; n <= 3; ++n) {
        const float time = (float)((likely * n + 147) / 148) / n + 0.05f * n;
        if (time < best) {
          best = time;
          a.tile_splits = a.tile_shares = n;
        }
      }
    }
  }
  a.own_splits = splits(items, a.tiles ? 296 : 148, 16);
  // us of a call with four warps and with one, 32 heads over 8, behind 2000 positions: rows with up to 100 own ones, 160 of them 52.9 and 48.7, 256 of them 77.5 and 68.8; with up to 800, 99 and 130,
  // 138 and 156; questions of 32 rows, five, 52.5 and 43.2, of 128 rows, two with up to 700, 116 and 68 (without blocks 118). Own positions are taken for few here: how many they are is known on
  // the device only, and rows of the many have one unit all the same (256 rows with 4000 own ones each 1010 us, 150 rows of which one is in no group and at position 30000 2455)
  a.own_warps = !a.tiles || !full ? 0 : items < 1184 ? 4 : 1;
  // Keys of a warp of the parts and the own kernels at most, by the room that slots have. With sums of a tile each 8 rows behind 4000 positions take 15.6 us, without 14.5
  const long prefix = a.wm ? std::min(most, a.tiles_from) / a.part_splits * a.wm / 4 : 0, own = most / a.own_splits / (a.own_warps == 1 ? 1 : 4);
  a.far = std::max(prefix, own) > 2048;
  return a;
}

template <int HD, int WM, bool FAR>
int launch_parts(const PrefixParams& p, long prefix_items, cudaStream_t s) {
  auto k = prefix_parts_kernel<HD, WM, FAR>;
  constexpr int smem = std::max(sizeof(Unit<HD, 4, 16 * WM, 3>), sizeof(Unit<HD, 4, 16, 3>));
  if (int rc = opt_in_smem_once<prefix_parts_kernel<HD, WM, FAR>>(smem)) return rc;
  const long items = prefix_items + (long)p.T * p.Hkv * p.own_splits;
  if (items > 0x7fffffff) return -1;
  return launch_chain(k, dim3((unsigned)items), dim3(NT), (size_t)smem, s, p, (int)prefix_items);
}
template <int HD, int W, int WM, bool FAR>
int launch_own(const PrefixParams& p, bf16* out, long ldo, cudaStream_t s) {
  auto k = prefix_own_kernel<HD, W, WM, FAR>;
  constexpr int rows = 4 / W, smem = std::max(rows * sizeof(Unit<HD, W, 16, OWN_STAGES>), sizeof(Unit<HD, 4, 16 * WM, OWN_STAGES>));
  if (int rc = opt_in_smem_once<prefix_own_kernel<HD, W, WM, FAR>>(smem)) return rc;
  return launch_chain(k, dim3((unsigned)((long)(p.T + rows - 1) / rows * p.Hkv)), dim3(NT), (size_t)smem, s, p, out, ldo);
}
template <int HD, bool FAR>
int launch_rest(const PrefixParams& p, const Plan& a, bf16* out, long ldo, cudaStream_t s) {
  if (a.own_warps == 4) return launch_own<HD, 4, 1, FAR>(p, out, ldo, s);
  if (a.own_warps == 1) return p.G <= 4 ? launch_own<HD, 1, 1, FAR>(p, out, ldo, s) : p.G <= 8 ? launch_own<HD, 1, 2, FAR>(p, out, ldo, s) : launch_own<HD, 1, 4, FAR>(p, out, ldo, s);
  const long parts = (long)a.part_tiles * p.Hkv * a.part_splits;
  if (int rc = a.wm == 4 ? launch_parts<HD, 4, FAR>(p, parts, s) : a.wm == 2 ? launch_parts<HD, 2, FAR>(p, parts, s) : launch_parts<HD, 1, FAR>(p, parts, s)) return rc;
  return launch_chain(prefix_merge_kernel<HD>, dim3((unsigned)((long)p.T * p.Hq)), dim3(NT), 0, s, p, out, ldo);
}
template <int HD>
int launch(const PrefixParams& p, const Plan& a, bf16* out, long ldo, cudaStream_t s) {
  const long tiles = (long)a.tile_tiles * p.Hkv;
  if ((long)a.part_tiles * p.Hkv * a.part_splits > 0x7fffffff || tiles * a.tile_splits > 0x7fffffff || (long)p.T * p.Hq > 0x7fffffff) return -1;
  if (a.tiles)
    if (int rc = launch_prefix_tiles(p, HD, tiles, s)) return rc;
  return a.far ? launch_rest<HD, true>(p, a, out, ldo, s) : launch_rest<HD, false>(p, a, out, ldo, s);
}

// Not 0, another one each time, and nothing that a scratch holds by chance: a count from the clock on, its bits mixed
unsigned long long next_number() {
  static std::atomic<uint64_t> calls{(uint64_t)std::chrono::system_clock::now().time_since_epoch().count()};
  uint64_t x = calls.fetch_add(1, std::memory_order_relaxed) * 0x9e3779b97f4a7c15ull;
  x = (x ^ (x >> 32)) * 0xd6e8feb86659fd93ull;
  return (x ^ (x >> 32)) | 1;
}

}  // namespace

extern "C" uint64_t ifab_shared_prefix_scratch(int T, int Hq, int Hkv, int head_dim, int groups) {
  if (T < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || groups < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  int most = 0;
  for (int with = 0; with < 2; ++with) {         // whatever the pages
    const Plan a = plan_of(T, Hkv, Hq / Hkv, head_dim, groups, with, 0x7fffffff);
    most = std::max(most, a.prefix_parts() + a.own_splits);
  }
  return ((uint64_t)T * Hq * most * (head_dim + 2) * sizeof(float) + sizeof(uint64_t) + 15) / 16 * 16;
}

extern "C" uint64_t ifab_shared_prefix_scratch_up_to(int T, int Hq, int Hkv, int head_dim, int groups) {
  uint64_t most = 0;
  for (int t = 1; t <= T; ++t) most = std::max(most, ifab_shared_prefix_scratch(t, Hq, Hkv, head_dim, groups));
  return most;
}

extern "C" int ifab_shared_prefix_launches(int T, int Hq, int Hkv, int head_dim, int groups, int page_tokens, int max_pages) {
  if (T < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || groups < 0 || (head_dim != 64 && head_dim != 128) || page_tokens < 1 || max_pages < 1) return -1;
  const Plan a = plan_of(T, Hkv, Hq / Hkv, head_dim, groups, page_tokens % 8 == 0, (long)max_pages * page_tokens);
  return a.tiles + (a.own_warps ? 1 : 2);
}

extern "C" int ifab_shared_prefix_attention(const void* q, long ldq, const void* k_cache, const void* v_cache, const int32_t* positions, const int32_t* slots, const int32_t* page_table,
                                            int num_slots, int max_pages, int page_tokens, int num_pages, const int32_t* groups, int num_groups, float scale, int T, int Hq, int Hkv,
                                            int head_dim, void* scratch, uint64_t scratch_bytes, void* out, long ldo, uint32_t* status, void* stream) {
  if (!(scale > 0.f) || scale > 2.35e38f) return -1;           // as a factor of powers of two it is finite
  if (!q || !k_cache || !v_cache || !positions || !slots || !page_table || !scratch || !out) return -1;
  if (T < 1 || T > 1 << 20 || Hkv < 1 || Hq < 1 || Hq % Hkv || Hq / Hkv > 16 || (head_dim != 64 && head_dim != 128) || num_groups < 0 || num_groups > 64 || (num_groups && !groups)) return -1;
  if (num_slots < 1 || max_pages < 1 || page_tokens < 1 || num_pages < 1 || (long)num_pages * page_tokens > 0x7fffffff || (long)max_pages * page_tokens > 0x7fffffff - 256) return -1;
  if (ldq % 8 || ldo % 8 || ((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)scratch | (uintptr_t)groups) % 16) return -1;
  const Plan a = plan_of(T, Hkv, Hq / Hkv, head_dim, num_groups, page_tokens % 8 == 0, (long)max_pages * page_tokens);
  if (ifab_shared_prefix_scratch(T, Hq, Hkv, head_dim, num_groups) > scratch_bytes) return -5;
  PrefixParams p;
  p.q = (const bf16*)q; p.ldq = ldq; p.k_cache = (const bf16*)k_cache; p.v_cache = (const bf16*)v_cache;
  p.positions = positions; p.slots = slots; p.page_table = page_table; p.group_list = groups;
  p.num_slots = num_slots; p.max_pages = max_pages; p.page_tokens = page_tokens; p.num_pages = num_pages; p.groups = num_groups;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  p.part_splits = a.part_splits; p.tile_splits = a.tile_splits; p.own_splits = a.own_splits; p.prefix_parts = a.prefix_parts(); p.tiles_from = a.tiles_from;
  p.tile_share = a.tile_share; p.tile_shares = std::max(1, a.tile_shares);
  p.parts = (float*)scratch;
  p.sums = (float2*)((float*)scratch + (uint64_t)T * Hq * (a.prefix_parts() + a.own_splits) * head_dim);
  p.status = status;
  p.word = (unsigned long long*)(p.sums + (uint64_t)T * Hq * (a.prefix_parts() + a.own_splits));
  p.number = a.tiles ? next_number() : 0;
  return head_dim == 64 ? launch<64>(p, a, (bf16*)out, ldo, (cudaStream_t)stream) : launch<128>(p, a, (bf16*)out, ldo, (cudaStream_t)stream);
}

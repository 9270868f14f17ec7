// Attention of query rows that share a long prefix: the prefix's keys and values are read once for all rows of a group, each row's own ones behind it as usual.
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k[j, h / G]) v[j, h / G],  j = 0 .. pos_t
//   positions j < n of a group's rows lie in the pages of the group's slot, j >= n in those of the row's own slot
//
// A softmax over two parts is put together from their maxima, sums and sums of values, so the parts are worked on by CTAs of their own, as are stretches of a long part:
//
//   parts kernel   one CTA per (tile of 16 WM rows x heads of a group, kv head, stretch of the prefix) and per (row, kv head, stretch of its own keys): m, l and O of each row and head into
//                  the scratch. Products on the tensor cores as m16n8k16, running maximum and sum in 32 bits, tiles of 64 keys through a ring in shared memory
//   merge kernel   one warp per (row, head): the stretches' parts, weighted by e^(m - largest m), over the sum
//
// With few rows this is bound by the bytes of the prefix; a tile of 64 rows and heads is where m16n8k16 keeps up with them.
#include <algorithm>

#include "mma16816.cuh"
#include "shared_prefix.cuh"

using namespace ifab;

namespace {

constexpr int KEYS = 64, STAGES = 3, WARPS = 4, NT = 32 * WARPS;

template <int HD>
struct Ring {
  static constexpr int ROW = HD * 2, CH = HD / 8, STAGE = 2 * KEYS * ROW, BYTES = STAGES * STAGE;
  static constexpr int SMEM = BYTES + WARPS * 16 * 8;          // behind the ring: maxima and sums of the warps
  static_assert(WARPS * 16 * HD * 4 <= BYTES, "the warps' results take the ring's place");
};

// One stretch of keys [begin, end) of the pages of `slot` against 16 WM (row, head) pairs. WM warps side by side have 16 pairs each, the others of a group of them other keys of a tile.
// `pair(i, &t, &h)`: pair i's row and head; false: nobody's
template <int HD, int WM, typename Pair>
__device__ __forceinline__ void attend(const PrefixParams& p, unsigned char* smem, int begin, int end, int slot, int kvh, int part, Pair pair) {
  using R = Ring<HD>;
  constexpr int WK = WARPS / WM, KW = KEYS / WK;                // warps of other keys, keys of a warp
  __shared__ int rows[STAGES + 1][KEYS];
  __shared__ int whole[STAGES + 1][2];
  __shared__ long pair_q[16 * WM], pair_part[16 * WM];          // where a pair's query and result lie, -1: nobody's
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c2 = (lane & 3) * 2;
  const int wm = warp % WM, wk = warp / WM;
  const uint32_t ring = smem_addr(smem);
  const long kv_elems = (long)p.Hkv * HD;
  const int tiles = (end - begin + KEYS - 1) / KEYS;
  // where the keys of tile i lie (two warps), -1: nowhere
  auto locate = [&](int i) {
    if (warp < 2 && i < tiles) {
      const int key = begin + i * KEYS + threadIdx.x;
      const int r = key < end ? p.row_of(key, slot) : -1;
      rows[i % (STAGES + 1)][threadIdx.x] = r;
      if (key < end && r < 0 && p.status) atomicOr(p.status, IFAB_STATUS_BAD_INDEX);
      const bool all = __all_sync(0xffffffffu, r >= 0);
      if (lane == 0) whole[i % (STAGES + 1)][warp] = all;
    }
  };
  auto load = [&](int i) {
    if (i < tiles) {
      const uint32_t dst0 = ring + (i % STAGES) * R::STAGE;
      const int ch = threadIdx.x % R::CH;
#pragma unroll
      for (int j = 0; j < KEYS * R::CH / NT; ++j) {
        const int key = threadIdx.x / R::CH + j * (NT / R::CH);
        const int r = rows[i % (STAGES + 1)][key];
        const long at = r < 0 ? 0 : r * kv_elems + (long)kvh * HD + ch * 8;
        const uint32_t dst = dst0 + key * R::ROW + ((ch ^ (key & 7)) << 4);
        copy16(dst, p.k_cache + at, r >= 0);
        copy16(dst + KEYS * R::ROW, p.v_cache + at, r >= 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) locate(i);
  if (threadIdx.x >= NT - 16 * WM) {
    const int i = threadIdx.x - (NT - 16 * WM);
    int t, h;
    const bool live = pair(i, &t, &h);
    pair_q[i] = live ? (long)t * p.ldq + (long)h * HD : -1;
    pair_part[i] = live ? p.part_of(t, h, part) : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(i);

  uint32_t q[HD / 16][4];
  {
    const bf16* src[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const long at = pair_q[wm * 16 + g + 8 * e];
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

  for (int i = 0; i < tiles; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();                             // tile i has landed for all threads, tile i - 1 is read
    load(i + STAGES - 1);
    const uint32_t kb = ring + (i % STAGES) * R::STAGE + wk * KW * R::ROW, vb = kb + KEYS * R::ROW;
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
        ldsm4(kb + key * R::ROW + ((ch ^ (key & 7)) << 4), b);
        mma16816(s[2 * n], q[kk][0], q[kk][1], q[kk][2], q[kk][3], b[0], b[1]);
        mma16816(s[2 * n + 1], q[kk][0], q[kk][1], q[kk][2], q[kk][3], b[2], b[3]);
      }
    const bool all = whole[i % (STAGES + 1)][0] && whole[i % (STAGES + 1)][1];
    float mn[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < KW / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= p.scale_log2;
        if (!all && rows[i % (STAGES + 1)][wk * KW + 8 * n + c2 + (e & 1)] < 0) s[n][e] = -INFINITY;
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
        s[n][e] = s[n][e] == -INFINITY ? PREFIX_LEAST_WEIGHT : prefix_weight(s[n][e] - m[e >> 1]);
        l[e >> 1] += s[n][e];
      }
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) two_terms(s[2 * kk + (j >> 1)][2 * (j & 1)], s[2 * kk + (j >> 1)][2 * (j & 1) + 1], &hi[j], &lo[j]);
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        uint32_t b[4];
        const int key = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), ch = 2 * j + (lane >> 4);
        ldsm4t(vb + key * R::ROW + ((ch ^ (key & 7)) << 4), b);
        mma16816(acc[2 * j], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
        mma16816(acc[2 * j + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
        mma16816(acc[2 * j], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
        mma16816(acc[2 * j + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
      }
    }
    __syncwarp();
    if (i + STAGES < tiles) locate(i + STAGES);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }
  if constexpr (WK > 1) {                        // warps of the same pairs and other keys: the first one adds up, over the ring
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* sm_acc = reinterpret_cast<float*>(smem) + warp * 16 * HD;
    float2* sm_ml = reinterpret_cast<float2*>(smem + R::BYTES);
    if ((lane & 3) == 0) {
      sm_ml[warp * 16 + g] = prefix_sums(m[0], l[0]);
      sm_ml[warp * 16 + g + 8] = prefix_sums(m[1], l[1]);
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      *reinterpret_cast<float2*>(sm_acc + g * HD + 8 * j + c2) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2*>(sm_acc + (g + 8) * HD + 8 * j + c2) = make_float2(acc[j][2], acc[j][3]);
    }
    __syncthreads();
    for (int i = warp; i < 16 * WM; i += WARPS) {
      const long at = pair_part[i];
      if (at < 0) continue;
      float w[WK], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < WK; ++k) M = fmaxf(M, w[k] = sm_ml[(k * WM + i / 16) * 16 + i % 16].x);
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        w[k] = w[k] == -INFINITY ? 0.f : exp2f(w[k] - M);
        L += w[k] * sm_ml[(k * WM + i / 16) * 16 + i % 16].y;
      }
      for (int c = lane * 2; c < HD; c += 64) {
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < WK; ++k) {
          const float2 a = *reinterpret_cast<const float2*>(reinterpret_cast<float*>(smem) + ((k * WM + i / 16) * 16 + i % 16) * HD + c);
          v.x += w[k] * a.x;
          v.y += w[k] * a.y;
        }
        *reinterpret_cast<float2*>(p.parts + at * HD + c) = v;
      }
      if (lane == 0) p.sums[at] = make_float2(M, L);
    }
  } else {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const long at = pair_part[wm * 16 + g + 8 * e];
      if (at < 0) continue;
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<float2*>(p.parts + at * HD + 8 * j + c2) = make_float2(acc[j][2 * e], acc[j][2 * e + 1]);
      if ((lane & 3) == 0) p.sums[at] = prefix_sums(m[e], l[e]);
    }
  }
}

// grid: prefix items (stretch fastest, then kv head, then tile), then own items (stretch, kv head, row)
template <int HD, int WM>
__global__ void __launch_bounds__(NT, 2) prefix_parts_kernel(PrefixParams p, int prefix_items) {
  extern __shared__ __align__(16) unsigned char smem[];
  grid_dep_launch();
  grid_dep_wait();
  int item = blockIdx.x;
  if (item < prefix_items) {
    const int split = item % p.prefix_splits, kvh = item / p.prefix_splits % p.Hkv;
    int tile = item / p.prefix_splits / p.Hkv, end = 0;
    PrefixGroup gr;
    for (int i = 0;; ++i) {
      if (i == p.groups) return;
      gr = p.group(i, &end);
      const int tiles = (gr.rows * p.G + 16 * WM - 1) / (16 * WM);
      if (tile < tiles) break;
      tile -= tiles;
    }
    const int per = p.per_split(gr.shared, p.prefix_splits), begin = split * per;
    if (begin >= gr.shared) return;
    attend<HD, WM>(p, smem, begin, min(begin + per, gr.shared), gr.slot, kvh, split, [&](int i, int* t, int* h) {
      const int x = tile * 16 * WM + i;
      if (x >= gr.rows * p.G) return false;
      *t = gr.first + x / p.G;
      *h = kvh * p.G + x % p.G;
      return p.sees(gr, *t);
    });
  } else {
    item -= prefix_items;
    const int split = item % p.own_splits, kvh = item / p.own_splits % p.Hkv, t0 = item / p.own_splits / p.Hkv;
    const PrefixOwn own = p.own(t0, p.naming(t0));
    const int per = p.per_split(own.end - own.begin, p.own_splits), begin = own.begin + split * per;
    if (begin >= own.end) return;
    attend<HD, 1>(p, smem, begin, min(begin + per, own.end), own.slot, kvh, p.streams * p.prefix_splits + split, [&](int i, int* t, int* h) {
      *t = t0;
      *h = kvh * p.G + i;
      return i < p.G;
    });
  }
}

// W warps per (row, head), each every W-th part, several parts' loads in flight
template <int HD, int W>
__global__ void __launch_bounds__(128) prefix_merge_kernel(PrefixParams p, bf16* out, long ldo) {
  constexpr int E = HD / 32, AT_ONCE = 4;
  __shared__ float sm[W > 1 ? W : 1][W > 1 ? HD + 1 : 1];
  grid_dep_launch();
  grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w0 = warp % W;
  const long pair = (long)blockIdx.x * (4 / W) + warp / W;
  const int t = (int)(pair / p.Hq), h = (int)(pair % p.Hq);
  if (t >= p.T || p.positions[t] < 0) return;    // (with W = 4 a whole CTA)
  const PrefixGroup gr = p.naming(t);
  const PrefixOwn own = p.own(t, gr);
  const int n = p.sees(gr, t) ? gr.shared : 0, own_n = own.end - own.begin;
  const int per = p.per_split(n, max(1, p.prefix_splits)), own_per = p.per_split(own_n, p.own_splits);
  const int ns = n > 0 ? (n + per - 1) / per * p.streams : 0, no = own_n > 0 ? (own_n + own_per - 1) / own_per : 0;
  const long base = p.part_of(t, h, 0);
  auto slot_of = [&](int i) { return base + (i < ns ? i : p.streams * p.prefix_splits + i - ns); };
  float M = -INFINITY;
  for (int i = lane; i < ns + no; i += 32) M = fmaxf(M, p.sums[slot_of(i)].x);
  M = warp_max(M);
  float v[E] = {}, L = 0.f;
  for (int i0 = w0; i0 < ns + no; i0 += AT_ONCE * W) {
    float2 ml[AT_ONCE], a[AT_ONCE][E / 2];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int i = i0 + k * W;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (i >= ns + no) continue;
      const long s = slot_of(i);
      ml[k] = p.sums[s];
#pragma unroll
      for (int e = 0; e < E / 2; ++e) a[k][e] = *reinterpret_cast<const float2*>(p.parts + s * HD + lane * E + 2 * e);
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const float w = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - M);
      if (w == 0.f) continue;                    // nothing, or an infinite value that weighs nothing
      L += w * ml[k].y;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        v[2 * e] += w * a[k][e].x;
        v[2 * e + 1] += w * a[k][e].y;
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sm[w0][lane * E + e] = v[e];
    if (lane == 0) sm[w0][HD] = L;
    __syncthreads();
    if (w0) return;
#pragma unroll
    for (int k = 1; k < W; ++k) {
      L += sm[k][HD];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] += sm[k][lane * E + e];
    }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;      // (a NaN among the scores stays one)
  bf16* dst = out + (long)t * ldo + (long)h * HD + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<__nv_bfloat162*>(dst + e) = __floats2bfloat162_rn(v[e] * inv, v[e + 1] * inv);
}

// how a call is shared out
struct Plan {
  int wm, tiles, prefix_splits, own_splits, streams, least;     // wm 0: the prefix on tcgen05
};
Plan plan_of(int T, int Hkv, int G, int groups, bool tiles) {          // tiles: pages that tcgen05's form takes
  Plan a{};
  auto splits = [](long items, long ctas, int most) { return (int)std::max(1l, std::min((long)most, (ctas + items - 1) / std::max(1l, items))); };
  const int rows = groups ? (T + groups - 1) / groups * G : 1;
  a.wm = rows <= 16 ? 1 : rows <= 32 ? 2 : tiles ? 0 : 4;
  a.streams = a.wm ? 1 : 2;
  const int tile = a.wm ? 16 * a.wm : 256;
  a.tiles = groups ? (int)std::max((long)groups, ((long)T * G - groups) / tile + groups) : 0;        // at most, however the rows are shared out
  a.prefix_splits = groups ? a.wm ? splits((long)a.tiles * Hkv, 296, 64) : std::max(1, std::min(148, (int)(148 / std::max(1l, (long)a.tiles * Hkv)))) : 0;
  a.own_splits = splits((long)T * Hkv, 296, 16);
  a.least = 128;
  return a;
}

template <int HD, int WM>
int launch_parts(const PrefixParams& p, long prefix_items, cudaStream_t s) {
  auto k = prefix_parts_kernel<HD, WM>;
  if (int rc = opt_in_smem(k, Ring<HD>::SMEM)) return rc;
  const long items = prefix_items + (long)p.T * p.Hkv * p.own_splits;
  if (items > 0x7fffffff) return -1;
  return launch_chain(k, dim3((unsigned)items), dim3(NT), (size_t)Ring<HD>::SMEM, s, p, (int)prefix_items);
}
template <int HD>
int launch(const PrefixParams& p, const Plan& a, bf16* out, long ldo, cudaStream_t s) {
  const long items = (long)a.tiles * p.Hkv * a.prefix_splits;
  if (items > 0x7fffffff) return -1;
  if (!a.wm)
    if (int rc = launch_prefix_tiles(p, HD, items, s)) return rc;
  if (int rc = a.wm == 4 ? launch_parts<HD, 4>(p, items, s) : a.wm == 2 ? launch_parts<HD, 2>(p, items, s) : launch_parts<HD, 1>(p, a.wm ? items : 0, s)) return rc;
  const long pairs = (long)p.T * p.Hq;
  if (a.streams * a.prefix_splits + a.own_splits > 4 && pairs <= 0x7fffffff) return launch_chain(prefix_merge_kernel<HD, 4>, dim3((unsigned)pairs), dim3(128), 0, s, p, out, ldo);
  return launch_chain(prefix_merge_kernel<HD, 1>, dim3((unsigned)((pairs + 3) / 4)), dim3(128), 0, s, p, out, ldo);
}

}  // namespace

extern "C" uint64_t ifab_shared_prefix_scratch(int T, int Hq, int Hkv, int head_dim, int groups) {
  if (T < 1 || Hkv < 1 || Hq % Hkv || groups < 0) return 0;
  const Plan a = plan_of(T, Hkv, Hq / Hkv, groups, true), b = plan_of(T, Hkv, Hq / Hkv, groups, false);
  return (uint64_t)T * Hq * (std::max(a.streams * a.prefix_splits, b.streams * b.prefix_splits) + a.own_splits) * (head_dim + 2) * sizeof(float);
}

extern "C" int ifab_shared_prefix_attention(const void* q, long ldq, const void* k_cache, const void* v_cache, const int32_t* positions, const int32_t* slots, const int32_t* page_table,
                                            int num_slots, int max_pages, int page_tokens, int num_pages, const int32_t* groups, int num_groups, float scale, int T, int Hq, int Hkv,
                                            int head_dim, void* scratch, uint64_t scratch_bytes, void* out, long ldo, uint32_t* status, void* stream) {
  if (T < 1 || T > 1 << 20 || Hkv < 1 || Hq < 1 || Hq % Hkv || Hq / Hkv > 16 || (head_dim != 64 && head_dim != 128) || num_groups < 0 || num_groups > 64 || (num_groups && !groups)) return -1;
  if (num_slots < 1 || max_pages < 1 || page_tokens < 1 || num_pages < 1 || (long)num_pages * page_tokens > 0x7fffffff || (long)max_pages * page_tokens > 0x7fffffff - 2 * KEYS) return -1;
  if (ldq % 8 || ldo % 8 || ((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)scratch | (uintptr_t)groups) % 16) return -1;
  const Plan a = plan_of(T, Hkv, Hq / Hkv, num_groups, page_tokens % 8 == 0);
  if (ifab_shared_prefix_scratch(T, Hq, Hkv, head_dim, num_groups) > scratch_bytes) return -5;
  PrefixParams p;
  p.q = (const bf16*)q; p.ldq = ldq; p.k_cache = (const bf16*)k_cache; p.v_cache = (const bf16*)v_cache;
  p.positions = positions; p.slots = slots; p.page_table = page_table; p.group_list = groups;
  p.num_slots = num_slots; p.max_pages = max_pages; p.page_tokens = page_tokens; p.num_pages = num_pages; p.groups = num_groups;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  p.prefix_splits = a.prefix_splits; p.own_splits = a.own_splits; p.streams = a.streams; p.least = a.least;
  p.parts = (float*)scratch;
  p.sums = (float2*)((float*)scratch + (uint64_t)T * Hq * (a.streams * a.prefix_splits + a.own_splits) * head_dim);
  p.status = status;
  return head_dim == 64 ? launch<64>(p, a, (bf16*)out, ldo, (cudaStream_t)stream) : launch<128>(p, a, (bf16*)out, ldo, (cudaStream_t)stream);
}

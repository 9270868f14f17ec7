// Products of many rows with 4-bit weights (int4.cuh) on tcgen05:  y[t][n] = sum_k x[t][k] w[n][k] (+ residual), or of a gate | up matrix silu(gate) up.
//
// The 128 rows of an MMA are weight rows, the tokens its columns. Weights become s (q - z) in registers, where a thread is a row, and go straight into tensor memory
// as the MMA's first operand: they do not pass through shared memory, whose bandwidth belongs to the tokens' tiles; codes do, 8 KB for 32 of weights. Two groups of four warps take the
// chunks of 128 columns in turn.
// The operands are f16, each row with a power of two of its own. A product s (q - z) has up to 13 bits: bf16 leaves 8 of them, and a gated unit's result was off by 1.6
// times its rounding; f16 leaves 11. Rows of x keep all their 8 bits: a launch ahead (rows_kernel) brings a row's largest magnitude to 2^14 .. 2^15, so that what falls below
// f16's normal range is off by 2^-40 of that at most, and a row of weights has its largest scale at 2^11 .. 2^12 (15 of them stay below 65504). Both powers are taken out of
// the f32 sums.
//   warp 0      copies of the tokens' tiles (64 columns, 128-byte swizzle)
//   warp 1      MMAs
//   warp 10     copies of codes, the first of them ahead of the wait for the preceding kernel
//   warps 2-9   weights into tensor memory; then 2-5 read the accumulator
// Up to 128 tokens: two CTAs an SM (128 columns of sums and four stages of 32 columns of weights each), so that one multiplies while the other starts or stores. More: tiles of
// up to 256 tokens, a CTA an SM, so that the weights become operands once (203 rows of 6144 by 4096 24.2 us, in tiles of 112 tokens 30).
// With few tiles the chunks along K are shared by the CTAs of a cluster, of any size up to eight (17 rows of 4096 by 4096 10.2 us, of 6144 by 4096 15; in powers of two 12.8 and
// 19.5, when all clusters did not run at once): each leaves its part of the sum in its shared memory as f32 and every CTA adds up a share of the tokens over
// distributed shared memory, in the order of the parts.
// Measured: 0.65 - 0.8 us a chunk and 12 us beside them, of which the launch ahead, the first loads and the cluster's sum are most: 203 rows of 6144 by 4096 24.2 us (the bf16
// product of the same sizes 25.1; 7 us of products), 64 of 2 x 16384 by 4096 37 (58), 203 of 4096 by 16384 37 (41). The products' pipe is busy for 28 % of an SM's time there,
// the issue slots for 34 %; a fifth stage, and signals without the delay, gave 2 % or less.
// Every wait is bounded. One that runs out raises the CTA's flag and the status word; the warps that read the accumulator then wait for what the CTA has started and
// leave NaN as their part of the sum.
#include <algorithm>

#include "int4_tc.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::tc;
using namespace ifab::int4;

namespace ifab::int4 {
int pair_product(const View& v, const void* rows, const float* factor, const bf16* residual, long ldr, void* y, long ldy, int out_f32, int T, int tok, int pairs,
                 uint32_t spin_limit, uint32_t* status, cudaStream_t s);      // int4_tc_pair.cu
}

namespace {

constexpr int FT = 128, BK = 64, TOK = 128, STAGES = 4, CHUNKS = 4, THREADS = 352;       // TOK: tokens of a tile, twice as many where it is wide
template <int GROUP, bool ZEROS, bool WIDE>
constexpr int SMEM = STAGES * (WIDE ? 2 : 1) * TOK * BK * 2 + CHUNKS * Units<GROUP, ZEROS>::BYTES + 1024 + 512;
constexpr uint32_t DRAIN = 4000000u;                 // limit of the waits for what a CTA that gives up has started
// Phases are told apart by parity (int4_tc_pair.cu): a slot of codes belongs to one group of warps, and a group's block before this one, at most three back, waited for the
// products STAGES blocks ahead of it
static_assert(CHUNKS % 2 == 0 && STAGES >= 3, "a group could take a phase for the one two ahead");
static_assert(TOK * FT * 4 <= STAGES * TOK * BK * 2, "the part of the sum takes the ring's place");

struct TcP {
  View v;
  void* y; long ldy; int out_f32;
  const bf16* residual; long ldr;
  const float* factor;           // of the rows of x
  int T, tok, splits;            // tokens of a tile (a multiple of 16), CTAs of a cluster
  uint32_t* status; uint32_t spin_limit;
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_part4(uint32_t addr, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
// D[tmem] (+)= A[tmem] * B[smem]; issued by ONE thread
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// rows of x in f16 by a power of two each, which `factor` takes out again. A CTA a row
__global__ void __launch_bounds__(256) rows_kernel(const bf16* x, long ldx, __half* out, long ldo, float* factor, int K) {
  __shared__ float red[8];
  grid_dep_launch();
  grid_dep_wait();
  const uint4* row = reinterpret_cast<const uint4*>(x + (long)blockIdx.x * ldx);
  uint4* to = reinterpret_cast<uint4*>(out + (long)blockIdx.x * ldo);
  constexpr int HELD = 4;              // pieces of eight columns that a thread keeps: rows of up to 8192 are read once
  const int pieces = K / 8, first = threadIdx.x;
  uint4 held[HELD];
  float most = 0.f;
  auto widest = [&](const uint4& u) {
    float f[8];
    unpack8(u, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]) <= 3.4028234e38f ? fabsf(f[e]) : 0.f);
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i) held[i] = first + i * 256 < pieces ? row[first + i * 256] : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < HELD; ++i) widest(held[i]);
  for (int c = first + HELD * 256; c < pieces; c += 256) widest(row[c]);
  most = warp_max(most);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
  most = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7])));
  const int e = exponent_of(most);
  const float by = power_of_two(min(14 - e, 126));
  if (threadIdx.x == 0) factor[blockIdx.x] = power_of_two(max(e - 14, -126));
  auto scaled = [&](const uint4& in) {
    float f[8];
    unpack8(in, f);
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2half2_rn(f[2 * j] * by, f[2 * j + 1] * by);
    return u;
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (first + i * 256 < pieces) to[first + i * 256] = scaled(held[i]);
  for (int c = first + HELD * 256; c < pieces; c += 256) to[c] = scaled(row[c]);
}

// grid (feature tiles x splits, token tiles), clusters of `splits` along x
template <int GROUP, bool ZEROS, bool WIDE>
__global__ void __launch_bounds__(THREADS, WIDE ? 1 : 2) int4_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, TcP p) {
  using U = Units<GROUP, ZEROS>;
  constexpr int MOST = WIDE ? 2 * TOK : TOK, STAGE = MOST * BK * 2;
  constexpr uint32_t COLS = 2 * MOST, A_COL = MOST;    // of tensor memory; first column of the weights' stages
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* ring = smem + STAGES * STAGE;         // chunks of units
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + CHUNKS * U::BYTES);
  uint64_t *weights = full + STAGES, *empty = weights + STAGES, *acc_full = empty + STAGES, *units_full = acc_full + 1, *units_empty = units_full + CHUNKS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(units_empty + CHUNKS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ float factors[MOST];
  volatile int* requested = abort_flag + 1;      // blocks whose copies were requested, once no more will be; until then -1
  const View& v = p.v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const bool gated = v.halves == 2;
  const int n0 = tile * (gated ? FT / 2 : FT), m0 = blockIdx.y * p.tok;
  const int c0 = (int)((long)v.chunks * part / p.splits), nc = (int)((long)v.chunks * (part + 1) / p.splits) - c0, nk = 2 * nc;      // chunks, blocks of 64 columns

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&weights[s], 4);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < CHUNKS; ++s) {
      mbar_init(&units_full[s], 1);
      mbar_init(&units_empty[s], 4);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    *requested = -1;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_x);
  }
  const int row = (warp & 3) * 32 + lane, group = (warp - 2) >> 2;
  // the tile of sixteen rows that is unit u of this CTA's (a tile beyond the matrix: its last one, whose results are not stored): gate rows first
  auto tile_of = [&](int u) { return min(n0 / TILE + (gated ? u & 3 : u), v.tiles - 1) + (gated && u >= 4 ? v.tiles : 0); };
  __syncthreads();
  // Codes are written by no kernel of the stream: the first ones are on their way ahead of the wait
  int chunk = 0;                                       // requested
  const unsigned char* from = v.at(tile_of(lane & 7), c0);
  auto request = [&]() {
    const int q = chunk % CHUNKS;
    if (lane == 0) mbar_expect_tx(&units_full[q], U::BYTES);
    __syncwarp();
    if (lane < 8) bulk_load(ring + q * U::BYTES + lane * U::UNIT, from + (long)chunk * U::UNIT, U::UNIT, &units_full[q]);
    ++chunk;
  };
  if (warp == 10)
    while (chunk < min(nc, CHUNKS)) request();
  RowOfWeights<GROUP, ZEROS> mine;
  if (warp >= 2 && warp < 10) {
    mine.start(v, row >> 4, row & 15);
    mine.scale(v.most[tile_of(row >> 4) * TILE + (row & 15)]);
  }
  grid_dep_wait();
  if (warp == 1) tmem_alloc(tmem_slot, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_launch();
  const uint32_t tmem_base = *tmem_slot;
  if (threadIdx.x < MOST && m0 + threadIdx.x < p.T) factors[threadIdx.x] = p.factor[m0 + threadIdx.x];

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int kb = 0; kb < nk; ++kb) {
      const int s = kb % STAGES;
      if (kb >= STAGES && !mbar_wait(&empty[s], (kb / STAGES - 1) & 1, p.spin_limit)) *abort_flag = 1;
      if (*abort_flag) break;
      mbar_expect_tx(&full[s], p.tok * BK * 2);
      tma_load_2d(smem + s * STAGE, &tmap_x, &full[s], (2 * c0 + kb) * BK, m0);
      issued = kb + 1;
    }
    *requested = issued;
    if (*abort_flag && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
  } else if (warp == 1) {                                // the whole warp walks and one lane issues, as among pairs
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const uint32_t idesc = umma_idesc_f16(FT, p.tok);
    const uint64_t first = umma_desc_sw128(smem_u32(smem));
    int s = 0;
    uint32_t parity = 0;
    bool ok = true;
#pragma unroll 1
    for (int kb = 0; kb < nk && ok; ++kb) {
      ok = mbar_wait(&full[s], parity, p.spin_limit) && mbar_wait(&weights[s], parity, p.spin_limit);
      ok = !__any_sync(0xffffffffu, !ok || *abort_flag);
      tc_fence_after();
      if (ok && elected) {
        const uint64_t db = first + (uint64_t)(s * (STAGE >> 4));
        const uint32_t a = tmem_base + A_COL + s * 32;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) umma_f16_ta(tmem_base, a + 8 * k, db + (uint64_t)(2 * k), idesc, kb > 0 || k > 0);
        umma_commit(&empty[s]);
      }
      if (++s == STAGES) s = 0, parity ^= 1;
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    }
    if (elected) umma_commit(acc_full);
  } else if (warp == 10) {
    while (chunk < nc) {
      if (!mbar_wait(&units_empty[chunk % CHUNKS], (chunk / CHUNKS - 1) & 1, p.spin_limit)) *abort_flag = 1;
      if (__any_sync(0xffffffffu, *abort_flag)) break;
      request();
    }
    // what has been requested lands before the CTA ends, whoever gives up
    for (int i = max(0, chunk - CHUNKS); i < chunk; ++i) mbar_wait(&units_full[i % CHUNKS], (i / CHUNKS) & 1, DRAIN);
  } else if (warp >= 2) {
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    int written = -1;                                    // a stage is signalled when the next one's operands are there
    auto settle = [&]() {
      if (written < 0) return;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&weights[written]);
    };
#pragma unroll 1
    for (int ch = group; ch < nc; ch += 2) {
      const int q = ch % CHUNKS;
      bool late = !mbar_wait(&units_full[q], (ch / CHUNKS) & 1, p.spin_limit);
      mine.load(ring + q * U::BYTES, row & 15);
      __syncwarp();
      if (lane == 0) mbar_arrive(&units_empty[q]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int kb = 2 * ch + b, s = kb % STAGES;
        uint32_t w[32];
        mine.block(b, w);
        settle();                                        // the block before this one
        if (kb >= STAGES) late |= !mbar_wait(&empty[s], (kb / STAGES - 1) & 1, p.spin_limit);
        tc_fence_after();
        tmem_st_32x32(tmem_base + A_COL + s * 32 + lanes, reinterpret_cast<const float*>(w));
        written = s;
      }
      if (late) *abort_flag = 1;
      if (__any_sync(0xffffffffu, *abort_flag)) {
        if (lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
        break;
      }
    }
    settle();
  }
  __syncwarp();
  // The accumulator complete, all copies have landed and all products have read the ring: it becomes this CTA's part of the sum, [tokens][128].
  float* sum = reinterpret_cast<float*>(smem);
  const int tokens = min(p.tok, p.T - m0);
  if (warp >= 2 && warp < 6) {
    const bool ready = mbar_wait(acc_full, 0, p.spin_limit);
    tc_fence_after();
    if (!ready) {
      *abort_flag = 1;
      if (lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    }
    const uint32_t tm = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    if (__any_sync(0xffffffffu, *abort_flag)) {
      for (uint32_t i = 0; i < DRAIN && *requested < 0; ++i) __nanosleep(64);
      const int n = *requested;
      for (int kb = max(0, n - STAGES); kb < n; ++kb) mbar_wait(&full[kb % STAGES], (kb / STAGES) & 1, DRAIN);
      mbar_wait(acc_full, 0, DRAIN);
      for (int t = 0; t < tokens; ++t) sum[t * FT + row] = __int_as_float(0x7fffffff);
    } else {
      const float out = mine.out();
      for (int t0 = 0; t0 < tokens; t0 += 32) {
        float f[32];
        tmem_ld_32x32(tm + (uint32_t)t0, f);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (t0 + i < tokens) sum[(t0 + i) * FT + row] = f[i] * out;
      }
    }
  }
  tc_fence_before();
  if (p.splits > 1) cluster_barrier();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, COLS);
  const uint32_t sum_at = smem_u32(sum);
  const int width = gated ? FT / 8 : FT / 4;         // pieces of four features of a token
  for (int i = threadIdx.x;; i += THREADS) {
    const int t = part + i / width * p.splits, f = i % width * 4, col = n0 + f;
    if (t >= tokens) break;
    if (col >= v.N) continue;
    float a[4] = {}, u[4] = {};
    for (int r = 0; r < p.splits; ++r) {
      const float4 x = p.splits > 1 ? ld_part4(sum_at + (t * FT + f) * 4, r) : *reinterpret_cast<const float4*>(sum + t * FT + f);
      a[0] += x.x, a[1] += x.y, a[2] += x.z, a[3] += x.w;
      if (gated) {
        const float4 z = p.splits > 1 ? ld_part4(sum_at + (t * FT + FT / 2 + f) * 4, r) : *reinterpret_cast<const float4*>(sum + t * FT + FT / 2 + f);
        u[0] += z.x, u[1] += z.y, u[2] += z.z, u[3] += z.w;
      }
    }
    const int live = min(4, v.N - col);
    const long m = m0 + t;
    const float factor = factors[t];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] *= factor;
      u[e] *= factor;
      if (gated) a[e] = gated_unit(a[e], u[e]);
      if (p.residual && e < live) a[e] += __bfloat162float(p.residual[m * p.ldr + col + e]);
    }
    if (p.out_f32) {
      float* out = reinterpret_cast<float*>(p.y) + m * p.ldy + col;
      if (live == 4 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) *reinterpret_cast<float4*>(out) = make_float4(a[0], a[1], a[2], a[3]);
      else
        for (int e = 0; e < live; ++e) out[e] = a[e];
    } else {
      bf16* out = reinterpret_cast<bf16*>(p.y) + m * p.ldy + col;
      if (live == 4 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(a[0], a[1]), hi = __floats2bfloat162_rn(a[2], a[3]);
        *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        for (int e = 0; e < live; ++e) out[e] = __float2bfloat16_rn(a[e]);
      }
    }
  }
  if (p.splits > 1) cluster_barrier();               // the parts stay until every CTA has read them
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

template <int GROUP, bool ZEROS, bool WIDE>
int launch(const CUtensorMap& tx, const TcP& p, dim3 grid, cudaStream_t s) {
  auto k = int4_tc_kernel<GROUP, ZEROS, WIDE>;
  constexpr int smem = SMEM<GROUP, ZEROS, WIDE>;
  static std::atomic<uint64_t> done;
  if (int rc = allow_smem(k, smem, device_now().id, done)) return rc;
  if (p.splits > 1) return launch_chain_cluster(k, grid, dim3(THREADS), (unsigned)p.splits, (size_t)smem, s, tx, p);
  return launch_chain(k, grid, dim3(THREADS), (size_t)smem, s, tx, p);
}
// Clusters of n CTAs that run at once: an SM's neighbours are not all free to join, and of 296 CTAs (two an SM) 279 run in threes, 259 in sevens; of 148, 135 and 105
template <bool WIDE>
int at_once(int n, const Device& dev) {
  static std::atomic<int> known[64][9];
  std::atomic<int>* have = dev.id < 64 ? &known[dev.id][n] : nullptr;
  if (have && have->load()) return have->load();
  auto k = int4_tc_kernel<128, false, WIDE>;
  static std::atomic<uint64_t> done;
  constexpr int smem = SMEM<128, false, WIDE>;
  int count = 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n * dev.sms), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  if (allow_smem(k, smem, dev.id, done) || cudaOccupancyMaxActiveClusters(&count, k, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  if (have) have->store(count);
  return count;
}
// CTAs along K: those that run at once, by the chunks that the busiest SM goes through and what a wave costs besides (start, first loads, cluster's sum: 10 us), counted in chunks.
// 2 and 6 chose the same or as good ones over 25 sizes of one wave, but two waves of shares where one of whole tiles is as fast
constexpr int WAVE_COST = 12;
template <bool WIDE>
int splits_of(int tiles, int chunks, const Device& dev, int* waves) {
  int best = 1;
  long least = 0;
  for (int n = 1; n <= 8 && (n == 1 || chunks >= 2 * n); ++n) {
    const int room = at_once<WIDE>(n, dev);
    if (!room) continue;
    const long waves_of_n = ceil_div(tiles, room), share = WIDE ? 1 : std::min(2, ceil_div(std::min(tiles, room) * n, dev.sms));
    const long cost = waves_of_n * (share * ceil_div(chunks, n) + WAVE_COST);
    if (!least || cost < least) least = cost, best = n, *waves = (int)waves_of_n;
  }
  return best;
}
template <int GROUP, bool ZEROS>
int launch_wide(const CUtensorMap& tx, const TcP& p, dim3 grid, cudaStream_t s) {
  return p.tok > TOK ? launch<GROUP, ZEROS, true>(tx, p, grid, s) : launch<GROUP, ZEROS, false>(tx, p, grid, s);
}

}  // namespace

// What a chunk of 128 columns costs a CTA's or a pair's tile: most of it whatever the tokens (0.80 us at 176 of them, 0.91 at 256; counted in tokens)
constexpr long CHUNK_COST = 480;
// Tokens of a pair's tile (int4_tc_pair.cu), the width whose waves of tiles over the pairs cost least, and that cost
static int pair_tokens(int T, int rows, int chunks, int pairs, long* cost) {
  int best = 0;
  for (int tok = 256; tok >= 128; tok -= 16) {
    const long now = ((long)ceil_div(rows, 2 * FT) * ceil_div(T, tok) + pairs - 1) / pairs * chunks * (tok + CHUNK_COST);
    if (!best || now < *cost) *cost = now, best = tok;
  }
  return best;
}

// bytes of the workspace of T rows
extern "C" uint64_t ifab_int4_gemm_scratch(int T, int K) { return T < 1 || K < 8 ? 0 : (uint64_t)T * K * 2 + ((uint64_t)T * 4 + 15) / 16 * 16; }

// x [T, K] in bf16, rows on 16 bytes; scratch: ifab_int4_gemm_scratch bytes on 16 bytes, for this call alone. The units are written by no kernel that may still run. spin_limit: polls of a wait.
extern "C" int ifab_int4_gemm(const IfabInt4* d, const void* x, long ldx, const void* residual, long ldr, void* y, long ldy, int out_f32, int T, void* scratch,
                              uint32_t spin_limit, uint32_t* status, void* stream) {
  TcP p{};
  if (view_of(d, &p.v) || T < 1 || !x || !y || !scratch || ((uintptr_t)x | (uintptr_t)scratch) % 16 || ldx % 8 || (p.v.halves == 2 && residual)) return -1;
  __half* rows = (__half*)scratch;
  float* factor = (float*)((char*)scratch + (uint64_t)T * p.v.K * 2);
  p.y = y, p.ldy = ldy, p.out_f32 = out_f32, p.residual = (const bf16*)residual, p.ldr = ldr, p.factor = factor, p.T = T, p.status = status;
  p.spin_limit = spin_limit;
  const Device dev = device_now();
  const int halves = p.v.halves, sms = dev.sms;
  cudaStream_t s = (cudaStream_t)stream;
  if (int rc = launch_chain(rows_kernel, dim3(T), dim3(256), 0, s, (const bf16*)x, ldx, rows, (long)p.v.K, factor, p.v.K)) return rc;
  const int wide = T > TOK, ty = ceil_div(T, wide ? 2 * TOK : TOK), tiles = ceil_div(p.v.N, halves == 2 ? FT / 2 : FT);
  p.tok = std::max(ceil_div(ceil_div(T, ty), 16) * 16, wide ? TOK + 16 : 16);
  int waves = 1;
  p.splits = (long)tiles * ty > 8l * sms ? 1 : wide ? splits_of<true>(tiles * ty, p.v.chunks, dev, &waves) : splits_of<false>(tiles * ty, p.v.chunks, dev, &waves);
  if (wide) {
    // Pairs, unless a tile a CTA whose K is shared costs less, a wave counted as twelve chunks, of which pairs have eight: 256 rows of 6144 by 4096 26 us (pairs 33), 512 of 4096 by 16384 64 (113);
    // 256 of 10240 by 4096 42 (36), 400 of 6144 by 4096 37 (35), 2048 of 1024 by 1024 22 (19)
    long cost = 0;
    const int tok = pair_tokens(T, p.v.N * halves, p.v.chunks, sms / 2, &cost);
    if ((long)tiles * ty > 8l * sms || cost <= waves * ((long)ceil_div(p.v.chunks, p.splits) * (p.tok + CHUNK_COST)) + (waves * WAVE_COST - 8) * (2 * TOK + CHUNK_COST))
      return pair_product(p.v, rows, factor, p.residual, ldr, y, ldy, out_f32, T, tok, (int)std::min<long>(sms / 2, (long)ceil_div(p.v.N * halves, 2 * FT) * ceil_div(T, tok)), spin_limit, status, s);
  }
  if (ty > 65535) return -1;
  CUtensorMap tx;          // of 16-bit elements: the type is the products' to know
  if (int rc = make_tmap_bf16_2d(&tx, rows, (uint64_t)T, (uint64_t)p.v.K, (uint64_t)p.v.K, (uint32_t)p.tok)) return rc;
  const dim3 grid(tiles * p.splits, ty);
  if (p.v.zeros) return p.v.group == 128 ? launch_wide<128, true>(tx, p, grid, s) : p.v.group == 64 ? launch_wide<64, true>(tx, p, grid, s) : launch_wide<32, true>(tx, p, grid, s);
  return p.v.group == 128 ? launch_wide<128, false>(tx, p, grid, s) : p.v.group == 64 ? launch_wide<64, false>(tx, p, grid, s) : launch_wide<32, false>(tx, p, grid, s);
}

// Products of many rows with 4-bit weights (int4.cuh) on pairs of SMs: int4_tc.cu's operands and results, for prompts long enough to fill the chip with tiles of 256 weight
// rows (a gate | up matrix: 128 features) by up to 256 tokens.
//
// A lone CTA with 128 weight rows loads 16 KB of tokens for 256 cycles of products, as much as an SM gets out of L2; a pair shares the tokens' tile, half in each CTA's
// shared memory (tcgen05.mma.cta_group::2), and each CTA brings its 128 rows of weights into its own tensor memory. One pair an SM pair walks the tiles; copies and
// weights of the next tile go on while this one's sums are stored.
//   warp 0       copies of this CTA's half of the tokens; both CTAs' bytes complete on the leader's barrier
//   warp 1       allocates tensor memory; in the leader, MMAs
//   warps 2-9    this CTA's weights into its tensor memory (256 columns: eight stages), signalled to the leader
//   warp 18      copies of this CTA's codes
//   warps 10-17  sums out of tensor memory (256 columns), two warps for 32 rows. A lane is a weight row, so that a token's results leave as 64 bytes a warp. Gate and up rows
//                lie in the two halves of a warp's rows, sixteen each: a lane gives every other token's value to its partner and has both of the others
// Every wait is bounded; one that runs out raises the CTA's flag and the status word, tiles that are not complete are stored as NaN, and both CTAs meet at the closing barrier.
#include <algorithm>
#include <type_traits>

#include "int4_tc.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::tc;
using namespace ifab::int4;

namespace {

constexpr int FT = 128, BK = 64, TOK = 256, STAGES = 8, CHUNKS = 6, THREADS = 608, READERS = 8;
constexpr int STAGE = TOK / 2 * BK * 2;
template <int GROUP, bool ZEROS>
constexpr int SMEM = STAGES * STAGE + CHUNKS * Units<GROUP, ZEROS>::BYTES + 1024 + 512;
constexpr uint32_t A_COL = 256;                      // first column of the weights' stages
constexpr uint32_t DRAIN = 4000000u;                 // limit of the waits for what a CTA that gives up has started
constexpr int RASTER = 8;                            // token tiles that pairs share weights over

struct PairP {
  View v;
  void* y; long ldy; int out_f32;
  const bf16* residual; long ldr;
  const float* factor;
  int T, tok;                    // tokens of a tile (a multiple of 16)
  uint32_t* status; uint32_t spin_limit;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_leader(const void* at) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(at)));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// as mbar_wait, for a barrier that the peer arrives on
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, uint32_t limit) {
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (i > 256) __nanosleep(64);
  }
  return false;
}
// this CTA's tile; its bytes go to the barrier at `bar` (the leader's)
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(m), "r"(bar),
               "r"(x), "r"(y)
               : "memory");
}
// D[tmem of both] (+)= A[tmem of both] * B[smem of both]; issued by ONE thread of the leader
__device__ __forceinline__ void umma_f16_pair_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// arrive on the barrier at this place in both CTAs once the products issued so far have completed
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
// tile t: token tiles fastest, in groups of RASTER, so that the pairs at work share weights and keep few tokens
__device__ __forceinline__ void tile_at(int t, int tiles_t, int tiles_n, int* tt, int* tn) {
  const int per = RASTER * tiles_n, g = t / per, within = t - g * per, first = g * RASTER, rows = min(RASTER, tiles_t - first);
  *tt = first + within % rows;
  *tn = within / rows;
}

template <bool F32>
__device__ __forceinline__ void put(void* y, long at, float v) {
  if (F32) reinterpret_cast<float*>(y)[at] = v;
  else reinterpret_cast<bf16*>(y)[at] = __float2bfloat16_rn(v);
}
// Tokens 0 .. live - 1 (of 32) of this lane's row; `f`: the sums, `factor`: of token `lane`; y and the residual from the first token's result on
template <bool GATED, bool F32, bool WHOLE>
__device__ __forceinline__ void store32(float (&f)[32], float out, float factor, void* y, long ldy, const bf16* residual, long ldr, int live, bool there, int lane) {
  if constexpr (GATED) {
    const bool up = lane >= 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float lo = f[2 * i] * out, hi = f[2 * i + 1] * out, got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, 16), by = __shfl_sync(0xffffffffu, factor, 2 * i + up);
      const float v = gated_unit((up ? got : lo) * by, (up ? hi : got) * by);
      if (there && (WHOLE || 2 * i + up < live)) put<F32>(y, (2 * i + up) * ldy, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) f[i] = f[i] * out * __shfl_sync(0xffffffffu, factor, i);
    if (!there) return;
    if (residual) {
      bf16 r[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = WHOLE || i < live ? residual[i * ldr] : __float2bfloat16_rn(0.f);
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] += __bfloat162float(r[i]);
    }
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (WHOLE || i < live) put<F32>(y, i * ldy, f[i]);
  }
}

// grid (2 * pairs), clusters of 2
template <int GROUP, bool ZEROS>
__global__ void __launch_bounds__(THREADS, 1) int4_tc_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, PairP p) {
  using U = Units<GROUP, ZEROS>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* ring = smem + STAGES * STAGE;                               // chunks of units
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + CHUNKS * U::BYTES);    // leader's: both halves of the tokens
  uint64_t* weights = full + STAGES;                                         // leader's: an arrival of every warp that wrote rows of the stage
  uint64_t* empty = weights + STAGES;                                        // each CTA's own, as acc_full
  uint64_t *acc_full = empty + STAGES, *acc_empty = acc_full + 1;            // acc_empty: leader's
  uint64_t *units_full = acc_empty + 1, *units_empty = units_full + CHUNKS;   // each CTA's own
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(units_empty + CHUNKS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const View& v = p.v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const bool gated = v.halves == 2;
  const int per_cta = gated ? FT / 2 : FT;               // columns of the result
  const int tiles_n = (v.N + 2 * per_cta - 1) / (2 * per_cta), tiles_t = (p.T + p.tok - 1) / p.tok, tiles = tiles_n * tiles_t, nc = v.chunks, nk = 2 * nc;

  // the tile of sixteen rows that is unit u of this CTA's part of a pair's tile (a tile beyond the matrix: its last one, whose results are not stored)
  auto tile_of = [&](int tn, int u) {
    const int at = (tn * 2 + rank) * (per_cta / TILE) + (gated ? u >> 1 : u);
    return min(at, v.tiles - 1) + (gated && (u & 1) ? v.tiles : 0);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&weights[s], 8);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < CHUNKS; ++s) {
      mbar_init(&units_full[s], 1);
      mbar_init(&units_empty[s], 4);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * READERS);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_x);
  }
  __syncthreads();
  grid_dep_wait();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();                                     // the peer's barriers and tensor memory exist before anything is signalled or issued
  tc_fence_after();
  grid_dep_launch();
  const uint32_t tmem_base = *tmem_slot, quarter = (uint32_t)((warp & 3) * 32) << 16;

  if (warp == 0 && lane == 0) {
    uint32_t it = 0;
    for (int t = pair; t < tiles && !*abort_flag; t += pairs) {
      int tt, tn;
      tile_at(t, tiles_t, tiles_n, &tt, &tn);
      const int m = tt * p.tok + rank * (p.tok / 2);
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % STAGES;
        if (it >= STAGES && !mbar_wait(&empty[s], (it / STAGES - 1) & 1, p.spin_limit)) *abort_flag = 1;
        if (*abort_flag) break;
        if (rank == 0) mbar_expect_tx(&full[s], p.tok * BK * 2);
        load_pair(smem + s * STAGE, &tmap_x, in_leader(&full[s]), kb * BK, m);
      }
    }
    if (*abort_flag && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    if (rank == 0)                                       // what has been requested lands before the CTAs end, whoever gives up
      for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, DRAIN);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    const uint32_t idesc = umma_idesc_f16(2 * FT, p.tok);
    uint32_t it = 0;
    int j = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs, ++j) {
      if (j && !wait_cluster(acc_empty, (j - 1) & 1, p.spin_limit)) { ok = false; break; }
      tc_fence_after();
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % STAGES;
        const uint32_t parity = (it / STAGES) & 1;
        if (!wait_cluster(&full[s], parity, p.spin_limit) || !wait_cluster(&weights[s], parity, p.spin_limit) || *abort_flag) { ok = false; break; }
        tc_fence_after();
        const uint64_t db = umma_desc_sw128(smem_u32(smem + s * STAGE));
        const uint32_t a = tmem_base + A_COL + s * 32;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) umma_f16_pair_ta(tmem_base, a + 8 * k, db + (uint64_t)(2 * k), idesc, kb > 0 || k > 0);
        commit_pair(&empty[s]);
      }
      commit_pair(acc_full);
    }
    if (!ok) {
      *abort_flag = 1;
      if (p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    }
  } else if (warp >= 2 && warp < 10) {
    const int group = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;
    RowOfWeights<GROUP, ZEROS> mine;
    mine.start(v, row >> 4, row & 15);
    uint32_t base = 0;                                   // chunks of the tiles ahead
    bool ok = true;
    // A stage is signalled when the next one's operands are there: the wait for its stores costs nothing then. (Each block signalled at once: a group of warps took 1400
    // cycles for a chunk, the products 1024.)
    int written = -1;
    auto settle = [&]() {
      if (written < 0) return;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(in_leader(&weights[written]));
    };
#pragma unroll 1
    for (int t = pair; t < tiles && ok; t += pairs, base += nc) {
      int tt, tn;
      tile_at(t, tiles_t, tiles_n, &tt, &tn);
      mine.scale(v.most[tile_of(tn, row >> 4) * TILE + (row & 15)]);
#pragma unroll 1
      for (int ch = group; ch < nc && ok; ch += 2) {
        const uint32_t ic = base + ch;
        const int q = ic % CHUNKS;
        bool late = !mbar_wait(&units_full[q], (ic / CHUNKS) & 1, p.spin_limit);
        mine.load(ring + q * U::BYTES, row & 15);
        __syncwarp();
        if (lane == 0) mbar_arrive(&units_empty[q]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint32_t it = 2 * ic + b;
          const int s = it % STAGES;
          uint32_t w[32];
          mine.block(b, w);
          settle();                                      // the block before this one
          if (it >= STAGES) late |= !mbar_wait(&empty[s], (it / STAGES - 1) & 1, p.spin_limit);
          tc_fence_after();
          tmem_st_32x32(tmem_base + A_COL + s * 32 + quarter, reinterpret_cast<const float*>(w));
          written = s;
        }
        if (late) *abort_flag = 1;
        ok = !__any_sync(0xffffffffu, *abort_flag);
      }
    }
    settle();
    if (!ok && lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
  } else if (warp == 18) {
    uint32_t ic = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      int tt, tn;
      tile_at(t, tiles_t, tiles_n, &tt, &tn);
      const unsigned char* from = v.at(tile_of(tn, lane & 7), 0);
      for (int ch = 0; ch < nc; ++ch, ++ic) {
        const int q = ic % CHUNKS;
        if (ic >= CHUNKS && !mbar_wait(&units_empty[q], (ic / CHUNKS - 1) & 1, p.spin_limit)) *abort_flag = 1;
        ok = !__any_sync(0xffffffffu, *abort_flag);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&units_full[q], U::BYTES);
        __syncwarp();
        if (lane < 8) bulk_load(ring + q * U::BYTES + lane * U::UNIT, from + (long)ch * U::UNIT, U::UNIT, &units_full[q]);
      }
    }
    for (uint32_t i = ic > CHUNKS ? ic - CHUNKS : 0; i < ic; ++i) mbar_wait(&units_full[i % CHUNKS], (i / CHUNKS) & 1, DRAIN);
  } else if (warp >= 10 && warp < 18) {
    const int half = (warp - 10) >> 2, row = (warp & 3) * 32 + lane;
    bool ok = true;
    int j = 0;
#pragma unroll 1
    for (int t = pair; t < tiles; t += pairs, ++j) {
      int tt, tn;
      tile_at(t, tiles_t, tiles_n, &tt, &tn);
      const int n0 = (tn * 2 + rank) * per_cta, n = n0 + (gated ? (row >> 5) * 16 + (lane & 15) : row), m = tt * p.tok, tokens = min(p.tok, p.T - m);
      const float out = power_of_two(exponent_of(v.most[tile_of(tn, row >> 4) * TILE + (row & 15)]) - 11);
      if (ok && !mbar_wait(acc_full, j & 1, p.spin_limit)) *abort_flag = 1;
      if (__any_sync(0xffffffffu, *abort_flag)) {
        if (ok && lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
        ok = false;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = half * 32; c < tokens; c += 64) {
        float f[32];
        if (ok) {
          tmem_ld_32x32(tmem_base + quarter + (uint32_t)c, f);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __int_as_float(0x7fffffff);
        }
        const int live = min(32, tokens - c);
        const float factor = lane < live ? p.factor[m + c + lane] : 0.f;
        const long first = (long)(m + c) * p.ldy + n;
        void* y = p.out_f32 ? (void*)(reinterpret_cast<float*>(p.y) + first) : (void*)(reinterpret_cast<bf16*>(p.y) + first);
        const bf16* residual = p.residual ? p.residual + (long)(m + c) * p.ldr + n : nullptr;
        const bool there = n < v.N;
        auto store = [&](auto g, auto f32) {
          if (live == 32) store32<decltype(g)::value, decltype(f32)::value, true>(f, out, factor, y, p.ldy, residual, p.ldr, 32, there, lane);
          else store32<decltype(g)::value, decltype(f32)::value, false>(f, out, factor, y, p.ldy, residual, p.ldr, live, there, lane);
        };
        using yes = std::true_type;
        using no = std::false_type;
        if (gated) p.out_f32 ? store(yes{}, yes{}) : store(yes{}, no{});
        else p.out_f32 ? store(no{}, yes{}) : store(no{}, no{});
      }
      tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) arrive_cluster(in_leader(acc_empty));
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

template <int GROUP, bool ZEROS>
int launch(const CUtensorMap& tx, const PairP& p, int pairs, cudaStream_t s) {
  auto k = int4_tc_pair_kernel<GROUP, ZEROS>;
  constexpr int smem = SMEM<GROUP, ZEROS>;
  if (int rc = opt_in_smem(k, smem)) return rc;
  return launch_chain_cluster(k, dim3(2 * pairs), dim3(THREADS), 2, (size_t)smem, s, tx, p);
}

}  // namespace

namespace ifab::int4 {

// Rows of x in f16 and their factors are int4_tc.cu's; arguments are checked there. pairs: of the device's SMs
int pair_product(const View& v, const void* rows, const float* factor, const bf16* residual, long ldr, void* y, long ldy, int out_f32, int T, int tok, int pairs, uint32_t spin_limit,
                 uint32_t* status, cudaStream_t s) {
  PairP p{v, y, ldy, out_f32, residual, ldr, factor, T, tok, status, spin_limit};
  CUtensorMap tx;          // of 16-bit elements
  if (int rc = make_tmap_bf16_2d(&tx, rows, (uint64_t)T, (uint64_t)v.K, (uint64_t)v.K, (uint32_t)(tok / 2))) return rc;
  if (v.zeros) return v.group == 128 ? launch<128, true>(tx, p, pairs, s) : v.group == 64 ? launch<64, true>(tx, p, pairs, s) : launch<32, true>(tx, p, pairs, s);
  return v.group == 128 ? launch<128, false>(tx, p, pairs, s) : v.group == 64 ? launch<64, false>(tx, p, pairs, s) : launch<32, false>(tx, p, pairs, s);
}

}  // namespace ifab::int4

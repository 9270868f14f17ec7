// Products of many rows with 4-bit weights (int4.cuh) on pairs of SMs: int4_tc.cu's operands and results, for prompts long enough to fill the chip with tiles of 256 weight
// rows (a gate | up matrix: 128 features) by up to 256 tokens.
//
// A lone CTA with 128 weight rows loads 16 KB of tokens for 256 cycles of products, as much as an SM gets out of L2; a pair shares the tokens' tile, half in each CTA's
// shared memory (tcgen05.mma.cta_group::2), and each CTA makes its 128 rows of weights. One pair an SM pair walks the tiles, with two sums in tensor memory: while one is
// stored, the next tile's products go into the other.
//   warp 0       copies of this CTA's half of the tokens; both CTAs' bytes complete on the leader's barrier
//   warp 1       allocates tensor memory; in the leader, MMAs
//   warp 2       copies of this CTA's codes
//   warps 3-10   this CTA's weights into its shared memory, signalled to the leader; two groups take the chunks of 128 columns in turn
//   warps 11-18  sums out of tensor memory, two warps for 32 rows. A lane is a weight row, so that a token's results leave as 64 bytes a warp. Gate and up rows lie in the two halves of a warp's
//                rows, sixteen each: a lane gives every other token's value to its partner and has both of the others
// Measured: 4096 rows of 2 x 16384 by 4096 803 - 820 us (the bf16 product of the same sizes 750; 1.1 TFLOP, 658 at the rate of a short burst), of 6144 by 4096 178 (152), 509 rows of the latter
// 35 (29). Long prompts are bound by the products at the clocks that the power limit leaves (their pipe is busy for 64 % of the time of 1024 rows, issue slots for 44 %);
// few tiles by 0.8 us a chunk, whatever their width, and 9.5 us beside. A thread has 96 registers; groups of 32, and of 64 with zero points, spill one.
// Weights go by way of shared memory: in tensor memory, where the MMA takes its first operand as well (int4_tc.cu), they leave no room for a second sum.
// Every wait is bounded; one that runs out raises the CTA's flag and the status word, tiles that are not complete are stored as NaN, and both CTAs meet at the closing barrier.
#include <algorithm>
#include <type_traits>

#include "int4_tc.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::tc;
using namespace ifab::int4;

namespace {

constexpr int FT = 128, BK = 64, TOK = 256, STAGES = 5, CHUNKS = 6, THREADS = 608, READERS = 8;
constexpr int W_BYTES = FT * BK * 2, STAGE = W_BYTES + TOK / 2 * BK * 2;      // weights, then tokens
template <int GROUP, bool ZEROS>
constexpr int SMEM = STAGES * STAGE + CHUNKS * Units<GROUP, ZEROS>::BYTES + 1024 + 512;
constexpr uint32_t SUM_COLS = 256;                   // of tensor memory
// A wait by parity tells a phase from the one before it only, so whoever waits has to know that the one before that is over. The groups that make operands know it by the order
// of the products: a group's block before this one, at most five back (three chunks apart where a tile has an odd number of them), waited for the products STAGES blocks ahead of
// it, whose own stage, and chunk of codes, were done with before.
static_assert(STAGES >= 5 && 2 * CHUNKS >= STAGES + 5, "a group could take a phase for the one two ahead");
constexpr uint32_t DRAIN = 4000000u;                 // limit of the waits for what a CTA that gives up has started
constexpr int QUIET = 2000;
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
// this CTA's tile; its bytes go to the barrier at `bar` (the leader's)
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* m, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(m), "r"(bar),
               "r"(x), "r"(y)
               : "memory");
}
// D[tmem of both] (+)= A[smem of both] * B[smem of both]; issued by ONE thread of the leader
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
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
// 32 lanes x 16 consecutive f32 columns
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
// Tokens 0 .. live - 1 (of 16) of this lane's row; `f`: the sums, `factor`: of token `lane & 15`; y and the residual from the first token's result on
template <bool GATED, bool F32, bool WHOLE>
__device__ __forceinline__ void store16(float (&f)[16], float out, float factor, void* y, long ldy, const bf16* residual, long ldr, int live, bool there, int lane) {
  if constexpr (GATED) {
    const bool up = lane >= 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lo = f[2 * i] * out, hi = f[2 * i + 1] * out, got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, 16), by = __shfl_sync(0xffffffffu, factor, 2 * i + up);
      const float v = gated_unit((up ? got : lo) * by, (up ? hi : got) * by);
      if (there && (WHOLE || 2 * i + up < live)) put<F32>(y, (2 * i + up) * ldy, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = f[i] * out * __shfl_sync(0xffffffffu, factor, i);
    if (!there) return;
    if (residual) {
      bf16 r[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = WHOLE || i < live ? residual[i * ldr] : __float2bfloat16_rn(0.f);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] += __bfloat162float(r[i]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (WHOLE || i < live) put<F32>(y, i * ldy, f[i]);
  }
}

// What lies behind the rings in shared memory
struct Signals {
  uint64_t full[STAGES];                             // leader's: both halves of the tokens, and an arrival of every warp that wrote weights
  uint64_t empty[STAGES];                            // each CTA's own, as acc_full
  uint64_t acc_full[2], acc_empty[2];                // of each sum; acc_empty: leader's
  uint64_t units_full[CHUNKS], units_empty[CHUNKS];  // each CTA's own
  uint64_t drained;
  uint32_t tmem_slot;
  int abort_flag;
};
// The second CTA, all threads: behind the last of what the leader signals to it. Where either gave up, tokens that it requested may still be under way, and their bytes count on
// the leader's barrier, in phases that may never end: they get QUIET microseconds, a thousand times what a copy takes. (A call, as its addresses spill where it is not: 4096 rows
// of 2 x 16384 by 4096 928 us with it, 957 without.)
__device__ __noinline__ void second_ends(int units) {
  extern __shared__ unsigned char smem_raw[];
  Signals* s = reinterpret_cast<Signals*>(((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023) + STAGES * STAGE + units);
  if (threadIdx.x < 32) mbar_wait(&s->drained, 0, DRAIN);
  if (__syncthreads_or(*(volatile int*)&s->abort_flag) && threadIdx.x < 32)
    for (int i = 0; i < QUIET; ++i) __nanosleep(1000);
}

// grid (2 * pairs), clusters of 2
template <int GROUP, bool ZEROS>
__global__ void __launch_bounds__(THREADS, 1) int4_tc_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, PairP p) {
  using U = Units<GROUP, ZEROS>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* ring = smem + STAGES * STAGE;                               // chunks of units
  Signals& sig = *reinterpret_cast<Signals*>(ring + CHUNKS * U::BYTES);
  uint64_t *full = sig.full, *empty = sig.empty, *acc_full = sig.acc_full, *acc_empty = sig.acc_empty, *units_full = sig.units_full, *units_empty = sig.units_empty;
  uint64_t* drained = &sig.drained;
  uint32_t* tmem_slot = &sig.tmem_slot;
  volatile int* abort_flag = &sig.abort_flag;
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
      mbar_init(&full[s], 1 + 8);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < CHUNKS; ++s) {
      mbar_init(&units_full[s], 1);
      mbar_init(&units_empty[s], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * READERS);
    }
    mbar_init(drained, 1);
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
        load_pair(smem + s * STAGE + W_BYTES, &tmap_x, in_leader(&full[s]), kb * BK, m);
      }
    }
    if (*abort_flag && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    if (rank == 0)                                       // what has been requested lands before the CTAs end, whoever gives up
      for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, DRAIN);
  } else if (warp == 1 && rank == 0) {
    // The whole warp walks and one lane issues: a block's products take 512 cycles, and with a lane alone on this path, two barriers to look at and stages by division the path
    // took 930.
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const uint32_t idesc = umma_idesc_f16(2 * FT, p.tok), at = smem_u32(smem);
    const uint64_t first = umma_desc_sw128(at);
    int s = 0, j = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs, ++j) {
      const uint32_t d = tmem_base + (j & 1) * SUM_COLS;
      ok = j < 2 || mbar_wait(&acc_empty[j & 1], ((j >> 1) - 1) & 1, p.spin_limit);
      tc_fence_after();
#pragma unroll 1
      for (int kb = 0; kb < nk && ok; ++kb) {
        ok = mbar_wait(&full[s], parity, p.spin_limit);
        tc_fence_after();
        if (ok && elected) {
          const uint64_t da = first + (uint64_t)(s * (STAGE >> 4)), db = da + (W_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) umma_f16_pair(d, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc, kb > 0 || k > 0);
          commit_pair(&empty[s]);
        }
        if (++s == STAGES) s = 0, parity ^= 1;
      }
      ok = !__any_sync(0xffffffffu, !ok || *abort_flag);
      if (ok && elected) commit_pair(&acc_full[j & 1]);
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) {
        uint32_t peers;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 1;" : "=r"(peers) : "r"(smem_u32(const_cast<int*>(abort_flag))));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peers), "r"(1) : "memory");
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        if (p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
      }
    }
    __syncwarp();
    // whoever gives up: products that were issued end before the CTAs do
    if (elected) commit_pair(drained);
    mbar_wait(drained, 0, DRAIN);
  } else if (warp >= 3 && warp < 11) {
    const int group = (warp - 3) >> 2, row = ((warp - 3) & 3) * 32 + lane;
    RowOfWeights<GROUP, ZEROS> mine;
    mine.start(v, row >> 4, row & 15);
    uint32_t base = 0;                                   // chunks of the tiles ahead
    bool ok = true;
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
          if (it >= STAGES) late |= !mbar_wait(&empty[s], (it / STAGES - 1) & 1, p.spin_limit);
          // a row of 128 bytes in pieces of 16, where the 128-byte swizzle has them
          uint4* to = reinterpret_cast<uint4*>(smem + s * STAGE + row * 128);
#pragma unroll
          for (int i = 0; i < 8; ++i) to[i ^ (row & 7)] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) arrive_cluster(in_leader(&full[s]));
        }
        if (late) *abort_flag = 1;
        ok = !__any_sync(0xffffffffu, *abort_flag);
      }
    }
    if (!ok && lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
  } else if (warp == 2) {
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
  } else if (warp >= 11) {
    const int half = (warp - 11) >> 2, row = (warp & 3) * 32 + lane;
    bool ok = true;
    int j = 0;
#pragma unroll 1
    for (int t = pair; t < tiles; t += pairs, ++j) {
      int tt, tn;
      tile_at(t, tiles_t, tiles_n, &tt, &tn);
      const int n0 = (tn * 2 + rank) * per_cta, n = n0 + (gated ? (row >> 5) * 16 + (lane & 15) : row), m = tt * p.tok, tokens = min(p.tok, p.T - m);
      const float out = power_of_two(exponent_of(v.most[tile_of(tn, row >> 4) * TILE + (row & 15)]) - 11);
      if (ok && !mbar_wait(&acc_full[j & 1], (j >> 1) & 1, p.spin_limit)) *abort_flag = 1;
      if (__any_sync(0xffffffffu, *abort_flag)) {
        if (ok && lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
        ok = false;
      }
      tc_fence_after();
#pragma unroll 1
      for (int c = half * 16; c < tokens; c += 32) {
        float f[16];
        if (ok) {
          tmem_ld_32x16(tmem_base + quarter + (j & 1) * SUM_COLS + (uint32_t)c, f);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = __int_as_float(0x7fffffff);
        }
        const int live = min(16, tokens - c);
        const float factor = (lane & 15) < live ? p.factor[m + c + (lane & 15)] : 0.f;
        const long first = (long)(m + c) * p.ldy + n;
        void* y = p.out_f32 ? (void*)(reinterpret_cast<float*>(p.y) + first) : (void*)(reinterpret_cast<bf16*>(p.y) + first);
        const bf16* residual = p.residual ? p.residual + (long)(m + c) * p.ldr + n : nullptr;
        const bool there = n < v.N;
        auto store = [&](auto g, auto f32) {
          if (live == 16) store16<decltype(g)::value, decltype(f32)::value, true>(f, out, factor, y, p.ldy, residual, p.ldr, 16, there, lane);
          else store16<decltype(g)::value, decltype(f32)::value, false>(f, out, factor, y, p.ldy, residual, p.ldr, live, there, lane);
        };
        using yes = std::true_type;
        using no = std::false_type;
        if (gated) p.out_f32 ? store(yes{}, yes{}) : store(yes{}, no{});
        else p.out_f32 ? store(no{}, yes{}) : store(no{}, no{});
      }
      tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) arrive_cluster(in_leader(&acc_empty[j & 1]));
    }
  }
  __syncwarp();
  if (cluster_rank() == 1) second_ends(CHUNKS * U::BYTES);
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
  static std::atomic<uint64_t> done;
  if (int rc = allow_smem(k, smem, device_now().id, done)) return rc;
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

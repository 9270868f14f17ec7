// Products of one to sixteen rows with 4-bit weights (int4.cuh):  y[t][n] = sum_k x[t][k] w[n][k] (+ residual), or of a gate | up matrix silu(gate) up.
//
// Bound by the stream of codes (half a byte a weight) as long as a weight costs little else: at 6.5 TB/s an SM has 2.8 lane operations for each. So no weight is made at all.
// A code q goes into the upper mantissa bits of a bf16 whose exponent makes it 16 + q, two codes in a rotation and a logical operation; weights are the sixteen rows of A of
// an m16n8k16, rows of x the eight columns of B, and what the offset and the zero point add to a group's sum, (16 + z) times the sum of x, is where that sum starts from
// (with the opposite sign). The sums of x come out of products with ones, once for all tiles of a CTA. The group's scale multiplies its f32 sum. Products are exact; sums run
// up to 24 |x| instead of 8 |x| a weight, which costs them two bits of f32; a result that comes out as no finite number is taken from the definition instead.
// A CTA has a share of the tiles of sixteen rows, and its eight warps share K: a warp takes every eighth run of one or two units, for all tiles of the CTA, so that its operands
// of x are loaded once, and normalised on the way. (A norm's factor into the sums instead saves the pass ahead, 1.5 us of 8 rows of 4096, but rounds the row differently from
// a norm of its own: results were off by twice their rounding.) Units come by bulk copies into a ring of the warp's own, the first ones ahead
// of the wait for the preceding kernel. (Loads ahead into registers waited for one another, whatever their number: 3.4 TB/s without any products.) Sums of the tiles lie in
// shared memory, a float4 a lane. What a unit costs is its instructions (two cycles of a scheduler for one on integers, eight for a product), so a ninth warp computes the
// copies' addresses and requests them, and a stage costs the others a look at its barrier and an arrival. The warps' sums are added in one order, and so a row's bits do not
// depend on the rows beside it.
// Few tiles and a long K: the units along K are shared by the CTAs of a cluster, whose sums are added over distributed shared memory.
// Measured, us (GB/s of codes and scales), weights not in L2: one row of 37888 by 8192 33.3 (4810; copies without products 6000), of 2 x 16384 by 4096 behind a norm 16.6 (4170), of 4096 by
// 16384 12.0, 4096 by 4096 4.6, 1024 by 1024 2.4; eight rows of these 21.9 (3170), 13.8, 5.3, 2.5; 16 of 4096 by 4096 7.7 (tiles on the tensor cores 9.9), 17 as two passes
// 11.8 (10.0). No pipe is full (one row of 2 x 16384 by 4096 under a profiler: issue slots 47 % and integers 54 % of the cycles of an SM at work, DRAM 38 %): what is left is latency. Four
// such warps a scheduler each wait at a stage's barrier, load from shared memory and go through a chain of eight dependent products a unit; a launch's start, first copies and last
// sums are 4 us of it. Two CTAs an SM leave a thread 96 registers, and 38 of the 108 forms spill (20 of them in groups of 32, up to 84 bytes; in groups of 128 up to 20).
#include <algorithm>

#include "int4.cuh"
#include "mma16816.cuh"
#include "tc_common.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::int4;

namespace {

constexpr int WARPS = 8, BARS = 17, LEFT = 16 * 8;      // BARS: words of a warp's barriers; LEFT: bytes from the first of them to its limit

struct RowsP {
  View v;
  const bf16* x; long ldx;
  const bf16* norm_w; float eps;
  const bf16* residual; long ldr;
  void* y; long ldy; int out_f32;
  int T;
  int groups, more, splits;      // CTAs (clusters) that share the tiles (pairs of them where gated), how many of them have one more than the others; CTAs of a cluster
  int most;                      // tiles of a CTA, at most
  int depth;                     // stages of a ring
  int wide;                      // units of a run: 2 also where they are taken one by one (J 1), so that sums are added in the same order
  uint32_t* status; uint32_t spin_limit;
};

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_part(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts_f4(uint32_t at, const float4& v) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void sts_u4(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t lds4(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds2(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v;
}
// 16 bytes that the preceding kernel has written (issued where it stands)
__device__ __forceinline__ uint4 ld_now16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void mma_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ bool ready(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// `left`: of the warp in shared memory, how many polls a wait may take; 0 once one ran out, and so nothing is waited for after it
__device__ __noinline__ bool wait_more(uint32_t bar, uint32_t parity, uint32_t left) {
  const uint32_t limit = lds4(left);
  for (uint32_t i = 0; i < limit; ++i) {
    if (ready(bar, parity)) return true;
    if (i > 256) __nanosleep(64);
  }
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(left), "r"(0u) : "memory");
  return false;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, uint32_t left) { return ready(bar, parity) || wait_more(bar, parity, left); }
// the warps that multiply (the ninth one is at its copies)
__device__ __forceinline__ void consumers() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); }

// One row: its factor out of the eight warps' sums of squares
__device__ __forceinline__ float factor_of_sums(const RowsP& p, const float* sums) {
  float ss = sums[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) ss += sums[w];
  return rsqrtf(ss / (float)p.v.K + p.eps);
}
// A norm's factor of the row of this lane's operands. One row: 256 threads add up its squares; more: a warp a row. In one order whatever the rows: of 256 threads' pieces of
// eight columns, 32 threads at a time. All loads of 4096 columns are under way at once.
__device__ __forceinline__ float factor_of(const RowsP& p, float* sums, float* inv, int warp, int lane, int most_rows) {
  const int pieces = p.v.K / 8;
  auto squares = [](const uint4& u, float& ss) {
    float f[8];
    unpack8(u, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
  };
  const uint4 none = make_uint4(0, 0, 0, 0);
  if (most_rows == 1) {
    float ss = 0.f;
    for (int i = warp * 32 + lane; i < pieces; i += 512) {
      const uint4 a = ld_now16(p.x + i * 8), b = i + 256 < pieces ? ld_now16(p.x + (i + 256) * 8) : none;
      squares(a, ss);
      squares(b, ss);
    }
    ss = warp_sum(ss);
    if (lane == 0) sums[warp] = ss;
    consumers();
    return factor_of_sums(p, sums);
  }
  float ss[WARPS] = {};
  if (warp < p.T) {
    const bf16* row = p.x + (long)warp * p.ldx;
    for (int i = lane; i < pieces; i += 512) {
      uint4 u[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) u[q] = i + q * 32 < pieces ? ld_now16(row + (i + q * 32) * 8) : none;
#pragma unroll
      for (int q = 0; q < 16; ++q) squares(u[q], ss[q % WARPS]);
    }
  }
#pragma unroll
  for (int q = 0; q < WARPS; ++q) ss[q] = warp_sum(ss[q]);
#pragma unroll
  for (int q = 1; q < WARPS; ++q) ss[0] += ss[q];
  if (lane == 0) inv[warp] = rsqrtf(ss[0] / (float)p.v.K + p.eps);
  consumers();
  return inv[lane >> 2];
}

// One result from the definition, in 64 bits: for sums that are not finite. 16 + q times an infinity and the offset's part of it are a NaN where q - z times it is an infinity, and
// (16 + q) x may pass f32's range where the result does not. `units`: of the tile; `r`: row of it; `gains`, `by`: the norm's (or null)
template <int GROUP, bool ZEROS, bool F16>
__device__ __noinline__ float from_definition(const unsigned char* units, int r, const bf16* x, int K, const bf16* gains, float by) {
  constexpr int NG = CHUNK / GROUP, UNIT = CODES + NG * (ZEROS ? 48 : 32);
  const int g = r & 7, h = r >> 3;
  double sum = 0.;
  for (int k = 0; k < K && sum == sum; k += 8) {      // (NaN stays NaN)
    const unsigned char* unit = units + (long)(k / CHUNK) * UNIT;
    const int group = k % CHUNK / GROUP;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(unit + (k >> 6 & 1) * 512 + code_at(g, k >> 3 & 3) + h * 8 + (k >> 5 & 1) * 4);
    const float s = scales_of(*reinterpret_cast<const uint16_t*>(unit + CODES + group * 32 + g * 4 + h * 2), F16).x;
    const int z = ZEROS ? unit[CODES + NG * 32 + group * 16 + g * 2 + h] : 8;
    for (int i = 0; i < 8; ++i) {
      const int q = (int)(__funnelshift_r(word, word, i / 2 * 4) >> (3 + i % 2 * 16) & 15u);
      float v = __bfloat162float(x[k + i]);
      if (gains) v = __bfloat162float(__float2bfloat16_rn(v * by * __bfloat162float(gains[k + i])));
      sum += (double)v * ((double)s * (q - z));
    }
  }
  return (float)sum;
}

// MR: most rows of x; J: units of a run; NORM: under a norm (asked for in the kernel, it cost the others 4 %: 8 rows of 8192 by 8192 13.2 us and 13.7)
template <int GROUP, bool ZEROS, bool F16, int MR, int J, bool NORM>
__global__ void __launch_bounds__(WARPS * 32 + 32, 2) int4_rows_kernel(RowsP p) {
  constexpr int NT = (MR + 7) / 8, RUNS = GROUP / 32, NG = 4 / RUNS, UNIT = CODES + NG * (ZEROS ? 48 : 32);      // runs of 32 columns of a group, groups of a unit, its bytes
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float sums[WARPS], inv[8];            // of a row's squares; the rows' factors
  __shared__ __align__(16) unsigned char runs_of_x[MR == 1 ? WARPS * 512 : 16];
  __shared__ uint64_t bars[WARPS * BARS];          // of a warp's stages: full, and eight further on empty; behind them the polls that its waits may take
  grid_dep_launch();
  const View& v = p.v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % p.splits, group = blockIdx.x / p.splits;
  const bool gated = v.halves == 2;
  const int fewest = v.tiles / p.groups, mine = fewest + (group < p.more), first = group * fewest + min(group, p.more);
  const int tiles = mine * v.halves;               // the CTA's: gate tiles, then up tiles
  const int chunk0 = (int)((long)v.chunks * split / p.splits), chunk1 = (int)((long)v.chunks * (split + 1) / p.splits);
  // the run behind the one that begins with unit r
  auto after = [&](int r) {
    if (J == 2 || p.wide == 1) return r + WARPS * p.wide;
    const int odd = (r - chunk0) & 1;
    return odd || r + 1 == chunk1 ? r - odd + WARPS * 2 : r + 1;
  };
  // sums: [warp][tile][rows of x by eight][lane], then the rings
  const uint32_t acc = smem_addr(smem) + (warp * p.most * NT * 32 + lane) * 16, rings = smem_addr(smem) + WARPS * p.most * NT * 512;
  const uint32_t bar = smem_addr(bars + warp * BARS);

  if (warp == WARPS && lane < WARPS) {
    for (int i = 0; i < p.depth; ++i) {
      tc::mbar_init(bars + lane * BARS + i, 1);
      tc::mbar_init(bars + lane * BARS + 8 + i, 1);
    }
    *reinterpret_cast<uint32_t*>(bars + lane * BARS + 16) = p.spin_limit;
    tc::mbar_fence_init();
  }
  __syncthreads();
  if (warp == WARPS) {
    // lane w requests the runs of warp w. Codes are written by no kernel of the stream: nothing to wait for
    if (lane < WARPS) {
      const uint32_t ring = rings + lane * p.depth * J * UNIT, full = smem_addr(bars + lane * BARS);
      const long row = (long)v.chunks * UNIT, up = (long)(v.tiles - mine) * row;      // from a tile to the next one, and to the first up tile besides
      int slot = 0, round = 0;
      bool ok = true;
      for (int rc = chunk0 + lane * p.wide; rc < chunk1 && ok; rc = after(rc)) {
        const unsigned char* from = v.units + (long)first * row + (long)rc * UNIT;
        const uint32_t bytes = J == 1 ? UNIT : min(J, chunk1 - rc) * UNIT;
        for (int i = 0; i < tiles; ++i, from += row) {
          if (gated && i == mine) from += up;
          // a warp that gave up gives its stages back all the same: nothing is requested into one whose last copy may not have landed
          if (round && (!wait_for(full + 64 + slot * 8, (round - 1) & 1, full + LEFT) || !lds4(full + LEFT))) { ok = false; break; }
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full + slot * 8), "r"(bytes) : "memory");
          asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ring + slot * J * UNIT), "l"(from), "r"(bytes),
                       "r"(full + slot * 8)
                       : "memory");
          if (++slot == p.depth) slot = 0, ++round;
        }
      }
    }
    __syncwarp();
  } else {
    for (int i = 0; i < tiles * NT; ++i) sts_f4(acc + i * 512, make_float4(0.f, 0.f, 0.f, 0.f));
    if (NORM)
      for (int i = threadIdx.x * 64; i < v.K; i += WARPS * 32 * 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.norm_w + i));
  }
  grid_dep_wait();

  bool late = p.spin_limit == 0;
  if (warp < WARPS) {
    const uint32_t ring = rings + warp * p.depth * J * UNIT + code_at(g, c), meta = CODES + g * 4 - code_at(g, c), end = ring + p.depth * J * UNIT;
    uint32_t at = ring, stage = bar, parity = 0;   // the stage at hand: this lane's first codes, and its barrier
    const int ch0 = chunk0 + warp * p.wide, k1 = min(v.K, chunk1 * CHUNK);      // the first run, the end of the CTA's columns
    uint4 b[J][NT][4];                             // operands: four runs of eight columns of a row of x a unit
    // eight columns under the norm, rounded as a norm of its own would leave them
    auto normed = [&](uint4& x, const uint4& gain, float by) {
      float f[8], w[8];
      unpack8(x, f);
      unpack8(gain, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = f[e] * by * w[e];
      x = pack8(f);
    };
    const uint4 none = make_uint4(0, 0, 0, 0);
    // One row: a lane has eight columns of a run, one run ahead, and the warp reads them from shared memory
    const uint32_t xs = smem_addr(runs_of_x) + warp * 512;
    uint4 ahead = none, gain = none;
    auto fetch = [&](int ch) {
      const int k = ch * CHUNK + lane * 8;
      const bool in = ch < chunk1 && lane < 16 * J && k < k1;
      ahead = in ? ld_now16(p.x + k) : none;
      if (NORM) gain = in ? *reinterpret_cast<const uint4*>(p.norm_w + k) : none;
    };
    if (MR == 1) fetch(ch0);
    const float by = NORM ? factor_of(p, sums, inv, warp, lane, MR) : 1.f;      // of this lane's row
    const bf16* xr[NT];                            // more: this lane's row (for rows behind the last one that one, whose results nothing stores), its first column
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] = p.x + (long)min(n * 8 + g, p.T - 1) * p.ldx + c * 8;
#pragma unroll 1
    for (int ch = ch0; ch < chunk1; ch = after(ch)) {
      if (MR == 1) {
        uint4 x = ahead;
        if (NORM) normed(x, gain, by);
        sts_u4(xs + lane * 16, x);
        fetch(after(ch));
        __syncwarp();
#pragma unroll
        for (int u = 0; u < J; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) b[u][0][i] = lds16(xs + (u * 16 + i * 4 + c) * 16);
        __syncwarp();
      } else {
        const int k0 = ch * CHUNK;
        if (NT == 1 && !NORM && k0 + J * CHUNK <= k1) {         // without the look at every column's place; with gains, or with two tiles of rows, the code's length costs more
                                                               // (8 rows of 4096 by 16384 14.4 us without, 13.7 with; of 2 x 16384 by 4096 under a norm 20.9 and 21.4)
#pragma unroll
          for (int u = 0; u < J; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) b[u][n][i] = ld_now16(xr[n] + k0 + u * CHUNK + i * 32);
        } else {
#pragma unroll
          for (int u = 0; u < J; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) b[u][n][i] = k0 + u * CHUNK + i * 32 + c * 8 < k1 ? ld_now16(xr[n] + k0 + u * CHUNK + i * 32) : none;
        }
        if (NORM) {
#pragma unroll
          for (int u = 0; u < J; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int k = k0 + u * CHUNK + i * 32 + c * 8;
              normed(b[u][0][i], k < k1 ? *reinterpret_cast<const uint4*>(p.norm_w + k) : none, by);
            }
        }
      }
      float sum[J][NT][NG][4];                     // of the groups' columns of x, rows 2 c and 2 c + 1, twice: times -24 without zero points
#pragma unroll
      for (int u = 0; u < J; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < NG; ++q) {
            constexpr uint32_t one = ZEROS ? 0x3f803f80u : 0xc1c0c1c0u;      // 1 or -24
#pragma unroll
            for (int r = q * RUNS; r < (q + 1) * RUNS; ++r) {
              if (r == q * RUNS) mma16816_alone(sum[u][n][q], one, one, one, one, b[u][n][r].x, b[u][n][r].y);
              else mma16816(sum[u][n][q], one, one, one, one, b[u][n][r].x, b[u][n][r].y);
              mma16816(sum[u][n][q], one, one, one, one, b[u][n][r].z, b[u][n][r].w);
            }
          }
      const bool whole = J == 1 || ch + 1 < chunk1;
      uint32_t to = acc;
#pragma unroll 1
      for (int i = 0; i < tiles; ++i, to += NT * 512) {
        late |= !wait_for(stage, parity, bar + LEFT);
        float4 so_far[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) so_far[n] = lds_f4(to + n * 512);
#pragma unroll
        for (int u = 0; u < J; ++u) {
          if (u == 1 && !whole) break;
          float part[NT][4];
          uint4 w;
#pragma unroll
          for (int r = 0; r < 4; ++r) {            // runs of 32 columns
            if (r % 2 == 0) w = lds16(at + u * UNIT + (r >> 1) * 512);
            const uint32_t wl = r & 1 ? w.y : w.x, wh = r & 1 ? w.w : w.z;
            const int q = r / RUNS;
            uint32_t al[4], ah[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) al[j] = pair_under(wl, j, 0x41804180u), ah[j] = pair_under(wh, j, 0x41804180u);      // 16 + q
            float lo = 1.f, hi = 1.f;              // -(16 + z)
            if (ZEROS && r % RUNS == 0) {
              const uint32_t z = lds2(at + u * UNIT + meta + NG * 32 + q * 16 - g * 2);
              lo = 8388592.f - __uint_as_float(0x4b000000u | (z & 255));
              hi = 8388592.f - __uint_as_float(0x4b000000u | z >> 8);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float(&x)[4] = sum[u][n][q];
              if (r % RUNS == 0 && ZEROS) {
                const float start[4] = {x[0] * lo, x[1] * lo, x[0] * hi, x[1] * hi};
                mma_from(part[n], start, al[0], ah[0], al[1], ah[1], b[u][n][r].x, b[u][n][r].y);
              } else if (r % RUNS == 0) {
                mma_from(part[n], x, al[0], ah[0], al[1], ah[1], b[u][n][r].x, b[u][n][r].y);
              } else {
                mma16816(part[n], al[0], ah[0], al[1], ah[1], b[u][n][r].x, b[u][n][r].y);
              }
              mma16816(part[n], al[2], ah[2], al[3], ah[3], b[u][n][r].z, b[u][n][r].w);
            }
            if (r % RUNS == RUNS - 1) {
              const float2 s = scales_of(lds4(at + u * UNIT + meta + q * 32), F16);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                so_far[n].x += s.x * part[n][0];
                so_far[n].y += s.x * part[n][1];
                so_far[n].z += s.y * part[n][2];
                so_far[n].w += s.y * part[n][3];
              }
            }
          }
        }
        __syncwarp();                              // the stage is read
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(stage + 64) : "memory");
#pragma unroll
        for (int n = 0; n < NT; ++n) sts_f4(to + n * 512, so_far[n]);
        at += J * UNIT;
        stage += 8;
        if (at == end) at = ring, stage = bar, parity ^= 1;
      }
    }
  }
  if (warp < WARPS && __any_sync(0xffffffffu, late)) {             // a copy that did not land: nothing of the tiles is right
    if (lane == 0 && p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
    const float nan = __int_as_float(0x7fffffff);
    for (int i = 0; i < tiles * NT; ++i) sts_f4(acc + i * 512, make_float4(nan, nan, nan, nan));
    // What was requested lands before its place is used for the sums below, or by another CTA: some milliseconds, a thousand times what a copy takes; nothing more is requested.
    // (A loop, or waits for each copy, in this place cost the kernels beside this one: a step of 24 layers, 1 row over 2000 positions, 750 us and 820)
    __nanosleep(1000000);
    __nanosleep(1000000);
    __nanosleep(1000000);
    __nanosleep(1000000);
  }
  __syncthreads();
  // the warps' sums, added up into [tile][16][rows of x] in the place of the rings
  constexpr int W = 8 * NT;
  const float* red = reinterpret_cast<const float*>(smem);
  const int step = p.most * NT * 128;
  float* part = reinterpret_cast<float*>(smem) + WARPS * step;
  for (int i = threadIdx.x; i < tiles * TILE * W; i += WARPS * 32 + 32) {
    const int t = i % W, r = i / W % TILE, tile = i / W / TILE;
    const float* f = red + ((tile * NT + (t >> 3)) * 32 + (r & 7) * 4 + ((t & 7) >> 1)) * 4 + (r >> 3) * 2 + (t & 1);
    part[i] = ((f[0] + f[step]) + (f[2 * step] + f[3 * step])) + ((f[4 * step] + f[5 * step]) + (f[6 * step] + f[7 * step]));
  }
  if (p.splits > 1) cluster_barrier();
  else __syncthreads();
  const int rows = mine * TILE;                    // of the result
  const uint32_t part_at = smem_addr(part);
  for (int i = threadIdx.x + split * (WARPS * 32 + 32); i < rows * p.T; i += p.splits * (WARPS * 32 + 32)) {
    const int r = i % rows, t = i / rows, n = first * TILE + r;
    if (n >= v.N) continue;
    const int at = r * W + t, up_at = at + rows * W;
    float a = 0.f, u = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      a += p.splits > 1 ? ld_part(part_at + at * 4, s) : part[at];
      if (gated) u += p.splits > 1 ? ld_part(part_at + up_at * 4, s) : part[up_at];
    }
    if (__builtin_expect(!(fabsf(a) <= 3.4028234e38f && fabsf(u) <= 3.4028234e38f), 0)) {      // no finite number: from the definition, unless a wait ran out
      bool right = true;
      for (int s = 0; s < p.splits * WARPS; ++s) {
        const uint32_t left = smem_addr(bars + s % WARPS * BARS) + LEFT;
        right = right && (p.splits > 1 ? __float_as_uint(ld_part(left, s / WARPS)) : lds4(left)) != 0;
      }
      if (right) {
        const bf16 *x = p.x + (long)t * p.ldx, *gains = NORM ? p.norm_w : nullptr;
        const int tile = first + r / TILE;
        const float by = !NORM ? 1.f : MR == 1 ? factor_of_sums(p, sums) : inv[t & 7];
        a = from_definition<GROUP, ZEROS, F16>(v.at(tile, 0), r % TILE, x, v.K, gains, by);
        if (gated) u = from_definition<GROUP, ZEROS, F16>(v.at(tile + v.tiles, 0), r % TILE, x, v.K, gains, by);
      }
    }
    if (gated) a = a / (1.f + __expf(-a)) * u;
    if (p.residual) a += __bfloat162float(p.residual[t * p.ldr + n]);
    if (p.out_f32) reinterpret_cast<float*>(p.y)[t * p.ldy + n] = a;
    else reinterpret_cast<bf16*>(p.y)[t * p.ldy + n] = __float2bfloat16_rn(a);
  }
  if (p.splits > 1) cluster_barrier();             // the sums stay until every CTA has read them
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// CTAs of a cluster that share K: the most an SM has to do (units of its tiles, at 24 ns of an SM's share of memory) is weighed against a cluster's two barriers and the trips
// between its CTAs, 1 us. Nothing of it goes by the rows, so that a row's bits do not either.
int splits_of(const View& v, int sms) {
  int best = 1;
  long least = 0;
  for (int s = 1; s <= 8 && s * WARPS <= std::max(v.chunks, WARPS); s *= 2) {
    const long cost = (long)ceil_div(v.tiles * s, sms) * v.halves * ceil_div(v.chunks, s) + (s > 1 ? 40 : 0);
    if (!least || cost < least) least = cost, best = s;
  }
  return best;
}
// Clusters of s CTAs that are counted on to run at once, two CTAs an SM: not all SMs of a part of the chip can be divided by four or eight. Of 148 SMs 148, 69 and 31 clusters of two,
// four and eight; the device has room for up to 71 and 33 of the latter
int at_once(int s, int sms) { return s <= 2 ? 2 * sms / s : s == 4 ? 2 * sms * 15 / 64 : 2 * sms * 6 / 56; }
constexpr int SMEM = 107 * 1024;                   // of a CTA, two of which share an SM (beside 5 KB that the kernel declares, and 1 KB each)

template <int GROUP, bool ZEROS, bool F16, int MR, int J, bool NORM>
int launch(RowsP p, cudaStream_t s) {
  constexpr int NT = (MR + 7) / 8, unit = CODES + CHUNK / GROUP * (ZEROS ? 48 : 32), tile = WARPS * NT * 512 + TILE * 8 * NT * 4;      // bytes of a tile's sums and their sum
  auto k = int4_rows_kernel<GROUP, ZEROS, F16, MR, J, NORM>;
  static std::atomic<uint64_t> done;
  const Device dev = device_now();
  const int sms = dev.sms, halves = p.v.halves;
  // as many CTAs as run at once, unless their tiles' sums are too many for them; those with one tile more come first, so that an SM has some of either kind
  p.groups = std::max(std::min(p.v.tiles, at_once(p.splits, sms)), ceil_div(p.v.tiles, (SMEM - WARPS * 3 * J * unit) / tile / halves));
  p.more = p.v.tiles % p.groups;
  p.most = (p.v.tiles / p.groups + (p.more > 0)) * halves;
  const int runs = ceil_div(ceil_div(p.v.chunks, p.splits), WARPS * p.wide) * (p.wide / J) * p.most;           // of a warp
  p.depth = std::max(1, std::min({runs, (SMEM - p.most * WARPS * NT * 512) / (WARPS * J * unit), 8}));
  const int smem = p.most * WARPS * NT * 512 + std::max(WARPS * p.depth * J * unit, p.most * TILE * 8 * NT * 4);
  if (int rc = allow_smem(k, SMEM, dev.id, done)) return rc;
  const dim3 grid(p.groups * p.splits);
  if (p.splits > 1) return launch_chain_cluster(k, grid, dim3(WARPS * 32 + 32), (unsigned)p.splits, (size_t)smem, s, p);
  return launch_chain(k, grid, dim3(WARPS * 32 + 32), (size_t)smem, s, p);
}
template <int GROUP, bool ZEROS, bool F16, int MR>
int launch_runs(RowsP p, cudaStream_t s) {
  p.splits = splits_of(p.v, device_now().sms);
  // runs of two units while every warp has one: a copy of 1 KB costs as much as one of two
  p.wide = ceil_div(p.v.chunks, p.splits) >= 2 * WARPS ? 2 : 1;
  if constexpr (MR <= 8) {
    if (p.norm_w) return p.wide == 2 ? launch<GROUP, ZEROS, F16, MR, 2, true>(p, s) : launch<GROUP, ZEROS, F16, MR, 1, true>(p, s);
    if (p.wide == 2) return launch<GROUP, ZEROS, F16, MR, 2, false>(p, s);
  }
  return launch<GROUP, ZEROS, F16, MR, 1, false>(p, s);
}
template <int GROUP, int MR>
int by_kind(const RowsP& p, cudaStream_t s) {
  if (p.v.zeros) return p.v.f16 ? launch_runs<GROUP, true, true, MR>(p, s) : launch_runs<GROUP, true, false, MR>(p, s);
  return p.v.f16 ? launch_runs<GROUP, false, true, MR>(p, s) : launch_runs<GROUP, false, false, MR>(p, s);
}
template <int MR>
int dispatch(const RowsP& p, cudaStream_t s) {
  return p.v.group == 128 ? by_kind<128, MR>(p, s) : p.v.group == 64 ? by_kind<64, MR>(p, s) : by_kind<32, MR>(p, s);
}

}  // namespace

// x [T, K] in bf16, rows on 16 bytes; norm_w: one to eight rows. The units are written by no kernel that may still run (ifab_int4_pack and ifab_int4_quantise see to it).
// spin_limit: polls of a wait for a copy.
extern "C" int ifab_int4_rows(const IfabInt4* d, const void* x, long ldx, const void* norm_w, float eps, const void* residual, long ldr, void* y, long ldy, int out_f32,
                              int T, uint32_t spin_limit, uint32_t* status, void* stream) {
  RowsP p{};
  if (view_of(d, &p.v) || T < 1 || !x || !y || ((uintptr_t)x | (uintptr_t)norm_w) % 16 || ldx % 8 || (norm_w && T > 8) || (p.v.halves == 2 && residual)) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  for (int t = 0; t < T; t += 16) {
    p.T = std::min(16, T - t);
    p.x = (const bf16*)x + t * ldx;
    p.ldx = ldx;
    p.norm_w = (const bf16*)norm_w;
    p.eps = eps;
    p.residual = residual ? (const bf16*)residual + t * ldr : nullptr;
    p.ldr = ldr;
    p.y = out_f32 ? (void*)((float*)y + t * ldy) : (void*)((bf16*)y + t * ldy);
    p.ldy = ldy;
    p.out_f32 = out_f32;
    p.status = status;
    p.spin_limit = spin_limit;
    if (int rc = p.T <= 1 ? dispatch<1>(p, s) : p.T <= 8 ? dispatch<8>(p, s) : dispatch<16>(p, s)) return rc;
  }
  return 0;
}

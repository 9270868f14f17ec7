// Products of one to sixteen rows with 4-bit weights (int4.cuh):  y[t][n] = sum_k x[t][k] w[n][k] (+ residual), or of a gate | up matrix silu(gate) up.
//
// Bound by the stream of codes (half a byte a weight) as long as a weight costs little else, so no weight becomes more than a bf16 difference q - z, which is exact:
// the products of a group are added up by the tensor cores (weights are the sixteen rows of A, rows of x the eight columns of B) and the group's scale multiplies
// their f32 sum. A CTA has up to eight tiles of sixteen rows; its eight warps take every eighth unit along K, with a ring of their own in shared memory (cp.async,
// no barrier among the warps), filled before the wait for the preceding kernel. Operands of x come from shared memory, where a CTA lays the columns of a segment
// once, normalised on the way. The warps' sums are added in one order, so a row's bits do not depend on the rows beside it.
// Few tiles and a long K: the units along K are shared by the CTAs of a cluster, whose sums are added over distributed shared memory.
#include <algorithm>

#include "int4.cuh"
#include "mma16816.cuh"
#include "tc_common.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::int4;

namespace {

constexpr int WARPS = 8, TB = 8;
constexpr int X_BYTES = 65536;                    // of shared memory for columns of x

struct RowsP {
  View v;
  const bf16* x; long ldx;
  const bf16* norm_w; float eps;
  const bf16* residual; long ldr;
  void* y; long ldy; int out_f32;
  int T;
  int groups, more, splits;      // CTAs (clusters) that share the tiles (pairs of them where gated), how many of them have one more than the others; CTAs of a cluster
  int cols;                      // columns of x in shared memory at a time
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

// MR: most rows of x
template <int GROUP, bool ZEROS, int MR>
struct RowsSmem {
  static constexpr int NT = (MR + 7) / 8, DEPTH = MR <= 2 ? 6 : 4;
  static constexpr int UNIT = CODES + CHUNK / GROUP * (ZEROS ? 48 : 32), RING = WARPS * DEPTH * UNIT;
  static constexpr int RED = WARPS * TB * TILE * 8 * NT * 4 + TB * TILE * 8 * NT * 4;         // takes the place of ring and rows
  static constexpr int bytes(int T, int cols) { return RING + T * (cols * 2 + 64) > RED ? RING + T * (cols * 2 + 64) : RED; }
};

template <int GROUP, bool ZEROS, int MR>
__global__ void __launch_bounds__(WARPS * 32, MR <= 8 ? 2 : 1) int4_rows_kernel(RowsP p) {
  using S = RowsSmem<GROUP, ZEROS, MR>;
  constexpr int NT = S::NT, DEPTH = S::DEPTH;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ float sums[WARPS * 8];
  grid_dep_launch();
  const View& v = p.v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % p.splits, group = blockIdx.x / p.splits;
  const bool gated = v.halves == 2;
  const int fewest = v.tiles / p.groups, mine = fewest + (group < p.more), first = group * fewest + min(group, p.more);
  const int tiles = mine * v.halves;               // the CTA's: gate tiles, then up tiles
  const int chunk0 = (int)((long)v.chunks * split / p.splits), chunk1 = (int)((long)v.chunks * (split + 1) / p.splits);
  const uint32_t ring = smem_addr(smem) + warp * DEPTH * S::UNIT, xs = smem_addr(smem) + S::RING;
  const int cols = p.cols, pitch = cols * 2 + 64;

  // the next unit to be requested: tile ri of chunk rc
  int rc = chunk0 + warp, ri = 0;
  const long row = (long)v.chunks * S::UNIT, up = (long)(v.tiles - mine) * row;      // from a tile to the next one, and to the first up tile besides
  const unsigned char* head = v.units + (long)first * row + (long)rc * S::UNIT + lane * 16;
  const unsigned char* from = head;
  auto request = [&](int slot) {
    if (rc < chunk1) {
      const uint32_t to = ring + slot * S::UNIT + lane * 16;
      copy16(to, from, true);
      copy16(to + 512, from + 512, true);
      if (lane < (S::UNIT - CODES) / 16) copy16(to + CODES, from + CODES, true);
      from += row;
      ++ri;
      if (gated && ri == mine) from += up;
      if (ri == tiles) {
        ri = 0;
        rc += WARPS;
        head += WARPS * S::UNIT;
        from = head;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < DEPTH; ++i) request(i);
  grid_dep_wait();

  float inv[NT == 1 ? MR : 1];                     // of the rows, where there is a norm
  if (NT == 1 && p.norm_w) {
    // MR 8: a warp a row; otherwise all of them every row. The sum of squares in one order whatever the rows: of 256 threads' pieces, 32 threads at a time
    constexpr int PIECES = MR == 8 ? WARPS : 1, STEP = MR == 8 ? 32 : 256;
    const int start = MR == 8 ? lane : threadIdx.x;
#pragma unroll
    for (int r = 0; r < (MR == 8 ? 1 : MR); ++r) {
      const int t = MR == 8 ? warp : r;
      float ss[PIECES] = {};
      if (t < p.T) {
        const bf16* xr = p.x + t * p.ldx;
        for (int i = start; i < v.K / 8; i += STEP * PIECES) {
          uint4 u[PIECES];
#pragma unroll
          for (int q = 0; q < PIECES; ++q) u[q] = i + q * STEP < v.K / 8 ? *reinterpret_cast<const uint4*>(xr + (i + q * STEP) * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int q = 0; q < PIECES; ++q) {
            float f[8];
            unpack8(u[q], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[q] += f[e] * f[e];
          }
        }
      }
#pragma unroll
      for (int q = 0; q < PIECES; ++q) ss[q] = warp_sum(ss[q]);
      if (lane == 0) {
        if (MR == 8) {
#pragma unroll
          for (int q = 1; q < PIECES; ++q) ss[0] += ss[q];
          sums[t] = ss[0];
        } else {
          sums[warp * 8 + t] = ss[0];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MR; ++t) {
      float s = sums[t];
      if (MR != 8)
#pragma unroll
        for (int w = 1; w < WARPS; ++w) s += sums[w * 8 + t];
      inv[t] = rsqrtf(s / (float)v.K + p.eps);
    }
  }
  // columns of a segment from chunk `at` on, zeros beyond K
  auto stage = [&](int at) {
    constexpr int HELD = MR < 8 ? MR : 8;          // rows whose pieces are on their way together
    const int pieces = cols / 8;
#pragma unroll 1
    for (int i = threadIdx.x; i < pieces; i += WARPS * 32) {
      const int k = at * CHUNK + i * 8;
      const bool in = k < v.K;
      uint4 gain = make_uint4(0, 0, 0, 0);
      if (NT == 1 && p.norm_w && in) gain = *reinterpret_cast<const uint4*>(p.norm_w + k);
#pragma unroll
      for (int t0 = 0; t0 < MR; t0 += HELD) {
        uint4 u[HELD];
#pragma unroll
        for (int t = 0; t < HELD; ++t) u[t] = in && t0 + t < p.T ? *reinterpret_cast<const uint4*>(p.x + (t0 + t) * p.ldx + k) : make_uint4(0, 0, 0, 0);
        if (NT == 1 && p.norm_w) {
          float w[8];
          unpack8(gain, w);
#pragma unroll
          for (int t = 0; t < HELD; ++t) {
            float f[8];
            unpack8(u[t], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = f[e] * inv[NT == 1 ? t : 0] * w[e];
            u[t] = pack8(f);
          }
        }
#pragma unroll
        for (int t = 0; t < HELD; ++t)
          if (t0 + t < p.T)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(xs + (t0 + t) * pitch + i * 16), "r"(u[t].x), "r"(u[t].y), "r"(u[t].z), "r"(u[t].w) : "memory");
      }
    }
  };

  float acc[TB][NT][4];
#pragma unroll
  for (int i = 0; i < TB; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][n][e] = 0.f;
  int slot = 0;
#pragma unroll 1
  for (int seg = chunk0; seg < chunk1; seg += cols / CHUNK) {
    if (seg > chunk0) __syncthreads();
    stage(seg);
    __syncthreads();
    const int end = min(chunk1, seg + cols / CHUNK);
#pragma unroll 1
    for (int ch = seg + warp; ch < end; ch += WARPS) {
      uint4 b[NT][4];                              // this lane's operands: four runs of eight columns of a row of x
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint32_t at = xs + (n * 8 + g) * pitch + (ch - seg) * CHUNK * 2 + c * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) b[n][i] = n * 8 + g < p.T ? lds16(at + i * 64) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < TB; ++i) {
        if (i >= tiles) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        __syncwarp();
        const uint32_t at = ring + slot * S::UNIT;
        float part[NT][4];
        uint4 w;
        uint32_t lo = less_of(8), hi = less_of(8);
#pragma unroll
        for (int r = 0; r < 4; ++r) {              // runs of 32 columns
          constexpr int RUNS = GROUP / 32;
          if (r % 2 == 0) w = lds16(at + (r >> 1) * 512 + code_at(g, c));
          if (ZEROS && r % RUNS == 0) {
            const uint32_t z = lds2(at + CODES + CHUNK / GROUP * 32 + r / RUNS * 16 + g * 2);
            lo = less_of(z & 255);
            hi = less_of(z >> 8);
          }
          const uint32_t wl = r & 1 ? w.y : w.x, wh = r & 1 ? w.w : w.z;
          uint32_t al[4], ah[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) al[j] = pair_of(wl, j, lo), ah[j] = pair_of(wh, j, hi);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (r % RUNS == 0) mma16816_alone(part[n], al[0], ah[0], al[1], ah[1], b[n][r].x, b[n][r].y);
            else mma16816(part[n], al[0], ah[0], al[1], ah[1], b[n][r].x, b[n][r].y);
            mma16816(part[n], al[2], ah[2], al[3], ah[3], b[n][r].z, b[n][r].w);
          }
          if (r % RUNS == RUNS - 1) {
            const float2 s = scales_of(lds4(at + CODES + r / RUNS * 32 + g * 4), v.f16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[i][n][0] += s.x * part[n][0];
              acc[i][n][1] += s.x * part[n][1];
              acc[i][n][2] += s.y * part[n][2];
              acc[i][n][3] += s.y * part[n][3];
            }
          }
        }
        __syncwarp();                              // the unit is read
        request(slot);
        slot = slot + 1 == DEPTH ? 0 : slot + 1;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // the warps' sums [warp][tile][16][rows of x], added up into [tile][16][rows of x]
  constexpr int W = 8 * NT;
  float* red = reinterpret_cast<float*>(smem);
  float* part = red + WARPS * TB * TILE * W;
#pragma unroll
  for (int i = 0; i < TB; ++i) {
    if (i >= tiles) break;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* to = red + ((warp * TB + i) * TILE + g) * W + n * 8 + 2 * c;
      *reinterpret_cast<float2*>(to) = make_float2(acc[i][n][0], acc[i][n][1]);
      *reinterpret_cast<float2*>(to + 8 * W) = make_float2(acc[i][n][2], acc[i][n][3]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tiles * TILE * W; i += WARPS * 32) {
    constexpr int STEP = TB * TILE * W;
    const float* f = red + i;
    part[i] = ((f[0] + f[STEP]) + (f[2 * STEP] + f[3 * STEP])) + ((f[4 * STEP] + f[5 * STEP]) + (f[6 * STEP] + f[7 * STEP]));
  }
  if (p.splits > 1) cluster_barrier();
  else __syncthreads();
  const int rows = mine * TILE;                    // of the result
  const uint32_t part_at = smem_addr(part);
  for (int i = threadIdx.x + split * WARPS * 32; i < rows * p.T; i += p.splits * WARPS * 32) {
    const int r = i % rows, t = i / rows, n = first * TILE + r;
    if (n >= v.N) continue;
    const int at = r * W + t, up_at = at + mine * TILE * W;
    float a = 0.f, u = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      a += p.splits > 1 ? ld_part(part_at + at * 4, s) : part[at];
      if (gated) u += p.splits > 1 ? ld_part(part_at + up_at * 4, s) : part[up_at];
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
// between its CTAs, 1 us, and against the barriers around every further segment of eight rows of x, 1.5 us. Nothing of it goes by the rows, so that a row's bits do not either.
int splits_of(const View& v, int sms) {
  int best = 1;
  long least = 0;
  for (int s = 1; s <= 8 && s * WARPS <= std::max(v.chunks, WARPS); s *= 2) {
    const int chunks = ceil_div(v.chunks, s);
    const long cost = (long)ceil_div(v.tiles * s, sms) * v.halves * chunks + (s > 1 ? 40 : 0) + 60 * (ceil_div(chunks * CHUNK, X_BYTES / 16) - 1);
    if (!least || cost < least) least = cost, best = s;
  }
  return best;
}

template <int GROUP, bool ZEROS, int MR>
int launch(RowsP p, cudaStream_t s) {
  using S = RowsSmem<GROUP, ZEROS, MR>;
  auto k = int4_rows_kernel<GROUP, ZEROS, MR>;
  const int sms = tc::device_sms();
  p.splits = splits_of(p.v, sms);
  // as many CTAs as run at once, two on an SM, unless their tiles are too many for them; those with one tile more come first, so that an SM has one of either kind
  p.groups = std::max(std::min(p.v.tiles, 2 * sms / p.splits), ceil_div(p.v.tiles, TB / p.v.halves));
  p.more = p.v.tiles % p.groups;
  p.cols = std::min(ceil_div(ceil_div(p.v.chunks, p.splits), WARPS) * WARPS * CHUNK, X_BYTES / 2 / MR / (WARPS * CHUNK) * (WARPS * CHUNK));
  if (int rc = (int)cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::bytes(MR, X_BYTES / 2 / MR))) return rc;
  const int smem = S::bytes(p.T, p.cols);
  const dim3 grid(p.groups * p.splits);
  if (p.splits > 1) return launch_chain_cluster(k, grid, dim3(WARPS * 32), (unsigned)p.splits, (size_t)smem, s, p);
  return launch_chain(k, grid, dim3(WARPS * 32), (size_t)smem, s, p);
}
template <int MR>
int dispatch(const RowsP& p, cudaStream_t s) {
  if (p.v.zeros) return p.v.group == 128 ? launch<128, true, MR>(p, s) : p.v.group == 64 ? launch<64, true, MR>(p, s) : launch<32, true, MR>(p, s);
  return p.v.group == 128 ? launch<128, false, MR>(p, s) : p.v.group == 64 ? launch<64, false, MR>(p, s) : launch<32, false, MR>(p, s);
}

}  // namespace

// x [T, K] in bf16, rows on 16 bytes; norm_w: one to eight rows. The units are written by no kernel that may still run (ifab_int4_pack and ifab_int4_quantise see to it).
extern "C" int ifab_int4_rows(const IfabInt4* d, const void* x, long ldx, const void* norm_w, float eps, const void* residual, long ldr, void* y, long ldy, int out_f32,
                              int T, void* stream) {
  RowsP p{};
  if (view_of(d, &p.v) || T < 1 || !x || !y || ((uintptr_t)x | (uintptr_t)norm_w) % 16 || ldx % 8 || (norm_w && T > 8) || (p.v.halves == 2 && residual)) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  for (int t = 0; t < T; t += 16) {
    p.T = min(16, T - t);
    p.x = (const bf16*)x + t * ldx;
    p.ldx = ldx;
    p.norm_w = (const bf16*)norm_w;
    p.eps = eps;
    p.residual = residual ? (const bf16*)residual + t * ldr : nullptr;
    p.ldr = ldr;
    p.y = out_f32 ? (void*)((float*)y + t * ldy) : (void*)((bf16*)y + t * ldy);
    p.ldy = ldy;
    p.out_f32 = out_f32;
    if (int rc = p.T <= 2 ? dispatch<2>(p, s) : p.T <= 8 ? dispatch<8>(p, s) : dispatch<16>(p, s)) return rc;
  }
  return 0;
}

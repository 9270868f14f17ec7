// 4-bit weights into their units (int4.cuh) and out of them.
//
//   quantise     s = bf16(max |w| / 7), z = 8, or with zero points lo = min(w, 0), hi = max(w, 0), s = bf16((hi - lo) / 15), z = rint(-lo / s) within 0 .. 15;
//                q = rint(w / s) + z within 0 .. 15, divisions and roundings as IEEE 754 has them (halves to even); where s is 0, so are the weights. A group that holds an
//                infinity or NaN gets a scale of NaN: what it multiplies is NaN, not something else.
//   pack         codes, scales and zero points of a checkpoint
//   dequantise   bf16(s (q - z))
// Bound by the bytes of the matrix. A warp has a unit: lane 4 g + c holds two runs of eight columns of rows g and g + 8 in both blocks; four lanes read 64 bytes of a row.
#include "int4.cuh"
#include "ifab_kernels.h"

using namespace ifab;
using namespace ifab::int4;

namespace {

__device__ __forceinline__ uint32_t word_of(const uint8_t* q) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= (uint32_t)q[2 * j] << (4 * j) | (uint32_t)q[2 * j + 1] << (4 * j + 16);
  return w << 3 | w >> 29;
}
// Rows' largest finite scales. The launch behind this one may read units ahead of its wait for the kernel before it (int4_rows.cu): this one is launched behind the end of the
// kernels that write them, and `settled_kernel` behind its own.
__global__ void __launch_bounds__(256) most_kernel(View v) {
  const int row = blockIdx.x * 256 + threadIdx.x, tile = row / TILE, r = row % TILE;
  if (tile >= v.halves * v.tiles) return;
  float most = 0.f;
  for (int ch = 0; ch < v.chunks; ++ch)
    for (int i = 0; i < v.groups(); ++i) {
      const float s = fabsf(scales_of(reinterpret_cast<const uint16_t*>(v.at(tile, ch) + CODES)[i * 16 + (r & 7) * 2 + (r >> 3)], v.f16).x);
      if (s <= 3.4028234e38f) most = fmaxf(most, s);
    }
  v.most[row] = most;
}
__global__ void settled_kernel() {}

struct Place {           // of a lane in its unit
  int tile, chunk, half, row0, g, c;
  __device__ __forceinline__ Place(const View& v, long unit) {
    const int lane = threadIdx.x & 31;
    tile = (int)(unit / v.chunks);
    chunk = (int)(unit - (long)tile * v.chunks);
    half = tile >= v.tiles;
    row0 = (tile - half * v.tiles) * TILE;
    g = lane >> 2;
    c = lane & 3;
  }
  // row of the matrix for row g + 8 h; -1: none
  __device__ __forceinline__ long row(const View& v, int h) const { return row0 + g + 8 * h < v.N ? (long)half * v.N + row0 + g + 8 * h : -1; }
  // first column of run r of four
  __device__ __forceinline__ int col(int r) const { return chunk * CHUNK + r * 32 + c * 8; }
};

template <int GROUP, bool ZEROS>
__global__ void __launch_bounds__(256) quantise_kernel(View v, const bf16* w, long ldw, long units) {
  grid_dep_wait();
  const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const Place at(v, unit);
  unsigned char* out = v.at(at.tile, at.chunk);
  float f[2][4][8];        // [row][run][column]
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long row = at.row(v, h);
      const int k = at.col(r);
      uint4 u = make_uint4(0, 0, 0, 0);
      if (row >= 0 && k < v.K) u = ld_stream16(w + row * ldw + k);
      unpack8(u, f[h][r]);
    }
  constexpr int RUNS = GROUP / 32;      // of a group
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r0 = 0; r0 < 4; r0 += RUNS) {
      float lo = 0.f, hi = 0.f;
      int bad = 0;
#pragma unroll
      for (int r = r0; r < r0 + RUNS; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = f[h][r][i];
          lo = fminf(lo, x);
          hi = fmaxf(hi, x);
          bad |= !(fabsf(x) <= 3.4028234e38f);
        }
#pragma unroll
      for (int o = 1; o < 4; o *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad |= __shfl_xor_sync(0xffffffffu, bad, o);
      }
      bf16 sb = __float2bfloat16_rn(ZEROS ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f));
      const float s = __bfloat162float(sb) == 0.f ? 1.f : __bfloat162float(sb);
      const float z = ZEROS ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 8.f;
#pragma unroll
      for (int r = r0; r < r0 + RUNS; ++r) {
        uint8_t q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = (uint8_t)(bad ? z : fminf(fmaxf(rintf(__fdiv_rn(f[h][r][i], s)) + z, 0.f), 15.f));
        *reinterpret_cast<uint32_t*>(out + (r >> 1) * 512 + code_at(at.g, at.c) + 8 * h + 4 * (r & 1)) = word_of(q);
      }
      if (at.c == 0) {
        const int group = r0 / RUNS;
        reinterpret_cast<bf16*>(out + CODES)[group * 16 + at.g * 2 + h] = bad ? __ushort_as_bfloat16(0x7fc0) : sb;
        if (ZEROS) (out + CODES + v.groups() * 32)[group * 16 + at.g * 2 + h] = (uint8_t)z;
      }
    }
}

__global__ void __launch_bounds__(256) pack_kernel(View v, const uint8_t* codes, long ldc, const uint16_t* scales, const uint8_t* zeros, long units) {
  grid_dep_wait();
  const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const Place at(v, unit);
  unsigned char* out = v.at(at.tile, at.chunk);
  const int per = (v.K + v.group - 1) / v.group;       // groups of a row
  for (int h = 0; h < 2; ++h) {
    const long row = at.row(v, h);
    for (int r = 0; r < 4; ++r) {
      uint8_t q[8];
      for (int i = 0; i < 8; ++i) {
        const int k = at.col(r) + i;
        q[i] = row < 0 ? 8 : k < v.K ? codes[row * ldc + k] & 15 : zeros ? zeros[row * per + min(k / v.group, per - 1)] & 15 : 8;
      }
      *reinterpret_cast<uint32_t*>(out + (r >> 1) * 512 + code_at(at.g, at.c) + 8 * h + 4 * (r & 1)) = word_of(q);
    }
    if (at.c < v.groups()) {
      const int group = at.chunk * v.groups() + at.c;
      const bool in = row >= 0 && group < per;
      reinterpret_cast<uint16_t*>(out + CODES)[at.c * 16 + at.g * 2 + h] = in ? scales[row * per + group] : 0;
      // a group beyond K: the zero point that its codes were given above
      if (v.zeros) (out + CODES + v.groups() * 32)[at.c * 16 + at.g * 2 + h] = row < 0 ? 8 : zeros[row * per + min(group, per - 1)] & 15;
    }
  }
}

__global__ void __launch_bounds__(256) dequantise_kernel(View v, bf16* w, long ldw, long units) {
  grid_dep_wait();
  const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const Place at(v, unit);
  const unsigned char* in = v.at(at.tile, at.chunk);
  uint4 u[2];              // [block]: row g's two runs, row g + 8's
  u[0] = ld_stream16(in + code_at(at.g, at.c));
  u[1] = ld_stream16(in + 512 + code_at(at.g, at.c));
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int group = r * 32 / v.group, k = at.col(r);
    const float2 s = scales_of(reinterpret_cast<const uint32_t*>(in + CODES)[group * 8 + at.g], v.f16);
    const uint4 b = u[r >> 1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long row = at.row(v, h);
      const uint32_t z = v.zeros ? (in + CODES + v.groups() * 32)[group * 16 + at.g * 2 + h] : 8;
      const uint32_t word = h ? (r & 1 ? b.w : b.z) : (r & 1 ? b.y : b.x);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t two = pair_under(word, j, 0x41804180u);          // 16 + q
        const float2 d = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two));
        f[2 * j] = (d.x - (float)(16 + z)) * (h ? s.y : s.x);
        f[2 * j + 1] = (d.y - (float)(16 + z)) * (h ? s.y : s.x);
      }
      if (row >= 0 && k < v.K) *reinterpret_cast<uint4*>(w + row * ldw + k) = pack8(f);
    }
  }
}

template <int GROUP>
int launch_quantise(const View& v, const bf16* w, long ldw, long units, cudaStream_t s) {
  return launch_chain(v.zeros ? quantise_kernel<GROUP, true> : quantise_kernel<GROUP, false>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, s, v, w, ldw, units);
}
int settle(const View& v, cudaStream_t s) {
  most_kernel<<<(v.halves * v.tiles * TILE + 255) / 256, 256, 0, s>>>(v);
  settled_kernel<<<1, 32, 0, s>>>();
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" uint64_t ifab_int4_bytes(int N, int K, int group, int zeros, int gated) {
  if (N < 1 || K < 8 || K % 8 || (group != 32 && group != 64 && group != 128)) return 0;
  return (uint64_t)((N + TILE - 1) / TILE) * (gated ? 2 : 1) * ((uint64_t)((K + CHUNK - 1) / CHUNK) * unit_bytes(group, zeros) + TILE * 4);
}

// w [N or 2 N, K] in bf16, rows on 16 bytes
extern "C" int ifab_int4_quantise(const IfabInt4* d, const void* w, long ldw, void* stream) {
  View v;
  if (view_of(d, &v) || v.f16 || !w || (uintptr_t)w % 16 || ldw % 8 || ldw < v.K) return -1;
  const long units = (long)v.halves * v.tiles * v.chunks;
  cudaStream_t s = (cudaStream_t)stream;
  const bf16* p = (const bf16*)w;
  int rc = v.group == 128 ? launch_quantise<128>(v, p, ldw, units, s) : v.group == 64 ? launch_quantise<64>(v, p, ldw, units, s) : launch_quantise<32>(v, p, ldw, units, s);
  return rc ? rc : settle(v, s);
}

// codes [N or 2 N, K] a byte each (low four bits), scales and zero points [N or 2 N, ceil(K / group)]
extern "C" int ifab_int4_pack(const IfabInt4* d, const uint8_t* codes, long ldc, const void* scales, const uint8_t* zeros, void* stream) {
  View v;
  if (view_of(d, &v) || !codes || !scales || (uintptr_t)scales % 2 || (v.zeros != 0) != (zeros != nullptr) || ldc < v.K) return -1;
  const long units = (long)v.halves * v.tiles * v.chunks;
  cudaStream_t s = (cudaStream_t)stream;
  int rc = launch_chain(pack_kernel, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, s, v, codes, ldc, (const uint16_t*)scales, zeros, units);
  return rc ? rc : settle(v, s);
}

// out [N or 2 N, K] in bf16, rows on 16 bytes
extern "C" int ifab_int4_dequantise(const IfabInt4* d, void* out, long ldo, void* stream) {
  View v;
  if (view_of(d, &v) || !out || (uintptr_t)out % 16 || ldo % 8 || ldo < v.K) return -1;
  const long units = (long)v.halves * v.tiles * v.chunks;
  return launch_chain(dequantise_kernel, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, v, (bf16*)out, ldo, units);
}

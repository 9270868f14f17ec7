// 4-bit weights into their units (int4.cuh) and out of them.
//
//   quantise     s = bf16(max |w| / 7), z = 8, or with zero points lo = min(w, 0), hi = max(w, 0), s = bf16((hi - lo) / 15), z = rint(-lo / s) within 0 .. 15;
//                q = rint(w / s) + z within 0 .. 15, divisions and roundings as IEEE 754 has them (halves to even); where s is 0, so are the weights. A group that holds an
//                infinity or NaN gets a scale of NaN: what it multiplies is NaN, not something else.
//   pack         codes, scales and zero points of a checkpoint
//   dequantise   bf16(s (q - z))
// Bound by the bytes of the matrix. A CTA has a tile of sixteen rows and its warps the units in turn, so that the rows' largest scales are at hand in the end: lane 4 g + c
// holds two runs of eight columns of rows g and g + 8 in both blocks; four lanes read 64 bytes of a row.
// Measured, 32768 x 4096 in groups of 64 with zero points: quantise 78 us in the kernel (4.4 TB/s of 6.5; instructions are issued in 61 % of the cycles, the rounding's seven a
// weight; with zero points 8 bytes a thread spill), without zero points and groups of 128 68 with the call; dequantise 58 (5.8 TB/s). 1024 x 4096: 16 and 6.5, the calls' own time.
// w / s is w times 1 / s and times what 1 / s was rounded off, off by 2^-45 ahead of its rounding to f32: a quotient that is half a step exactly comes out so, and others are
// 2^-10 and more away from it, as w and s have eight bits. Scales below 2^-126 and above 2^100 divide.
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
// The launch behind a linear may read units ahead of its wait for the kernel before it (int4_rows.cu): this one is launched behind the end of the kernels that write them
__global__ void settled_kernel() {}

// rows' largest finite scales, out of the warps' (lane 4 g: rows g and g + 8) into v.most; all threads of the CTA
__device__ __forceinline__ void keep_most(const View& v, int tile, float (&most)[2]) {
  __shared__ float all[8][TILE];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((lane & 3) == 0) {
    all[warp][lane >> 2] = most[0];
    all[warp][(lane >> 2) + 8] = most[1];
  }
  __syncthreads();
  if (threadIdx.x < TILE) {
    float m = 0.f;
    for (int w = 0; w < 8; ++w) m = fmaxf(m, all[w][threadIdx.x]);
    v.most[tile * TILE + threadIdx.x] = m;
  }
}

struct Place {           // of a lane in its unit
  int tile, chunk, half, row0, g, c;
  __device__ __forceinline__ Place(const View& v, int tile_, int chunk_) {
    const int lane = threadIdx.x & 31;
    tile = tile_;
    chunk = chunk_;
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
__global__ void __launch_bounds__(256, 4) quantise_kernel(View v, const bf16* w, long ldw) {
  grid_dep_wait();
  float most[2] = {0.f, 0.f};
#pragma unroll 1
  for (int chunk = threadIdx.x >> 5; chunk < v.chunks; chunk += 8) {
    const Place at(v, blockIdx.x, chunk);
    unsigned char* out = v.at(at.tile, at.chunk);
    uint4 u[2][4];           // [row][run]
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const long row = at.row(v, h);
        const int k = at.col(r);
        u[h][r] = make_uint4(0, 0, 0, 0);
        if (row >= 0 && k < v.K) u[h][r] = ld_stream16(w + row * ldw + k);
      }
    constexpr int RUNS = GROUP / 32;      // of a group
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r0 = 0; r0 < 4; r0 += RUNS) {
        // the smallest and the largest, NaN where there is one
        __nv_bfloat162 two_lo = __float2bfloat162_rn(0.f), two_hi = two_lo;
#pragma unroll
        for (int r = r0; r < r0 + RUNS; ++r) {
          const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&u[h][r]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            two_lo = __hmin2_nan(two_lo, x[i]);
            two_hi = __hmax2_nan(two_hi, x[i]);
          }
        }
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
          two_lo = __hmin2_nan(two_lo, __shfl_xor_sync(0xffffffffu, two_lo, o));
          two_hi = __hmax2_nan(two_hi, __shfl_xor_sync(0xffffffffu, two_hi, o));
        }
        const float lo = __bfloat162float(__hmin_nan(two_lo.x, two_lo.y)), hi = __bfloat162float(__hmax_nan(two_hi.x, two_hi.y));
        const bool bad = !(fabsf(lo) <= 3.4028234e38f && fabsf(hi) <= 3.4028234e38f);
        float range = ZEROS ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f);
        if (ZEROS && range > 3.4028234e38f) range = 2.f * __fdiv_rn(0.5f * hi - 0.5f * lo, 15.f);      // hi - lo passes f32's range, a fifteenth of it does not
        const bf16 sb = __float2bfloat16_rn(range);
        const float s = __bfloat162float(sb) == 0.f ? 1.f : __bfloat162float(sb), by = __frcp_rn(s);
        const int z = ZEROS && !bad ? (int)fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 8;
        const float rest = fmaf(-s, by, 1.f) * by, top = (float)(15 - z);
        const bool plain = s < 1.1754944e-38f || s > 1.2676506e30f || bad;      // 1 / s is no number to multiply by, or (above 2^100) what it was rounded off is none
#pragma unroll
        for (int r = r0; r < r0 + RUNS; ++r) {
          constexpr float SHIFT = 12582912.f;              // 1.5 2^23: a number near it has its nearest integer in its last bits, halves to even
          float f[8];
          unpack8(u[h][r], f);
          uint32_t word = (z - 0x4b400000u) * 0x11111111u;
          if (plain) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = bad ? 0.f : fminf(fmaxf(__fdiv_rn(f[i], s), -(float)z), top);
          } else {
            // without zero points a quotient is at most 7 (1 + 2^-8), with them at least -(z + 1/2)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              f[i] = fmaf(f[i], by, f[i] * rest);
              if (ZEROS) f[i] = fminf(f[i], top);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) word += __float_as_uint(f[i] + SHIFT) << ((i >> 1) * 4 + (i & 1) * 16);
          *reinterpret_cast<uint32_t*>(out + (r >> 1) * 512 + code_at(at.g, at.c) + 8 * h + 4 * (r & 1)) = word << 3 | word >> 29;
        }
        if (at.c == 0) {
          const int group = r0 / RUNS;
          reinterpret_cast<bf16*>(out + CODES)[group * 16 + at.g * 2 + h] = bad ? __ushort_as_bfloat16(0x7fc0) : sb;
          if (ZEROS) (out + CODES + v.groups() * 32)[group * 16 + at.g * 2 + h] = (uint8_t)z;
        }
        if (!bad) most[h] = fmaxf(most[h], __bfloat162float(sb));
      }
  }
  keep_most(v, blockIdx.x, most);
}

__global__ void __launch_bounds__(256) pack_kernel(View v, const uint8_t* codes, long ldc, const uint16_t* scales, const uint8_t* zeros) {
  grid_dep_wait();
  float most[2] = {0.f, 0.f};
  const int per = (v.K + v.group - 1) / v.group;       // groups of a row
  for (int chunk = threadIdx.x >> 5; chunk < v.chunks; chunk += 8)
    for (int h = 0; h < 2; ++h) {
      const Place at(v, blockIdx.x, chunk);
      unsigned char* out = v.at(at.tile, at.chunk);
      const long row = at.row(v, h);
      for (int r = 0; r < 4; ++r) {
        uint8_t q[8];
        for (int i = 0; i < 8; ++i) {
          const int k = at.col(r) + i;
          q[i] = row < 0 ? 8 : k < v.K ? codes[row * ldc + k] & 15 : zeros ? zeros[row * per + min(k / v.group, per - 1)] & 15 : 8;
        }
        *reinterpret_cast<uint32_t*>(out + (r >> 1) * 512 + code_at(at.g, at.c) + 8 * h + 4 * (r & 1)) = word_of(q);
      }
      float widest = 0.f;
      if (at.c < v.groups()) {
        const int group = at.chunk * v.groups() + at.c;
        const bool in = row >= 0 && group < per;
        if (in) widest = fabsf(scales_of(scales[row * per + group], v.f16).x);
        reinterpret_cast<uint16_t*>(out + CODES)[at.c * 16 + at.g * 2 + h] = in ? scales[row * per + group] : 0;
        // a group beyond K: the zero point that its codes were given above
        if (v.zeros) (out + CODES + v.groups() * 32)[at.c * 16 + at.g * 2 + h] = row < 0 ? 8 : zeros[row * per + min(group, per - 1)] & 15;
      }
      if (!(widest <= 3.4028234e38f)) widest = 0.f;
      for (int o = 1; o < 4; o *= 2) widest = fmaxf(widest, __shfl_xor_sync(0xffffffffu, widest, o));
      most[h] = fmaxf(most[h], widest);
    }
  keep_most(v, blockIdx.x, most);
}

__global__ void __launch_bounds__(256) dequantise_kernel(View v, bf16* w, long ldw, long units) {
  grid_dep_wait();
  const long unit = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const Place at(v, (int)(unit / v.chunks), (int)(unit % v.chunks));
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
int launch_quantise(const View& v, const bf16* w, long ldw, cudaStream_t s) {
  return launch_chain(v.zeros ? quantise_kernel<GROUP, true> : quantise_kernel<GROUP, false>, dim3(v.halves * v.tiles), dim3(256), 0, s, v, w, ldw);
}
int settle(cudaStream_t s) {
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
  cudaStream_t s = (cudaStream_t)stream;
  const bf16* p = (const bf16*)w;
  int rc = v.group == 128 ? launch_quantise<128>(v, p, ldw, s) : v.group == 64 ? launch_quantise<64>(v, p, ldw, s) : launch_quantise<32>(v, p, ldw, s);
  return rc ? rc : settle(s);
}

// codes [N or 2 N, K] a byte each (low four bits), scales and zero points [N or 2 N, ceil(K / group)]
extern "C" int ifab_int4_pack(const IfabInt4* d, const uint8_t* codes, long ldc, const void* scales, const uint8_t* zeros, void* stream) {
  View v;
  if (view_of(d, &v) || !codes || !scales || (uintptr_t)scales % 2 || (v.zeros != 0) != (zeros != nullptr) || ldc < v.K) return -1;
  cudaStream_t s = (cudaStream_t)stream;
  int rc = launch_chain(pack_kernel, dim3(v.halves * v.tiles), dim3(256), 0, s, v, codes, ldc, (const uint16_t*)scales, zeros);
  return rc ? rc : settle(s);
}

// out [N or 2 N, K] in bf16, rows on 16 bytes
extern "C" int ifab_int4_dequantise(const IfabInt4* d, void* out, long ldo, void* stream) {
  View v;
  if (view_of(d, &v) || !out || (uintptr_t)out % 16 || ldo % 8 || ldo < v.K) return -1;
  const long units = (long)v.halves * v.tiles * v.chunks;
  return launch_chain(dequantise_kernel, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, v, (bf16*)out, ldo, units);
}

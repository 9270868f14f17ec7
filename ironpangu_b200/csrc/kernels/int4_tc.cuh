// What the tensor-core forms of the 4-bit linears share (int4_tc.cu, int4_tc_pair.cu): a thread's row of the matrix as f16 operands.
#pragma once
#include "int4.cuh"
#include "tc_common.cuh"

namespace ifab::int4 {

// eight weights of a word in f16: 1024 + q is an f16 whose last four bits are q, and the difference is exact. less: twice -(1024 + z), s2: twice the scale
__device__ __forceinline__ void weights_of(uint32_t word, uint32_t less, uint32_t s2, uint32_t* out) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t d = ((word >> (4 * j)) & 0x000f000fu) | 0x64006400u;
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(d) : "r"(less));
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(out[j]) : "r"(d), "r"(s2));
  }
}
// the exponent of a magnitude within -112 .. 127, so that its powers below are normal f32
__device__ __forceinline__ int exponent_of(float most) { return max(min((int)(__float_as_uint(most) >> 23) - 127, 127), -112); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// kind::f16 instruction descriptor: f16 x f16 -> f32, both operands K-major
__device__ __forceinline__ uint32_t umma_idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

// A thread's row of the matrix, chunk by chunk: codes, scales and zero points of the next chunk are on the way while the last one's become operands.
template <int GROUP, bool ZEROS>
struct RowOfWeights {
  const unsigned char* unit;         // of the row's tile, first chunk
  int step, f16, g, h;
  float by;                          // the row's power of two
  uint2 next[8], codes[8];
  uint16_t next_s[CHUNK / GROUP];
  uint8_t next_z[CHUNK / GROUP];
  uint32_t s2[CHUNK / GROUP], less[CHUNK / GROUP];

  // row `r` (of sixteen) of tile `tile`
  __device__ __forceinline__ void start(const View& v, int tile, int r) {
    unit = v.at(tile, 0);
    step = v.unit;
    f16 = v.f16;
    g = r & 7;
    h = r >> 3;
    by = power_of_two(11 - exponent_of(v.most[tile * TILE + r]));
  }
  __device__ __forceinline__ float out() const { return __uint_as_float((254u << 23) - __float_as_uint(by)); }       // 1 / by
  __device__ __forceinline__ void fetch(int chunk) {
    const unsigned char* at = unit + (long)chunk * step;
#pragma unroll
    for (int i = 0; i < 8; ++i) next[i] = *reinterpret_cast<const uint2*>(at + (i >> 2) * 512 + code_at(g, i & 3) + h * 8);
#pragma unroll
    for (int i = 0; i < CHUNK / GROUP; ++i) {
      next_s[i] = *reinterpret_cast<const uint16_t*>(at + CODES + i * 32 + g * 4 + h * 2);
      next_z[i] = ZEROS ? at[CODES + CHUNK / GROUP * 32 + i * 16 + g * 2 + h] : 8;
    }
  }
  // what was fetched last becomes the chunk at hand
  __device__ __forceinline__ void turn() {
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[i] = next[i];
#pragma unroll
    for (int i = 0; i < CHUNK / GROUP; ++i) {
      const __half2 s = __float2half2_rn(scales_of(next_s[i], f16).x * by);
      s2[i] = *reinterpret_cast<const uint32_t*>(&s);
      less[i] = 0xe400e400u | next_z[i] | next_z[i] << 16;
    }
  }
  // block b (64 columns) of the chunk at hand: 32 pairs in the order of the columns
  __device__ __forceinline__ void block(int b, uint32_t (&w)[32]) const {
    const int lo = GROUP == 128 ? 0 : GROUP == 64 ? b : 2 * b, hi = GROUP == 32 ? lo + 1 : lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      weights_of(codes[4 * b + i].x, less[lo], s2[lo], w + 4 * i);
      weights_of(codes[4 * b + i].y, less[hi], s2[hi], w + 16 + 4 * i);
    }
  }
};

}  // namespace ifab::int4

// What the tensor-core forms of the 4-bit linears share (int4_tc.cu, int4_tc_pair.cu): a thread's row of the matrix as f16 operands.
#pragma once
#include "int4.cuh"
#include "tc_common.cuh"

namespace ifab::int4 {

// eight weights of a word in f16: 128 + q is an f16 with q in bits 3 .. 6, and the difference is exact. less: twice -(128 + z), s2: twice the scale
__device__ __forceinline__ void weights_of(uint32_t word, uint32_t less, uint32_t s2, uint32_t* out) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t d = pair_under(word, j, 0x58005800u);
    asm("add.rn.f16x2 %0, %0, %1;" : "+r"(d) : "r"(less));
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(out[j]) : "r"(d), "r"(s2));
  }
}
// the exponent of a magnitude within -112 .. 127, so that its powers below are normal f32
__device__ __forceinline__ int exponent_of(float most) { return max(min((int)(__float_as_uint(most) >> 23) - 127, 127), -112); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// kind::f16 instruction descriptor: f16 x f16 -> f32, both operands K-major
__device__ __forceinline__ uint32_t umma_idesc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }

// Units of a chunk of 128 rows in shared memory: eight of them back to back, brought by bulk copies. (With the codes of the next chunk in registers, a warp's other waits -
// for its stores into tensor memory, for the barriers - waited for those loads too: 4096 rows of 2 x 16384 by 4096 1.28 ms, with copies 1.06.)
template <int GROUP, bool ZEROS>
struct Units {
  static constexpr int UNIT = CODES + CHUNK / GROUP * (ZEROS ? 48 : 32), BYTES = 8 * UNIT;
};
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(bytes), "r"(tc::smem_u32(bar)) : "memory");
}

// silu(a) u, off by a few steps of f32: the exponential is at most 1 and the divisor between 1 and 2
__device__ __forceinline__ float gated_unit(float a, float u) {
  const float e = __expf(-fabsf(a));
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return (a >= 0.f ? a : a * e) * r * u;
}

// A thread's row (of 128) in a chunk
template <int GROUP, bool ZEROS>
struct RowOfWeights {
  using U = Units<GROUP, ZEROS>;
  float by;                          // the row's power of two
  int at, f16;                       // of the row in a chunk's units
  uint2 codes[8];
  uint32_t s2[CHUNK / GROUP], less[CHUNK / GROUP];

  // unit `u` of the eight, row `r` of its sixteen
  __device__ __forceinline__ void start(const View& v, int u, int r) {
    at = u * U::UNIT + (r >> 3) * 8;
    f16 = v.f16;
  }
  __device__ __forceinline__ void scale(float most) { by = power_of_two(11 - exponent_of(most)); }
  __device__ __forceinline__ float out() const { return __uint_as_float((254u << 23) - __float_as_uint(by)); }       // 1 / by
  __device__ __forceinline__ void load(const unsigned char* chunk, int r) {
    const int g = r & 7, h = r >> 3;
    const unsigned char* unit = chunk + at - h * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[i] = *reinterpret_cast<const uint2*>(chunk + at + (i >> 2) * 512 + code_at(g, i & 3));
#pragma unroll
    for (int i = 0; i < CHUNK / GROUP; ++i) {
      const __half2 s = __float2half2_rn(scales_of(*reinterpret_cast<const uint16_t*>(unit + CODES + i * 32 + g * 4 + h * 2), f16).x * by);
      const uint32_t z = ZEROS ? unit[CODES + CHUNK / GROUP * 32 + i * 16 + g * 2 + h] : 8;
      s2[i] = *reinterpret_cast<const uint32_t*>(&s);
      less[i] = 0xd800d800u | z << 3 | z << 19;
    }
  }
  // block b (64 columns) of the chunk: 32 pairs in the order of the columns
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

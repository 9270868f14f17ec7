// Weights of 4 bits with a scale (and a zero point) per group of columns:  w[n][k] = s[n][k / G] (q[n][k] - z[n][k / G]), q and z in 0 .. 15, z = 8 without zero points.
//
// A unit holds 16 rows by 128 columns in one piece of memory, codes first, then its scales and zero points, so that whoever multiplies streams one range of
// bytes: 1024 bytes of codes and 32 a group of scales (16 a group of zero points); units of a tile of 16 rows follow one another along K. Rows and columns beyond
// the matrix have the code of the value zero, groups beyond it a scale of zero. A packed gate | up matrix is two halves of whole tiles.
//   codes    block of 64 columns b (512 bytes), columns 8 c .. 8 c + 7 and 32 + 8 c .. of it (c < 4), rows g and g + 8 (g < 8): 16 bytes at b 512 + c 128 +
//            (g ^ 2 c) 16, row g's 8 bytes first, a word for each run of eight columns. A warp whose lane is 4 g + c reads a block without meeting a bank twice and
//            has the operands of four m16n8k16 products (with K permuted alike in the other operand), each of columns of one group; threads that are rows read
//            128 bytes in a row for a fixed c.
//   a word   columns k .. k + 7: rotated right by 4 j, column k + 2 j in bits 3 .. 6 and column k + 2 j + 1 in bits 19 .. 22, the upper mantissa bits of two bf16. That way
//            three rotations make four pairs.
//   scales   [group][g][row g, row g + 8], 16 bits each (bf16 or f16); zero points the same in bytes
// Behind the units: per row the largest of its finite scales, in f32.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace ifab::int4 {

constexpr int TILE = 16, CHUNK = 128, CODES = 1024;          // rows and columns of a unit, bytes of its codes

struct View {
  unsigned char* units;
  float* most;                      // [halves * tiles * 16]: a row's largest finite scale
  int N, K, group, zeros, f16;      // N: rows of one half where gated
  int halves, tiles, chunks, unit;  // tiles of one half, units of a tile, bytes of a unit
  __host__ __device__ int groups() const { return CHUNK / group; }
  __device__ __forceinline__ unsigned char* at(int tile, int chunk) const { return units + ((long)tile * chunks + chunk) * unit; }
};
__host__ __device__ inline int unit_bytes(int group, int zeros) { return CODES + CHUNK / group * (zeros ? 48 : 32); }

// host: SMs of the current device, and a kernel's dynamic shared memory, asked for and set once a device (each a part of a microsecond of a launch's three)
struct Device {
  int id, sms;
};
inline Device device_now() {
  static std::atomic<int> known[64];
  Device d{0, 0};
  cudaGetDevice(&d.id);
  const bool kept = d.id >= 0 && d.id < 64;
  if (kept) d.sms = known[d.id].load(std::memory_order_relaxed);
  if (!d.sms) {
    if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, d.id) != cudaSuccess || d.sms < 1) d.sms = 148;
    if (kept) known[d.id].store(d.sms, std::memory_order_relaxed);
  }
  return d;
}
template <typename Kernel>
inline int allow_smem(Kernel kernel, int bytes, int device, std::atomic<uint64_t>& done) {
  const bool kept = device >= 0 && device < 64;
  if (kept && (done.load(std::memory_order_relaxed) >> device & 1)) return 0;
  if (int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return rc;
  if (kept) done.fetch_or(1ull << device, std::memory_order_relaxed);
  return 0;
}

// host: the view of a descriptor; 0 or -1
inline int view_of(const IfabInt4* d, View* v) {
  if (!d || !d->units || (uintptr_t)d->units % 16 || d->N < 1 || d->K < 8 || d->K % 8 || (d->group != 32 && d->group != 64 && d->group != 128)) return -1;
  *v = View{(unsigned char*)d->units, nullptr, d->N, d->K, d->group, d->zeros != 0, d->f16 != 0, d->gated ? 2 : 1, (d->N + TILE - 1) / TILE, (d->K + CHUNK - 1) / CHUNK,
            unit_bytes(d->group, d->zeros)};
  v->most = (float*)(v->units + (uint64_t)v->halves * v->tiles * v->chunks * v->unit);
  return 0;
}

__device__ __forceinline__ int code_at(int g, int c) { return c * 128 + ((g ^ (2 * c)) << 4); }

// pair j of a word, its codes eight times in the lower bits of two 16-bit numbers with `high` above them
__device__ __forceinline__ uint32_t pair_under(uint32_t word, int j, uint32_t high) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(j ? __funnelshift_r(word, word, 4 * j) : word), "r"(0x00780078u), "r"(high));       // (a & b) | c
  return v;
}
__device__ __forceinline__ float2 scales_of(uint32_t two, int f16) {
  if (f16) return __half22float2(*reinterpret_cast<const __half2*>(&two));
  return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}

}  // namespace ifab::int4

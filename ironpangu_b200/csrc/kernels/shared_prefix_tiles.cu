// The prefix part of the attention of rows that share it (shared_prefix.cu) on tcgen05, for more query rows and heads than m16n8k16 keeps up with.
//
// One CTA per (up to 256 pairs of rows and heads over a kv head, kv head, stretch of the prefix), with two streams of 128 pairs by 128 keys each that take turns on the tensor cores, so that one
// multiplies while the other is between its products: the two halves of the pairs, or where a group has 128 pairs at most, the even and the odd tiles of keys.
//
//   warps 0-3, 4-7   a stream's softmax, a pair a thread: scores out of tensor memory, weights against the pair's reference maximum (which moves only where a maximum exceeds it by 8 powers
//                    of two; then the sums of values are rescaled in place), weights back as two bf16 terms in the scores' place
//   warp 8           tensor memory and the products: S = Q K^T with both operands from shared memory, O += P V with P from tensor memory. V lies as it does in its pages, so it is an operand whose
//                    columns run along the keys' rows (MN-major)
//   warps 12, 13     keys, values into rings of tiles in shared memory, 128-byte swizzle: a lane a box of rows of one page. (By cp.async an SM took in 19 bytes a cycle, however many were under way:
//                    1024 rows over 16384 positions 814 us.)
//
// What each thread of a tile costs is balanced: 1536 cycles of products (a third of them for the weights' second terms, without which the result would be off by half as much again as its own
// rounding) and about as many instructions of softmax.
// Every wait is bounded. One that runs out raises the CTA's flag and the status word; the products that were issued end before the CTA does, and its part of the results becomes NaN.
#include "shared_prefix.cuh"
#include "tc_common.cuh"

using namespace ifab;
using namespace ifab::tc;

namespace {

constexpr int TILE = 128, NT = 512;
// The tensor core cuts off what does not fit a sum: values of one sign lose 1.1e-8 of their sum a key (measured: 16384 keys 1.8e-4, 262144 3.1e-3). So a sum goes on for FOLD tiles (4096 keys: 2^-14.4)
// and is then added, rounded to nearest, to what the part in the scratch has. 1024 rows behind 16384 positions 436 us, with 8192 keys 424, with 2048 451, in one sum 420
constexpr int FOLD = 32;
constexpr uint32_t SPIN_LIMIT = 4000000u;

template <int HD>
struct Layout {
  static constexpr int PANELS = HD / 64, PANEL = TILE * 128, BYTES = PANELS * PANEL;        // 64 columns of 128 rows; a tile of queries, keys or values
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int Q = 0, K = Q + 2 * BYTES, V = K + STAGES * BYTES, BARS = V + STAGES * BYTES, FOLD_BUF = BARS + 512, SMEM = FOLD_BUF + 8 * 4096 + 1024;
};
template <int STAGES>
struct Bars {
  uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_ready[2], o_full[2], cut, drained;
  uint32_t tmem;
  int abort, holes;
};

// D[tmem] (+)= A B with A in shared or in tensor memory, and a commit, by the one lane that is elected. The whole warp comes by: operands that are the same in all lanes lie in uniform registers
// then, where a lane's own would have to be brought there for every product (94 cycles a product, 64 of them its own, while the other warps compute)
__device__ __forceinline__ void umma_elected(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ta_elected(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_elected(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// MN-major with 128-byte swizzle: rows of 64 columns; eight rows further 1024 bytes, 64 columns further a panel
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, int panel_bytes) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(panel_bytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// lane l of the warp writes 16 consecutive columns of its row
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
      "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// pairs of floats
__device__ __forceinline__ uint64_t both(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t twice(float a) { return both(a, a); }
__device__ __forceinline__ void halves(uint64_t v, float* a, float* b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float power_of_2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A warp's parts: what they have times `carry` (first: they have nothing), and the sums of values in tensor memory, a pair a lane; `to`: where the pair's part lies, negative: nobody's. 32 columns at a
// time by way of `buf`, so that eight lanes write a pair's 128 bytes, and without a look at what is there where that stays as it is: 1024 rows behind 16384 positions, a sum of 2048 keys, 522 us with a
// pair a lane, 490 with loads, 451. A call of its own, so that the loop around it has its registers to itself
template <int HD>
__device__ __noinline__ void fold(uint32_t o_addr, unsigned char* buf, float* parts, long to, bool first, float carry) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < HD; c += 32) {
    float v[32];
    tmem_ld_32x32(o_addr + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(buf + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 4 * i + (lane >> 3);
      const long dst = __shfl_sync(0xffffffffu, to, row);
      const float by = __shfl_sync(0xffffffffu, carry, row);
      float4 sum = *reinterpret_cast<const float4*>(buf + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
      float4* part = reinterpret_cast<float4*>(parts + max(dst, 0l) + c + (lane & 7) * 4);
      if (dst < 0) continue;
      if (first) {
        *part = sum;
      } else if (by == 1.f) {                    // without waiting for what is there (a place is one thread's, whose additions follow one another)
        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(part), "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w) : "memory");
      } else {
        float4 had;
        asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(had.x), "=f"(had.y), "=f"(had.z), "=f"(had.w) : "l"(part) : "memory");
        *part = make_float4(fmaf(had.x, by, sum.x), fmaf(had.y, by, sum.y), fmaf(had.z, by, sum.z), fmaf(had.w, by, sum.w));
      }
    }
    __syncwarp();
  }
}

template <int HD>
__global__ void __launch_bounds__(NT, 1) prefix_tiles_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, PrefixParams p, int items, int box) {
  using L = Layout<HD>;
  constexpr int ST = L::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  auto* B = reinterpret_cast<Bars<ST>*>(smem + L::BARS);
  volatile int* abort_flag = &B->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&B->k_full[s], 1);
      mbar_init(&B->v_full[s], 1);
      mbar_init(&B->k_empty[s], 1);
      mbar_init(&B->v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&B->s_full[x], 1);
      mbar_init(&B->p_ready[x], 4);
      mbar_init(&B->o_full[x], 1);
    }
    mbar_init(&B->cut, 1);
    mbar_init(&B->drained, 1);
    B->abort = B->holes = 0;
    mbar_fence_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  grid_dep_wait();
  if (blockIdx.x == 0 && tid == 0) p.hand_on();

  // this CTA's work
  const int item = blockIdx.x % items, split = blockIdx.x / items, kvh = item % p.Hkv;          // (the last stretch, which may be shorter, last)
  int tile = item / p.Hkv, end_rows = 0;
  PrefixGroup gr{0, 0, 0, 0};
  for (int i = 0; i < p.groups; ++i) {
    gr = p.group(i, &end_rows);
    const int tiles = (gr.rows * p.G + 2 * TILE - 1) / (2 * TILE);
    if (tile < tiles) break;
    tile -= tiles;
    gr = PrefixGroup{0, 0, 0, 0};
  }
  if (p.tiles_from && !p.by_tiles()) gr = PrefixGroup{0, 0, 0, 0};         // they are the parts kernel's
  const int per = p.per_tile_split(gr.shared), begin = split * per, end = begin + min(per, gr.shared - begin);       // (whole stretches may pass 32 bits)
  // parts of rows that do not see the prefix, or that the stretches leave over, are nothing: the merge kernel goes by their sums alone
  for (int x = tile * 2 * TILE + tid; x < min((tile + 1) * 2 * TILE, gr.rows * p.G); x += NT) {
    const int t = gr.first + x / p.G;
    const long at = p.part_of(t, kvh * p.G + x % p.G, 2 * split);
    if (begin >= end || !p.sees(gr, t)) p.sums[at] = p.sums[at + 1] = make_float2(-INFINITY, 0.f);
    if (split == 0)
      for (int i = 2 * p.tile_splits; i < p.prefix_parts; ++i) p.sums[at + i] = make_float2(-INFINITY, 0.f);
  }
  if (begin >= end) return;                      // (dependents may start then, as below)
  if (warp == 8) tmem_alloc(&B->tmem, 512);      // S of the streams at 0 and 128, O at 256 and 384. Ahead of the launch of dependents, which might hold some and wait for this kernel
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B->tmem;
  grid_dep_launch();
  const int x0 = tile * 2 * TILE, pairs = gr.rows * p.G, nt = (end - begin + TILE - 1) / TILE;
  const bool two = pairs - x0 > TILE;            // two halves of pairs, or two streams of keys
  const int units = two ? 2 * nt : nt;           // products of scores: unit u is stream u & 1

  for (int i = begin / p.page_tokens + tid; i <= (end - 1) / p.page_tokens; i += NT)
    if (p.row_of(i * p.page_tokens, gr.slot) < 0) B->holes = 1;
  // queries: a pair is a row of 128-byte lines, chunk c of a line at c ^ (row % 8)
  for (int i = tid; i < (two ? 2 : 1) * TILE * (HD / 8); i += NT) {
    const int row = i / (HD / 8), c = i % (HD / 8), x = x0 + row;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (x < pairs) v = *reinterpret_cast<const uint4*>(p.q + (long)(gr.first + x / p.G) * p.ldq + (long)(kvh * p.G + x % p.G) * HD + c * 8);
    const int r = row % TILE;
    *reinterpret_cast<uint4*>(smem + L::Q + row / TILE * L::BYTES + (c >> 3) * L::PANEL + (r >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
  }
  fence_proxy_async_smem();
  __syncthreads();
  auto fail = [&]() {
    *abort_flag = 1;
    if (p.status) atomicOr(p.status, IFAB_STATUS_MBAR_TIMEOUT);
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int X = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16, s_addr = tmem + lane_addr + X * 128, o_addr = tmem + lane_addr + 256 + X * 128;
    const int steps = two ? nt : (nt - X + 1) / 2;
    const bool holes = B->holes;
    auto part_at = [&]() {                       // of this thread's pair; -1: nobody's
      const int x = x0 + (two ? X * TILE : 0) + r;
      return x < pairs && p.sees(gr, gr.first + x / p.G) ? p.part_of(gr.first + x / p.G, kvh * p.G + x % p.G, 2 * split) : -1l;
    };
    auto add_up = [&](bool first, float carry) {
      const long at = part_at();
      fold<HD>(o_addr, smem + L::FOLD_BUF + warp * 4096, p.parts, at < 0 ? -1 : (at + (two ? 0 : X)) * HD, first, carry);
    };
    float m_ref = -INFINITY, l = 0.f, carry = 1.f;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&B->s_full[X], j & 1, SPIN_LIMIT) && !*abort_flag)) { ok = false; break; }
      tc_fence_after();
      const int key0 = begin + (two ? j : 2 * j + X) * TILE;
      if (holes || key0 + TILE > end) {          // keys that are not there: their scores are put out in place
#pragma unroll 1
        for (int c = 0; c < TILE; c += 16) {
          uint32_t s[16], there = 0;
          tmem_ld_32x16(s_addr + c, s);
          tmem_ld_wait();
#pragma unroll 1
          for (int i = 0; i < 16; ++i) there |= (uint32_t)(key0 + c + i < end && !(holes && p.row_of(key0 + c + i, gr.slot) < 0)) << i;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (!(there >> i & 1)) s[i] = 0xff800000u;
          tmem_st_32x16(s_addr + c, s);
        }
        tmem_st_wait();
      }
      // Two passes over the scores, 64 and 32 at a time: all 128 in registers made a loop of 40 KB, and the warps waited for instructions
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < TILE; c += 64) {
        float s[64];
        tmem_ld_32x32(s_addr + c, s);
        tmem_ld_32x32(s_addr + c + 32, s + 32);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      const bool moved = top > m_ref + 8.f, fresh = j % FOLD == 0;       // also for the first key (m_ref = -inf)
      if (fresh && j > 0) {                      // the product before has ended: these scores follow it in the pipe
        add_up(j == FOLD, carry);
        carry = 1.f;
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float corr = moved ? exp2f(m_ref - top) : 1.f;
        l *= corr;
        carry *= corr;
        if (moved) m_ref = top;
        if (!fresh) {
#pragma unroll 1
          for (int c = 0; c < HD; c += 16) {
            uint32_t v[16];
            tmem_ld_32x16(o_addr + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
            tmem_st_32x16(o_addr + c, v);
          }
        }
      }
      const float from = m_ref == -INFINITY ? 0.f : m_ref;
      const uint64_t scale2 = twice(p.scale_log2), from2 = twice(-from), above2 = twice(1.f + 0x1p-20f);
      uint64_t sum[2] = {0, 0};
      // 32 scores become 16 words of first terms and 16 of second terms, in their own place
#pragma unroll 1
      for (int c = 0; c < TILE; c += 64) {
        float s[64];
        tmem_ld_32x32(s_addr + c, s);
        tmem_ld_32x32(s_addr + c + 32, s + 32);
        tmem_ld_wait();
#pragma unroll
        for (int half = 0; half < 64; half += 32) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            // two weights at a time: the first term is cut off, the second one is what that leaves and 2^-20 of the weight, so that no weight has one of 0
            float a, b;
            halves(fma2(both(s[half + 2 * i], s[half + 2 * i + 1]), scale2, from2), &a, &b);
            a = power_of_2(a);
            b = power_of_2(b);
            const uint64_t ab = both(a, b);
            sum[i & 1] = add2(sum[i & 1], ab);
            float ra, rb;
            halves(fma2(ab, above2, both(-__uint_as_float(__float_as_uint(a) & 0xffff0000u), -__uint_as_float(__float_as_uint(b) & 0xffff0000u))), &ra, &rb);
            hi[i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
            lo[i] = __byte_perm(__float_as_uint(ra), __float_as_uint(rb), 0x7632);
          }
          tmem_st_32x16(s_addr + c + half, hi);
          tmem_st_32x16(s_addr + c + half + 16, lo);
        }
      }
      float even, odd;
      halves(add2(sum[0], sum[1]), &even, &odd);
      l += even + odd;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->p_ready[X]);
    }
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&B->o_full[X], 0, SPIN_LIMIT) && !*abort_flag);
    tc_fence_after();
    if (!ok && lane == 0) fail();
    const long at = part_at();
    if (ok && steps > FOLD) {
      add_up(false, carry);
    } else if (ok && steps > 0) {              // (a pair a lane: by way of shared memory 27 rows in three groups take 41 us, so 39.5)
      float* to = p.parts + (at + (two ? 0 : X)) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float v[32];
        tmem_ld_32x32(o_addr + c, v);
        tmem_ld_wait();
        if (at >= 0)
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(to + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
    if (at >= 0) {
      p.sums[at + (two ? 0 : X)] = !ok ? make_float2(INFINITY, NAN) : steps > 0 ? prefix_sums(m_ref, l) : make_float2(-INFINITY, 0.f);
      if (two) p.sums[at + 1] = make_float2(-INFINITY, 0.f);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 8) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(TILE, TILE), idesc_o = umma_idesc_bf16(TILE, HD) | 1u << 16;      // V's columns run along the rows
      const auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
      const uint32_t base = uniform(smem_u32(smem)), tm = uniform(tmem), all = uniform((uint32_t)units);
      const bool pair = uniform(two);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, SPIN_LIMIT)); };
      auto keys = [&](uint32_t u) {
        const uint32_t kt = pair ? u >> 1 : u;
        return wait(&B->k_full[kt % ST], (kt / ST) & 1);
      };
      auto scores = [&](uint32_t u) {
        const uint32_t kt = pair ? u >> 1 : u, X = u & 1, s = kt % ST;
        const uint64_t da = umma_desc_sw128(base + L::Q + (pair ? X : 0) * L::BYTES), db = umma_desc_sw128(base + L::K + s * L::BYTES);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) umma_elected(tm + X * 128, da + (uint64_t)((k >> 2) * (L::PANEL >> 4) + (k & 3) * 2), db + (uint64_t)((k >> 2) * (L::PANEL >> 4) + (k & 3) * 2), idesc_s, k > 0);
        commit_elected(&B->s_full[X]);
        if (!pair || X == 1) commit_elected(&B->k_empty[s]);
      };
      bool ok = true;
      for (uint32_t u = 0; u < min(2u, all) && ok; ++u) {
        ok = keys(u);
        tc_fence_after();
        if (ok) scores(u);
      }
      for (uint32_t u = 0; u < all && ok; ++u) {
        const uint32_t kt = pair ? u >> 1 : u, X = u & 1, s = kt % ST, j = u >> 1;
        // the weights come last: what else is waited for costs the pipe nothing then
        if (!wait(&B->v_full[s], (kt / ST) & 1) || (u + 2 < all && !keys(u + 2)) || *abort_flag || !wait(&B->p_ready[X], j & 1)) { ok = false; break; }
        tc_fence_after();
        const uint64_t dv = desc_rows(base + L::V + s * L::BYTES, L::PANEL);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)
            umma_ta_elected(tm + 256 + X * 128, tm + X * 128 + (k >> 1) * 32 + term * 16 + (k & 1) * 8, dv + (uint64_t)(k * (16 * 128 >> 4)), idesc_o, j % FOLD > 0 || term > 0 || k > 0);
        if (!pair || X == 1) commit_elected(&B->v_empty[s]);
        if (u + 2 >= all) commit_elected(&B->o_full[X]);
        if (u + 2 < all) scores(u + 2);
      }
      if (!ok) {
        if (lane == 0) fail();
        commit_elected(&B->drained);
        mbar_wait(&B->drained, 0, SPIN_LIMIT);
      }
    } else if (warp == 12 || warp == 13) {
      // a warp for keys, one for values; a lane a box (rows of one page, 64 columns). A page that is not there is asked for behind the caches' end: zeros
      const bool values = warp == 13;
      const CUtensorMap* map = values ? &map_v : &map_k;
      uint64_t *full = values ? B->v_full : B->k_full, *empty = values ? B->v_empty : B->k_empty;
      unsigned char* ring = smem + (values ? L::V : L::K);
      const int b = lane / L::PANELS, panel = lane % L::PANELS;
      const bool mine = b < TILE / box;
      static_assert(TILE / 8 * L::PANELS <= 32, "a lane a box");
      auto row_at = [&](int kt) {                // of this lane's box; the caches' end: there is none
        const int key = begin + kt * TILE + b * box, row = mine && kt < nt && key < end ? p.row_of(key, gr.slot) : -2;
        return row >= 0 ? row : p.num_pages * p.page_tokens - 1 - row;
      };
      bool ok = true;
      int next = row_at(0), issued = 0;
      for (int kt = 0; kt < nt; ++kt) {
        const int s = kt % ST, row = next;
        if (kt >= ST && !__all_sync(0xffffffffu, mbar_wait(&empty[s], (kt / ST - 1) & 1, SPIN_LIMIT) && !*abort_flag)) { ok = false; break; }
        const bool cut = values && kt == nt - 1 && (end - begin) % TILE;       // rows behind the stretch: whatever they hold, it must not count
        uint64_t* bar = cut ? &B->cut : &full[s];
        if (lane == 0) mbar_expect_tx(bar, L::BYTES);
        __syncwarp();
        if (mine) tma_load_2d(ring + s * L::BYTES + panel * L::PANEL + b * box * 128, map, bar, kvh * HD + panel * 64, row);
        issued = kt + 1;
        if (row == p.num_pages * p.page_tokens && p.status) atomicOr(p.status, IFAB_STATUS_BAD_INDEX);
        next = row_at(kt + 1);
        if (cut) {
          if (!__all_sync(0xffffffffu, mbar_wait(&B->cut, 0, SPIN_LIMIT))) { ok = false; break; }
          const int live = end - begin - kt * TILE;
          for (int i = lane; i < (TILE - live) * L::PANELS * 8; i += 32) {
            const int key = live + i / (L::PANELS * 8), c = i % (L::PANELS * 8);
            *reinterpret_cast<uint4*>(ring + s * L::BYTES + (c >> 3) * L::PANEL + key * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[s]);
        }
      }
      if (!ok) {                                 // what was requested lands before the CTA ends
        if (lane == 0) fail();
        for (int j = max(0, issued - ST); j < issued; ++j)
          if (!(values && j == nt - 1 && (end - begin) % TILE)) mbar_wait(&full[j % ST], (j / ST) & 1, SPIN_LIMIT);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
int launch(const PrefixParams& p, long items, cudaStream_t s) {
  auto k = prefix_tiles_kernel<HD>;
  if (int rc = opt_in_smem_once<prefix_tiles_kernel<HD>>(Layout<HD>::SMEM)) return rc;
  int box = TILE;                                // rows of a box: they never pass a page's end
  while (p.page_tokens % box) box /= 2;
  const uint64_t rows = (uint64_t)p.num_pages * p.page_tokens, cols = (uint64_t)p.Hkv * HD;
  CUtensorMap map_k, map_v;
  if (int rc = make_tmap_bf16_2d(&map_k, p.k_cache, rows, cols, cols, (uint32_t)box)) return rc;
  if (int rc = make_tmap_bf16_2d(&map_v, p.v_cache, rows, cols, cols, (uint32_t)box)) return rc;
  return launch_chain(k, dim3((unsigned)(items * p.tile_splits)), dim3(NT), (size_t)Layout<HD>::SMEM, s, map_k, map_v, p, (int)items, box);
}

}  // namespace

namespace ifab {
int launch_prefix_tiles(const PrefixParams& p, int head_dim, long items, cudaStream_t s) {
  if (p.page_tokens % 8) return -1;
  return head_dim == 64 ? launch<64>(p, items, s) : launch<128>(p, items, s);
}
}  // namespace ifab

// The prefix part of the attention of rows that share it (shared_prefix.cu) on tcgen05, for more query rows and heads than m16n8k16 keeps up with.
//
// One CTA per (up to 256 pairs of rows and heads over a kv head, kv head, stretch of the prefix), with two streams of 128 pairs by 128 keys each that take turns on the tensor cores, so that one
// multiplies while the other is between its products: the two halves of the pairs, or where a group has 128 pairs at most, the even and the odd tiles of keys.
//
//   warps 0-3, 4-7   a stream's softmax, a pair a thread: scores out of tensor memory, weights against the pair's reference maximum (which moves only where a maximum exceeds it by 8 powers
//                    of two; then the sums of values are rescaled in place), weights back as two bf16 terms in the scores' place
//   warp 8           tensor memory and the products: S = Q K^T with both operands from shared memory, O += P V with P from tensor memory. V lies as it does in its pages, so it is an operand whose
//                    columns run along the keys' rows (MN-major)
//   warps 12-15      keys and values into rings of tiles in shared memory, 128-byte swizzle, by cp.async: a key's row may lie in any page, and one that is not there is read as zeros
//
// What each thread of a tile costs is balanced: 1536 cycles of products (a third of them for the weights' second terms, without which the result would be off by half as much again as its own
// rounding) and about as many instructions of softmax.
// Every wait is bounded. One that runs out raises the CTA's flag and the status word; the products that were issued end before the CTA does, and its part of the results becomes NaN.
#include "shared_prefix.cuh"
#include "tc_common.cuh"

using namespace ifab;
using namespace ifab::tc;

namespace {

constexpr int TILE = 128, NT = 512, PRODUCERS = 128;
constexpr uint32_t SPIN_LIMIT = 4000000u;

template <int HD>
struct Layout {
  static constexpr int PANELS = HD / 64, PANEL = TILE * 128, BYTES = PANELS * PANEL;        // 64 columns of 128 rows; a tile of queries, keys or values
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int Q = 0, K = Q + 2 * BYTES, V = K + STAGES * BYTES, BARS = V + STAGES * BYTES, SMEM = BARS + 512 + 1024;
};
template <int STAGES>
struct Bars {
  uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_ready[2], o_full[2], drained;
  uint32_t tmem;
  int abort, holes;
};

// D[tmem] (+)= A[tmem] * B[smem]; issued by one thread
__device__ __forceinline__ void umma_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"((uint32_t)accumulate)
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
__device__ __forceinline__ void copy16_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

template <int HD>
__global__ void __launch_bounds__(NT, 1) prefix_tiles_kernel(PrefixParams p) {
  using L = Layout<HD>;
  constexpr int ST = L::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  auto* B = reinterpret_cast<Bars<ST>*>(smem + L::BARS);
  volatile int* abort_flag = &B->abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&B->k_full[s], PRODUCERS / 32);
      mbar_init(&B->v_full[s], PRODUCERS / 32);
      mbar_init(&B->k_empty[s], 1);
      mbar_init(&B->v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&B->s_full[x], 1);
      mbar_init(&B->p_ready[x], 4);
      mbar_init(&B->o_full[x], 1);
    }
    mbar_init(&B->drained, 1);
    B->abort = B->holes = 0;
    mbar_fence_init();
  }
  if (warp == 8) tmem_alloc(&B->tmem, 512);      // S of the streams at 0 and 128, O at 256 and 384. Ahead of the launch of dependents, which might hold some and wait for this kernel
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B->tmem;
  grid_dep_launch();
  grid_dep_wait();

  // this CTA's work
  const int split = blockIdx.x % p.prefix_splits, kvh = blockIdx.x / p.prefix_splits % p.Hkv;
  int tile = blockIdx.x / p.prefix_splits / p.Hkv, end_rows = 0;
  PrefixGroup gr{0, 0, 0, 0};
  for (int i = 0; i < p.groups; ++i) {
    gr = p.group(i, &end_rows);
    const int tiles = (gr.rows * p.G + 2 * TILE - 1) / (2 * TILE);
    if (tile < tiles) break;
    tile -= tiles;
    gr.shared = 0;
  }
  const int per = p.per_split(gr.shared, p.prefix_splits), begin = split * per, end = min(begin + per, gr.shared);
  if (begin >= end) {
    if (warp == 8) tmem_dealloc(tmem, 512);
    return;
  }
  const int x0 = tile * 2 * TILE, pairs = gr.rows * p.G, nt = (end - begin + TILE - 1) / TILE;
  const bool two = pairs - x0 > TILE;            // two halves of pairs, or two streams of keys
  const int units = two ? 2 * nt : nt;           // products of scores: unit u is stream u & 1
  const long kv_elems = (long)p.Hkv * HD;

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
    float m_ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&B->s_full[X], j & 1, SPIN_LIMIT) && !*abort_flag)) { ok = false; break; }
      tc_fence_after();
      float s[TILE];
#pragma unroll
      for (int c = 0; c < TILE; c += 32) tmem_ld_32x32(s_addr + c, s + c);
      tmem_ld_wait();
      const int key0 = begin + (two ? j : 2 * j + X) * TILE;
      if (holes || key0 + TILE > end) {
#pragma unroll
        for (int c = 0; c < TILE; c += 32) {
          uint32_t there = 0;
#pragma unroll 1
          for (int i = 0; i < 32; ++i) there |= (uint32_t)(key0 + c + i < end && !(holes && p.row_of(key0 + c + i, gr.slot) < 0)) << i;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(there >> i & 1)) s[c + i] = -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < TILE; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      const bool moved = top > m_ref + 8.f;      // also for the first key (m_ref = -inf)
      if (__any_sync(0xffffffffu, moved)) {
        const float corr = moved ? exp2f(m_ref - top) : 1.f;
        l *= corr;
        if (moved) m_ref = top;
        if (j > 0) {                             // the product before has ended: these scores follow it in the pipe
#pragma unroll
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
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < TILE; c += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float a = prefix_weight(fmaf(s[c + 2 * i], p.scale_log2, -from)), b = prefix_weight(fmaf(s[c + 2 * i + 1], p.scale_log2, -from));
          sum[(2 * i) & 3] += a;
          sum[(2 * i + 1) & 3] += b;
          two_terms(a, b, &hi[i], &lo[i]);
        }
        tmem_st_32x16(s_addr + c / 2, hi);
        tmem_st_32x16(s_addr + 64 + c / 2, lo);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->p_ready[X]);
    }
    if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait(&B->o_full[X], 0, SPIN_LIMIT) && !*abort_flag);
    tc_fence_after();
    if (!ok && lane == 0) fail();
    const int x = x0 + (two ? X * TILE : 0) + r;
    const bool mine = x < pairs && p.sees(gr, gr.first + x / p.G);
    const long at = mine ? p.part_of(gr.first + x / p.G, kvh * p.G + x % p.G, 2 * split) : 0;
    if (ok && steps > 0) {
      float* to = p.parts + (at + (two ? 0 : X)) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float v[32];
        tmem_ld_32x32(o_addr + c, v);
        tmem_ld_wait();
        if (mine)
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(to + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
      }
    }
    if (mine) {
      p.sums[at + (two ? 0 : X)] = !ok ? make_float2(INFINITY, NAN) : steps > 0 ? prefix_sums(m_ref, l) : make_float2(-INFINITY, 0.f);
      if (two) p.sums[at + 1] = make_float2(-INFINITY, 0.f);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 8 && lane == 0) {
      constexpr uint32_t idesc_s = umma_idesc_bf16(TILE, TILE), idesc_o = umma_idesc_bf16(TILE, HD) | 1u << 16;      // V's columns run along the rows
      auto scores = [&](int u) {
        const int kt = two ? u >> 1 : u, X = u & 1, s = kt % ST;
        if (!mbar_wait(&B->k_full[s], (kt / ST) & 1, SPIN_LIMIT) || *abort_flag) return false;
        tc_fence_after();
        const uint32_t qa = smem_u32(smem + L::Q + (two ? X : 0) * L::BYTES), ka = smem_u32(smem + L::K + s * L::BYTES);
#pragma unroll
        for (int pp = 0; pp < L::PANELS; ++pp) {
          const uint64_t da = umma_desc_sw128(qa + pp * L::PANEL), db = umma_desc_sw128(ka + pp * L::PANEL);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_bf16(tmem + X * 128, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc_s, pp > 0 || k > 0);
        }
        umma_commit(&B->s_full[X]);
        if (!two || X == 1) umma_commit(&B->k_empty[s]);
        return true;
      };
      bool ok = true;
      for (int u = 0; u < min(2, units) && ok; ++u) ok = scores(u);
      for (int u = 0; u < units && ok; ++u) {
        const int kt = two ? u >> 1 : u, X = u & 1, s = kt % ST, j = u >> 1;
        if (!mbar_wait(&B->p_ready[X], j & 1, SPIN_LIMIT) || !mbar_wait(&B->v_full[s], (kt / ST) & 1, SPIN_LIMIT) || *abort_flag) { ok = false; break; }
        tc_fence_after();
        const uint64_t dv = desc_rows(smem_u32(smem + L::V + s * L::BYTES), L::PANEL);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int k = 0; k < TILE / 16; ++k)
            umma_ta(tmem + 256 + X * 128, tmem + X * 128 + term * 64 + k * 8, dv + (uint64_t)(k * (16 * 128 >> 4)), idesc_o, j > 0 || term > 0 || k > 0);
        if (!two || X == 1) umma_commit(&B->v_empty[s]);
        if (u + 2 >= units) umma_commit(&B->o_full[X]);
        if (u + 2 < units) ok = scores(u + 2);
      }
      if (!ok) {
        fail();
        umma_commit(&B->drained);
        mbar_wait(&B->drained, 0, SPIN_LIMIT);
      }
    } else if (warp >= 12) {
      // groups of copies: keys, then values, tile by tile. A group that has landed is told to the tensor cores' thread, by a warp for its share
      const int pw = warp - 12;
      constexpr int CH = HD / 8, PENDING = 3;
      int issued = 0, told = 0;
      auto tell = [&](int until) {
        fence_proxy_async_smem();
        __syncwarp();
        for (; told < until; ++told)
          if (lane == 0) mbar_arrive(told & 1 ? &B->v_full[(told >> 1) % ST] : &B->k_full[(told >> 1) % ST]);
      };
      auto row_at = [&](int kt) {
        const int pos = begin + kt * TILE + pw * 32 + lane;
        if (kt >= nt || pos >= end) return -1;
        const int row = p.row_of(pos, gr.slot);
        if (row < 0 && p.status) atomicOr(p.status, IFAB_STATUS_BAD_INDEX);
        return row;
      };
      bool ok = true;
      int next = row_at(0);
      for (int kt = 0; kt < nt && ok; ++kt) {
        const int row = next, s = kt % ST;
        next = row_at(kt + 1);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint64_t* empty = part ? &B->v_empty[s] : &B->k_empty[s];
          if (kt >= ST && !__all_sync(0xffffffffu, mbar_try_wait(empty, (kt / ST - 1) & 1))) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            tell(issued);
            if (!__all_sync(0xffffffffu, mbar_wait(empty, (kt / ST - 1) & 1, SPIN_LIMIT) && !*abort_flag)) { ok = false; break; }
          }
          const bf16* cache = (part ? p.v_cache : p.k_cache) + (long)kvh * HD;
          const uint32_t to = smem_u32(smem + (part ? L::V : L::K) + s * L::BYTES);
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const int k = i * (32 / CH) + lane / CH, c = lane % CH, at = __shfl_sync(0xffffffffu, row, k), key = pw * 32 + k;
            copy16_zero(to + (c >> 3) * L::PANEL + (key >> 3) * 1024 + (key & 7) * 128 + (((c & 7) ^ (key & 7)) << 4), cache + (at < 0 ? 0 : at * kv_elems + c * 8), at >= 0);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          ++issued;
          asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
          if (issued - PENDING > told) tell(issued - PENDING);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (ok) tell(issued);
      else if (lane == 0) fail();
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
  if (int rc = opt_in_smem(k, Layout<HD>::SMEM)) return rc;
  return launch_chain(k, dim3((unsigned)items), dim3(NT), (size_t)Layout<HD>::SMEM, s, p);
}

}  // namespace

namespace ifab {
int launch_prefix_tiles(const PrefixParams& p, int head_dim, long items, cudaStream_t s) { return head_dim == 64 ? launch<64>(p, items, s) : launch<128>(p, items, s); }
}  // namespace ifab

// Attention over the paged 4-bit KV cache for many rows a sequence (prompts,
// chunks of prompts), on the tensor cores (tcgen05).
//
// Rows are (query, head of the kv head's group): 128 of them a tile, two tiles
// a CTA, so a dequantised block of 128 tokens serves 256 rows.  Per block:
//   S_t = Q_t K^T            f16 x f16 -> f32 in tensor memory
//   P_t = 2^(c S_t - ref)    one thread a row; f16, written over S_t
//   O_t = O_t + P_t V        P from tensor memory, f32 accumulators there
// Roles: two warpgroups of softmax threads (a tile each; their threads also
// bring the query rows in and write the results), one warpgroup that
// dequantises K and V into two shared-memory stages, one warp that issues the
// products.  The issuing thread takes whatever is ready of the two tiles, so
// one tile's products run while the other tile's softmax does.
//
// Numbers: K, V, Q and P are f16 (11 bits; one rounding each).  Q is scaled by
// a power of two per row, K per block and V by a power of two that follows the
// largest scale seen, so that range is not lost; O is rescaled when that power
// or a row's softmax reference moves, the latter only when a score passes it by
// 8 in powers of two.  Weights below 2^-31 of the reference count as zero.
// K's values keep the order of the packed row (Q is permuted alike); V's too
// (the results are put in order on the way out).
//
// A V group that holds NaN is zero in the product and reaches the rows that
// see its token by hand, so that 0 * NaN does not reach the others.
#include <limits.h>

#include "kv_attn.cuh"

namespace rc {

constexpr int kPrRows = 128;                         // rows of a tile, tokens of a block
constexpr int kPrThreads = 13 * 32;
constexpr int kPrInfo = 4;                           // blocks whose exponents are kept
constexpr uint32_t kPrTmemCols = 512;

template <int NJ>
struct PrLayout {
  static constexpr int D = 32 * NJ, halves = D / 64;              // 128-byte column blocks of a row
  static constexpr int tile = kPrRows * D * 2;
  static constexpr int o_q = 0, o_k = 2 * tile, o_v = o_k + 2 * tile;
  static constexpr int o_poison = o_v + 2 * tile;                 // [kPrInfo][128] group masks of NaN values
  static constexpr int o_info = o_poison + kPrInfo * kPrRows;     // [kPrInfo]{K exponent, V exponent, poisoned, -}
  static constexpr int o_red = o_info + kPrInfo * 16;             // [2][4 warps]{K, V}
  static constexpr int o_bar = o_red + 64;
  static constexpr int n_bars = 16;
  static constexpr int o_misc = o_bar + 8 * n_bars;               // tensor memory address, abort word
  static constexpr int bytes = o_misc + 16 + 1024;                // and the alignment
  static constexpr uint32_t s_col = 0, o_col = 2 * kPrRows;       // tensor memory: S0 S1 O0 O1
};

__device__ __forceinline__ void pr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pr_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pr_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Operand tiles in the 128-byte swizzle: rows 128 B apart, 8-row groups 1024 B
// apart; 64-value column blocks one tile half apart.
__device__ __forceinline__ uint64_t pr_desc(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// f32 accumulator, f16 operands, M = 128; B K-major (QK^T) or N-major (PV).
__device__ constexpr uint32_t pr_idesc(int n, bool b_n_major) {
  return (1u << 4) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPrRows >> 4) << 24);
}
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void pr_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void pr_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void pr_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// The rows of an item and the blocks of tokens they see.
struct PrItem {
  int b, head, flat0;                     // sequence, kv head, first row of the item's 256
  int first, rows, rows_do, len;
  int lo, sinks, sink_blocks, blk_lo, blocks;
};
__device__ __forceinline__ int pr_block(const PrItem &it, int j) {   // first token of the j-th block
  return (j < it.sink_blocks ? j : it.blk_lo + j - it.sink_blocks) * kPrRows;
}

// Item blockIdx.x: sequences in order, a sequence's last rows (the longest
// items) first, kv heads innermost.  Computed by warp 0, shared by all.
__device__ __forceinline__ bool pr_item(const AttnParams &p, int lane, PrItem &it) {
  const int rows_item = 2 * kPrRows;
  int i = blockIdx.x;
  for (int b0 = 0; b0 < p.b.n_seqs; b0 += 32) {
    int first = 0, rows = 0, rows_do = 0, len = 0, n = 0;
    if (b0 + lane < p.b.n_seqs) {
      attn_seq(p, b0 + lane, first, rows, rows_do, len);
      n = (int)(((long long)rows_do * p.group + rows_item - 1) / rows_item) * p.g.heads;
    }
    int run = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    const unsigned in = __ballot_sync(0xffffffffu, i < run);
    if (in) {
      const int src = __ffs(in) - 1;
      const int start = __shfl_sync(0xffffffffu, run - n, src), count = __shfl_sync(0xffffffffu, n, src);
      it.b = b0 + src;
      it.first = __shfl_sync(0xffffffffu, first, src);
      it.rows = __shfl_sync(0xffffffffu, rows, src);
      it.rows_do = __shfl_sync(0xffffffffu, rows_do, src);
      it.len = __shfl_sync(0xffffffffu, len, src);
      const int r = i - start;
      it.head = r % p.g.heads;
      it.flat0 = (count / p.g.heads - 1 - r / p.g.heads) * rows_item;
      const int base = it.len - it.rows;                                   // position of row 0
      const int p_first = base + it.flat0 / p.group;
      const int p_last = base + min(it.rows_do - 1, (it.flat0 + rows_item - 1) / p.group);
      it.lo = p.window > 0 ? max(0, p_first - p.window + 1) : 0;
      it.sinks = p.window > 0 ? min(p.sinks, it.lo) : 0;
      it.blk_lo = it.lo / kPrRows;
      it.sink_blocks = min((it.sinks + kPrRows - 1) / kPrRows, it.blk_lo);
      const int end = p_last < 0 ? 0 : (p_last + kPrRows) / kPrRows;       // blocks up to the last visible token
      it.blocks = p_last < 0 ? 0 : it.sink_blocks + max(0, end - it.blk_lo);
      return true;
    }
    i -= __shfl_sync(0xffffffffu, run, 31);
  }
  return false;
}

// Exponents of 128 tokens' params: the larger of the scales' and of minima more than 2^19 times as large.
template <int NJ>
__device__ __forceinline__ int pr_exponent(const uint32_t (&par)[NJ]) {
  int e = 0;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int se = (par[j] >> 7) & 0xFF, me = (par[j] >> 23) & 0xFF;
    if (se != 0xFF && me != 0xFF) e = max(e, max(se, me - 19));
  }
  return e;
}
__device__ __forceinline__ int pr_shift(int e) { return max(-126, min(122 - e, 106)); }

template <int N>
__device__ __forceinline__ void ldg_words(const uint8_t *p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = __ldcg(reinterpret_cast<const uint4 *>(p + 4 * i));
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else {
    const uint2 v = __ldcg(reinterpret_cast<const uint2 *>(p));
    w[0] = v.x, w[1] = v.y;
  }
}

// Eight codes of a word into four f16x2 {nibble i, nibble i + 4}, scaled.
__device__ __forceinline__ uint4 pr_unpack(uint32_t w, uint32_t s2, uint32_t m2) {
  return make_uint4(hfma2((w << 4) & 0x00F000F0u, s2, m2), hfma2(w & 0x00F000F0u, s2, m2),
                    hfma2((w >> 4) & 0x00F000F0u, s2, m2), hfma2((w >> 8) & 0x00F000F0u, s2, m2));
}

// 16-byte chunk c of row r of a swizzled tile.
__device__ __forceinline__ uint32_t pr_chunk(int r, int c) {
  return (uint32_t)((c >> 3) * (kPrRows * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

struct PrBars {
  uint32_t q, kfull, kempty, vfull, vempty, sfull, pfull, odone, drain;
};

__device__ __forceinline__ bool pr_wait(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  while (!*abort) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (global_timer_ns() - t0 > 1000000000ull) {
      *abort = 1;
      atomicCAS(err, 0, kErrWaitTimeout);
    }
  }
  return false;
}
__device__ __forceinline__ bool pr_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  return __all_sync(0xffffffffu, pr_wait(bar, parity, abort, err));
}

template <int NJ>
__global__ void __launch_bounds__(kPrThreads, 1) rc_kv_prompt_kernel(const __grid_constant__ AttnParams p) {
  using L = PrLayout<NJ>;
  constexpr int D = L::D;
  extern __shared__ uint8_t pr_raw[];
  __shared__ PrItem s_item;
  __shared__ int s_have;
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pr_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar0 = smem_addr(sm + L::o_bar);
  const PrBars bars{bar0, bar0 + 8, bar0 + 24, bar0 + 40, bar0 + 56, bar0 + 72, bar0 + 88, bar0 + 104, bar0 + 120};
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + L::o_misc);
  volatile int *abort = reinterpret_cast<volatile int *>(sm + L::o_misc + 4);
  int4 *info = reinterpret_cast<int4 *>(sm + L::o_info);
  uint8_t *poison = sm + L::o_poison;
  pdl_launch_dependents();
  pdl_wait_prior();
  if (warp == 0) {
    PrItem it;
    const bool have = pr_item(p, lane, it);
    if (lane == 0) {
      s_have = have;
      if (have) s_item = it;
      *abort = 0;
      const int tiles = have && (it.rows_do * p.group - it.flat0) > kPrRows ? 2 : 1;
      mbar_init(bars.q, kPrRows * 2);
      for (int s = 0; s < 2; ++s) {
        mbar_init(bars.kfull + 8 * s, kPrRows);
        mbar_init(bars.kempty + 8 * s, tiles);
        mbar_init(bars.vfull + 8 * s, kPrRows);
        mbar_init(bars.vempty + 8 * s, tiles);
        mbar_init(bars.sfull + 8 * s, 1);
        mbar_init(bars.pfull + 8 * s, kPrRows);
        mbar_init(bars.odone + 8 * s, 1);
      }
      mbar_init(bars.drain, 1);
      mbar_fence_init();
    }
  }
  __syncthreads();
  if (!s_have) return;
  const PrItem it = s_item;
  const int tiles = it.rows_do * p.group - it.flat0 > kPrRows ? 2 : 1;
  if (warp == 12 && it.blocks) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kPrTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pr_fence_before();
  __syncthreads();
  pr_fence_after();
  const uint32_t tmem = it.blocks ? *tmem_slot : 0;

  if (warp < 8) {
    // ------------------------------------------------- query rows, softmax --
    const int t = warp >> 2, row = tid & (kPrRows - 1);
    const int flat = it.flat0 + t * kPrRows + row, qi = flat / p.group;
    const bool live = qi < it.rows_do;
    const int pos = it.len - it.rows + qi;
    const size_t head_at = (size_t)(it.head * p.group + flat % p.group) * D;
    float l = 0.f;
    int fv = 0;
    uint32_t nan_groups = 0;
    if (it.blocks) {
      float c_row;
      {
        uint4 w[4 * NJ];
#pragma unroll
        for (int i = 0; i < 4 * NJ; ++i) w[i] = make_uint4(0, 0, 0, 0);
        if (live) {
          const uint4 *src = reinterpret_cast<const uint4 *>(p.q + (size_t)(it.first + qi) * p.ldq + head_at);
#pragma unroll
          for (int i = 0; i < 4 * NJ; ++i) w[i] = __ldcg(src + i);
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4 * NJ; ++i) {
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7FFFu, (u[e] >> 16) & 0x7FFFu));
        }
        const int sh = top < (15u << 7) ? 126 : 141 - (int)(top >> 7);
        const float mul = p.scale_log2 < 0.f ? -pow2f(sh) : pow2f(sh);   // the sign of the scale goes into Q
        c_row = pow2f(-sh) * fabsf(p.scale_log2);
#pragma unroll
        for (int i = 0; i < 4 * NJ; ++i) {
          // dims 8i .. 8i+7 = 32j + 8q ..: chunk q * NJ + j
          const int j = i / 4, q = i % 4;
          const float x[8] = {bf16_lo_f32(w[i].x) * mul, bf16_hi_f32(w[i].x) * mul, bf16_lo_f32(w[i].y) * mul,
                              bf16_hi_f32(w[i].y) * mul, bf16_lo_f32(w[i].z) * mul, bf16_hi_f32(w[i].z) * mul,
                              bf16_lo_f32(w[i].w) * mul, bf16_hi_f32(w[i].w) * mul};
          *reinterpret_cast<uint4 *>(sm + L::o_q + t * L::tile + pr_chunk(row, q * NJ + j)) =
              make_uint4(pack_f16x2(x[0], x[4]), pack_f16x2(x[1], x[5]), pack_f16x2(x[2], x[6]), pack_f16x2(x[3], x[7]));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(bars.q);
      if (t < tiles) {
        const uint32_t lane_at = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_at = tmem + lane_at + L::s_col + t * kPrRows, o_at = tmem + lane_at + L::o_col + t * D;
        // positions of the tile's rows, for the blocks that need no mask
        const int base = it.len - it.rows, last_flat = it.rows_do * p.group - 1;
        const int p_min = base + min(it.flat0 + t * kPrRows, last_flat) / p.group;
        const int p_max = base + min(it.flat0 + t * kPrRows + kPrRows - 1, last_flat) / p.group;
        float ref = -INFINITY;
        bool ok = true;
        for (int j = 0; j < it.blocks && ok; ++j) {
          const int t0 = pr_block(it, j);
          const bool masked = !(t0 + kPrRows - 1 <= p_min &&
                                (p.window <= 0 || t0 > p_max - p.window || t0 + kPrRows <= p.sinks));
          const int c_hi = pos - t0, c_lo = p.window > 0 ? c_hi - p.window : INT_MIN, c_sink = p.sinks - t0;
          ok = pr_wait_warp(bars.sfull + 8 * t, j & 1, abort, p.err);
          if (!ok) break;
          pr_fence_after();
          const int4 f = info[j % kPrInfo];
          const float c = c_row * pow2f(-f.x);
          float top = -INFINITY;
          uint32_t v[32];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            pr_ld32(s_at + 32 * k, v);
            pr_wait_ld();
            float a[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (masked) {
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int col = 32 * k + e;
                const bool see = col <= c_hi && (col > c_lo || col < c_sink);
                a[e & 3] = fmaxf(a[e & 3], see ? __uint_as_float(v[e]) : -INFINITY);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) a[e & 3] = fmaxf(a[e & 3], __uint_as_float(v[e]));
            }
            top = fmaxf(top, fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
          }
          const float x_top = top == -INFINITY ? -INFINITY : top * c;
          const bool move = x_top > ref + kAttnSlack;
          if (__any_sync(0xffffffffu, move || (j > 0 && f.y != fv))) {
            float by = 1.f;
            if (move) {
              by = exp2f(ref - x_top);
              ref = x_top;
            }
            l *= by;
            if (j > 0) {
              by *= pow2f(max(f.y - fv, -126));
              ok = pr_wait_warp(bars.odone + 8 * t, (j - 1) & 1, abort, p.err);
              if (!ok) break;
              pr_fence_after();
#pragma unroll 1
              for (int k = 0; k < D / 32; ++k) {
                pr_ld32(o_at + 32 * k, v);
                pr_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * by);
                pr_st32(o_at + 32 * k, v);
              }
              pr_wait_st();
            }
          }
          fv = f.y;
          const float minus = ref == -INFINITY ? 0.f : kAttnLift - ref;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            pr_ld32(s_at + 32 * k, v);
            pr_wait_ld();
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float x0 = fmaf(__uint_as_float(v[e]), c, minus), x1 = fmaf(__uint_as_float(v[e + 1]), c, minus);
              if (masked) {
                const int col = 32 * k + e;
                if (!(col <= c_hi && (col > c_lo || col < c_sink))) x0 = -INFINITY;
                if (!(col + 1 <= c_hi && (col + 1 > c_lo || col + 1 < c_sink))) x1 = -INFINITY;
              }
              x0 = ex2(x0);
              x1 = ex2(x1);
              sum[(e >> 1) & 3] += x0 + x1;
              w[e / 2] = pack_f16x2(x0, x1);
            }
            pr_st16(s_at + 16 * k, w);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          if (f.z) {
            // groups of this block that hold NaN, in tokens that this row sees
            for (int col = 0; col < kPrRows; ++col) {
              const bool see = col <= c_hi && (col > c_lo || col < c_sink);
              if (see) nan_groups |= poison[(j % kPrInfo) * kPrRows + col];
            }
          }
          pr_wait_st();
          pr_fence_before();
          mbar_arrive(bars.pfull + 8 * t);
        }
        if (ok) ok = pr_wait_warp(bars.odone + 8 * t, (it.blocks - 1) & 1, abort, p.err);
        pr_fence_after();
        if (ok) {
          // columns 8W + 2i + o hold dim 32 (j + o) + 4 g + i, W = (g NJ + j) / 2; 32 columns cover 16 / NJ g's
          const float r = l == 0.f ? 0.f : 1.f / l, un = pow2f(-fv);
          uint16_t *dst = p.out + (size_t)(it.first + qi) * p.ldo + head_at;
#pragma unroll 1
          for (int k = 0; k < D / 32; ++k) {
            uint32_t v[32];
            pr_ld32(o_at + 32 * k, v);
            pr_wait_ld();
            if (live) {
              constexpr int kPer = 8 / NJ;               // g's of 32 columns
#pragma unroll
              for (int j = 0; j < NJ; ++j) {
                const float bad = (nan_groups >> j) & 1 ? NAN : 0.f;
                uint32_t w[2 * kPer];
#pragma unroll
                for (int g = 0; g < kPer; ++g) {
                  const int c0 = 8 * ((g * NJ + j) / 2) + (j & 1);
                  float x[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[c0 + 2 * i]) * r * un + bad;
                  w[2 * g] = f32_to_bf16_rne(x[0]) | ((uint32_t)f32_to_bf16_rne(x[1]) << 16);
                  w[2 * g + 1] = f32_to_bf16_rne(x[2]) | ((uint32_t)f32_to_bf16_rne(x[3]) << 16);
                }
#pragma unroll
                for (int g = 0; g < 2 * kPer; g += 4)
                  *reinterpret_cast<uint4 *>(dst + 32 * j + 4 * kPer * k + 2 * g) = make_uint4(w[g], w[g + 1], w[g + 2], w[g + 3]);
              }
            }
          }
        }
      }
    } else if (live && t < tiles) {
      uint4 *dst = reinterpret_cast<uint4 *>(p.out + (size_t)(it.first + qi) * p.ldo + head_at);
#pragma unroll
      for (int i = 0; i < 4 * NJ; ++i) dst[i] = make_uint4(0, 0, 0, 0);
    }
  } else if (warp < 12 && it.blocks) {
    // --------------------------------------------------------- dequantise --
    const int row = tid & (kPrRows - 1), w4 = warp & 3;
    uint32_t kc[4 * NJ], vc[4 * NJ], kp[NJ], vp[NJ];
    int2 *red = reinterpret_cast<int2 *>(sm + L::o_red);
    auto fetch = [&](int j) {   // this thread's token of block j; zeros where nobody sees it
      const int tok = pr_block(it, j) + row;
      const uint8_t *blk = nullptr;
      if (tok < it.len && (tok >= it.lo || tok < it.sinks)) blk = kv_head_block(p.g, p.b, it.b, tok, it.head, p.err);
      if (blk) {
        const int at = tok & (p.g.page - 1);
        ldg_words<NJ>(blk + p.g.kp_off + at * NJ * 4, kp);
        ldg_words<NJ>(blk + p.g.vp_off + at * NJ * 4, vp);
        ldg_words<4 * NJ>(blk + at * (D / 2), kc);
        ldg_words<4 * NJ>(blk + p.g.vc_off + at * (D / 2), vc);
      } else {
#pragma unroll
        for (int i = 0; i < NJ; ++i) kp[i] = vp[i] = 0;
#pragma unroll
        for (int i = 0; i < 4 * NJ; ++i) kc[i] = vc[i] = 0;
      }
    };
    int v_exp = 0;
    fetch(0);
    // Every warp goes through every block's barrier, also after a wait has given up.
    for (int j = 0; j < it.blocks; ++j) {
      const int s = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      // the block's exponents
      uint32_t mask = 0;
#pragma unroll
      for (int i = 0; i < NJ; ++i)
        if (((vp[i] >> 7) & 0xFF) == 0xFF || ((vp[i] >> 23) & 0xFF) == 0xFF) mask |= 1u << i, vp[i] = 0;
      const int ke = (int)__reduce_max_sync(0xffffffffu, (uint32_t)pr_exponent<NJ>(kp));
      const int ve = (int)__reduce_max_sync(0xffffffffu, (uint32_t)pr_exponent<NJ>(vp)) | (__any_sync(0xffffffffu, mask != 0) ? 0x1000 : 0);
      if (lane == 0) red[s * 4 + w4] = make_int2(ke, ve);
      asm volatile("bar.sync 2, %0;" ::"n"(kPrRows) : "memory");
      int k_exp = 0, bad = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int2 e = red[s * 4 + i];
        k_exp = max(k_exp, e.x);
        v_exp = max(v_exp, e.y & 0xFFF);
        bad |= e.y >> 12;
      }
      const int fk = pr_shift(k_exp), fvv = pr_shift(v_exp);
      if (pr_wait_warp(bars.kempty + 8 * s, ph ^ 1, abort, p.err)) {
        if (bad) poison[(j % kPrInfo) * kPrRows + row] = (uint8_t)mask;
        if (row == 0) info[j % kPrInfo] = make_int4(fk, fvv, bad, 0);
        const float up = pow2f(fk), up20 = up * 0x1p20f;
        uint8_t *dst = sm + L::o_k + s * L::tile;
#pragma unroll
        for (int g = 0; g < NJ; ++g) {
          const uint32_t s2 = pack_f16x2(bf16_lo_f32(kp[g]) * up20, bf16_lo_f32(kp[g]) * up20);
          const uint32_t m2 = pack_f16x2(bf16_hi_f32(kp[g]) * up, bf16_hi_f32(kp[g]) * up);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(dst + pr_chunk(row, q * NJ + g)) = pr_unpack(kc[q * NJ + g], s2, m2);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bars.kfull + 8 * s);
      }
      if (pr_wait_warp(bars.vempty + 8 * s, ph ^ 1, abort, p.err)) {
        const float up = pow2f(fvv), up20 = up * 0x1p20f;
        uint8_t *dst = sm + L::o_v + s * L::tile;
#pragma unroll
        for (int g = 0; g < NJ; g += 2) {
          const uint32_t s2 = pack_f16x2(bf16_lo_f32(vp[g]) * up20, bf16_lo_f32(vp[g + 1]) * up20);
          const uint32_t m2 = pack_f16x2(bf16_hi_f32(vp[g]) * up, bf16_hi_f32(vp[g + 1]) * up);
#pragma unroll
          for (int q = 0; q < 8; ++q)   // word (q NJ + g) / 2 of the row
            *reinterpret_cast<uint4 *>(dst + pr_chunk(row, (q * NJ + g) / 2)) = pr_unpack(vc[(q * NJ + g) / 2], s2, m2);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bars.vfull + 8 * s);
      }
      if (j + 1 < it.blocks) fetch(j + 1);
    }
  } else if (warp == 12 && it.blocks && lane == 0) {
    // ------------------------------------------------------------ products --
    constexpr uint32_t id_s = pr_idesc(kPrRows, false), id_o = pr_idesc(D, true);
    constexpr uint32_t kBlock = kPrRows * 128;           // a 64-value column block of a tile
    const uint32_t q_at = smem_addr(sm + L::o_q), k_at = smem_addr(sm + L::o_k), v_at = smem_addr(sm + L::o_v);
    int at[2] = {0, 0};                                   // block of a tile's next product
    bool scored[2] = {false, false};                      // its S is issued
    bool q_ready = false;
    uint64_t t_last = global_timer_ns();
    while (at[0] < it.blocks || (tiles == 2 && at[1] < it.blocks)) {
      bool any = false;
      if (!q_ready) q_ready = mbar_try_wait(bars.q, 0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int j = at[t], s = j & 1;
        if (t >= tiles || j >= it.blocks || !q_ready) continue;
        const uint32_t ph = (j >> 1) & 1;
        if (!scored[t]) {
          if (!mbar_try_wait(bars.kfull + 8 * s, ph) || (j > 0 && !mbar_try_wait(bars.odone + 8 * t, (j - 1) & 1))) continue;
          pr_fence_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k >> 2) * kBlock + (k & 3) * 32;
            pr_mma_ss(tmem + L::s_col + t * kPrRows, pr_desc(q_at + t * L::tile + off, 16), pr_desc(k_at + s * L::tile + off, 16),
                      id_s, k > 0);
          }
          pr_commit(bars.sfull + 8 * t);
          pr_commit(bars.kempty + 8 * s);
          scored[t] = true;
        } else {
          if (!mbar_try_wait(bars.pfull + 8 * t, j & 1) || !mbar_try_wait(bars.vfull + 8 * s, ph)) continue;
          pr_fence_after();
#pragma unroll
          for (int k = 0; k < kPrRows / 16; ++k)
            pr_mma_ts(tmem + L::o_col + t * D, tmem + L::s_col + t * kPrRows + 8 * k,
                      pr_desc(v_at + s * L::tile + k * 2048, kBlock), id_o, j > 0 || k > 0);
          pr_commit(bars.odone + 8 * t);
          pr_commit(bars.vempty + 8 * s);
          scored[t] = false;
          ++at[t];
        }
        any = true;
      }
      const uint64_t now = global_timer_ns();
      if (any) t_last = now;
      else if (*abort) break;
      else if (now - t_last > 2000000000ull) {
        *abort = 1;
        atomicCAS(p.err, 0, kErrWaitTimeout);
        break;
      }
    }
    pr_commit(bars.drain);                                // whatever was issued has ended before the memory is given back
    mbar_wait_bounded(bars.drain, 0);
  }
  __syncwarp();
  pr_fence_before();
  __syncthreads();
  if (warp == 12 && it.blocks) {
    pr_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kPrTmemCols));
  }
}

template <int NJ>
static int prompt_launch(rc_ctx *ctx, const AttnParams &a, cudaStream_t s) {
  using L = PrLayout<NJ>;
  auto kernel = rc_kv_prompt_kernel<NJ>;
  // an upper bound of the items: whole 256-row items of all rows, and a cut one for each sequence
  const long long items = ((long long)a.b.n_rows * a.group / (2 * kPrRows) + a.b.n_seqs) * a.g.heads;
  RC_CHECK_ARG(items <= INT_MAX, "rc_kv_attend: the batch is too large");
  static std::atomic<bool> ready[64];
  if (ctx->device >= 64 || !ready[ctx->device].load(std::memory_order_relaxed)) {
    RC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::bytes));
    if (ctx->device < 64) ready[ctx->device].store(true, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)items);
  cfg.blockDim = dim3(kPrThreads);
  cfg.dynamicSmemBytes = L::bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  RC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return RC_OK;
}

int kv_attend_prompt(rc_ctx *ctx, const AttnParams &a, cudaStream_t s) {
  return a.g.dim == 128 ? prompt_launch<4>(ctx, a, s) : prompt_launch<2>(ctx, a, s);
}

}  // namespace rc

// Attention over the paged 4-bit KV cache for many rows a sequence (prompts,
// chunks of prompts), on the tensor cores (tcgen05).
//
// Rows are (query, head of the kv head's group): 128 of them a tile, two tiles
// a CTA, so a dequantised block of 128 tokens serves 256 rows.  Per block:
//   S_t = Q_t K^T            f16 x f16 -> f32 in tensor memory
//   P_t = 2^(c S_t - ref)    one thread a row; f16, to tensor memory
//   O_t = O_t + P_t V        P from tensor memory, f32 accumulators there
// Roles: eight softmax warps (a tile for four of them, one thread a row; they
// also write the results), four warps that make K f16 in shared memory and four
// for V (and Q, a tile each), one that copies the packed K and V in, one that
// issues the products, one that finds the items.  A row's scores are read into
// registers at once (setmaxnreg takes them from the other roles), which frees the
// tensor memory of S for the other tile's scores: the two tiles share one S and
// have a P each, and a tile's next scores are there when its softmax comes for
// them.  CTAs are persistent and every role goes straight from one item to the
// next, so the next item's query rows and blocks come in while the last one's
// results go out.  Items after the first are claimed by turns (dealt in fixed
// rounds, six ragged prompts took 28 us for 20, and one of 4096 139 for 141).  The loops of the other roles are rolled and short on purpose:
// together with a larger text they outgrew the instruction cache, and each of
// them, the issuing warp first, ran at the speed of its misses.
//
// Numbers: K, V, Q and P are f16 (11 bits; one rounding each).  Q is scaled by
// a power of two per row, K per block and V by a power of two that follows the
// largest scale seen, so that range is not lost; O is rescaled when that power
// or a row's softmax reference moves, the latter only when a score passes it by
// 8 in powers of two.  A key below 2^-9 of the largest scale of its block, and a
// value below 2^-9 of the largest seen, has fewer bits: it is good to 2^-20 of that
// scale.  Weights below 2^-21 of the reference have fewer bits (good to 2^-32 of it),
// and below 2^-31 they count as zero, while the sum of the weights has them all.
// K's values keep the order of the packed row (Q is permuted alike); V's too
// (the results are put in order on the way out).
//
// A V group that holds NaN is zero in the product and reaches the rows that
// see its token by hand, so that 0 * NaN does not reach the others.
//
// Measured: 4096 rows of 32 heads over 4 kv heads of 128, causal, 142 us in a graph
// of 30 calls (970 TFLOP/s of visible pairs, 59% of the matrix peak) and 158 after a
// tenth of a second of them, at the power cap (872; 1.73 GHz); chunks of 2048 and
// 1416 rows of 32 heads over 8 that see 4096 tokens and 16 sinks 230 us (61%) and
// 259; six prompts of 117 to 701 tokens, 16 heads of 64, 20 us.  Bound by the chain
// of a block: scores (640 cycles), their way into registers (300), maximum (500),
// weights (1700; without the exponentials the prompt took 125 us, without making K
// and V 132, with half the products 141), values (530).  S and P in one place, and S
// for each tile, was slower (188 us): then a tile's chain has no overlap.  A short
// prompt pays 7 us before its first score: items, rows, codes.
#include <limits.h>

#include "kv_attn.cuh"

namespace rc {

constexpr int kPrRows = 128;                         // rows of a tile, tokens of a block
constexpr int kPrThreads = 640;
// Registers: the softmax warpgroups get what the others leave of 640 x 96.
constexpr int kPrRegsSoftmax = 160, kPrRegsMake = 56, kPrRegsIssue = 48;
static_assert(2 * kPrRegsSoftmax + 2 * kPrRegsMake + kPrRegsIssue == 5 * 96, "setmaxnreg draws on the launch's registers");
constexpr int kPrInfo = 4;                           // blocks whose exponents are kept
constexpr int kPrRaw = 3;                            // packed K and V blocks (by turns) on their way in
constexpr uint32_t kPrTmemCols = 512;
// The rows of an item and the blocks of tokens they see.
struct PrItem {
  int b, head, flat0;                     // sequence (-1: no more items), kv head, first of the item's 256 rows
  int first, rows, rows_do, len;
  int lo, sinks, sink_blocks, blk_lo, blocks;
  int tiles;
};

template <int NJ>
struct PrLayout {
  static constexpr int D = 32 * NJ;
  static constexpr int tile = kPrRows * D * 2;
  static constexpr int o_q = 0, o_k = 2 * tile, o_v = o_k + 2 * tile;
  static constexpr int o_poison = o_v + 2 * tile;                 // [kPrInfo][K, V][128] groups that hold NaN (V), bit 7 for any of K
  static constexpr int o_info = o_poison + 2 * kPrInfo * kPrRows; // [kPrInfo]{exponent, poisoned} of K and of V
  static constexpr int o_red = o_info + kPrInfo * 16;             // [K, V][2][4 warps] exponents
  static constexpr int o_crow = o_red + 64;                       // [2 items][256] score scales, NaN for a row that is
  static constexpr int o_item = o_crow + 2 * 2 * kPrRows * 4;     // [2] items
  static constexpr int o_bar = o_item + 2 * 64;
  static constexpr int n_bars = 30 + 2 * kPrRaw;
  static constexpr int o_misc = o_bar + 8 * n_bars;               // tensor memory address, abort word
  static constexpr int o_prefix = o_misc + 16;                    // [n_seqs / 32 + 1] items of the sequences before
  static constexpr int o_raw = (o_prefix + (kKvMaxSeqs / 32 + 1) * 4 + 127) / 128 * 128;
  static constexpr int raw = kPrRows * D * 5 / 8;                 // packed K or V of a block
  static constexpr int bytes = o_raw + kPrRaw * raw;
  static constexpr uint32_t s_col = 0, p_col = kPrRows, o_col = 2 * kPrRows;   // tensor memory: S, P0 P1, O0 O1
};
static_assert(sizeof(PrItem) <= 64, "an item's slot");
static_assert(PrLayout<4>::bytes <= kGemvSmemLimit, "shared memory of an SM");

__device__ __forceinline__ void pr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool pr_elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void pr_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Waits for the loads; ``v`` (the last one's values) is touched so that nothing uses it earlier.
__device__ __forceinline__ void pr_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                 "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void pr_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Descriptor of an operand tile in the 128-byte swizzle: rows 128 B apart, 8-row groups 1024 B apart, 64-value column
// blocks ``lead`` bytes apart (for an N-major tile).  The low word; the high one is the same for all.
__device__ __forceinline__ uint32_t pr_desc(uint32_t saddr, uint32_t lead) {
  return ((saddr >> 4) & 0x3FFF) | ((lead >> 4) << 16);
}
constexpr uint32_t kPrDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
// f32 accumulator, f16 operands, M = 128; B K-major (QK^T) or N-major (PV).
__device__ constexpr uint32_t pr_idesc(int n, bool b_n_major) {
  return (1u << 4) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPrRows >> 4) << 24);
}
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kPrDescHigh));
}
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kPrDescHigh));
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
__device__ __forceinline__ void pr_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ int pr_block(const PrItem &it, int j) {   // first token of the j-th block
  return (j < it.sink_blocks ? j : it.blk_lo + j - it.sink_blocks) * kPrRows;
}
__device__ __forceinline__ int pr_items(const AttnParams &p, int rows_do) {
  return (rows_do * p.group + 2 * kPrRows - 1) / (2 * kPrRows) * p.g.heads;
}

// Item i: sequences in order, a sequence's last rows (the longest items) first, kv heads innermost.  By a warp:
// ``prefix`` has the items before every 32nd sequence.
__device__ __forceinline__ PrItem pr_item(const AttnParams &p, const int *prefix, int i, int lane) {
  int lo = 0, hi = (p.b.n_seqs - 1) / 32;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  PrItem it;
  it.first = it.rows = it.rows_do = it.len = 0;
  if (32 * lo + lane < p.b.n_seqs) attn_seq(p, 32 * lo + lane, it.first, it.rows, it.rows_do, it.len);
  const int mine = pr_items(p, it.rows_do);
  int run = mine;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  i -= prefix[lo];
  const int src = __ffs(__ballot_sync(0xffffffffu, i < run)) - 1;      // there is one: i < all items
  it.b = 32 * lo + src;
  it.first = __shfl_sync(0xffffffffu, it.first, src);
  it.rows = __shfl_sync(0xffffffffu, it.rows, src);
  it.rows_do = __shfl_sync(0xffffffffu, it.rows_do, src);
  it.len = __shfl_sync(0xffffffffu, it.len, src);
  const int count = __shfl_sync(0xffffffffu, mine, src), r = i - __shfl_sync(0xffffffffu, run - mine, src);
  it.head = r % p.g.heads;
  it.flat0 = (count / p.g.heads - 1 - r / p.g.heads) * 2 * kPrRows;
  it.tiles = it.rows_do * p.group - it.flat0 > kPrRows ? 2 : 1;
  const int base = it.len - it.rows;                                   // position of row 0
  const int p_first = base + attn_row(p, it.flat0);
  const int p_last = base + min(it.rows_do - 1, attn_row(p, it.flat0 + 2 * kPrRows - 1));
  it.lo = attn_window_lo(p, p_first);
  it.sinks = p.window > 0 ? min(p.sinks, it.lo) : 0;
  it.blk_lo = it.lo / kPrRows;
  it.sink_blocks = min((it.sinks + kPrRows - 1) / kPrRows, it.blk_lo);
  const int end = p_last < 0 ? 0 : p_last / kPrRows + 1;               // blocks up to the last visible token
  it.blocks = p_last < 0 ? 0 : it.sink_blocks + max(0, end - it.blk_lo);
  return it;
}
// Token t is visible to a row of the item.
__device__ __forceinline__ bool pr_seen_by_item(const PrItem &it, int t) { return t < it.len && (t >= it.lo || t < it.sinks); }

// Exponents of a token's params: the larger of the scales' and of minima more than 2^19 times as large.
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
// The power that brings the largest scale below 2^-4; 2^20 of it more, which the codes take, is an f16 then.  Down to
// -132, more than pow2f has in one factor.
__device__ __forceinline__ int pr_shift(int e) { return min(122 - e, 106); }

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
  uint32_t item_full, item_empty, q_full, q_empty, k_full, k_empty, v_full, v_empty, s_full, p_full, o_done, o_empty, drain, vote, s_free, claim, raw_full, raw_empty;
};

// Of columns 32 k .. 32 k + 31, those a row sees: column <= c_hi, and > c_lo or < c_sink.
__device__ __forceinline__ uint32_t pr_seen(int k, int c_hi, int c_lo, int c_sink) {
  const int hi = c_hi - 32 * k, lo = max(c_lo, -64) - 32 * k, sk = c_sink - 32 * k;
  const uint32_t upto = hi < 0 ? 0u : hi >= 31 ? ~0u : (2u << hi) - 1u;
  const uint32_t past = lo < 0 ? ~0u : lo >= 31 ? 0u : ~((2u << lo) - 1u);
  const uint32_t first = sk <= 0 ? 0u : sk >= 32 ? ~0u : (1u << sk) - 1u;
  return upto & (past | first);
}

__device__ __forceinline__ void pr_touch(uint32_t (&v)[32]) {   // nothing uses v before this point
  asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                 "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void pr_ld8(uint32_t addr, uint32_t *v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void pr_scale8(uint32_t addr, float by) {
  uint32_t v[8];
  pr_ld8(addr, v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])
               :
               : "memory");
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * by);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ uint64_t pr_pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void pr_split(uint64_t v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t pr_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t pr_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <int NJ>
__global__ void __launch_bounds__(kPrThreads, 1) rc_kv_prompt_kernel(const __grid_constant__ AttnParams p) {
  using L = PrLayout<NJ>;
  constexpr int D = L::D;
  extern __shared__ __align__(1024) uint8_t pr_raw[];
  uint8_t *sm = pr_raw;
  if (smem_addr(sm) & 1023) {   // the swizzled tiles start on their pattern; there is no room to move them
    atomicCAS(p.err, 0, kErrWaitTimeout);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar0 = smem_addr(sm + L::o_bar);
  const PrBars bars{bar0,       bar0 + 16,  bar0 + 32,  bar0 + 48,  bar0 + 64,  bar0 + 80, bar0 + 96,
                    bar0 + 112, bar0 + 128, bar0 + 144, bar0 + 160, bar0 + 176, bar0 + 192, bar0 + 208, bar0 + 224, bar0 + 232, bar0 + 240, bar0 + 240 + 8 * kPrRaw};
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + L::o_misc);
  volatile int *abort = reinterpret_cast<volatile int *>(sm + L::o_misc + 4);
  int4 *info = reinterpret_cast<int4 *>(sm + L::o_info);
  uint8_t *poison = sm + L::o_poison;
  float *crow = reinterpret_cast<float *>(sm + L::o_crow);
  int *prefix = reinterpret_cast<int *>(sm + L::o_prefix);
  if (tid == 0) {
    *abort = 0;
    for (int s = 0; s < 2; ++s) {
      mbar_init(bars.item_full + 8 * s, 1);
      mbar_init(bars.item_empty + 8 * s, 19);            // softmax, operands, copies, scores, values
      mbar_init(bars.q_full + 8 * s, kPrRows);
      mbar_init(bars.q_empty + 8 * s, 1);
      mbar_init(bars.k_full + 8 * s, kPrRows + 4);   // K's rows, and V's exponent from four warps
      mbar_init(bars.k_empty + 8 * s, 1);
      mbar_init(bars.v_full + 8 * s, kPrRows);
      mbar_init(bars.v_empty + 8 * s, 1);
      mbar_init(bars.s_full + 8 * s, 1);
      mbar_init(bars.p_full + 8 * s, 4);
      mbar_init(bars.o_done + 8 * s, 1);
      mbar_init(bars.o_empty + 8 * s, 4);
    }
    mbar_init(bars.drain, 1);
    mbar_init(bars.drain + 8, 1);
    mbar_init(bars.vote, 4);
    mbar_init(bars.vote + 8, 4);
    mbar_init(bars.s_free, 4);
    mbar_init(bars.claim, 1);
    for (int s = 0; s < kPrRaw; ++s) {
      mbar_init(bars.raw_full + 8 * s, 1);
      mbar_init(bars.raw_empty + 8 * s, 4);
    }
    mbar_fence_init();
  }
  pdl_launch_dependents();
  pdl_wait_prior();
  // items of every 32 sequences, then of all before them
#pragma unroll 1
  for (int b0 = 32 * warp; b0 < p.b.n_seqs; b0 += kPrThreads) {
    int first, rows, rows_do = 0, len;
    if (b0 + lane < p.b.n_seqs) attn_seq(p, b0 + lane, first, rows, rows_do, len);
    const int all = (int)__reduce_add_sync(0xffffffffu, (uint32_t)pr_items(p, rows_do));
    if (lane == 0) prefix[b0 / 32 + 1] = all;
  }
  __syncthreads();
  if (tid == 0) {
    prefix[0] = 0;
#pragma unroll 1
    for (int g = 0; g < (p.b.n_seqs + 31) / 32; ++g) prefix[g + 1] += prefix[g];
  } else if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kPrTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pr_fence_before();
  __syncthreads();
  pr_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto item_done = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bars.item_empty + 8 * (k & 1));
  };

  if (warp < 8) {
    // ------------------------------------------------------------- softmax --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrRegsSoftmax));
    // from a shuffle with a fixed lane, so that addresses and loop state are known to be the warp's and leave the
    // threads' registers to the scores (spilled, the block loop takes a fifth longer)
    const int wu = __shfl_sync(0xffffffffu, warp, 0), t = wu >> 2, row = tid & (kPrRows - 1);
    const uint32_t lane_at = __shfl_sync(0xffffffffu, tmem, 0) + ((uint32_t)(32 * (wu & 3)) << 16);
    const uint32_t s_at = lane_at + L::s_col, p_at = lane_at + L::p_col + t * (kPrRows / 2), o_at = lane_at + L::o_col + t * D;
    const uint32_t bar_s = bars.s_full + 8 * t, bar_p = bars.p_full + 8 * t, bar_o = bars.o_done + 8 * t;
    int n = 0, done = 0;                                  // blocks of all items so far; this tile's
#pragma unroll 1
    for (int k = 0;; ++k) {
      if (!attn_wait(bars.item_full + 8 * (k & 1), (k >> 1) & 1, abort, p.err)) break;
      const PrItem *it = reinterpret_cast<const PrItem *>(sm + L::o_item + 64 * (k & 1));
      if (it->b < 0) break;
      const int blocks = it->blocks;
      if (t < it->tiles) {
        const int flat0 = it->flat0 + t * kPrRows, base = it->len - it->rows;
        // positions: of this row, and of the tile's rows, for the blocks that need no mask
        const int last_flat = it->rows_do * p.group - 1;
        const int pos = base + attn_row(p, flat0 + row);
        const int p_min = base + attn_row(p, min(flat0, last_flat));
        const int p_max = base + attn_row(p, min(flat0 + kPrRows - 1, last_flat));
        // blocks clear_lo .. clear_hi - 1 are seen whole by every row of the tile
        const int skip = it->blk_lo - it->sink_blocks;
        const int clear_lo = p.window <= 0 ? 0 : max(it->sink_blocks, (max(p_max - p.window, -1) + kPrRows) / kPrRows - skip);
        const int clear_hi = (p_min + 1) / kPrRows - skip;
        float ref = -INFINITY, l = 0.f;
        int fv = 0;
        uint32_t nan_groups = 0;
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < blocks; ++j, ++done) {
          const bool masked = j < clear_lo || j >= clear_hi;
          ok = attn_wait(bar_s, done & 1, abort, p.err);
          if (!ok) break;
          pr_fence_after();
          uint32_t v[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) pr_ld32(s_at + 32 * i, v[i]);
          pr_wait_ld(v[0]);
          pr_touch(v[1]);
          pr_touch(v[2]);
          pr_touch(v[3]);
          pr_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars.s_free);
          const int4 f = info[(n + j) % kPrInfo];
          const float c = fmaxf(crow[(k & 1) * 2 * kPrRows + t * kPrRows + row] * pow2f(-f.x >> 1) * pow2f(-f.x - (-f.x >> 1)), 0x1p-126f);   // above 0 (also of NaN): a hidden score is -Inf
          const int t0 = pr_block(*it, j);
          const int c_hi = pos - t0, c_lo = p.window > 0 ? c_hi - p.window : INT_MIN, c_sink = p.sinks - t0;
          if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t seen = pr_seen(i, c_hi, c_lo, c_sink);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen >> e & 1)) v[i][e] = 0xFF800000u;
            }
          }
          float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              top4[(e >> 1) & 3] = fmaxf(fmaxf(top4[(e >> 1) & 3], __uint_as_float(v[i][e])), __uint_as_float(v[i][e + 1]));
          const float x_top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * c;
          // the tile's last values are done: P may be written, O changed
          if (done > 0) {
            ok = attn_wait(bar_o, (done - 1) & 1, abort, p.err);
            if (!ok) break;
            pr_fence_after();
          }
          if (__any_sync(0xffffffffu, x_top > ref + kAttnSlack || f.z != fv)) {
            float by = 1.f;
            if (x_top > ref + kAttnSlack) {
              by = exp2f(ref - x_top);
              ref = x_top;
            }
            l *= by;
            if (j > 0) {
              by *= pow2f(max(f.z - fv, -126));
#pragma unroll 1
              for (int i = 0; i < D / 8; ++i) pr_scale8(o_at + 8 * i, by);
            }
            fv = f.z;
          }
          const float minus = ref == -INFINITY ? 0.f : kAttnLift - ref;
          const uint64_t c2 = pr_pair(c, c), m2 = pr_pair(minus, minus);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float x0, x1;
              pr_split(pr_fma2(pr_pair(__uint_as_float(v[i][e]), __uint_as_float(v[i][e + 1])), c2, m2), x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              sum[(e >> 1) & 1] = pr_add2(sum[(e >> 1) & 1], pr_pair(x0, x1));
              w[e / 2] = pack_f16x2(x0, x1);
            }
            pr_st16(p_at + 16 * i, w);
          }
          float s0, s1;
          pr_split(pr_add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
          if (f.y | f.w) {
            // groups of this block that hold NaN, in tokens that this row sees
#pragma unroll 1
            for (int col = 0; col < kPrRows; ++col) {
              const bool see = col <= c_hi && (col > c_lo || col < c_sink);
              const uint8_t *m = poison + (n + j) % kPrInfo * 2 * kPrRows + col;
              if (see) nan_groups |= m[0] ? (1u << NJ) - 1u : m[kPrRows];
            }
          }
          pr_wait_st();
          pr_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p);
        }
        // results; zeros where there are no blocks
        if (blocks && ok) ok = attn_wait(bar_o, (done - 1) & 1, abort, p.err);
        if (ok) {
          pr_fence_after();
          const int flat = flat0 + row, qi = attn_row(p, flat);
          const bool live = qi < it->rows_do;
          uint16_t *dst = p.out + (size_t)(it->first + qi) * p.ldo + (size_t)(it->head * p.group + flat - qi * p.group) * D;
          // a query that is not finite, unless its row is empty (any other sees its own token)
          if (blocks && pos >= 0 && isnan(crow[(k & 1) * 2 * kPrRows + t * kPrRows + row])) nan_groups = (1u << NJ) - 1u;
          const float r = (l == 0.f ? 0.f : 1.f / l) * pow2f(-(fv >> 1)), un = pow2f((fv >> 1) - fv);   // with V's power, in two factors
          const unsigned long long mine = live ? reinterpret_cast<unsigned long long>(dst) : 0ull;
          // columns 8W + 2i + o hold dim 32 (j + o) + 4 g + i, W = (g NJ + j) / 2; two of the 32-value groups at a time
#pragma unroll 1
          for (int jj = 0; jj < NJ; jj += 2) {
            uint32_t v[2][32];
            if (blocks) {
#pragma unroll
              for (int g = 0; g < 8; ++g) pr_ld8(o_at + 4 * (g * NJ + jj), &v[g / 4][8 * (g % 4)]);
              pr_wait_ld(v[0]);
              pr_touch(v[1]);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[0][e] = v[1][e] = 0;
            }
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const float bad = (nan_groups >> (jj + o)) & 1 ? NAN : 0.f;
              uint32_t u[4][4];                           // 16 bytes of the row each
#pragma unroll
              for (int g = 0; g < 8; ++g) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(__uint_as_float(v[g / 4][8 * (g % 4) + 2 * e + o]) * r, un, bad);
                u[g / 2][2 * (g % 2)] = pack_bf16x2(x[0], x[1]);
                u[g / 2][2 * (g % 2) + 1] = pack_bf16x2(x[2], x[3]);
              }
              // four lanes transpose their rows' quarters, so that a store writes 64 bytes of a row
#pragma unroll
              for (int m = 1; m < 4; m *= 2)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (!(x & m))
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const bool odd = lane & m;
                      const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? u[x][e] : u[x + m][e], m);
                      if (odd) u[x][e] = got;
                      else u[x + m][e] = got;
                    }
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const unsigned long long to = __shfl_sync(0xffffffffu, mine, (lane & 28) + m);
                if (to) *reinterpret_cast<uint4 *>(to + 64 * (jj + o) + 16 * (lane & 3)) = make_uint4(u[m][0], u[m][1], u[m][2], u[m][3]);
              }
            }
          }
          if (blocks) {
            pr_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars.o_empty + 8 * t);
          }
        }
      }
      n += blocks;
      item_done(k);
    }
  } else if (warp < 16) {
    // -------------------------------------------------- operands as f16 --
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrRegsMake));
    const int wu = __shfl_sync(0xffffffffu, warp, 0), kv = (wu - 8) >> 2;                       // 0: K and tile 0's Q; 1: V and tile 1's Q
    const int row = tid & (kPrRows - 1), w4 = wu & 3;
    int *red = reinterpret_cast<int *>(sm + L::o_red) + 8 * kv;
    const uint32_t bar_full = (kv ? bars.v_full : bars.k_full), bar_empty = (kv ? bars.v_empty : bars.k_empty);

    // this row's codes and params within a packed block: the pages' parts one after the other
    const uint32_t sub = (uint32_t)(row >> p.g.log2_page) * (p.g.head_bytes / 2);
    const uint32_t o_codes = sub + (row & (p.g.page - 1)) * (D / 2);
    const uint32_t o_par = sub + p.g.kp_off + (row & (p.g.page - 1)) * (NJ * 4);
    int n = 0, uses = 0;                                  // blocks so far; items of the tile so far
    int exp = 0;
#pragma unroll 1
    for (int k = 0;; item_done(k), ++k) {
      if (!attn_wait(bars.item_full + 8 * (k & 1), (k >> 1) & 1, abort, p.err)) break;
      const PrItem &it = *reinterpret_cast<const PrItem *>(sm + L::o_item + 64 * (k & 1));
      if (it.b < 0) break;
      if (it.blocks == 0) continue;
      // the item's query rows, 4 NJ lanes a row
      const int t = kv;
      if (t < it.tiles && attn_wait(bars.q_empty + 8 * t, (uses++ & 1) ^ 1, abort, p.err)) {
        constexpr int kLanes = 4 * NJ, kAtOnce = 4;
        const int i = row % kLanes;                       // dims 8i .. 8i+7 = 32j + 8q ..: chunk q * NJ + j
#pragma unroll 1
        for (int r0 = row / kLanes; r0 < kPrRows; r0 += kAtOnce * (kPrRows / kLanes)) {
          uint4 w[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int flat = it.flat0 + t * kPrRows + r0 + u * (kPrRows / kLanes), qi = attn_row(p, flat);
            w[u] = make_uint4(0, 0, 0, 0);
            if (r0 + u * (kPrRows / kLanes) < kPrRows && qi < it.rows_do)
              w[u] = __ldcg(reinterpret_cast<const uint4 *>(p.q + (size_t)(it.first + qi) * p.ldq +
                                                            (size_t)(it.head * p.group + flat - qi * p.group) * D) + i);
          }
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) {
            const int r = r0 + u * (kPrRows / kLanes);
            const uint32_t x4[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(x4[e] & 0x7FFFu, (x4[e] >> 16) & 0x7FFFu));
#pragma unroll
            for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int sh = top < (15u << 7) ? 126 : 141 - (int)(top >> 7);   // largest value to [2^14, 2^15)
            // the sign of the score scale goes into Q, and a scale of zero (the factor of the scores is above zero); a row
            // that is not finite gives NaN, not its products
            const float mul = top >= 0x7F80u || p.scale_log2 == 0.f ? 0.f : p.scale_log2 < 0.f ? -pow2f(sh) : pow2f(sh);
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[2 * e] = top >= 0x7F80u ? 0.f : bf16_lo_f32(x4[e]) * mul;
              x[2 * e + 1] = top >= 0x7F80u ? 0.f : bf16_hi_f32(x4[e]) * mul;
            }
            if (r < kPrRows) {
              *reinterpret_cast<uint4 *>(sm + L::o_q + t * L::tile + pr_chunk(r, (i % 4) * NJ + i / 4)) =
                  make_uint4(pack_f16x2(x[0], x[4]), pack_f16x2(x[1], x[5]), pack_f16x2(x[2], x[6]), pack_f16x2(x[3], x[7]));
              if (i == 0)
                crow[(k & 1) * 2 * kPrRows + t * kPrRows + r] = top >= 0x7F80u ? NAN : pow2f(-sh) * fabsf(p.scale_log2);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bars.q_full + 8 * t);
      }

#pragma unroll 1
      for (int j = 0; j < it.blocks; ++j, ++n) {
        const int s = n & 1, slot = (2 * n + kv) % kPrRaw;
        const uint8_t *raw = sm + L::o_raw + slot * L::raw;
        const bool seen = pr_seen_by_item(it, pr_block(it, j) + row);
        if (!attn_wait(bars.raw_full + 8 * slot, (2 * n + kv) / kPrRaw & 1, abort, p.err)) break;
        uint32_t par[NJ];
        lds_words<NJ>(raw + o_par, par);
        // the block's exponents; a NaN group is zero and told to the rows that see it
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
          if (!seen) par[i] = 0;
          if (((par[i] >> 7) & 0xFF) == 0xFF || ((par[i] >> 23) & 0xFF) == 0xFF) mask |= kv ? 1u << i : 0x80u, par[i] = 0;
        }
        const int e = (int)__reduce_max_sync(0xffffffffu, (uint32_t)pr_exponent<NJ>(par)) |
                      (__any_sync(0xffffffffu, mask != 0) ? 0x1000 : 0);
        if (lane == 0) {
          red[s * 4 + w4] = e;
          mbar_arrive(bars.vote + 8 * kv);
        }
        if (!attn_wait(bars.vote + 8 * kv, n & 1, abort, p.err)) break;
        if (j == 0 || !kv) exp = 0;                       // V's follows the largest of the item, K's is the block's own
        int bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          exp = max(exp, red[s * 4 + i] & 0xFFF);
          bad |= red[s * 4 + i] >> 12;
        }
        const int f = pr_shift(exp);
        auto tell = [&] {
          poison[((n % kPrInfo) * 2 + kv) * kPrRows + row] = (uint8_t)mask;
          if (row == 0) *(reinterpret_cast<int2 *>(info + n % kPrInfo) + kv) = make_int2(f, bad);
        };
        if (kv) {
          // K's barrier waits for it too, so that the scores' one tells the softmax of both.  It is in this block's
          // phase: V's packed block n takes the slot of K's n - 1, so K's n - 2 has been made.
          static_assert(kPrRaw <= 3, "V two blocks ahead of K");
          tell();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars.k_full + 8 * s);
        }
        if (!attn_wait(bar_empty + 8 * s, ((n >> 1) & 1) ^ 1, abort, p.err)) break;
        if (!kv) tell();                                  // not before: block n - 4's may still be read
        // four words of codes at a time, each with its {scale, min}
        const float up = pow2f(f >> 1) * pow2f(f - (f >> 1)), up20 = up * 0x1p20f;
        uint32_t s2[4], m2[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          // a K word is of group w % NJ; a V word holds groups 2 (w % (NJ / 2)) and the next
          const uint32_t lo = kv ? par[2 * (w % (NJ / 2))] : par[w % NJ], hi = kv ? par[2 * (w % (NJ / 2)) + 1] : par[w % NJ];
          s2[w] = pack_f16x2(bf16_lo_f32(lo) * up20, bf16_lo_f32(hi) * up20);
          m2[w] = pack_f16x2(bf16_hi_f32(lo) * up, bf16_hi_f32(hi) * up);
        }
        uint8_t *dst = sm + (kv ? L::o_v : L::o_k) + s * L::tile + row * 128;
#pragma unroll 1
        for (int i0 = 0; i0 < NJ; ++i0) {
          const int i = NJ == 4 ? i0 ^ ((row >> 1) & 3) : i0 ^ ((row >> 2) & 1);   // rows of eight lanes at eight banks
          uint32_t w[4];
          lds_words<4>(raw + o_codes + 16 * i, w);
          // chunks 4 i .. 4 i + 3 of the row
          uint8_t *half = dst + (i >> 1) * (kPrRows * 128);
          const uint32_t x = (uint32_t)((4 * i ^ row) & 7) << 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) *reinterpret_cast<uint4 *>(half + (x ^ (e << 4))) = pr_unpack(w[e], s2[e], m2[e]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(bar_full + 8 * s);
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.raw_empty + 8 * slot);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrRegsIssue));
    if (warp == 17) {
      // ----------------------------------------------------------- items --
      const int total = prefix[(p.b.n_seqs + 31) / 32];
#pragma unroll 1
      for (int k = 0;; ++k) {
        if (!attn_wait(bars.item_empty + 8 * (k & 1), ((k >> 1) & 1) ^ 1, abort, p.err)) break;
        // the first item by the CTA's number, the next ones by turns, claimed when the last one's copies are on their way
        int i = blockIdx.x;
        if (k > 0) {
          if (!attn_wait(bars.claim, (k - 1) & 1, abort, p.err)) break;
          if (lane == 0) i = (int)gridDim.x + atomicAdd(p.turns, 1);
          i = __shfl_sync(0xffffffffu, i, 0);
        }
        PrItem it;
        it.b = -1;
        if (i < total) it = pr_item(p, prefix, i, lane);
        if (lane == 0) {
          *reinterpret_cast<PrItem *>(sm + L::o_item + 64 * (k & 1)) = it;
          mbar_arrive(bars.item_full + 8 * (k & 1));
        }
        __syncwarp();
        if (i >= total) break;
      }
      // no claim comes after a CTA's last: the last CTA to get here leaves the counters at zero
      if (lane == 0 && atomicAdd(p.turns + 1, 1) == (int)gridDim.x - 1) p.turns[0] = p.turns[1] = 0;
    } else if (warp == 18) {
      // ------------------------------------------------- packed K and V --
      const uint32_t part = p.g.head_bytes / 2;           // K or V of a page
      int h = 0;                                          // packed blocks asked for: K, V, K, ...
      bool ok = true;
#pragma unroll 1
      for (int k = 0; ok; item_done(k), ++k) {
        ok = attn_wait(bars.item_full + 8 * (k & 1), (k >> 1) & 1, abort, p.err);
        if (!ok) break;
        const PrItem &it = *reinterpret_cast<const PrItem *>(sm + L::o_item + 64 * (k & 1));
        if (it.b < 0) break;
#pragma unroll 1
        for (int j = 0; j < it.blocks && ok; ++j) {
          // lane l: page l of the block, unless nobody sees its tokens
          const int t = pr_block(it, j) + (lane << p.g.log2_page);
          const uint8_t *src = nullptr;
          if (lane < kPrRows >> p.g.log2_page && t < it.len && (t + p.g.page > it.lo || t < it.sinks))
            src = kv_head_block(p.g, p.b, it.b, t, it.head, p.err);
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, src != nullptr)) * part;
#pragma unroll 1
          for (int v = 0; v < 2; ++v, ++h) {
            const int slot = h % kPrRaw;
            ok = attn_wait(bars.raw_empty + 8 * slot, (h / kPrRaw & 1) ^ 1, abort, p.err);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(bars.raw_full + 8 * slot, bytes);
            __syncwarp();
            if (src)
              bulk_copy_g2s_plain(smem_addr(sm + L::o_raw + slot * L::raw) + lane * part, src + (v ? part : 0), part,
                                  bars.raw_full + 8 * slot);
          }
        }
        if (lane == 0) mbar_arrive(bars.claim);
      }
      // copies in flight land before the CTA leaves: the last phase of each slot that had one, with a limit
      for (int i = max(0, h - kPrRaw); i < h; ++i) mbar_wait_bounded_warp(bars.raw_full + 8 * (i % kPrRaw), i / kPrRaw & 1);
    } else {
      // -------------------------------------------------------- products --
      // Two warps: 16 issues the scores, 19 the values (one warp's instructions for both took longer than the products).
      const bool is_v = warp == 19;
      constexpr uint32_t id_s = pr_idesc(kPrRows, false), id_o = pr_idesc(D, true);
      constexpr uint32_t kBlock = kPrRows * 128;          // a 64-value column block of a tile
      const uint32_t q_at = smem_addr(sm + L::o_q), k_at = smem_addr(sm + L::o_k), v_at = smem_addr(sm + L::o_v);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      uint32_t items = 0, any = 0, made = 0, valued = 0;  // by tile (bit t): parity of its items, whether there were any ...
      int n = 0;                                          // ... of its values; scores of both tiles; blocks
      bool ok = true;
      // the whole warp takes every step and one thread is elected for the products: their operands stay in uniform registers
#pragma unroll 1
      for (int k = 0; ok; item_done(k), ++k) {
        ok = attn_wait(bars.item_full + 8 * (k & 1), (k >> 1) & 1, abort, p.err);
        if (!ok) break;
        const PrItem *it = reinterpret_cast<const PrItem *>(sm + L::o_item + 64 * (k & 1));
        if (it->b < 0) break;
        const int tiles = __shfl_sync(0xffffffffu, it->tiles, 0), blocks = __shfl_sync(0xffffffffu, it->blocks, 0);
#pragma unroll 1
        for (int j = 0; j < blocks && ok; ++j, ++n) {
          const int s = n & 1;
          const uint32_t ph = (n >> 1) & 1;
#pragma unroll 1
          for (int t = 0; t < tiles && ok; ++t) {
            if (!is_v) {
              if (j == 0) {
                ok = attn_wait(bars.q_full + 8 * t, (items >> t) & 1, abort, p.err);
                items ^= 1u << t;
              }
              if (t == 0) ok = ok && attn_wait(bars.k_full + 8 * s, ph, abort, p.err);
              // the tiles share S: the last scores have been read
              if (made) ok = ok && attn_wait(bars.s_free, (made - 1) & 1, abort, p.err);
              if (!ok) break;
              ++made;
              pr_fence_after();
              if (pr_elect()) {
                const uint32_t da = pr_desc(q_at + t * L::tile, 16), db = pr_desc(k_at + s * L::tile, 16);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                  const uint32_t off = ((i >> 2) * kBlock + (i & 3) * 32) >> 4;
                  pr_mma_ss(tm + L::s_col, da + off, db + off, id_s, i > 0);
                }
                pr_commit(bars.s_full + 8 * t);
                if (t == tiles - 1) pr_commit(bars.k_empty + 8 * s);
                if (j == blocks - 1) pr_commit(bars.q_empty + 8 * t);
              }
            } else {
              if (j == 0) {
                // the tile's previous results have been read
                if ((any >> t) & 1) ok = attn_wait(bars.o_empty + 8 * t, ((items >> t) & 1) ^ 1, abort, p.err);
                any |= 1u << t;
                items ^= 1u << t;
              }
              if (t == 0) ok = ok && attn_wait(bars.v_full + 8 * s, ph, abort, p.err);
              ok = ok && attn_wait(bars.p_full + 8 * t, (valued >> t) & 1, abort, p.err);
              if (!ok) break;
              valued ^= 1u << t;
              pr_fence_after();
              if (pr_elect()) {
                const uint32_t d = tm + L::o_col + t * D, at = tm + L::p_col + t * (kPrRows / 2);
                const uint32_t db = pr_desc(v_at + s * L::tile, kBlock);
#pragma unroll
                for (int i = 0; i < kPrRows / 16; ++i) pr_mma_ts(d, at + 8 * i, db + i * (2048 >> 4), id_o, j > 0 || i > 0);
                pr_commit(bars.o_done + 8 * t);
                if (t == tiles - 1) pr_commit(bars.v_empty + 8 * s);
              }
            }
            __syncwarp();
          }
        }
      }
      if (pr_elect()) pr_commit(bars.drain + 8 * is_v);   // whatever was issued has ended before the memory is given back
      mbar_wait_bounded_warp(bars.drain + 8 * is_v, 0);
    }
  }
  __syncwarp();
  pr_fence_before();
  __syncthreads();
  if (warp == 16) {
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
  cfg.gridDim = dim3((unsigned)(items < ctx->sm_count ? items : ctx->sm_count));
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

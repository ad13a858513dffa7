// Attention over the paged 4-bit KV cache for few rows a sequence (decode).
//
//   s_t = scale * q . k_t,  o = sum_t softmax_t(s) v_t   over the visible t
//
// The cached tokens are read once (5 bits a value); a kv head's query heads,
// and the rows of a sequence when there are several, are the columns of the
// products, eight (NB = 1) or sixteen (NB = 2) at a time.
//
// Scores.  K rows are the A operand as 4-bit codes: a nibble masked into an
// f16 register is the exact subnormal code * 2^-24 (nibbles 1 and 3 of a
// half-word come out 16 times larger, and their columns of q are 1/16).  The
// query is scaled by a power of two per column so that its f16 is exact down
// to 2^-29 of its largest value.  A group's product is scaled afterwards:
// s = sum_j scale_j * (codes_j . q_j) + min_j * sum(q_j); the minima's term is a
// product of its own, the bf16 minima with the sums split into three bf16 parts.
// Output.  The contraction runs over tokens, so a value's scale cannot be
// applied to the product: V is dequantised to f16 in registers, min + scale *
// code in one rounding (the code again as a subnormal operand of the packed
// multiply-add), and P is f16 too: 2^-12 of a term each, the only roundings
// below 32 bits.  V is brought to about 1 at most by a power of two that follows
// the largest scale seen, so a value below 2^-9 of that scale has fewer bits (it
// is good to 2^-20 of the scale); P has 7 bits at least, and weights below 2^-64
// of a reference are zero.  Its codes are read in the transposed fragment order
// by byte permutes of two tokens' words, P is transposed in registers (movmatrix).
// The softmax reference of a column moves only when a score passes it by 8
// (in powers of two), so the sums are rescaled a few times a chunk at most.
//
// Work.  A sequence's visible tokens (its sinks, then its window) are cut into
// stages of 128 and the stages into chunks whose number depends on their own
// count alone, so a row's bytes do not depend on the batch.  Items (sequence,
// kv head, column block, chunk) are dealt in runs over a persistent grid, so
// that a CTA keeps its query columns over several chunks; it finds them from the
// device's lengths.  One warp finds the items and streams the stages (K and V of
// one kv head, one bulk copy a page) into a ring, four warps take 32 tokens of
// a stage each.  A row of one chunk is written directly; else each chunk leaves
// (maximum, sum, values) in scratch and the last one to arrive joins them in
// chunk order.
//
// Measured (32 query heads, 4 kv heads of 128): 64 sequences of 65 to 8191 tokens
// 62.4 us (170 MB: 2.7 TB/s, 43% of the copy rate), two of 111870 and 131072 tokens
// 52.8 us (156 MB, 46%), one of 333 tokens 7.7 us.  Neither memory (a third of its
// cycles) nor issue (0.53 a cycle) is full: the registers allow three computing warps
// a scheduler, and these do not cover one another's chains of dependent steps (codes,
// score products, weights, value products).  450 warp instructions for 16 tokens of a
// kv head, a third of them to unpack the codes.  The forms for heads of 128 spill 12
// to 144 bytes a thread.
#include <limits.h>

#include "kv_attn.cuh"

namespace rc {

constexpr int kDcWarps = 4;                       // computing warps
constexpr int kDcThreads = 32 * (kDcWarps + 1);   // and one that copies
constexpr int kDcStage = 128;                     // tokens of a stage
// A chunk is an eighth of the stages, but four to six of them (512 to 768
// tokens: smaller ones cost more in partial results than they give in balance),
// and a 256th where that is more.  us with at least 1 / 2 / 3 / 4 / 5: one
// sequence of 333 tokens 8.9 / 9.2 / 8.1 / 7.9 / 7.9, 64 of up to 8191 tokens
// 68.7 / 65.1 / 66.5 / 62.6 / 62.2, 32 that see 1028 tokens 21.6 / 21.8 / 21.2 /
// 21.0 / 21.8 (one of 1024 takes 11.4 with 4 and 10.0 with 2); two of up to 131072
// with at most 6 / 8 / 10: 54.0 / 60.8 / 56.9.
constexpr int kDcMinStages = 4, kDcMaxStages = 6, kDcMaxChunks = 256;
constexpr int kDcFan = 16;                        // partial results joined at a time
constexpr int kDcGroups = (kDcMaxChunks + kDcFan - 1) / kDcFan;

__host__ __device__ constexpr int dc_min(int a, int b) { return a < b ? a : b; }
__host__ __device__ constexpr int dc_max(int a, int b) { return a > b ? a : b; }
__host__ __device__ constexpr int dc_ceil(int a, int b) { return (a + b - 1) / b; }
// Stages of a chunk of a sequence of ``stages``.
__host__ __device__ constexpr int dc_per_chunk(int stages) {
  return dc_max(dc_min(dc_max(dc_ceil(stages, 8), kDcMinStages), kDcMaxStages), dc_ceil(stages, kDcMaxChunks));
}
// The most chunks of a sequence of up to ``stages``: eight while they grow, then those of the largest constant chunk.
__host__ __device__ constexpr int dc_most_chunks(int stages) {
  return dc_max(dc_min(dc_ceil(stages, kDcMinStages), 8), dc_min(dc_ceil(stages, kDcMaxStages), kDcMaxChunks));
}
constexpr bool dc_holds(int stages) {
  for (int s = 1; s <= stages; ++s)
    if (dc_ceil(s, dc_per_chunk(s)) > dc_most_chunks(s) || dc_most_chunks(s) < dc_most_chunks(s - 1)) return false;
  return true;
}
static_assert(dc_holds(4 * kDcMaxChunks * kDcMaxStages), "the partial results of a sequence have room");

struct DcParams {
  AttnParams a;
  int cbs;            // column blocks of max_q rows
  int chunks, slots;  // partials of one (sequence, head, column block): its chunks', then, if any, its groups'
  float *part;        // [n_seqs][heads][cbs][slots][cols * (D + 2)]
  int *count;         // [n_seqs][heads][cbs][1 + groups] arrivals, zero between launches
};

// What a sequence's items need.
struct DcSeq {
  int first, rows, rows_do, len;   // first row, rows, rows computed (at most max_q), tokens
  int lo, sinks;                   // visible to some row: t >= lo or t < sinks
  int n_sink, stages, per_chunk, n_chunks;
  __device__ int cost() const { return stages + n_chunks; }   // of one column block, in stages: an item costs one more
};

__device__ __forceinline__ DcSeq dc_seq(const AttnParams &p, int b) {
  DcSeq s;
  attn_seq(p, b, s.first, s.rows, s.rows_do, s.len);
  s.lo = attn_window_lo(p, s.len - s.rows);
  s.sinks = p.window > 0 ? min(p.sinks, s.lo) : 0;
  const int first = s.lo / kDcStage;
  s.n_sink = min((s.sinks + kDcStage - 1) / kDcStage, first);
  s.stages = s.n_sink + (s.len + kDcStage - 1) / kDcStage - first;
  s.per_chunk = dc_per_chunk(s.stages);
  s.n_chunks = max(1, (s.stages + s.per_chunk - 1) / s.per_chunk);
  return s;
}

struct DcItem {
  int b, head, cb, chunk, n_chunks;      // b < 0: no more items
  int first, rows, rows_do, len, lo, sinks;
  int v0, v1, n_sink;                    // stages v0 .. v1 - 1 of the sequence
};
static_assert(sizeof(DcItem) <= 64, "an item's slot");

__device__ __forceinline__ int dc_stage(const DcItem &it, int v) {   // first token of stage v
  return (v < it.n_sink ? v : it.lo / kDcStage + v - it.n_sink) * kDcStage;
}
__device__ __forceinline__ bool dc_seen(const DcItem &it, int t) { return t < it.len && (t >= it.lo || t < it.sinks); }

// The items in order: sequences, kv heads, column blocks, chunks.  ``at`` is the cost of all items before the present one.
struct DcWalk {
  DcSeq s;
  int b, cell, cells, chunk, at;

  __device__ __forceinline__ void load(const AttnParams &p, int nc, int seq) {
    b = seq;
    s = dc_seq(p, seq);
    cells = (s.rows_do * p.group + nc - 1) / nc * p.g.heads;
  }
  // To the first item with at least ``cost`` before it.
  __device__ __forceinline__ void seek(const AttnParams &p, const int *prefix, int nc, int cost) {
    int lo = 0, hi = p.b.n_seqs - 1;   // the last sequence that starts at or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= cost) lo = mid;
      else hi = mid - 1;
    }
    load(p, nc, lo);
    const int off = cost - prefix[lo];
    cell = off / s.cost();
    chunk = (off - cell * s.cost() + s.per_chunk) / (s.per_chunk + 1);
    at = prefix[lo] + cell * s.cost() + chunk * (s.per_chunk + 1);
    settle(p, nc);
  }
  // Past the end of a column block, of a sequence (which may have no rows).
  __device__ __forceinline__ void settle(const AttnParams &p, int nc) {
    if (cell < cells && chunk >= s.n_chunks) {
      at += s.cost() - chunk * (s.per_chunk + 1);
      chunk = 0;
      ++cell;
    }
    while (cell >= cells && b + 1 < p.b.n_seqs) {
      load(p, nc, b + 1);
      cell = 0;
    }
  }
  __device__ __forceinline__ void next(const AttnParams &p, int nc) {
    ++chunk;
    at += s.per_chunk + 1;
    settle(p, nc);
  }
  __device__ __forceinline__ DcItem item(const AttnParams &p) const {
    DcItem it;
    it.b = b;
    const int cbs = cells / p.g.heads;
    it.head = cell / cbs;
    it.cb = cell - it.head * cbs;
    it.chunk = chunk;
    it.n_chunks = s.n_chunks;
    it.first = s.first, it.rows = s.rows, it.rows_do = s.rows_do, it.len = s.len;
    it.lo = s.lo, it.sinks = s.sinks, it.n_sink = s.n_sink;
    it.v0 = chunk * s.per_chunk;
    it.v1 = min(s.stages, it.v0 + s.per_chunk);
    return it;
  }
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void dc_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kDcWarps) : "memory"); }

template <int NJ, int NB>
struct DcLayout {
  static constexpr int D = 32 * NJ, cols = 8 * NB;
  static constexpr int stage = kDcStage * D * 5 / 4;
  static constexpr int stages = NJ == 4 ? (NB == 1 ? 2 : 3) : (NB == 1 ? 5 : 6);
  static constexpr int join = kDcWarps * cols * D * 4;                       // the warps' values of one item
  static_assert(join >= cols * kDcFan * 12, "the joined parts' (reference, sum) and shares lie there too");
  static constexpr int o_scratch = stages * stage;
  static constexpr int o_vpar = o_scratch + join;                            // [warps][2][8 token pairs][NJ]{scale, min} f16x2
  static constexpr int vpar = 2 * 8 * NJ * 8;
  static constexpr int o_ml = o_vpar + kDcWarps * vpar;                      // [2][warps][cols]
  static constexpr int o_item = o_ml + 2 * kDcWarps * cols * 4;              // [2]
  static constexpr int o_bar = o_item + 2 * 64;
  static constexpr int o_flags = o_bar + 16 * stages + 32;
  static constexpr int o_prefix = o_flags + 16;
  static int bytes(int n_seqs) { return o_prefix + (n_seqs + 1) * 4; }
};

// True in every thread of the CTA that arrives last of n; it then sees what the
// others wrote before they arrived (and leaves the counter at zero).  One thread's
// releasing add after the barrier covers the CTA's writes.
__device__ __forceinline__ bool dc_arrive_last(int *count, int n, volatile int *s_last, int tid) {
  dc_sync();
  if (tid == 0) {
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    *s_last = before == n - 1;
    if (before == n - 1) *count = 0;
  }
  dc_sync();
  return *s_last;
}

// Of a sum of weights (0: no token was seen), to 2 ulp.
__device__ __forceinline__ float dc_inverse(float sum) { return sum == 0.f ? 0.f : __fdividef(1.f, sum); }

// Joins n <= kDcFan partial results, each a mean of values with the reference and sum of its weights, in order;
// sink(column, value, 4 means, reference, sum).
template <int NJ, int NB, typename Sink>
__device__ __forceinline__ void dc_join(const float *src, int n, float *scratch, int tid, Sink sink) {
  constexpr int D = 32 * NJ, NC = 8 * NB;
  constexpr size_t kSlot = (size_t)NC * (D + 2);
  float2 *ml = reinterpret_cast<float2 *>(scratch);   // [part][column]
  float *share = scratch + 2 * kDcFan * NC;           // [part][column] weights, all of one reference
  dc_sync();
  for (int e = tid; e < n * NC; e += 32 * kDcWarps)
    ml[e] = __ldcg(reinterpret_cast<const float2 *>(src + (e / NC) * kSlot + (size_t)NC * D) + e % NC);
  dc_sync();
  for (int e = tid; e < n * NC; e += 32 * kDcWarps) {
    float top = -INFINITY;
    for (int c = 0; c < n; ++c) top = fmaxf(top, ml[c * NC + e % NC].x);
    share[e] = (top == -INFINITY ? 1.f : exp2f(ml[e].x - top)) * ml[e].y;
  }
  dc_sync();
#pragma unroll 1
  for (int e = tid; e < NC * D / 4; e += 32 * kDcWarps) {
    const int col = e / (D / 4), d = 4 * (e % (D / 4));
    float4 v[kDcFan];
#pragma unroll
    for (int c = 0; c < kDcFan; ++c)
      v[c] = c < n ? __ldcg(reinterpret_cast<const float4 *>(src + c * kSlot + (size_t)col * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    for (int c = 0; c < n; ++c) top = fmaxf(top, ml[c * NC + col].x), sum += share[c * NC + col];
    const float r = dc_inverse(sum);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kDcFan; ++c) {
      if (c >= n) break;
      const float f = share[c * NC + col] * r;
      acc.x = fmaf(f, v[c].x, acc.x), acc.y = fmaf(f, v[c].y, acc.y), acc.z = fmaf(f, v[c].z, acc.z), acc.w = fmaf(f, v[c].w, acc.w);
    }
    sink(col, d, acc, top, sum);
  }
}

// MULTI: the rows of a sequence have masks of their own.
template <int NJ, int NB, bool MULTI>
__global__ void __launch_bounds__(kDcThreads, NB == 1 ? 3 : 2) rc_kv_decode_kernel(const __grid_constant__ DcParams p) {
  using L = DcLayout<NJ, NB>;
  constexpr int D = L::D, NC = L::cols;
  extern __shared__ __align__(128) uint8_t sm[];
  const AttnParams &a = p.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t bar_full = smem_addr(sm + L::o_bar), bar_empty = bar_full + 8 * L::stages;
  const uint32_t bar_item = bar_empty + 8 * L::stages, bar_taken = bar_item + 16;
  volatile int *abort = reinterpret_cast<volatile int *>(sm + L::o_flags);
  int *s_last = reinterpret_cast<int *>(sm + L::o_flags) + 1;
  volatile int *s_go = reinterpret_cast<volatile int *>(sm + L::o_flags) + 2;
  int *prefix = reinterpret_cast<int *>(sm + L::o_prefix);
  if (tid == 0) {
    *abort = 0;
    for (int i = 0; i < L::stages; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, kDcWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_item + 8 * i, 1);
      mbar_init(bar_taken + 8 * i, kDcWarps);
    }
    mbar_fence_init();
  }
  pdl_launch_dependents();
  pdl_wait_prior();
  // cost of every sequence's items, then their prefix sums
#pragma unroll 1
  for (int b = tid; b < a.b.n_seqs; b += kDcThreads) {
    const DcSeq s = dc_seq(a, b);
    prefix[b + 1] = s.cost() * a.g.heads * ((s.rows_do * a.group + NC - 1) / NC);
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < a.b.n_seqs; b0 += 32) {
      int v = b0 + lane < a.b.n_seqs ? prefix[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < a.b.n_seqs) prefix[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  int slot = 0;
  uint32_t phase = 0;                                     // of the ring's current round

  if (warp == kDcWarps) {
    // ----------------------------------------------------- items, copies --
    // this CTA's items: those that start in its share of the whole cost
    const long long total = prefix[a.b.n_seqs];
    const int end = (int)(total * (blockIdx.x + 1) / gridDim.x);
    const uint64_t policy = policy_evict_first();         // unless other column blocks come for the same tokens
    bool ok = true;
    DcWalk w;
    w.seek(a, prefix, NC, (int)(total * blockIdx.x / gridDim.x));
#pragma unroll 1
    for (int k = 0; ok; ++k, w.next(a, NC)) {
      DcItem it;
      it.b = -1;
      if (w.cell < w.cells && w.at < end) it = w.item(a);
      ok = attn_wait(bar_taken + 8 * (k & 1), ((k >> 1) & 1) ^ 1, abort, a.err);
      if (!ok) break;
      if (lane == 0) {
        *reinterpret_cast<DcItem *>(sm + L::o_item + 64 * (k & 1)) = it;
        mbar_arrive(bar_item + 8 * (k & 1));
      }
      if (it.b < 0) break;
#pragma unroll 1
      for (int v = it.v0; v < it.v1 && ok; ++v) {
        // lane l: page l of the stage, unless nobody sees its tokens
        const int t = dc_stage(it, v) + (lane << a.g.log2_page);
        const uint8_t *src = nullptr;
        if (lane < kDcStage >> a.g.log2_page && t < it.len && (t + a.g.page > it.lo || t < it.sinks))
          src = kv_head_block(a.g, a.b, it.b, t, it.head, a.err);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, src != nullptr)) * a.g.head_bytes;
        ok = attn_wait(bar_empty + 8 * slot, phase ^ 1, abort, a.err);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(bar_full + 8 * slot, bytes);
        __syncwarp();
        if (src) {
          const uint32_t dst = smem_addr(sm + slot * L::stage) + lane * a.g.head_bytes;
          if (p.cbs == 1) bulk_copy_g2s(dst, src, a.g.head_bytes, bar_full + 8 * slot, policy);
          else bulk_copy_g2s_plain(dst, src, a.g.head_bytes, bar_full + 8 * slot);
        }
        if (++slot == L::stages) slot = 0, phase ^= 1;
      }
    }
    // copies in flight land before the CTA leaves: each slot's last phase, with a limit
    for (int i = 0; i < L::stages; ++i) mbar_wait_bounded_warp(bar_full + 8 * i, i < slot ? phase : phase ^ 1);
    return;
  }

  // --------------------------------------------------------------- compute --
  const int g = lane >> 2, q4 = lane & 3;
  const int f_row = g ^ ((g >> 1) & 1);                  // token of row g among 8 (spreads V's rows over the banks)
  const int v_tok = 2 * q4 ^ (q4 & 1);                   // tokens v_tok and v_tok ^ 1 are columns 2 q4 and 2 q4 + 1
  const int vp_tok = 2 * (lane / NJ % 8) ^ (lane / NJ & 1);   // of lane = pair * NJ + group: the pair's first token
  uint8_t *vpar = sm + L::o_vpar + warp * L::vpar;
  float *s_o = reinterpret_cast<float *>(sm + L::o_scratch);
  float *s_m = reinterpret_cast<float *>(sm + L::o_ml), *s_l = s_m + kDcWarps * NC;
  // this warp's two 16-token groups within a stage: codes and params of K; V's lie half a head block further
  const uint32_t half = a.g.head_bytes / 2;
  uint32_t o_kc[2], o_kp[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int t = 32 * warp + 16 * r, at = t & (a.g.page - 1);
    o_kc[r] = (uint32_t)(t >> a.g.log2_page) * a.g.head_bytes + at * (D / 2);
    o_kp[r] = (uint32_t)(t >> a.g.log2_page) * a.g.head_bytes + a.g.kp_off + at * NJ * 4;
  }
  // query columns: B fragments of column 8 nb + g, of its group sums, score scales of columns 8 nb + 2 q4, + 1
  uint32_t qb[NB][2 * NJ][2], qm[NB][2];
  float cs[NB][2];
  int pos[NB][2];
  int cell_b = -1, cell_head = 0, cell_cb = 0;

#pragma unroll 1
  for (int k = 0;; ++k) {
    // one warp's verdict for all, so that they meet at the barriers below also when a wait has given up; past this
    // barrier the last item's scratch is free
    if (warp == 0) {
      const bool ok = attn_wait(bar_item + 8 * (k & 1), (k >> 1) & 1, abort, a.err);
      if (lane == 0) *s_go = ok && reinterpret_cast<const DcItem *>(sm + L::o_item + 64 * (k & 1))->b >= 0;
    }
    dc_sync();
    if (!*s_go) break;
    DcItem it = *reinterpret_cast<const DcItem *>(sm + L::o_item + 64 * (k & 1));
    it.v0 = __shfl_sync(0xffffffffu, it.v0, 0), it.v1 = __shfl_sync(0xffffffffu, it.v1, 0), it.n_sink = __shfl_sync(0xffffffffu, it.n_sink, 0);
    it.lo = __shfl_sync(0xffffffffu, it.lo, 0), it.len = __shfl_sync(0xffffffffu, it.len, 0), it.sinks = __shfl_sync(0xffffffffu, it.sinks, 0);
    it.rows = __shfl_sync(0xffffffffu, it.rows, 0);
    it.b = __shfl_sync(0xffffffffu, it.b, 0), it.head = __shfl_sync(0xffffffffu, it.head, 0), it.cb = __shfl_sync(0xffffffffu, it.cb, 0), it.chunk = __shfl_sync(0xffffffffu, it.chunk, 0), it.n_chunks = __shfl_sync(0xffffffffu, it.n_chunks, 0), it.first = __shfl_sync(0xffffffffu, it.first, 0), it.rows_do = __shfl_sync(0xffffffffu, it.rows_do, 0);

    if (lane == 0) mbar_arrive(bar_taken + 8 * (k & 1));

    if (it.b != cell_b || it.head != cell_head || it.cb != cell_cb) {
      cell_b = it.b, cell_head = it.head, cell_cb = it.cb;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int flat = it.cb * NC + 8 * nb + g, qi = attn_row(a, flat);
        uint4 w[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) w[j] = make_uint4(0, 0, 0, 0);
        if (qi < it.rows_do) {
          const uint16_t *src = a.q + (size_t)(it.first + qi) * a.ldq + (it.head * a.group + flat - qi * a.group) * D + 8 * q4;
#pragma unroll
          for (int j = 0; j < NJ; ++j) w[j] = __ldcg(reinterpret_cast<const uint4 *>(src + 32 * j));
        }
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, max(u[e] & 0x7FFFu, (u[e] >> 16) & 0x7FFFu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int sh = top < (15u << 7) ? 126 : 141 - (int)(top >> 7);   // largest value to [2^14, 2^15)
        // the sign of the scale goes into q, and a scale of zero: the factor of the scores cannot be zero
        const float mul = a.scale_log2 < 0.f ? -pow2f(sh) : a.scale_log2 > 0.f ? pow2f(sh) : 0.f;
        uint32_t part[3][NJ];                             // group sums, 2^-24 as the codes, in three bf16
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float x[8] = {bf16_lo_f32(w[j].x) * mul, bf16_hi_f32(w[j].x) * mul, bf16_lo_f32(w[j].y) * mul,
                              bf16_hi_f32(w[j].y) * mul, bf16_lo_f32(w[j].z) * mul, bf16_hi_f32(w[j].z) * mul,
                              bf16_lo_f32(w[j].w) * mul, bf16_hi_f32(w[j].w) * mul};
          qb[nb][2 * j][0] = pack_f16x2(x[0], x[4]);
          qb[nb][2 * j][1] = pack_f16x2(x[1] * 0.0625f, x[5] * 0.0625f);
          qb[nb][2 * j + 1][0] = pack_f16x2(x[2], x[6]);
          qb[nb][2 * j + 1][1] = pack_f16x2(x[3] * 0.0625f, x[7] * 0.0625f);
          float gs = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
          gs += __shfl_xor_sync(0xffffffffu, gs, 1);
          gs += __shfl_xor_sync(0xffffffffu, gs, 2);
          gs *= 0x1p-24f;
#pragma unroll
          for (int e = 0; e < 3; ++e) {
            part[e][j] = pack_bf16x2(gs, 0.f);
            gs -= bf16_lo_f32(part[e][j]);
          }
        }
        // rows of that product: part 0, 1, 2 of the NJ groups; lane q4 holds rows 2 q4, + 1 and 8 + 2 q4, + 1
        if constexpr (NJ == 4) {
          const uint32_t hi = q4 & 1 ? part[0][2] | part[0][3] << 16 : part[0][0] | part[0][1] << 16;
          const uint32_t mid = q4 & 1 ? part[1][2] | part[1][3] << 16 : part[1][0] | part[1][1] << 16;
          const uint32_t low = q4 & 1 ? part[2][2] | part[2][3] << 16 : part[2][0] | part[2][1] << 16;
          qm[nb][0] = q4 & 2 ? mid : hi;
          qm[nb][1] = q4 & 2 ? 0u : low;
        } else {
          const uint32_t pick = q4 == 0 ? part[0][0] | part[0][1] << 16 : q4 == 1 ? part[1][0] | part[1][1] << 16
                                                                                : part[2][0] | part[2][1] << 16;
          qm[nb][0] = q4 == 3 ? 0u : pick;
          qm[nb][1] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int from = 4 * (2 * q4 + c), ci = attn_row(a, it.cb * NC + 8 * nb + 2 * q4 + c);
          // above 0, so that a hidden score is -Inf
          cs[nb][c] = fmaxf(pow2f(-__shfl_sync(0xffffffffu, sh, from)) * 0x1p24f * fabsf(a.scale_log2), 0x1p-126f);
          pos[nb][c] = ci < it.rows_do ? it.len - it.rows + ci : -1;
        }
      }
    }

    // m: softmax references; over: raw scores from which they move
    float o[NB][2 * NJ][4], m[NB][2], over[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int c = 0; c < 2; ++c) m[nb][c] = over[nb][c] = -INFINITY, l[nb][c] = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * NJ; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
    }
    int vexp = -1;      // exponent field of the largest V scale so far; V's f16 carry 2^fexp
    int fexp = 0;
    float up = 1.f;     // 2^fexp

#pragma unroll 1
    for (int v = it.v0; v < it.v1; ++v) {
      const bool ready = attn_wait(bar_full + 8 * slot, phase, abort, a.err);
      const int tw = dc_stage(it, v) + 32 * warp;        // this warp's 32 tokens
      if (ready && tw < it.len && (tw + 32 > it.lo || tw < it.sinks)) {
        const uint8_t *st = sm + slot * L::stage;
        bool full = tw + 31 <= it.len - it.rows && (tw + 31 < it.sinks || tw >= (MULTI ? max(it.lo, it.len - a.window) : it.lo));
        if (MULTI && a.window <= 0) full = tw + 31 <= it.len - it.rows;

        // raw scores of rows f_row, f_row + 8 of the two groups in columns 2 q4, 2 q4 + 1
        float x[2][NB][2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t k0[NJ], k1[NJ], p0[NJ], p1[NJ], n0[2], n1[2];
          const uint8_t *kp = st + o_kp[r] + f_row * NJ * 4;
          lds_words<NJ>(st + o_kc[r] + f_row * (D / 2) + q4 * NJ * 4, k0);
          lds_words<NJ>(st + o_kc[r] + (f_row + 8) * (D / 2) + q4 * NJ * 4, k1);
          lds_words<NJ>(kp, p0);
          lds_words<NJ>(kp + 8 * NJ * 4, p1);
          lds_words<2>(kp + (NJ == 4 ? (q4 & 1) * 8 : 0), n0);
          lds_words<2>(kp + 8 * NJ * 4 + (NJ == 4 ? (q4 & 1) * 8 : 0), n1);
          const uint32_t m0 = __byte_perm(n0[0], n0[1], 0x7632), m1 = __byte_perm(n1[0], n1[1], 0x7632);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            mma_bf16_16816(d, m0, m1, m0, m1, qm[nb][0], qm[nb][1]);
#pragma unroll
            for (int c = 0; c < 2; ++c) x[r][nb][0][c] = d[c], x[r][nb][1][c] = d[2 + c];
          }
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const float s0 = bf16_lo_f32(p0[j]), s1 = bf16_lo_f32(p1[j]);
            const uint32_t h0 = k0[j] >> 8, h1 = k1[j] >> 8;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float d[4];
              mma_f16_16816_zero(d, k0[j] & 0x000F000Fu, k1[j] & 0x000F000Fu, k0[j] & 0x00F000F0u, k1[j] & 0x00F000F0u,
                                 qb[nb][2 * j][0], qb[nb][2 * j][1]);
              mma_f16_16816(d, h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, qb[nb][2 * j + 1][0],
                            qb[nb][2 * j + 1][1]);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                x[r][nb][0][c] = fmaf(s0, d[c], x[r][nb][0][c]);
                x[r][nb][1][c] = fmaf(s1, d[2 + c], x[r][nb][1][c]);
              }
            }
          }
        }
        // V params of this lane's (token pair, group)
        uint32_t vp[2][2] = {{0, 0}, {0, 0}};
        if (lane < 8 * NJ) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t *src = st + o_kp[r] + half + lane % NJ * 4;
            vp[r][0] = *reinterpret_cast<const uint32_t *>(src + vp_tok * NJ * 4);
            vp[r][1] = *reinterpret_cast<const uint32_t *>(src + (vp_tok ^ 1) * NJ * 4);
          }
        }
        if (!full) {
          // what lies in the slots of tokens that nobody sees may be anything
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int ta = tw + 16 * r + f_row, tb = ta + 8;
            const bool seen_a = dc_seen(it, ta), seen_b = dc_seen(it, tb);
            if (!dc_seen(it, tw + 16 * r + vp_tok)) vp[r][0] = 0;
            if (!dc_seen(it, tw + 16 * r + (vp_tok ^ 1))) vp[r][1] = 0;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                bool va = seen_a, vb = seen_b;
                if (MULTI) {
                  va = ta <= pos[nb][c] && (a.window <= 0 || ta > pos[nb][c] - a.window || ta < a.sinks);
                  vb = tb <= pos[nb][c] && (a.window <= 0 || tb > pos[nb][c] - a.window || tb < a.sinks);
                }
                if (!va) x[r][nb][0][c] = -INFINITY;
                if (!vb) x[r][nb][1][c] = -INFINITY;
              }
          }
        }
        // a score past its reference, a V scale past the largest (or a minimum 2^19 times as large), a NaN group
        bool odd = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            odd = odd || fmaxf(fmaxf(x[0][nb][0][c], x[0][nb][1][c]), fmaxf(x[1][nb][0][c], x[1][nb][1][c])) > over[nb][c];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            odd = odd || (int)(vp[r][i] & 0x7FFFu) >= (vexp + 1) << 7 || (int)((vp[r][i] >> 16) & 0x7FFFu) >= (vexp + 20) << 7;
        if (__any_sync(0xffffffffu, odd)) {
          uint32_t bad[2] = {0, 0};   // NaN groups of a 16-token group: bit j (row f_row), NJ + j (row f_row + 8)
          int ve = 0;
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // the NaN of a group reaches the columns that see its token by hand, below; the products get zeros
              const bool mine = ((vp[r][i] >> 7) & 0xFF) == 0xFF || ((vp[r][i] >> 23) & 0xFF) == 0xFF;
              const uint32_t who = __ballot_sync(0xffffffffu, mine);
              const int pair = f_row >> 1;
              // token f_row is entry i of its pair when i matches its place there
              if ((((2 * pair) ^ (pair & 1)) ^ f_row) == i) {
                bad[r] |= (who >> (pair * NJ)) & ((1u << NJ) - 1u);
                bad[r] |= ((who >> ((pair + 4) * NJ)) & ((1u << NJ) - 1u)) << NJ;
              }
              if (mine) vp[r][i] = 0;
              ve = max(ve, max((int)((vp[r][i] >> 7) & 0xFF), (int)((vp[r][i] >> 23) & 0xFF) - 19));
            }
          ve = max(vexp, (int)__reduce_max_sync(0xffffffffu, (uint32_t)ve));
          const int fe = min(122 - ve, 106);              // the largest scale below 2^-4; 2^(fe + 20) in range
          const float vf = vexp < 0 ? 0.f : pow2f(max(fe - fexp, -126));
          vexp = ve;
          fexp = fe;
          up = pow2f(fe >> 1) * pow2f(fe - (fe >> 1));    // down to 2^-132
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(fmaxf(x[0][nb][0][c], x[0][nb][1][c]), fmaxf(x[1][nb][0][c], x[1][nb][1][c]));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              float al = 1.f;
              if (mx > over[nb][c]) {
                mx *= cs[nb][c];
                al = exp2f(m[nb][c] - mx);
                m[nb][c] = mx;
                over[nb][c] = (mx + kAttnSlack) / cs[nb][c];
              }
              l[nb][c] *= al;
              const float of = al * vf;
              uint32_t nan = 0;
#pragma unroll
              for (int r = 0; r < 2; ++r)
                nan |= (x[r][nb][0][c] == -INFINITY ? 0u : bad[r]) | (x[r][nb][1][c] == -INFINITY ? 0u : bad[r] >> NJ);
              nan |= __shfl_xor_sync(0xffffffffu, nan, 4);
              nan |= __shfl_xor_sync(0xffffffffu, nan, 8);
              nan |= __shfl_xor_sync(0xffffffffu, nan, 16);
#pragma unroll
              for (int j = 0; j < 2 * NJ; ++j) {
                const float f = (nan >> (j / 2)) & 1 ? NAN : of;
                o[nb][j][c] *= f, o[nb][j][2 + c] *= f;
              }
            }
        }
        if (lane < 8 * NJ) {
          const float up20 = up * 0x1p20f;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *reinterpret_cast<uint2 *>(vpar + (r * 8 * NJ + lane) * 8) =
                make_uint2(pack_f16x2(bf16_lo_f32(vp[r][0]) * up20, bf16_lo_f32(vp[r][1]) * up20),
                           pack_f16x2(bf16_hi_f32(vp[r][0]) * up, bf16_hi_f32(vp[r][1]) * up));
        }
        // Weights, over the scores.  Those below 2^-24 of the reference would lose their bits in f16: when there are
        // any, they get a pass of their own, 2^32 times larger, into sums that are 2^32 times larger meanwhile.
        uint32_t least = ~0u;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float minus = m[nb][c] == -INFINITY ? 0.f : kAttnLift - m[nb][c];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float w = ex2(fmaf(x[r][nb][h][c], cs[nb][c], minus));
                x[r][nb][h][c] = w;
                l[nb][c] += w;
                least = min(least, __float_as_uint(w) - 1u);   // zeros, and NaN, are large here
              }
          }
        const bool faint = __any_sync(0xffffffffu, least < __float_as_uint(0x1p-17f) - 1u);
        uint32_t b0[2][NB], b1[2][NB];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            float (&w)[2][2] = x[r][nb];
            if (!faint) {
              b0[r][nb] = pack_f16x2(w[0][0], w[0][1]);
              b1[r][nb] = pack_f16x2(w[1][0], w[1][1]);
            } else {
              b0[r][nb] = pack_f16x2(w[0][0] < 0x1p-17f ? 0.f : w[0][0], w[0][1] < 0x1p-17f ? 0.f : w[0][1]);
              b1[r][nb] = pack_f16x2(w[1][0] < 0x1p-17f ? 0.f : w[1][0], w[1][1] < 0x1p-17f ? 0.f : w[1][1]);
            }
            b0[r][nb] = movmatrix(b0[r][nb]);
            b1[r][nb] = movmatrix(b1[r][nb]);
          }
        __syncwarp();
#pragma unroll 1
        for (bool again = faint;; again = false) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t va[NJ / 2], vb[NJ / 2], vc[NJ / 2], vd[NJ / 2];
            const uint8_t *vs = st + o_kc[r] + half + g * NJ * 2;
            lds_words<NJ / 2>(vs + v_tok * (D / 2), va);
            lds_words<NJ / 2>(vs + (v_tok ^ 1) * (D / 2), vb);
            lds_words<NJ / 2>(vs + (v_tok + 8) * (D / 2), vc);
            lds_words<NJ / 2>(vs + ((v_tok + 8) ^ 1) * (D / 2), vd);
#pragma unroll
            for (int jj = 0; jj < NJ; jj += 2) {
              uint32_t pl[4], ph[4];                      // {scale, min} of groups jj, jj + 1: tokens below 8, above
              lds_words<4>(vpar + (r * 8 * NJ + q4 * NJ + jj) * 8, pl);
              lds_words<4>(vpar + (r * 8 * NJ + (q4 + 4) * NJ + jj) * 8, ph);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint32_t r0 = __byte_perm(va[jj / 2], vb[jj / 2], u ? 0x7632 : 0x5410);
                const uint32_t r1 = __byte_perm(vc[jj / 2], vd[jj / 2], u ? 0x7632 : 0x5410);
                uint32_t y[4][2];                         // values 0 .. 3 of the lane's word, tokens below 8 and above
                y[0][0] = hfma2((r0 << 4) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
                y[1][0] = hfma2(r0 & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
                y[2][0] = hfma2((r0 >> 4) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
                y[3][0] = hfma2((r0 >> 8) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
                y[0][1] = hfma2((r1 << 4) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
                y[1][1] = hfma2(r1 & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
                y[2][1] = hfma2((r1 >> 4) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
                y[3][1] = hfma2((r1 >> 8) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                  mma_f16_16816(o[nb][2 * (jj + u)], y[0][0], y[1][0], y[0][1], y[1][1], b0[r][nb], b1[r][nb]);
                  mma_f16_16816(o[nb][2 * (jj + u) + 1], y[2][0], y[3][0], y[2][1], y[3][1], b0[r][nb], b1[r][nb]);
                }
              }
            }
          }
          if (!faint) break;
          const float by = again ? 0x1p32f : 0x1p-32f;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int j = 0; j < 2 * NJ; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nb][j][e] *= by;
            if (again) {
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float u[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                  for (int c = 0; c < 2; ++c) u[h][c] = x[r][nb][h][c] < 0x1p-17f ? x[r][nb][h][c] * 0x1p32f : 0.f;
                b0[r][nb] = movmatrix(pack_f16x2(u[0][0], u[0][1]));
                b1[r][nb] = movmatrix(pack_f16x2(u[1][0], u[1][1]));
              }
            }
          }
          if (!again) break;
        }
      }
      __syncwarp();
      if (ready && lane == 0) mbar_arrive(bar_empty + 8 * slot);
      if (++slot == L::stages) slot = 0, phase ^= 1;
    }

    // ---- this warp's share to shared memory, divided by its weights: these are up to 2^15 each, and their sum of values
    // near the largest number has no 32-bit form
    const float un0 = pow2f(-(fexp >> 1)), un1 = pow2f(-(fexp - (fexp >> 1)));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * nb + 2 * q4 + c;
        float ls = l[nb][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, x);
        if (g == 0) s_m[warp * NC + col] = m[nb][c], s_l[warp * NC + col] = ls;
        const float r = dc_inverse(ls);
#pragma unroll
        for (int j = 0; j < 2 * NJ; ++j)
          *reinterpret_cast<float2 *>(s_o + (warp * NC + col) * D + 32 * (j / 2) + 4 * g + 2 * (j % 2)) =
              make_float2(o[nb][j][c] * r * un0 * un1, o[nb][j][2 + c] * r * un0 * un1);
      }
    dc_sync();

    // ---- the four shares joined: written out, or left for the sequence's last chunk
    const size_t cell = ((size_t)it.b * a.g.heads + it.head) * p.cbs + it.cb;
    constexpr size_t kSlot = (size_t)NC * (D + 2);
    for (int e = tid; e < NC * D / 4; e += 32 * kDcWarps) {
      const int col = e / (D / 4), d = 4 * (e % (D / 4));
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kDcWarps; ++w) top = fmaxf(top, s_m[w * NC + col]);
      float fl[kDcWarps];
#pragma unroll
      for (int w = 0; w < kDcWarps; ++w) {
        fl[w] = (top == -INFINITY ? 1.f : exp2f(s_m[w * NC + col] - top)) * s_l[w * NC + col];
        sum += fl[w];
      }
      const float r = dc_inverse(sum);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kDcWarps; ++w) {
        const float f = fl[w] * r;
        const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * NC + col) * D + d);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      }
      if (it.n_chunks == 1) {
        attn_write4(a, it.first, it.rows_do, it.cb * NC + col, it.head, D, d, acc);
      } else {
        float *dst = p.part + (cell * p.slots + it.chunk) * kSlot;
        __stcg(reinterpret_cast<float4 *>(dst + (size_t)col * D + d), acc);
        if (d == 0) __stcg(reinterpret_cast<float2 *>(dst + (size_t)NC * D + 2 * col), make_float2(top, sum));
      }
    }
    if (it.n_chunks > 1) {
      // the last chunk of a group joins the group, the last group's joiner the row; always in order
      float *cell_part = p.part + cell * p.slots * kSlot;
      int *count = p.count + cell * (kDcGroups + 1);
      const int groups = (it.n_chunks + kDcFan - 1) / kDcFan, grp = it.chunk / kDcFan;
      if (dc_arrive_last(count + 1 + grp, min(kDcFan, it.n_chunks - grp * kDcFan), s_last, tid)) {
        const float *src = cell_part + (size_t)grp * kDcFan * kSlot;
        const int n = min(kDcFan, it.n_chunks - grp * kDcFan);
        if (groups == 1) {
          dc_join<NJ, NB>(src, n, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
            attn_write4(a, it.first, it.rows_do, it.cb * NC + col, it.head, D, d, acc);
          });
        } else {
          float *mid = cell_part + (size_t)p.chunks * kSlot;
          dc_join<NJ, NB>(src, n, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
            float *dst = mid + grp * kSlot;
            __stcg(reinterpret_cast<float4 *>(dst + (size_t)col * D + d), acc);
            if (d == 0) __stcg(reinterpret_cast<float2 *>(dst + (size_t)NC * D + 2 * col), make_float2(top, sum));
          });
          if (dc_arrive_last(count, groups, s_last, tid))
            dc_join<NJ, NB>(mid, groups, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
              attn_write4(a, it.first, it.rows_do, it.cb * NC + col, it.head, D, d, acc);
            });
        }
      }
    }
  }
}

template <int NJ, int NB, bool MULTI>
static int decode_launch(rc_ctx *ctx, DcParams &p, int max_q, cudaStream_t s) {
  using L = DcLayout<NJ, NB>;
  const AttnParams &a = p.a;
  const long long stages = ((long long)a.b.cols * a.g.page + kDcStage - 1) / kDcStage + 1;   // one more: a window cuts two
  p.cbs = (int)(((long long)max_q * a.group + L::cols - 1) / L::cols);
  p.chunks = stages < 2 * kDcMaxChunks * kDcMaxStages ? dc_most_chunks((int)stages) : kDcMaxChunks;
  p.slots = p.chunks + (p.chunks > kDcFan ? dc_ceil(p.chunks, kDcFan) : 0);
  const long long cells = (long long)a.b.n_seqs * a.g.heads * p.cbs;
  RC_CHECK_ARG(cells * (stages + kDcMaxChunks) <= INT_MAX, "rc_kv_attend: the batch is too large");
  int rc = ensure_attn_scratch(ctx, (size_t)cells * p.slots * L::cols * (L::D + 2) * sizeof(float), (size_t)cells * (kDcGroups + 1));
  if (rc) return rc;
  p.part = static_cast<float *>(ctx->attn_part);
  p.count = ctx->attn_count;
  auto kernel = rc_kv_decode_kernel<NJ, NB, MULTI>;
  // CTAs an SM holds, by device and by the batch's share of shared memory
  static std::atomic<int> resident[64][kKvMaxSeqs / 256 + 1];
  const int bucket = a.b.n_seqs / 256, smem = L::bytes(256 * bucket + 255);
  int per_sm = ctx->device < 64 ? resident[ctx->device][bucket].load(std::memory_order_relaxed) : 0;
  if (!per_sm) {
    RC_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmemLimit));
    RC_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kDcThreads, smem));
    RC_CHECK_ARG(per_sm >= 1, "rc_kv_attend: the decode kernel does not fit an SM");
    if (ctx->device < 64) resident[ctx->device][bucket].store(per_sm, std::memory_order_relaxed);
  }
  const long long items = cells * p.chunks, cap = (long long)ctx->sm_count * per_sm;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items < cap ? items : cap));
  cfg.blockDim = dim3(kDcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  RC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
  return RC_OK;
}

int kv_attend_decode(rc_ctx *ctx, const AttnParams &a, int max_q, cudaStream_t s) {
  DcParams p{};
  p.a = a;
  // eight columns when a sequence has no more; sixteen halve the passes over the cache otherwise
  const bool wide = (long long)max_q * a.group > 8, multi = a.b.q_off != nullptr && max_q > 1;
  if (a.g.dim == 128) {
    if (multi) return wide ? decode_launch<4, 2, true>(ctx, p, max_q, s) : decode_launch<4, 1, true>(ctx, p, max_q, s);
    return wide ? decode_launch<4, 2, false>(ctx, p, max_q, s) : decode_launch<4, 1, false>(ctx, p, max_q, s);
  }
  if (multi) return wide ? decode_launch<2, 2, true>(ctx, p, max_q, s) : decode_launch<2, 1, true>(ctx, p, max_q, s);
  return wide ? decode_launch<2, 2, false>(ctx, p, max_q, s) : decode_launch<2, 1, false>(ctx, p, max_q, s);
}

}  // namespace rc

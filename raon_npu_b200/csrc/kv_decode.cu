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
// s = sum_j scale_j * (codes_j . q_j) + min_j * sum(q_j), all in 32 bits.
// Output.  The contraction runs over tokens, so a value's scale cannot be
// applied to the product: V is dequantised to f16 in registers, min + scale *
// code in one rounding (the code again as a subnormal operand of the packed
// multiply-add), and P is f16 too: 2^-12 of a term each, the only roundings
// below 32 bits.  V is brought to about 1 at most by a power of two that follows
// the largest scale seen.  Its codes are read in the transposed fragment order
// by byte permutes of two tokens' words, P is transposed in registers (movmatrix).
// The softmax reference of a column moves only when a score passes it by 8
// (in powers of two), so the sums are rescaled a few times a chunk at most.
//
// Work.  A sequence is cut into chunks of tokens whose size depends on its own
// visible length alone, so a row's bytes do not depend on the batch.  Items
// (sequence, chunk, kv head, column block) are dealt over a persistent grid;
// every CTA finds its items from the device's lengths.  One warp streams 64
// tokens (K and V of one kv head, one bulk copy a page) into a ring of stages,
// four warps take 16 tokens each.  A row of one chunk is written directly;
// else each chunk leaves (maximum, sum, values) in scratch and the last one to
// arrive joins them in chunk order.
#include <limits.h>

#include "kv_attn.cuh"

namespace rc {

constexpr int kDcWarps = 4;                       // computing warps
constexpr int kDcThreads = 32 * (kDcWarps + 1);   // and one that copies
constexpr int kDcStage = 64;                      // tokens of a stage
constexpr int kDcChunk = 256;                     // smallest chunk ...
constexpr int kDcMaxChunk = 1024;                 // ... and the largest that more than 16 of a length are cut for
constexpr int kDcMaxChunks = 128;                 // chunks of a visible length ...
constexpr int kDcChunkSlots = kDcMaxChunks + 3;   // ... and those a window and sinks cut at their ends
constexpr int kDcFan = 16;                        // partial results joined at a time
constexpr int kDcGroups = (kDcChunkSlots + kDcFan - 1) / kDcFan;

struct DcParams {
  AttnParams a;
  int cbs;            // column blocks of max_q rows
  int slots;          // partials of one (sequence, head, column block): its chunks', then its groups'
  float *part;        // [n_seqs][heads][cbs][slots][cols * (D + 2)]
  int *count;         // [n_seqs][heads][cbs][1 + groups] arrivals, zero between launches
};

// What a sequence's items need.
struct DcSeq {
  int first, rows, rows_do, len;   // first row, rows, rows computed (at most max_q), tokens
  int lo, sinks;                   // visible to some row: t >= lo or t < sinks
  int chunk, n_sink, c_lo, n_chunks;
};

__device__ __forceinline__ DcSeq dc_seq(const AttnParams &p, int b) {
  DcSeq s;
  attn_seq(p, b, s.first, s.rows, s.rows_do, s.len);
  s.lo = p.window > 0 ? max(0, s.len - s.rows - p.window + 1) : 0;
  s.sinks = p.window > 0 ? min(p.sinks, s.lo) : 0;
  const int span = s.len - s.lo + s.sinks;
  s.chunk = kDcChunk;
  while (s.chunk < kDcMaxChunk && span > 16 * s.chunk) s.chunk *= 2;
  while (s.chunk < span / kDcMaxChunks + (span % kDcMaxChunks != 0)) s.chunk *= 2;
  s.c_lo = s.lo / s.chunk;
  s.n_sink = min((s.sinks + s.chunk - 1) / s.chunk, s.c_lo);
  s.n_chunks = max(1, s.n_sink + (s.len + s.chunk - 1) / s.chunk - s.c_lo);
  return s;
}

// Stage of tokens t0 .. t0 + 63 holds a visible token.
__device__ __forceinline__ bool dc_stage_visible(const DcSeq &s, int t0) {
  return t0 < s.len && (t0 + kDcStage > s.lo || t0 < s.sinks);
}

__device__ __forceinline__ bool dc_seen(const DcSeq &s, int t) { return t < s.len && (t >= s.lo || t < s.sinks); }

struct DcItem {
  int b, chunk, head, cb;   // chunk: index among the sequence's chunks
};

__device__ __forceinline__ DcItem dc_item(const int *prefix, int n_seqs, int heads, int nc, int i, DcSeq &s,
                                          const AttnParams &p) {
  int lo = 0, hi = n_seqs - 1;   // the last sequence whose first item is <= i
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  DcItem it;
  it.b = lo;
  s = dc_seq(p, lo);
  const int cbs = (s.rows_do * p.group + nc - 1) / nc;
  int r = i - prefix[lo];
  it.cb = r % cbs;
  r /= cbs;
  it.head = r % heads;
  it.chunk = r / heads;
  return it;
}

__device__ __forceinline__ int dc_chunk_start(const DcSeq &s, int i) {
  return (i < s.n_sink ? i : s.c_lo + i - s.n_sink) * s.chunk;
}

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
  static constexpr int stages = NJ == 4 ? (NB == 1 ? 5 : 7) : (NB == 1 ? 8 : 12);
  static constexpr int join = kDcWarps * cols * D * 4;                       // the warps' values of one item
  static_assert(join >= cols * kDcFan * 8, "the joined parts' (reference, sum) lie there too");
  static constexpr int o_scratch = stages * stage;
  static constexpr int o_vpar = o_scratch + join;                         // [warps][8 token pairs][NJ]{scale, min} f16x2
  static constexpr int vpar = 8 * NJ * 8;
  static constexpr int o_ml = o_vpar + kDcWarps * vpar;                      // [2][warps][cols]
  static constexpr int o_bar = o_ml + 2 * kDcWarps * cols * 4;
  static constexpr int o_flags = o_bar + 16 * stages;
  static constexpr int o_prefix = o_flags + 16;
  static int bytes(int n_seqs) { return o_prefix + (n_seqs + 1) * 4; }
};

// The CTA's writes are out; true in every thread of the CTA that arrives last
// of n, which then sees the others' writes (and finds the counter at zero again).
__device__ __forceinline__ bool dc_arrive_last(int *count, int n, volatile int *s_last, int tid) {
  __threadfence();
  dc_sync();
  if (tid == 0) {
    const bool last = atomicAdd(count, 1) == n - 1;
    *s_last = last;
    if (last) *count = 0;
  }
  dc_sync();
  if (!*s_last) return false;
  __threadfence();
  return true;
}

// Joins n <= kDcFan partial results in order; sink(column, value, 4 sums, reference, sum).
template <int NJ, int NB, typename Sink>
__device__ __forceinline__ void dc_join(const float *src, int n, float *scratch, int tid, Sink sink) {
  constexpr int D = 32 * NJ, NC = 8 * NB;
  constexpr size_t kSlot = (size_t)NC * (D + 2);
  float2 *ml = reinterpret_cast<float2 *>(scratch);   // [part][column]
  dc_sync();
  for (int e = tid; e < n * NC; e += 32 * kDcWarps)
    ml[e] = __ldcg(reinterpret_cast<const float2 *>(src + (e / NC) * kSlot + (size_t)NC * D) + e % NC);
  dc_sync();
#pragma unroll 1
  for (int e = tid; e < NC * D / 4; e += 32 * kDcWarps) {
    const int col = e / (D / 4), d = 4 * (e % (D / 4));
    float4 v[kDcFan];
#pragma unroll
    for (int c = 0; c < kDcFan; ++c)
      v[c] = c < n ? __ldcg(reinterpret_cast<const float4 *>(src + c * kSlot + (size_t)col * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    for (int c = 0; c < n; ++c) top = fmaxf(top, ml[c * NC + col].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kDcFan; ++c) {
      if (c >= n) break;
      const float2 x = ml[c * NC + col];
      const float f = top == -INFINITY ? 1.f : exp2f(x.x - top);
      sum = fmaf(f, x.y, sum);
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
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar_full = smem_addr(sm + L::o_bar), bar_empty = bar_full + 8 * L::stages;
  volatile int *abort = reinterpret_cast<volatile int *>(sm + L::o_flags);
  int *s_last = reinterpret_cast<int *>(sm + L::o_flags) + 1;
  int *prefix = reinterpret_cast<int *>(sm + L::o_prefix);
  if (tid == 0) {
    *abort = 0;
    for (int i = 0; i < L::stages; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, kDcWarps);
    }
    mbar_fence_init();
  }
  pdl_launch_dependents();
  pdl_wait_prior();
  // items of every sequence, then their prefix sums
  for (int b = tid; b < a.b.n_seqs; b += kDcThreads) {
    const DcSeq s = dc_seq(a, b);
    prefix[b + 1] = s.n_chunks * a.g.heads * ((s.rows_do * a.group + NC - 1) / NC);
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
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
  const int items = prefix[a.b.n_seqs];
  const int unit = min(a.g.page, kDcStage);              // tokens of one block of a stage
  const int unit_bytes = unit * D * 5 / 4, half = unit_bytes / 2;
  int slot = 0;
  uint32_t phase = 0;                                     // of the ring's current round

  if (warp == kDcWarps) {
    // ------------------------------------------------------------ copies --
    const uint64_t policy = policy_evict_first();
    bool ok = true;
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
      DcSeq s;
      const DcItem it = dc_item(prefix, a.b.n_seqs, a.g.heads, NC, i, s, a);
      const int t_start = dc_chunk_start(s, it.chunk), t_end = min(s.len, t_start + s.chunk);
      for (int t0 = t_start; t0 < t_end && ok; t0 += kDcStage) {
        if (!dc_stage_visible(s, t0)) continue;
        // lane l: page l of the stage (or, of a page larger than a stage, its l-th part)
        const bool whole = a.g.page <= kDcStage;
        const int n = whole ? kDcStage / unit : 4;
        const int t = whole ? t0 + lane * unit : t0;
        bool mine = lane < n && t < s.len && (t + unit > s.lo || t < s.sinks);
        const uint8_t *src = nullptr;
        if (mine) {
          src = kv_head_block(a.g, a.b, it.b, t, it.head, a.err);
          mine = src != nullptr;
        }
        uint32_t bytes = unit_bytes, at = lane * unit_bytes;
        if (!whole) {
          const uint32_t c = kDcStage * D / 2, m = kDcStage * NJ * 4, second = t0 & (a.g.page - 1) ? 1 : 0;
          bytes = lane & 1 ? m : c;
          at = (lane >> 1) * half + (lane & 1) * c;
          if (mine) src += (lane >> 1 ? a.g.vc_off : 0) + (lane & 1 ? a.g.kp_off : 0) + second * bytes;
        }
        ok = attn_wait(bar_empty + 8 * slot, phase ^ 1, abort, a.err);
        if (!ok) break;
        const uint32_t total = __reduce_add_sync(0xffffffffu, mine ? bytes : 0u);
        if (lane == 0) mbar_arrive_expect_tx(bar_full + 8 * slot, total);
        __syncwarp();
        if (mine) bulk_copy_g2s(smem_addr(sm + slot * L::stage + at), src, bytes, bar_full + 8 * slot, policy);
        if (++slot == L::stages) slot = 0, phase ^= 1;
      }
    }
    if (!ok) {
      // copies in flight land before the CTA leaves; the slots not yet reused are waited for, each with a limit
      for (int i = 0; i < L::stages; ++i) {
        const int k = (slot + i) % L::stages;
        const uint32_t ph = k < slot ? phase : phase ^ 1;
        mbar_wait_bounded_warp(bar_full + 8 * k, ph);
      }
    }
    return;
  }

  // --------------------------------------------------------------- compute --
  const int g = lane >> 2, q4 = lane & 3;
  const int f_row = g ^ ((g >> 1) & 1);                  // token of row g among 8 (spreads V's rows over the banks)
  const int sub = 16 * warp / unit, within = 16 * warp % unit;
  const int o_kc = sub * unit_bytes + within * (D / 2), o_kp = sub * unit_bytes + unit * (D / 2) + within * NJ * 4;
  const int v_tok = 2 * q4 ^ (q4 & 1);                   // tokens v_tok and v_tok ^ 1 are columns 2 q4 and 2 q4 + 1
  const int vp_tok = 2 * (lane / NJ % 8) ^ (lane / NJ & 1);   // of lane = pair * NJ + group: the pair's first token
  uint8_t *vpar = sm + L::o_vpar + warp * L::vpar;
  float *s_o = reinterpret_cast<float *>(sm + L::o_scratch);
  float *s_m = reinterpret_cast<float *>(sm + L::o_ml), *s_l = s_m + kDcWarps * NC;

  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    DcSeq s;
    const DcItem it = dc_item(prefix, a.b.n_seqs, a.g.heads, NC, i, s, a);
    const int t_start = dc_chunk_start(s, it.chunk), t_end = min(s.len, t_start + s.chunk);

    // query columns: column 8 nb + g of this lane's B fragments
    uint32_t qb[NB][2 * NJ][2];
    float qs[NB][NJ][2], cs[NB][2];                      // group sums and score scales of columns 8 nb + 2 q4, + 1
    int pos[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int flat = it.cb * NC + 8 * nb + g, qi = attn_row(a, flat);
      uint4 w[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) w[j] = make_uint4(0, 0, 0, 0);
      if (qi < s.rows_do) {
        const uint16_t *src = a.q + (size_t)(s.first + qi) * a.ldq + (it.head * a.group + flat - qi * a.group) * D + 8 * q4;
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
      const float mul = pow2f(sh);
      float gs[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float x[8] = {bf16_lo_f32(w[j].x) * mul, bf16_hi_f32(w[j].x) * mul, bf16_lo_f32(w[j].y) * mul,
                            bf16_hi_f32(w[j].y) * mul, bf16_lo_f32(w[j].z) * mul, bf16_hi_f32(w[j].z) * mul,
                            bf16_lo_f32(w[j].w) * mul, bf16_hi_f32(w[j].w) * mul};
        qb[nb][2 * j][0] = pack_f16x2(x[0], x[4]);
        qb[nb][2 * j][1] = pack_f16x2(x[1] * 0.0625f, x[5] * 0.0625f);
        qb[nb][2 * j + 1][0] = pack_f16x2(x[2], x[6]);
        qb[nb][2 * j + 1][1] = pack_f16x2(x[3] * 0.0625f, x[7] * 0.0625f);
        gs[j] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        gs[j] += __shfl_xor_sync(0xffffffffu, gs[j], 1);
        gs[j] += __shfl_xor_sync(0xffffffffu, gs[j], 2);
        gs[j] *= 0x1p-24f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * q4 + c), col = it.cb * NC + 8 * nb + 2 * q4 + c;
#pragma unroll
        for (int j = 0; j < NJ; ++j) qs[nb][j][c] = __shfl_sync(0xffffffffu, gs[j], from);
        cs[nb][c] = pow2f(-__shfl_sync(0xffffffffu, sh, from)) * 0x1p24f * a.scale_log2;
        const int ci = attn_row(a, col);
        pos[nb][c] = ci < s.rows_do ? s.len - s.rows + ci : -1;
      }
    }

    float o[NB][2 * NJ][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int c = 0; c < 2; ++c) m[nb][c] = -INFINITY, l[nb][c] = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * NJ; ++j) o[nb][j][0] = o[nb][j][1] = o[nb][j][2] = o[nb][j][3] = 0.f;
    }
    int vexp = -1;      // exponent field of the largest V scale so far; V's f16 carry 2^fexp
    int fexp = 0;

    for (int t0 = t_start; t0 < t_end; t0 += kDcStage) {
      if (!dc_stage_visible(s, t0)) continue;
      const bool ready = attn_wait(bar_full + 8 * slot, phase, abort, a.err);
      const int tw = t0 + 16 * warp;                     // this warp's 16 tokens
      if (ready && tw < s.len && (tw + 16 > s.lo || tw < s.sinks)) {
        const uint8_t *st = sm + slot * L::stage;
        bool full = tw + 15 <= s.len - s.rows && (tw + 15 < s.sinks || tw >= (MULTI ? max(s.lo, s.len - a.window) : s.lo));
        if (MULTI && a.window <= 0) full = tw + 15 <= s.len - s.rows;
        const int ta = tw + f_row, tb = ta + 8;

        // scores of rows f_row, f_row + 8 in columns 2 q4, 2 q4 + 1
        float x[NB][2][2];
        {
          uint32_t k0[NJ], k1[NJ], p0[NJ], p1[NJ];
          lds_words<NJ>(st + o_kc + f_row * (D / 2) + q4 * NJ * 4, k0);
          lds_words<NJ>(st + o_kc + (f_row + 8) * (D / 2) + q4 * NJ * 4, k1);
          lds_words<NJ>(st + o_kp + f_row * NJ * 4, p0);
          lds_words<NJ>(st + o_kp + (f_row + 8) * NJ * 4, p1);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) x[nb][0][0] = x[nb][0][1] = x[nb][1][0] = x[nb][1][1] = 0.f;
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const float sc0 = bf16_lo_f32(p0[j]), mn0 = bf16_hi_f32(p0[j]);
            const float sc1 = bf16_lo_f32(p1[j]), mn1 = bf16_hi_f32(p1[j]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float d[4];
              mma_f16_16816_zero(d, k0[j] & 0x000F000Fu, k1[j] & 0x000F000Fu, k0[j] & 0x00F000F0u, k1[j] & 0x00F000F0u,
                                 qb[nb][2 * j][0], qb[nb][2 * j][1]);
              mma_f16_16816(d, (k0[j] >> 8) & 0x000F000Fu, (k1[j] >> 8) & 0x000F000Fu, (k0[j] >> 8) & 0x00F000F0u,
                            (k1[j] >> 8) & 0x00F000F0u, qb[nb][2 * j + 1][0], qb[nb][2 * j + 1][1]);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                x[nb][0][c] = fmaf(sc0, d[c], fmaf(mn0, qs[nb][j][c], x[nb][0][c]));
                x[nb][1][c] = fmaf(sc1, d[2 + c], fmaf(mn1, qs[nb][j][c], x[nb][1][c]));
              }
            }
          }
        }
        // V params of this lane's (token pair, group)
        uint32_t vp[2] = {0, 0};
        if (lane < 8 * NJ) {
          const uint8_t *src = st + o_kp + half + lane % NJ * 4;
          vp[0] = *reinterpret_cast<const uint32_t *>(src + vp_tok * NJ * 4);
          vp[1] = *reinterpret_cast<const uint32_t *>(src + (vp_tok ^ 1) * NJ * 4);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) x[nb][0][c] *= cs[nb][c], x[nb][1][c] *= cs[nb][c];
        if (!full) {
          // what lies in the slots of tokens that nobody sees may be anything
          const bool seen_a = dc_seen(s, ta), seen_b = dc_seen(s, tb);
          if (!dc_seen(s, tw + vp_tok)) vp[0] = 0;
          if (!dc_seen(s, tw + (vp_tok ^ 1))) vp[1] = 0;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              bool va = seen_a, vb = seen_b;
              if (MULTI) {
                va = ta <= pos[nb][c] && (a.window <= 0 || ta > pos[nb][c] - a.window || ta < a.sinks);
                vb = tb <= pos[nb][c] && (a.window <= 0 || tb > pos[nb][c] - a.window || tb < a.sinks);
              }
              if (!va) x[nb][0][c] = -INFINITY;
              if (!vb) x[nb][1][c] = -INFINITY;
            }
        }
        bool over = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) over = over || fmaxf(x[nb][0][c], x[nb][1][c]) > m[nb][c] + kAttnSlack;
        // exponents: of the scales, and of minima more than 2^19 times as large
        int ve = 0;
        bool poison = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int se = (vp[i] >> 7) & 0xFF, me = (vp[i] >> 23) & 0xFF;
          poison = poison || se == 0xFF || me == 0xFF;
          ve = max(ve, max(se, me - 19));
        }
        over = over || ve > vexp || poison;
        uint32_t bad = 0;   // NaN groups: bit j (row f_row), NJ + j (row f_row + 8)
        if (__any_sync(0xffffffffu, over)) {
          if (__any_sync(0xffffffffu, poison)) {
            // the NaN of a group reaches the columns that see its token by hand, below; the products get zeros
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool mine = ((vp[i] >> 7) & 0xFF) == 0xFF || ((vp[i] >> 23) & 0xFF) == 0xFF;
              const uint32_t who = __ballot_sync(0xffffffffu, mine);
              const int tok = f_row, pair = f_row >> 1;
              // token f_row is entry i of its pair when i matches its place there
              if ((((2 * pair) ^ (pair & 1)) ^ tok) == i) {
                bad |= (who >> (pair * NJ)) & ((1u << NJ) - 1u);
                bad |= ((who >> ((pair + 4) * NJ)) & ((1u << NJ) - 1u)) << NJ;
              }
              if (mine) vp[i] = 0;
            }
            ve = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) ve = max(ve, max((int)((vp[i] >> 7) & 0xFF), (int)((vp[i] >> 23) & 0xFF) - 19));
          }
          ve = max(vexp, (int)__reduce_max_sync(0xffffffffu, (uint32_t)ve));
          const int fe = min(122 - ve, 106);            // the largest scale below 2^-4; 2^(fe + 20) in range
          const float vf = vexp < 0 ? 0.f : pow2f(max(fe - fexp, -126));
          vexp = ve;
          fexp = fe;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float mx = fmaxf(x[nb][0][c], x[nb][1][c]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              float al = 1.f;
              if (mx > m[nb][c] + kAttnSlack) {
                al = exp2f(m[nb][c] - mx);
                m[nb][c] = mx;
              }
              l[nb][c] *= al;
              const float of = al * vf;
              uint32_t nan = (x[nb][0][c] == -INFINITY ? 0u : bad) | (x[nb][1][c] == -INFINITY ? 0u : bad >> NJ);
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
        float w[NB][2][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float ref = m[nb][c] == -INFINITY ? 0.f : m[nb][c] - kAttnLift;
            w[nb][0][c] = ex2(x[nb][0][c] - ref);
            w[nb][1][c] = ex2(x[nb][1][c] - ref);
            l[nb][c] += w[nb][0][c] + w[nb][1][c];
          }
        if (lane < 8 * NJ) {
          const float up = pow2f(fexp >> 1) * pow2f(fexp - (fexp >> 1)), up20 = up * 0x1p20f;   // 2^fexp: down to 2^-132
          *reinterpret_cast<uint2 *>(vpar + lane * 8) =
              make_uint2(pack_f16x2(bf16_lo_f32(vp[0]) * up20, bf16_lo_f32(vp[1]) * up20),
                         pack_f16x2(bf16_hi_f32(vp[0]) * up, bf16_hi_f32(vp[1]) * up));
        }
        // Weights below 2^-24 of the reference would lose their bits in f16: when there are any, they get a second
        // pass of their own, 2^32 times larger, into sums that are 2^32 times larger meanwhile.
        uint32_t b0[NB], b1[NB];
        bool faint = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            faint = faint || (w[nb][0][c] < 0x1p-17f && w[nb][0][c] > 0.f) || (w[nb][1][c] < 0x1p-17f && w[nb][1][c] > 0.f);
        faint = __any_sync(0xffffffffu, faint);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float u[2][2];
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) u[r][c] = faint && w[nb][r][c] < 0x1p-17f ? 0.f : w[nb][r][c];
          b0[nb] = movmatrix(pack_f16x2(u[0][0], u[0][1]));
          b1[nb] = movmatrix(pack_f16x2(u[1][0], u[1][1]));
        }
        __syncwarp();
        uint32_t va[(NJ + 1) / 2], vb[(NJ + 1) / 2], vc[(NJ + 1) / 2], vd[(NJ + 1) / 2];
        lds_words<NJ / 2>(st + o_kc + half + v_tok * (D / 2) + g * NJ * 2, va);
        lds_words<NJ / 2>(st + o_kc + half + (v_tok ^ 1) * (D / 2) + g * NJ * 2, vb);
        lds_words<NJ / 2>(st + o_kc + half + (v_tok + 8) * (D / 2) + g * NJ * 2, vc);
        lds_words<NJ / 2>(st + o_kc + half + ((v_tok + 8) ^ 1) * (D / 2) + g * NJ * 2, vd);
#pragma unroll 1
        for (bool again = faint;; again = false) {
#pragma unroll
        for (int jj = 0; jj < NJ; jj += 2) {
          uint32_t pl[4], ph[4];                          // {scale, min} of groups jj, jj + 1: tokens below 8, above
          lds_words<4>(vpar + (q4 * NJ + jj) * 8, pl);
          lds_words<4>(vpar + ((q4 + 4) * NJ + jj) * 8, ph);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t r0 = __byte_perm(va[jj / 2], vb[jj / 2], u ? 0x7632 : 0x5410);
            const uint32_t r1 = __byte_perm(vc[jj / 2], vd[jj / 2], u ? 0x7632 : 0x5410);
            uint32_t v[4][2];                             // values 0 .. 3 of the lane's word, tokens below 8 and above
            v[0][0] = hfma2((r0 << 4) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
            v[1][0] = hfma2(r0 & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
            v[2][0] = hfma2((r0 >> 4) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
            v[3][0] = hfma2((r0 >> 8) & 0x00F000F0u, pl[2 * u], pl[2 * u + 1]);
            v[0][1] = hfma2((r1 << 4) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
            v[1][1] = hfma2(r1 & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
            v[2][1] = hfma2((r1 >> 4) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
            v[3][1] = hfma2((r1 >> 8) & 0x00F000F0u, ph[2 * u], ph[2 * u + 1]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              mma_f16_16816(o[nb][2 * (jj + u)], v[0][0], v[1][0], v[0][1], v[1][1], b0[nb], b1[nb]);
              mma_f16_16816(o[nb][2 * (jj + u) + 1], v[2][0], v[3][0], v[2][1], v[3][1], b0[nb], b1[nb]);
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
            float u[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
              for (int c = 0; c < 2; ++c) u[r][c] = w[nb][r][c] < 0x1p-17f ? w[nb][r][c] * 0x1p32f : 0.f;
            b0[nb] = movmatrix(pack_f16x2(u[0][0], u[0][1]));
            b1[nb] = movmatrix(pack_f16x2(u[1][0], u[1][1]));
          }
        }
        if (!again) break;
        }
      }
      __syncwarp();
      if (ready && lane == 0) mbar_arrive(bar_empty + 8 * slot);
      if (++slot == L::stages) slot = 0, phase ^= 1;
    }

    // ---- this warp's share to shared memory
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
#pragma unroll
        for (int j = 0; j < 2 * NJ; ++j)
          *reinterpret_cast<float2 *>(s_o + (warp * NC + col) * D + 32 * (j / 2) + 4 * g + 2 * (j % 2)) =
              make_float2(o[nb][j][c] * un0 * un1, o[nb][j][2 + c] * un0 * un1);
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
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kDcWarps; ++w) {
        const float mw = s_m[w * NC + col], f = mw == top && top == -INFINITY ? 1.f : exp2f(mw - top);
        const float4 v = *reinterpret_cast<const float4 *>(s_o + (w * NC + col) * D + d);
        sum = fmaf(f, s_l[w * NC + col], sum);
        acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
      }
      if (s.n_chunks == 1) {
        attn_write4(a, s.first, s.rows_do, it.cb * NC + col, it.head, D, d, acc, sum);
      } else {
        float *dst = p.part + (cell * p.slots + it.chunk) * kSlot;
        __stcg(reinterpret_cast<float4 *>(dst + (size_t)col * D + d), acc);
        if (d == 0) __stcg(reinterpret_cast<float2 *>(dst + (size_t)NC * D + 2 * col), make_float2(top, sum));
      }
    }
    if (s.n_chunks > 1) {
      // the last chunk of a group joins the group, the last group's joiner the row; always in order
      float *cell_part = p.part + cell * p.slots * kSlot;
      int *count = p.count + cell * (kDcGroups + 1);
      const int groups = (s.n_chunks + kDcFan - 1) / kDcFan, grp = it.chunk / kDcFan;
      if (dc_arrive_last(count + 1 + grp, min(kDcFan, s.n_chunks - grp * kDcFan), s_last, tid)) {
        const float *src = cell_part + (size_t)grp * kDcFan * kSlot;
        const int n = min(kDcFan, s.n_chunks - grp * kDcFan);
        if (groups == 1) {
          dc_join<NJ, NB>(src, n, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
            attn_write4(a, s.first, s.rows_do, it.cb * NC + col, it.head, D, d, acc, sum);
          });
        } else {
          float *mid = cell_part + (size_t)(p.slots - kDcGroups) * kSlot;
          dc_join<NJ, NB>(src, n, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
            float *dst = mid + grp * kSlot;
            __stcg(reinterpret_cast<float4 *>(dst + (size_t)col * D + d), acc);
            if (d == 0) __stcg(reinterpret_cast<float2 *>(dst + (size_t)NC * D + 2 * col), make_float2(top, sum));
          });
          if (dc_arrive_last(count, groups, s_last, tid))
            dc_join<NJ, NB>(mid, groups, s_o, tid, [&](int col, int d, float4 acc, float top, float sum) {
              attn_write4(a, s.first, s.rows_do, it.cb * NC + col, it.head, D, d, acc, sum);
            });
        }
      }
    }
    dc_sync();   // the scratch is the next item's
  }
}

template <int NJ, int NB, bool MULTI>
static int decode_launch(rc_ctx *ctx, DcParams &p, int max_q, cudaStream_t s) {
  using L = DcLayout<NJ, NB>;
  const AttnParams &a = p.a;
  const long long max_len = (long long)a.b.cols * a.g.page, chunks = (max_len + kDcChunk - 1) / kDcChunk;
  p.cbs = (int)(((long long)max_q * a.group + L::cols - 1) / L::cols);
  p.slots = (int)(chunks < kDcChunkSlots ? chunks : kDcChunkSlots) + kDcGroups;
  const long long cells = (long long)a.b.n_seqs * a.g.heads * p.cbs;
  RC_CHECK_ARG(cells * p.slots <= INT_MAX, "rc_kv_attend: the batch is too large");
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
  const long long items = cells * p.slots, cap = (long long)ctx->sm_count * per_sm;
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

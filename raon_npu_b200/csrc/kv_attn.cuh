// What the attention kernels over the 4-bit KV cache share.
#pragma once

#include <atomic>

#include "kv_internal.cuh"

namespace rc {

constexpr float kAttnSlack = 8.f;   // how far a score may pass a row's softmax reference, log2
constexpr float kAttnLift = 7.f;    // weights are 2^(score - reference + lift): at most 2^15

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// a * b + c in f16, one rounding; subnormal operands are exact.
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// 2^x to 2 ulp of 32 bits; results below 2^-126 are zero.
__device__ __forceinline__ float ex2(float x) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
  return d;
}
// Words from shared memory, in loads of up to 16 bytes.
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t *p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
}

// A wait for a phase of an mbarrier that gives up after about a second of
// clock cycles, or when another warp has (``abort``), so that every role runs
// to its end: by one thread, and by a warp with one verdict for all lanes.
__device__ __forceinline__ bool attn_wait1(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  bool there = mbar_try_wait(bar, parity);
  if (!there) {
    const uint32_t t0 = (uint32_t)clock();
    while (!(there = mbar_try_wait(bar, parity))) {
      if ((uint32_t)clock() - t0 > 2000000000u) {
        *abort = 1;
        atomicCAS(err, 0, kErrWaitTimeout);
      }
      if (*abort) break;
    }
  }
  return there;
}
__device__ __forceinline__ bool attn_wait(uint32_t bar, uint32_t parity, volatile int *abort, int *err) {
  return __all_sync(0xffffffffu, attn_wait1(bar, parity, abort, err));
}

struct AttnParams {
  KvGeom g;
  KvBatchDev b;
  const uint16_t *q;
  int ldq, group;        // query heads of a kv head
  FastDiv by_group;
  int max_q;
  float scale_log2;      // scale * log2(e): scores are in powers of two
  int window, sinks;
  uint16_t *out;
  int ldo;
  int *turns;            // items claimed by a prompt call, CTAs that are done; zero between calls
  int *err;
};

// Rows of a sequence and kv head are numbered row * group + head in the group;
// within these limits FastDiv is exact.
constexpr int kAttnMaxGroup = 256;
constexpr long long kAttnMaxFlat = 1 << 24;
__device__ __forceinline__ int attn_row(const AttnParams &p, int flat) { return (int)fdiv((uint32_t)flat, p.by_group); }

// First row, rows and tokens of a sequence; rows_do: the rows that are
// computed.  Values that do not fit the buffers set the error word and are cut.
__device__ __forceinline__ void attn_seq(const AttnParams &p, int b, int &first, int &rows, int &rows_do, int &len) {
  len = __ldcg(p.b.kv_len + b);
  first = b;
  rows = 1;
  bool bad = false;
  if (p.b.q_off) {
    first = __ldcg(p.b.q_off + b);
    const int end = __ldcg(p.b.q_off + b + 1);
    rows = end - first;
    if (first < 0 || end < first || end > p.b.n_rows) bad = true, rows = 0;
  }
  rows_do = rows;
  if (rows > p.max_q) bad = true, rows_do = p.max_q;
  const long long room = (long long)p.b.cols << p.g.log2_page;
  if (len > room) bad = true, len = (int)room;
  if (len < 0) len = 0;
  if (bad) atomicCAS(p.err, 0, kErrKvRange);
}

// First token of the window of the row at ``pos``, which may be negative (an
// empty row) and the window anything up to the largest int: no sum of the two.
__device__ __forceinline__ int attn_window_lo(const AttnParams &p, int pos) {
  return p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
}

// Values d .. d+3 of query column ``flat`` (row * group + head in the group)
// of a sequence.
__device__ __forceinline__ void attn_write4(const AttnParams &p, int first, int rows_do, int flat, int head, int D, int d,
                                            float4 v) {
  const int qi = attn_row(p, flat);
  if (qi >= rows_do) return;
  uint16_t *dst = p.out + (size_t)(first + qi) * p.ldo + (head * p.group + flat - qi * p.group) * D + d;
  *reinterpret_cast<uint2 *>(dst) =
      make_uint2(f32_to_bf16_rne(v.x) | ((uint32_t)f32_to_bf16_rne(v.y) << 16),
                 f32_to_bf16_rne(v.z) | ((uint32_t)f32_to_bf16_rne(v.w) << 16));
}

int kv_attend_decode(rc_ctx *ctx, const AttnParams &a, int max_q, cudaStream_t s);   // kv_decode.cu
int kv_attend_prompt(rc_ctx *ctx, const AttnParams &a, cudaStream_t s);              // kv_prompt.cu

}  // namespace rc

// What the attention kernels over the 4-bit KV cache share.
#pragma once

#include "kv_internal.cuh"

namespace rc {

struct AttnParams {
  KvGeom g;
  KvBatchDev b;
  const uint16_t *q;
  int ldq, group;        // query heads of a kv head
  int max_q;
  float scale_log2;      // scale * log2(e): scores are in powers of two
  int window, sinks;
  uint16_t *out;
  int ldo;
  int *err;
};

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

// Values d .. d+3 of query column ``flat`` (row * group + head in the group)
// of a sequence: acc / sum, zeros when nothing was seen.
__device__ __forceinline__ void attn_write4(const AttnParams &p, int first, int rows_do, int flat, int head, int D, int d,
                                            float4 acc, float sum) {
  const int qi = flat / p.group;
  if (qi >= rows_do) return;
  const float r = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t *dst = p.out + (size_t)(first + qi) * p.ldo + (head * p.group + flat % p.group) * D + d;
  *reinterpret_cast<uint2 *>(dst) =
      make_uint2(f32_to_bf16_rne(acc.x * r) | ((uint32_t)f32_to_bf16_rne(acc.y * r) << 16),
                 f32_to_bf16_rne(acc.z * r) | ((uint32_t)f32_to_bf16_rne(acc.w * r) << 16));
}

int kv_attend_decode(rc_ctx *ctx, const AttnParams &a, int max_q, cudaStream_t s);   // kv_decode.cu

}  // namespace rc

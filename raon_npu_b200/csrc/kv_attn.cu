// Attention over the paged 4-bit KV cache.
//
//   s_t = scale * q . k_t,  o = sum_t softmax_t(s) v_t   over the visible t
//
// One CTA per (row, query head): each warp takes every fourth visible token,
// keeps the running maximum, sum and weighted values of its share in 32 bits,
// and the four shares are joined at the end.
#include <limits.h>

#include "kv_internal.cuh"

namespace rc {

constexpr int kAttnWarps = 4;

struct AttnParams {
  KvGeom g;
  KvBatchDev b;
  const uint16_t *q;
  int ldq, q_heads;
  float scale;
  int window, sinks;
  uint16_t *out;
  int ldo;
  int *err;
};

template <int E>
__device__ __forceinline__ void row_values(const uint8_t *codes, uint32_t par, float (&v)[E]) {
  const float sc = bf16_lo_f32(par), mn = bf16_hi_f32(par);
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    v[2 * i] = fmaf(sc, (float)(codes[i] & 15), mn);
    v[2 * i + 1] = fmaf(sc, (float)(codes[i] >> 4), mn);
  }
}

template <int E>
__global__ void __launch_bounds__(32 * kAttnWarps) rc_kv_attend_kernel(const __grid_constant__ AttnParams p) {
  constexpr int D = 32 * E, NJ = D / kKvGroup;
  __shared__ float s_m[kAttnWarps], s_l[kAttnWarps], s_o[kAttnWarps][D];
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d0 = lane * E;
  const int r = blockIdx.x, h = blockIdx.y, kvh = h / (p.q_heads / p.g.heads);
  int seq, pos;
  if (!kv_find_row(p.b, r, lane, seq, pos)) return;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = bf16_to_f32(p.q[(size_t)r * p.ldq + h * D + d0 + e]), o[e] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;       // first token of the window
  const int sinks = p.window > 0 ? min(p.sinks, lo) : 0;
  const int n = pos < 0 ? 0 : sinks + pos + 1 - lo;
  for (int i = warp; i < n; i += kAttnWarps) {
    const int t = i < sinks ? i : lo + i - sinks;
    const uint8_t *blk = kv_head_block(p.g, p.b, seq, t, kvh, p.err);
    if (!blk) continue;
    const int tp = t & (p.g.page - 1);
    float k[E], v[E];
    row_values<E>(blk + (size_t)tp * (D / 2) + kv_k_byte(d0, NJ),
                  reinterpret_cast<const uint32_t *>(blk + p.g.kp_off)[tp * NJ + d0 / kKvGroup], k);
    row_values<E>(blk + p.g.vc_off + (size_t)tp * (D / 2) + kv_v_byte(d0, NJ),
                  reinterpret_cast<const uint32_t *>(blk + p.g.vp_off)[tp * NJ + d0 / kKvGroup], v);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= p.scale;
    const float mn = fmaxf(m, s), a = m == mn ? 1.f : expf(m - mn), w = expf(s - mn);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * v[e];
    m = mn;
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][d0 + e] = o[e];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_m[w]);
  float f[kAttnWarps];
  for (int w = 0; w < kAttnWarps; ++w) {
    f[w] = s_m[w] == -INFINITY && s_l[w] == 0.f ? 0.f : expf(s_m[w] - top);
    total += f[w] * s_l[w];
  }
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float acc = 0.f;
    for (int w = 0; w < kAttnWarps; ++w) acc += f[w] * s_o[w][d];
    p.out[(size_t)r * p.ldo + h * D + d] = n > 0 ? f32_to_bf16_rne(acc / total) : 0;
  }
}

}  // namespace rc

using namespace rc;

extern "C" int rc_kv_attend(rc_kv *kv, int layer, const uint16_t *q_dev, int ldq, int q_heads, int n_rows,
                            const int32_t *table_dev, int cols, int ld_table,
                            const int32_t *kv_len_dev, const int32_t *q_off_dev, int n_seqs, int max_q, float scale, int window, int sinks,
                            uint16_t *out_dev, int ldo, void *stream) {
  RC_CHECK_ARG(kv && q_dev && out_dev, "rc_kv_attend: NULL argument");
  int rc = kv_check_batch("rc_kv_attend", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(q_heads >= kv->heads && q_heads % kv->heads == 0 && q_heads <= 4096,
               "rc_kv_attend: %d query heads over %d kv heads", q_heads, kv->heads);
  RC_CHECK_ARG(max_q >= 1, "rc_kv_attend: max_q %d", max_q);
  RC_CHECK_ARG(ldq >= q_heads * kv->dim && ldo >= q_heads * kv->dim, "rc_kv_attend: rows of %d and %d values, %d are needed",
               ldq, ldo, q_heads * kv->dim);
  RC_CHECK_ARG(ldq % 8 == 0 && ldo % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(out_dev)) & 15) == 0,
               "rc_kv_attend: rows must start on 16-byte boundaries");
  RC_CHECK_ARG(scale == scale && window >= 0 && sinks >= 0, "rc_kv_attend: scale must be a number, window and sinks not negative");
  if (n_rows == 0 || n_seqs == 0) return RC_OK;
  RC_CUDA_TRY(cudaSetDevice(kv->ctx->device));
  AttnParams p{};
  p.g = kv_geom(kv, layer);
  p.b = KvBatchDev{table_dev, kv_len_dev, q_off_dev, cols, ld_table, n_seqs, n_rows};
  p.q = q_dev;
  p.ldq = ldq;
  p.q_heads = q_heads;
  p.scale = scale;
  p.window = window;
  p.sinks = sinks;
  p.out = out_dev;
  p.ldo = ldo;
  p.err = kv->ctx->err;
  const dim3 grid(n_rows, q_heads);
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  if (kv->dim == 128) rc_kv_attend_kernel<4><<<grid, 32 * kAttnWarps, 0, s>>>(p);
  else rc_kv_attend_kernel<2><<<grid, 32 * kAttnWarps, 0, s>>>(p);
  RC_CUDA_TRY(cudaGetLastError());
  return RC_OK;
}

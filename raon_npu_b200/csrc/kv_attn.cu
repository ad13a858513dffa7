// Attention over the paged 4-bit KV cache: the entry point.
#include "kv_attn.cuh"

using namespace rc;

// Rows of a sequence and kv head above which a call goes to the tensor-memory
// kernel.  The decode kernel reads the cache once per 16 rows, split over as many
// CTAs as there are; the other one once per 256, by one CTA a kv head.  Which is
// faster turns on the number of sequences and kv heads, and a row's bytes must not,
// so the rule is on the rows alone.  us, decode / prompt, 4096 tokens, heads of 128:
//               1 sequence, 4 kv heads   1, 16 kv heads   8, 4 kv heads   8, 16 kv heads
//    16 rows           16.8 / 57.3         19.2 / 58.0      20.0 / 58.6      57.3 / 60.5
//    32 rows           17.8 / 57.5         19.8 / 57.9      32.5 / 58.7      95.1 / 60.9
//    64 rows           19.2 / 57.5         32.2 / 58.1      57.7 / 59.0     182.8 / 61.4
//   128 rows           19.7 / 58.0         57.4 / 58.5      93.0 / 59.8     360.4 / 63.0
//   256 rows           32.1 / 67.0         93.3 / 68.2     179.4 / 69.6     710.0 / 74.2
//  1024 rows           92.7 / 67.8        358.5 / 69.5     700.7 / 73.1    2832.9 / 248.5
// 255 favours single sequences and few heads (two to three times faster up to there)
// at the price of batches: they cross at 64 rows for 8 sequences of 4 kv heads, at 16
// for 8 of 16, which lose near ten times just below the limit.  The decode kernel also
// keeps weights below 2^-31 of the largest.
constexpr long long kPromptRows = 255;

extern "C" int rc_kv_attend(rc_kv *kv, int layer, const uint16_t *q_dev, int ldq, int q_heads, int n_rows,
                            const int32_t *table_dev, int cols, int ld_table,
                            const int32_t *kv_len_dev, const int32_t *q_off_dev, int n_seqs, int max_q, float scale, int window, int sinks,
                            uint16_t *out_dev, int ldo, void *stream) {
  RC_CHECK_ARG(kv && ((q_dev && out_dev) || n_rows == 0), "rc_kv_attend: NULL argument");
  int rc = kv_check_batch("rc_kv_attend", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(q_heads >= kv->heads && q_heads % kv->heads == 0 && q_heads <= 4096,
               "rc_kv_attend: %d query heads over %d kv heads", q_heads, kv->heads);
  RC_CHECK_ARG(max_q >= 1, "rc_kv_attend: max_q %d", max_q);
  const int group = q_heads / kv->heads;
  RC_CHECK_ARG(group <= kAttnMaxGroup && (long long)max_q * group <= kAttnMaxFlat,
               "rc_kv_attend: %d query heads a kv head (at most %d), %d rows a sequence (rows x heads at most %lld)", group,
               kAttnMaxGroup, max_q, kAttnMaxFlat);
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
  p.group = group;
  p.by_group = make_fastdiv((uint32_t)group);
  p.max_q = q_off_dev ? max_q : 1;
  p.scale_log2 = scale * 1.44269504088896340736f;
  p.window = window;
  p.sinks = sinks;
  p.out = out_dev;
  p.ldo = ldo;
  p.turns = kv->ctx->attn_turns;
  p.err = kv->ctx->err;
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  return (long long)p.max_q * p.group > kPromptRows ? kv_attend_prompt(kv->ctx, p, s) : kv_attend_decode(kv->ctx, p, p.max_q, s);
}

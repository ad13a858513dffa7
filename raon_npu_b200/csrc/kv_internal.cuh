// Definitions shared by the KV cache translation units: the pool's geometry,
// the batch description and the arithmetic of one cached row.
#pragma once
#include <limits.h>


#include "rc_device.cuh"
#include "rc_internal.cuh"

struct rc_kv {
  rc_ctx *ctx;
  int layers, pages, heads, dim, page, log2_page;
  uint8_t *pool;
  int owned;             // the pool is this cache's own allocation
  size_t head_bytes, page_bytes, layer_bytes;
};

namespace rc {

constexpr int kKvGroup = 32;        // values per (scale, min)
constexpr int kKvMaxSeqs = 4096;    // sequences of one batch

// The calls of a step are chained by programmatic dependent launch, so a
// neighbour's CTA may have filled this SM's L1 with lines that the previous
// call rewrote: whatever earlier calls write (tables, lengths, queries, the
// cache) is read past L1 (ld.cg, bulk copies).

// One layer of a pool.  A head block: K codes, K params, V codes, V params.
struct KvGeom {
  uint8_t *base;
  int pages, heads, dim, page, log2_page;
  uint32_t head_bytes, kp_off, vc_off, vp_off;
  size_t page_bytes;
};

struct KvBatchDev {
  const int32_t *table;
  const int32_t *kv_len;
  const int32_t *q_off;   // null: one row per sequence
  int cols, ld;           // entries and stride of a table row
  int n_seqs, n_rows;
};

inline KvGeom kv_geom(const rc_kv *kv, int layer) {
  KvGeom g;
  g.base = kv->pool + (size_t)layer * kv->layer_bytes;
  g.pages = kv->pages;
  g.heads = kv->heads;
  g.dim = kv->dim;
  g.page = kv->page;
  g.log2_page = kv->log2_page;
  g.head_bytes = (uint32_t)kv->head_bytes;
  g.kp_off = (uint32_t)(kv->page * kv->dim / 2);
  g.vc_off = (uint32_t)(kv->head_bytes / 2);
  g.vp_off = g.vc_off + g.kp_off;
  g.page_bytes = kv->page_bytes;
  return g;
}

int kv_check_batch(const char *what, const rc_kv *kv, int layer, int n_rows, const int32_t *table, int cols, int ld,
                   const int32_t *kv_len, const int32_t *q_off, int n_seqs);   // kv_cache.cu

// Sequence and position of row r, found by one warp together (every lane gets
// the answer).  False for a row of no sequence.
__device__ __forceinline__ bool kv_find_row(const KvBatchDev &b, int r, int lane, int &seq, int &pos) {
  if (!b.q_off) {
    if (r >= b.n_seqs) return false;
    seq = r;
    pos = __ldcg(b.kv_len + r) - 1;
    return true;
  }
  int last_len = 0;                 // of the window before
  for (int k0 = 0; k0 <= b.n_seqs; k0 += 32) {
    const int k = k0 + lane, off = k <= b.n_seqs ? __ldcg(b.q_off + k) : INT_MAX, len = k < b.n_seqs ? __ldcg(b.kv_len + k) : 0;
    const unsigned m = __ballot_sync(0xffffffffu, k <= b.n_seqs && off <= r);
    if (m != 0xffffffffu) {
      const int n = __popc(m);      // offsets of this window <= r
      seq = k0 + n - 1;
      if (seq < 0 || seq >= b.n_seqs) return false;
      const int hi = __shfl_sync(0xffffffffu, off, n);
      pos = __shfl_sync(0xffffffffu, len, (n - 1) & 31);
      pos = (n ? pos : last_len) - hi + r;
      return true;
    }
    last_len = __shfl_sync(0xffffffffu, len, 31);
  }
  return false;
}

// Head block of (page of position pos, head); null, with the error word set,
// when the position lies outside the table or the page outside the pool.
__device__ __forceinline__ uint8_t *kv_head_block(const KvGeom &g, const KvBatchDev &b, int seq, int pos, int head,
                                                  int *err) {
  const int pi = pos >> g.log2_page;
  const int id = pi < b.cols ? __ldcg(b.table + (size_t)seq * b.ld + pi) : -1;
  if (id < 0 || id >= g.pages) {
    atomicCAS(err, 0, kErrKvRange);
    return nullptr;
  }
  return g.base + (size_t)id * g.page_bytes + (size_t)head * g.head_bytes;
}

// Byte of a K or V row that holds value d in its nibble d % 2.
__device__ __forceinline__ int kv_k_byte(int d, int nj) { return (((d % 32) / 8) * nj + d / 32) * 4 + (d % 8) / 2; }
__device__ __forceinline__ int kv_v_byte(int d, int nj) { return (((d % 32) / 4) * nj + d / 32) * 2 + (d % 4) / 2; }

}  // namespace rc

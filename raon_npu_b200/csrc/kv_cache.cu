// The paged 4-bit KV cache: its pool, the append of new rows (head norms,
// rotation, quantisation), the read-back and the page moves.
#include <limits.h>

#include "kv_internal.cuh"

namespace rc {

// ----------------------------------------------------------------- append --
// A warp takes some heads of one row (``per_warp``: one when there are few
// rows, up to eight when there are many, so that the row's position, its rotation
// and the norm weights are fetched once for all of them); a lane holds E = D / 32
// consecutive values, the next head's come in while this one is computed.
// Bound by memory: about 10 operations a value.  Query heads are computed in 32
// bits and rounded once to bf16.  Key heads are computed and quantised in 64
// bits (a code on the other side of a rounding boundary is off by a whole step);
// the FP64 work of one head in q_heads / kv_heads + 2 hides under the loads.
// Value heads are taken as they come, so their codes are found in 32 bits and
// only those near a boundary in 64.
constexpr int kKvWarps = 8;
constexpr int kAppendMaxHeads = 8;

struct AppendParams {
  KvGeom g;
  KvBatchDev b;
  const void *x;
  int ldx, q_heads;
  const uint16_t *q_norm, *k_norm;
  float eps;
  const float *rope;
  int rope_rows, rope_dim, interleaved;
  uint16_t *q_out;
  int ldq;
  int per_warp, parts;   // heads of a warp, warps of a row
  int *err;
};

template <int E, bool F32>
__device__ __forceinline__ void load_lane(const void *x, size_t at, float (&v)[E]) {
  if constexpr (F32) {
    const float *p = static_cast<const float *>(x) + at;
    if constexpr (E == 4) {
      const float4 w = __ldcg(reinterpret_cast<const float4 *>(p));
      v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
      const float2 w = __ldcg(reinterpret_cast<const float2 *>(p));
      v[0] = w.x, v[1] = w.y;
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(x) + at;
    if constexpr (E == 4) {
      const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(p));
      v[0] = bf16_lo_f32(w.x), v[1] = bf16_hi_f32(w.x), v[2] = bf16_lo_f32(w.y), v[3] = bf16_hi_f32(w.y);
    } else {
      const uint32_t w = __ldcg(reinterpret_cast<const uint32_t *>(p));
      v[0] = bf16_lo_f32(w), v[1] = bf16_hi_f32(w);
    }
  }
}

__device__ __forceinline__ float inv_sqrt(float v) { return 1.f / sqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// A lane's part of the rotation of a row: cos and sin of its values' pairs.
template <int E>
struct RopeLane {
  float c[E], s[E];   // of value e; interleaved pairs use the even entries
  int half;           // rope_dim / 2; 0: no rotation

  __device__ __forceinline__ void load(const float *row, int rd, bool interleaved, int lane) {
    half = rd / 2;
    const int d0 = lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = interleaved ? (d0 + e) / 2 : d0 + e < half ? d0 + e : d0 + e - half;
      c[e] = d0 < rd ? row[i] : 1.f;
      s[e] = d0 < rd ? row[half + i] : 0.f;
    }
  }
};

// RMS norm of a head with the lane's weights w (norm: whether there are any), then the rotation of its first values.
template <int E, typename T>
__device__ __forceinline__ void norm_rope(T (&v)[E], bool norm, const float (&w)[E], float eps, const RopeLane<E> &rope,
                                          bool interleaved, int lane) {
  if (norm) {
    T ss = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) ss += v[e] * v[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T r = inv_sqrt(ss / (T)(32 * E) + (T)eps);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] * r * (T)w[e];
  }
  if (!rope.half) return;
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const T c = rope.c[e], s = rope.s[e], a = v[e], b = v[e + 1];
      v[e] = a * c - b * s;
      v[e + 1] = a * s + b * c;
    }
  } else {
    const int off = rope.half / E;   // lanes between the two values of a pair (rope_dim is a multiple of 8)
    const bool first = lane < off, second = !first && lane < 2 * off;
    const int partner = first ? lane + off : second ? lane - off : lane;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const T other = __shfl_sync(0xffffffffu, v[e], partner), c = rope.c[e], s = rope.s[e];
      if (first) v[e] = v[e] * c - other * s;
      if (second) v[e] = v[e] * c + other * s;
    }
  }
}

// The q4nx group rule in 64 bits: {scale, min} of a group from its extremes.  False when it has no finite form.
__device__ __forceinline__ bool group_scale(double lo, double hi, float &sc, float &mn) {
  mn = bf16_floor_f32(__double2float_rd(lo));
  const double base = (double)mn, span = hi - base;
  sc = bf16_ceil_f64(span / 15.0);
  if (isfinite(sc) && base + 15.0 * (double)sc < hi) sc = bf16_next_up(sc);   // one step covers the rounding of the quotient
  if (span == 0.0) sc = 0.f;
  return isfinite(sc) && isfinite(mn);
}
__device__ __forceinline__ uint32_t group_code(double v, double base, float sc) {
  const double q = sc > 0.f ? rint((v - base) / (double)sc) : 0.0;
  return (uint32_t)(q < 0.0 ? 0.0 : q > 15.0 ? 15.0 : q);
}

// Codes of a lane's values and the group's {scale, min}, over the 32 / E lanes of a group; a group without a finite
// form becomes {0, NaN} (and false is returned).  T = float: the codes in 32 bits, which are those of 64 unless the
// quotient lies within 1e-3 of a boundary or the numbers are extreme.
template <int E, typename T>
__device__ __forceinline__ bool quantise_group(const T (&v)[E], uint32_t (&code)[E], uint32_t &param) {
  constexpr int kLanes = kKvGroup / E;
  bool fine = true;
  T lo = v[0], hi = v[0];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    fine = fine && isfinite(v[e]);
    lo = v[e] < lo ? v[e] : lo;
    hi = v[e] > hi ? v[e] : hi;
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    const T a = __shfl_xor_sync(0xffffffffu, lo, o), b = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  const int lane = threadIdx.x & 31;
  const unsigned mine = ((1u << kLanes) - 1u) << (lane & ~(kLanes - 1));
  fine = (__ballot_sync(0xffffffffu, fine) & mine) == mine;
  float sc, mn;
  fine = group_scale((double)lo, (double)hi, sc, mn) && fine;
  const T inv = sc > 0.f ? (T)1 / (T)sc : (T)0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const T d = v[e] - (T)mn, t = d * inv, q = rint(t);
    const T near = sizeof(T) == 4 ? (T)1e-3 : (T)1e-6;   // of a boundary: the exact quotient decides
    const bool sure = fabs(fabs(t - q) - (T)0.5) > near && (sizeof(T) == 8 || (fabs(d) < (T)1e38 && sc > 1e-30f));
    code[e] = sure ? (uint32_t)(q < (T)0 ? (T)0 : q > (T)15 ? (T)15 : q) : 0u;
    if (!sure) code[e] = group_code((double)v[e], (double)mn, sc);
    if (!fine) code[e] = 0u;
  }
  param = fine ? (__float_as_uint(sc) >> 16) | (__float_as_uint(mn) & 0xFFFF0000u) : 0x7FC00000u;
  return fine;
}

template <int E, bool F32>
__global__ void __launch_bounds__(32 * kKvWarps) rc_kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int D = 32 * E, NJ = D / kKvGroup;
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x & 31, d0 = lane * E;
  const int n_heads = p.q_heads + 2 * p.g.heads;
  const long long item = (long long)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
  const int r = (int)(item / p.parts), h0 = (int)(item - (long long)r * p.parts) * p.per_warp;
  const int h1 = min(h0 + p.per_warp, n_heads);
  if (r >= p.b.n_rows) return;
  const size_t x_at = (size_t)r * p.ldx + d0;
  float next[E];
  load_lane<E, F32>(p.x, x_at + (size_t)h0 * D, next);
  float wq[E], wk[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    wq[e] = p.q_norm && h0 < p.q_heads ? bf16_to_f32(p.q_norm[d0 + e]) : 1.f;
    wk[e] = p.k_norm && h1 > p.q_heads ? bf16_to_f32(p.k_norm[d0 + e]) : 1.f;
  }
  int seq, pos;
  if (!kv_find_row(p.b, r, lane, seq, pos)) return;
  RopeLane<E> rope;
  rope.half = 0;
  if (p.rope && pos >= 0 && h0 < p.q_heads + p.g.heads) {
    if (pos >= p.rope_rows) {
      if (lane == 0) atomicCAS(p.err, 0, kErrKvRange);
      return;
    }
    rope.load(p.rope + (size_t)pos * p.rope_dim, p.rope_dim, p.interleaved, lane);
  }
  uint8_t *page = h1 > p.q_heads && pos >= 0 ? kv_head_block(p.g, p.b, seq, pos, 0, p.err) : nullptr;
  const int t = pos & (p.g.page - 1);
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = next[e];
    if (h + 1 < h1) load_lane<E, F32>(p.x, x_at + (size_t)(h + 1) * D, next);
    if (h < p.q_heads) {
      norm_rope<E, float>(x, p.q_norm != nullptr, wq, p.eps, rope, p.interleaved, lane);
      uint16_t *out = p.q_out + (size_t)r * p.ldq + h * D + d0;
      uint32_t w[E / 2];
#pragma unroll
      for (int e = 0; e < E; e += 2)
        w[e / 2] = f32_to_bf16_rne(x[e]) | ((uint32_t)f32_to_bf16_rne(x[e + 1]) << 16);
      if constexpr (E == 4) *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t *>(out) = w[0];
      continue;
    }
    if (!page) return;
    const bool is_v = h >= p.q_heads + p.g.heads;
    uint32_t code[E], param;
    bool fine;
    if (is_v) {
      fine = quantise_group<E, float>(x, code, param);
    } else {
      double k[E];
#pragma unroll
      for (int e = 0; e < E; ++e) k[e] = x[e];
      norm_rope<E, double>(k, p.k_norm != nullptr, wk, p.eps, rope, p.interleaved, lane);
      fine = quantise_group<E, double>(k, code, param);
    }
    if (!fine) atomicCAS(p.err, 0, kErrKvNonFinite);
    uint8_t *blk = page + (size_t)(h - p.q_heads - (is_v ? p.g.heads : 0)) * p.g.head_bytes;
    uint8_t *codes = blk + (is_v ? p.g.vc_off : 0) + t * (D / 2) + (is_v ? kv_v_byte(d0, NJ) : kv_k_byte(d0, NJ));
    if constexpr (E == 4)
      *reinterpret_cast<uint16_t *>(codes) = (uint16_t)(code[0] | (code[1] << 4) | (code[2] << 8) | (code[3] << 12));
    else
      *codes = (uint8_t)(code[0] | (code[1] << 4));
    if (d0 % kKvGroup == 0)
      reinterpret_cast<uint32_t *>(blk + (is_v ? p.g.vp_off : p.g.kp_off))[t * NJ + d0 / kKvGroup] = param;
  }
}

// ------------------------------------------------------------------- read --
// One warp per (row, kv head, K or V): min + scale * code in 32 bits (one
// rounding: scale * code is exact), rounded to bf16.
template <int E>
__global__ void __launch_bounds__(32 * kKvWarps)
    rc_kv_read_kernel(const __grid_constant__ KvGeom g, const __grid_constant__ KvBatchDev b, uint16_t *k_out,
                      uint16_t *v_out, int *err) {
  constexpr int D = 32 * E, NJ = D / kKvGroup;
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x & 31, d0 = lane * E;
  const long long item = (long long)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
  const int r = (int)(item / (2 * g.heads)), i = (int)(item - (long long)r * 2 * g.heads);
  const int kv = i >= g.heads ? 1 : 0, h = i - kv * g.heads;
  if (r >= b.n_rows) return;
  int seq, pos;
  if (!kv_find_row(b, r, lane, seq, pos)) return;
  const uint8_t *blk = pos >= 0 ? kv_head_block(g, b, seq, pos, h, err) : nullptr;
  const int t = pos & (g.page - 1);
  uint32_t w[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) w[e] = 0;
  if (blk) {
    const uint8_t *codes = blk + (kv ? g.vc_off : 0) + t * (D / 2) + (kv ? kv_v_byte(d0, NJ) : kv_k_byte(d0, NJ));
    const uint32_t par = __ldcg(reinterpret_cast<const uint32_t *>(blk + (kv ? g.vp_off : g.kp_off)) + t * NJ + d0 / kKvGroup);
    uint32_t nib;
    if constexpr (E == 4) nib = __ldcg(reinterpret_cast<const uint16_t *>(codes));
    else nib = __ldcg(codes);
    const float sc = bf16_lo_f32(par), mn = bf16_hi_f32(par);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      const float a = fmaf(sc, (float)(nib >> (8 * e) & 15), mn), c = fmaf(sc, (float)(nib >> (8 * e + 4) & 15), mn);
      w[e] = f32_to_bf16_rne(a) | ((uint32_t)f32_to_bf16_rne(c) << 16);
    }
  }
  uint16_t *out = (kv ? v_out : k_out) + ((size_t)r * g.heads + h) * D + d0;
  if constexpr (E == 4) *reinterpret_cast<uint2 *>(out) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t *>(out) = w[0];
}

// ------------------------------------------------------------- page moves --
// Copy blocks move kMoveChunk bytes of one page of one layer; table blocks
// rewrite table entries through a hash of the moves in shared memory, built
// kMoveHash moves at a time (a destination is never a source, so one pass's
// new entries are left alone by the next).
constexpr int kMoveThreads = 256;
constexpr int kMoveChunk = 16384;
constexpr int kMoveHash = 2048;
constexpr int kMoveSlots = 2 * kMoveHash;
constexpr int kMoveEntries = 4096;   // table entries per block

struct MoveParams {
  uint8_t *pool;
  size_t layer_bytes, page_bytes;
  int pages, n, chunks;
  const int32_t *src, *dst;
  int32_t *table;
  int rows, cols, ld;
  int *err;
};

__device__ __forceinline__ uint32_t move_slot(int id) { return ((uint32_t)id * 2654435761u) >> 20; }   // 12 bits
static_assert(kMoveSlots == 4096, "move_slot gives 12 bits");

__global__ void __launch_bounds__(kMoveThreads) rc_kv_move_kernel(const __grid_constant__ MoveParams p) {
  __shared__ int keys[kMoveSlots], vals[kMoveSlots];
  pdl_launch_dependents();
  pdl_wait_prior();
  const int copies = p.n * p.chunks;
  if ((int)blockIdx.x < copies) {
    const int m = blockIdx.x / p.chunks, c = blockIdx.x % p.chunks;
    const int src = __ldcg(p.src + m), dst = __ldcg(p.dst + m);
    if ((unsigned)src >= (unsigned)p.pages || (unsigned)dst >= (unsigned)p.pages) {
      if (threadIdx.x == 0) atomicCAS(p.err, 0, kErrKvRange);
      return;
    }
    uint8_t *layer = p.pool + (size_t)blockIdx.y * p.layer_bytes;
    const size_t at = (size_t)c * kMoveChunk;
    const uint4 *a = reinterpret_cast<const uint4 *>(layer + (size_t)src * p.page_bytes + at);
    uint4 *b = reinterpret_cast<uint4 *>(layer + (size_t)dst * p.page_bytes + at);
    const int n16 = (int)((p.page_bytes - at < kMoveChunk ? p.page_bytes - at : kMoveChunk) / 16);
    constexpr int kPer = kMoveChunk / 16 / kMoveThreads;
    uint4 v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = threadIdx.x + i * kMoveThreads;
      if (k < n16) v[i] = __ldcg(a + k);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = threadIdx.x + i * kMoveThreads;
      if (k < n16) __stcs(b + k, v[i]);
    }
    return;
  }
  if (blockIdx.y) return;
  const long long e0 = (long long)((int)blockIdx.x - copies) * kMoveEntries, total = (long long)p.rows * p.cols;
  for (int m0 = 0; m0 < p.n; m0 += kMoveHash) {
    for (int i = threadIdx.x; i < kMoveSlots; i += kMoveThreads) keys[i] = -1;
    __syncthreads();
    for (int m = m0 + threadIdx.x; m < p.n && m < m0 + kMoveHash; m += kMoveThreads) {
      const int src = __ldcg(p.src + m), dst = __ldcg(p.dst + m);
      if ((unsigned)src >= (unsigned)p.pages || (unsigned)dst >= (unsigned)p.pages) continue;
      uint32_t s = move_slot(src);
      while (atomicCAS(keys + s, -1, src) != -1) s = (s + 1) % kMoveSlots;   // at most half full
      vals[s] = dst;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kMoveEntries && e0 + i < total; i += kMoveThreads) {
      int32_t *e = p.table + (e0 + i) / p.cols * p.ld + (e0 + i) % p.cols;
      const int id = __ldcg(e);
      if (id < 0) continue;
      for (uint32_t s = move_slot(id); keys[s] != -1; s = (s + 1) % kMoveSlots)
        if (keys[s] == id) {
          *e = vals[s];
          break;
        }
    }
    __syncthreads();
  }
}

int kv_check_batch(const char *what, const rc_kv *kv, int layer, int n_rows, const int32_t *table, int cols, int ld,
                   const int32_t *kv_len, const int32_t *q_off, int n_seqs) {
  RC_CHECK_ARG(layer >= 0 && layer < kv->layers, "%s: layer %d of %d", what, layer, kv->layers);
  RC_CHECK_ARG(table && kv_len, "%s: NULL table or kv_len", what);
  RC_CHECK_ARG(n_seqs >= 0 && n_seqs <= kKvMaxSeqs, "%s: %d sequences (0..%d)", what, n_seqs, kKvMaxSeqs);
  RC_CHECK_ARG(n_rows >= 0, "%s: %d rows", what, n_rows);
  RC_CHECK_ARG(q_off || n_rows == n_seqs, "%s: %d rows for %d sequences without q_off", what, n_rows, n_seqs);
  RC_CHECK_ARG(cols >= 1 && ld >= cols, "%s: a table of %d columns, stride %d", what, cols, ld);
  return RC_OK;
}

template <typename... Args>
static int launch(void (*kernel)(Args...), dim3 grid, dim3 block, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  RC_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return RC_OK;
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace rc

using namespace rc;

extern "C" {

int rc_kv_pool_bytes(int layers, int pages, int kv_heads, int head_dim, int page_size, size_t *out) {
  RC_CHECK_ARG(out, "rc_kv_pool_bytes: out is NULL");
  *out = 0;
  RC_CHECK_ARG(layers >= 1 && pages >= 1 && kv_heads >= 1, "KV cache: layers (%d), pages (%d) and kv_heads (%d) must be positive",
               layers, pages, kv_heads);
  RC_CHECK_ARG(layers <= 65535 && kv_heads <= 1024, "KV cache: at most 65535 layers and 1024 kv heads");
  RC_CHECK_ARG(head_dim == 64 || head_dim == 128, "KV cache: head_dim is 64 or 128, not %d", head_dim);
  RC_CHECK_ARG(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128,
               "KV cache: page_size is 16, 32, 64 or 128, not %d", page_size);
  const size_t page = (size_t)kv_heads * page_size * head_dim * 5 / 4;
  RC_CHECK_ARG((size_t)pages <= SIZE_MAX / page / (size_t)layers, "KV cache: the pool's size overflows");
  *out = page * (size_t)pages * (size_t)layers;
  return RC_OK;
}

int rc_kv_create(rc_ctx *ctx, int layers, int pages, int kv_heads, int head_dim, int page_size, void *pool_dev,
                 size_t pool_bytes, rc_kv **out) {
  RC_CHECK_ARG(ctx && out, "rc_kv_create: NULL argument");
  *out = nullptr;
  size_t need = 0;
  int rc = rc_kv_pool_bytes(layers, pages, kv_heads, head_dim, page_size, &need);
  if (rc) return rc;
  RC_CHECK_ARG(!pool_dev || pool_bytes >= need, "rc_kv_create: the pool has %zu bytes, %zu are needed", pool_bytes, need);
  RC_CHECK_ARG(aligned16(pool_dev), "rc_kv_create: the pool must be 16-byte aligned");
  RC_CUDA_TRY(cudaSetDevice(ctx->device));
  rc_kv *kv = static_cast<rc_kv *>(calloc(1, sizeof(rc_kv)));
  if (!kv) {
    set_error("rc_kv_create: out of host memory");
    return RC_ERR_CUDA;
  }
  kv->ctx = ctx;
  kv->layers = layers;
  kv->pages = pages;
  kv->heads = kv_heads;
  kv->dim = head_dim;
  kv->page = page_size;
  while ((1 << kv->log2_page) < page_size) ++kv->log2_page;
  kv->head_bytes = (size_t)page_size * head_dim * 5 / 4;
  kv->page_bytes = kv->head_bytes * kv_heads;
  kv->layer_bytes = kv->page_bytes * pages;
  kv->pool = static_cast<uint8_t *>(pool_dev);
  if (!pool_dev) {
    cudaError_t e = cudaMalloc(&kv->pool, need);
    if (e != cudaSuccess) {
      free(kv);
      set_error("rc_kv_create: %s (%zu bytes)", cudaGetErrorString(e), need);
      return RC_ERR_CUDA;
    }
    kv->owned = 1;
  }
  *out = kv;
  return RC_OK;
}

int rc_kv_destroy(rc_kv *kv) {
  if (!kv) return RC_OK;
  cudaSetDevice(kv->ctx->device);
  if (kv->owned) {
    cudaDeviceSynchronize();   // calls may sit on caller streams
    cudaFree(kv->pool);
  }
  free(kv);
  return RC_OK;
}

int rc_kv_append(rc_kv *kv, int layer, const void *x_dev, int x_dtype, int ldx, int q_heads, int n_rows,
                 const int32_t *table_dev, int cols, int ld_table, const int32_t *kv_len_dev,
                 const int32_t *q_off_dev, int n_seqs, const uint16_t *q_norm_dev, const uint16_t *k_norm_dev, float eps,
                 const float *rope_dev, int rope_rows, int rope_dim, int interleaved, uint16_t *q_out_dev, int ldq,
                 void *stream) {
  RC_CHECK_ARG(kv && x_dev, "rc_kv_append: NULL argument");
  int rc = kv_check_batch("rc_kv_append", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(x_dtype == RC_DTYPE_BF16 || x_dtype == RC_DTYPE_F32, "rc_kv_append: unknown dtype %d", x_dtype);
  RC_CHECK_ARG(q_heads >= 0 && q_heads <= 4096, "rc_kv_append: %d query heads", q_heads);
  RC_CHECK_ARG(q_heads == 0 || q_out_dev, "rc_kv_append: q_out is NULL");
  const long long width = (long long)(q_heads + 2 * kv->heads) * kv->dim;
  RC_CHECK_ARG(ldx >= width, "rc_kv_append: rows of %d values, %lld are needed", ldx, width);
  RC_CHECK_ARG(q_heads == 0 || ldq >= q_heads * kv->dim, "rc_kv_append: q_out rows of %d values, %d are needed", ldq,
               q_heads * kv->dim);
  RC_CHECK_ARG(ldx % 8 == 0 && ldq % 8 == 0 && aligned16(x_dev) && aligned16(q_out_dev),
               "rc_kv_append: rows must start on 16-byte boundaries");
  RC_CHECK_ARG(!rope_dev || (rope_rows >= 1 && rope_dim >= 8 && rope_dim <= kv->dim && rope_dim % 8 == 0),
               "rc_kv_append: rope_dim %d must be a multiple of 8 up to head_dim (and rope_rows, %d, positive)", rope_dim,
               rope_rows);
  RC_CHECK_ARG(eps >= 0.f, "rc_kv_append: eps must not be negative");
  if (n_rows == 0 || n_seqs == 0) return RC_OK;
  RC_CUDA_TRY(cudaSetDevice(kv->ctx->device));
  AppendParams p{};
  p.g = kv_geom(kv, layer);
  p.b = KvBatchDev{table_dev, kv_len_dev, q_off_dev, cols, ld_table, n_seqs, n_rows};
  p.x = x_dev;
  p.ldx = ldx;
  p.q_heads = q_heads;
  p.q_norm = q_norm_dev;
  p.k_norm = k_norm_dev;
  p.eps = eps;
  p.rope = rope_dev;
  p.rope_rows = rope_rows;
  p.rope_dim = rope_dim;
  p.interleaved = interleaved;
  p.q_out = q_out_dev;
  p.ldq = ldq;
  p.err = kv->ctx->err;
  // as many heads a warp as leave 64 warps an SM
  const int heads = q_heads + 2 * kv->heads;
  const long long spare = (long long)n_rows * heads / (64ll * kv->ctx->sm_count);
  p.per_warp = spare < 1 ? 1 : spare < kAppendMaxHeads ? (int)spare : kAppendMaxHeads;
  p.parts = (heads + p.per_warp - 1) / p.per_warp;
  const long long blocks = ((long long)n_rows * p.parts + kKvWarps - 1) / kKvWarps;
  RC_CHECK_ARG(blocks <= INT_MAX, "rc_kv_append: too many rows (%d)", n_rows);
  const dim3 grid((unsigned)blocks), block(32 * kKvWarps);
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  const bool f32 = x_dtype == RC_DTYPE_F32;
  if (kv->dim == 128) return f32 ? launch(rc_kv_append_kernel<4, true>, grid, block, s, p) : launch(rc_kv_append_kernel<4, false>, grid, block, s, p);
  return f32 ? launch(rc_kv_append_kernel<2, true>, grid, block, s, p) : launch(rc_kv_append_kernel<2, false>, grid, block, s, p);
}

int rc_kv_read(rc_kv *kv, int layer, int n_rows, const int32_t *table_dev, int cols, int ld_table,
               const int32_t *kv_len_dev, const int32_t *q_off_dev, int n_seqs, uint16_t *k_out_dev, uint16_t *v_out_dev, void *stream) {
  RC_CHECK_ARG(kv && k_out_dev && v_out_dev, "rc_kv_read: NULL argument");
  int rc = kv_check_batch("rc_kv_read", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(aligned16(k_out_dev) && aligned16(v_out_dev), "rc_kv_read: buffers must be 16-byte aligned");
  if (n_rows == 0 || n_seqs == 0) return RC_OK;
  RC_CUDA_TRY(cudaSetDevice(kv->ctx->device));
  const KvGeom g = kv_geom(kv, layer);
  const KvBatchDev b{table_dev, kv_len_dev, q_off_dev, cols, ld_table, n_seqs, n_rows};
  const long long blocks = ((long long)n_rows * 2 * kv->heads + kKvWarps - 1) / kKvWarps;
  RC_CHECK_ARG(blocks <= INT_MAX, "rc_kv_read: too many rows (%d)", n_rows);
  const dim3 grid((unsigned)blocks), block(32 * kKvWarps);
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  return kv->dim == 128 ? launch(rc_kv_read_kernel<4>, grid, block, s, g, b, k_out_dev, v_out_dev, kv->ctx->err)
                        : launch(rc_kv_read_kernel<2>, grid, block, s, g, b, k_out_dev, v_out_dev, kv->ctx->err);
}

int rc_kv_move_pages(rc_kv *kv, const int32_t *src_dev, const int32_t *dst_dev, int n, int32_t *table_dev, int rows,
                     int cols, int ld_table, void *stream) {
  RC_CHECK_ARG(kv, "rc_kv_move_pages: NULL cache");
  RC_CHECK_ARG(n >= 0 && n <= kv->pages, "rc_kv_move_pages: %d moves in a pool of %d pages", n, kv->pages);
  RC_CHECK_ARG(!table_dev || (rows >= 0 && cols >= 0 && ld_table >= cols), "rc_kv_move_pages: bad table shape [%d][%d], stride %d",
               rows, cols, ld_table);
  if (n == 0) return RC_OK;
  RC_CHECK_ARG(src_dev && dst_dev, "rc_kv_move_pages: NULL moves");
  RC_CUDA_TRY(cudaSetDevice(kv->ctx->device));
  MoveParams p{};
  p.pool = kv->pool;
  p.layer_bytes = kv->layer_bytes;
  p.page_bytes = kv->page_bytes;
  p.pages = kv->pages;
  p.n = n;
  p.chunks = (int)((kv->page_bytes + kMoveChunk - 1) / kMoveChunk);
  p.src = src_dev;
  p.dst = dst_dev;
  p.table = table_dev;
  p.rows = rows;
  p.cols = cols;
  p.ld = ld_table;
  p.err = kv->ctx->err;
  const long long entries = table_dev ? (long long)rows * cols : 0;
  const long long blocks = (long long)n * p.chunks + (entries + kMoveEntries - 1) / kMoveEntries;
  RC_CHECK_ARG(blocks <= INT_MAX, "rc_kv_move_pages: too many moves (%d)", n);
  return launch(rc_kv_move_kernel, dim3((unsigned)blocks, (unsigned)kv->layers), dim3(kMoveThreads),
                pick_stream(kv->ctx, stream), p);
}

}  // extern "C"

// The paged 4-bit KV cache: its pool, the append of new rows (head norms,
// rotation, quantisation), the read-back and the page moves.
#include <limits.h>

#include "kv_internal.cuh"

namespace rc {

// ----------------------------------------------------------------- append --
// A lane holds 8 consecutive values, so a warp holds 256 / D heads (a unit).  A
// warp takes units of one row: one when there are few rows, up to four, all
// asked for at once, when there are many, so that the row's position, its
// rotation and the norm weights are fetched once for all of them and enough
// loads are in flight.  Query
// heads are computed in 32 bits and rounded once to bf16.  Key heads are
// normalised, rotated and scaled in 64 bits (a code on the other side of a
// rounding boundary is off by a whole step), value heads are taken as they come;
// the codes of both are found in 32 bits and those near a boundary once more in
// 64.  A block is one warp, so that the room of a short one (queries) is free
// before a long one (keys) ends: with the read-back below, 4096 rows of 32 + 4 + 4
// heads of 128 took 47 us so, with blocks of two warps 50 and of eight 65.
// Measured: those rows in 30 us (86 MB in and out: 2.9 TB/s, 45% of the copy rate)
// and 10 for the read-back; 16 rows of a decode step in 5.3 us with it.  Neither
// memory (15% of its cycles) nor issue (0.60 a cycle, 250 instructions for a unit of
// 256 values) is full: 19 warps an SM do not cover the latency of a unit's steps, the
// 64-bit ones above all, and with few rows that of four dependent loads: the row's
// sequence, its page and rotation, the values.  The forms for f32 rows spill 72 bytes
// a thread (in 80 registers).
constexpr int kAppendUnits = 4, kAppendCtas = 24;

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
  int units_q, units_kv;       // units of a warp
  int parts_q, parts;          // warps for the queries of a row, for the row
  int *err;
};

template <bool F32>
struct Raw8 {
  uint4 a, b;   // 8 bf16 in a, or 8 f32
  __device__ __forceinline__ void load(const void *x, size_t at) {
    if constexpr (F32) {
      a = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const float *>(x) + at));
      b = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const float *>(x) + at) + 1);
    } else {
      a = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + at));
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (F32) {
      const uint32_t u[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]), v[4 + i] = __uint_as_float(u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo_f32(w[i]), v[2 * i + 1] = bf16_hi_f32(w[i]);
    }
  }
};

__device__ __forceinline__ uint32_t bf16x2_rn(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint4 bf16x8_rn(const float (&v)[8]) {
  return make_uint4(bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3]), bf16x2_rn(v[4], v[5]), bf16x2_rn(v[6], v[7]));
}

__device__ __forceinline__ float inv_sqrt(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return rsqrt(v); }

// A lane's part of the rotation of a row: v = c * v + s * (its pair's other value).
struct RopeLane {
  float c[8], s[8];
  int partner;        // lane of the other values; this one when a pair lies within the lane (interleaved)
  bool any;

  __device__ __forceinline__ void load(const float *row, int rd, bool interleaved, int lane, int d0) {
    const int half = rd / 2, off = half / 8;   // rope_dim is a multiple of 16
    any = true;
    partner = interleaved || d0 >= rd ? lane : d0 < half ? lane + off : lane - off;
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, s[e] = 0.f;
    if (d0 >= rd) return;
    if (interleaved) {
      const float4 a = __ldcg(reinterpret_cast<const float4 *>(row + d0 / 2)),
                   b = __ldcg(reinterpret_cast<const float4 *>(row + half + d0 / 2));
      const float cs[4] = {a.x, a.y, a.z, a.w}, sn[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = cs[e / 2], s[e] = e % 2 ? sn[e / 2] : -sn[e / 2];
    } else {
      const float4 *at = reinterpret_cast<const float4 *>(row + (d0 < half ? d0 : d0 - half));
      const float4 a0 = __ldcg(at), a1 = __ldcg(at + 1), b0 = __ldcg(at + half / 4), b1 = __ldcg(at + half / 4 + 1);
      const float cs[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
      const float sn[8] = {b0.x, b0.y, b0.z, b0.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = cs[e], s[e] = d0 < half ? -sn[e] : sn[e];
    }
  }
};

// RMS norm of a head with the lane's weights w (norm: whether it has one), then the rotation (turn: whether it turns).
template <int kLanes, typename T>
__device__ __forceinline__ void norm_rope(T (&v)[8], bool norm, bool any_norm, const uint4 &w, float eps,
                                          const RopeLane &rope, bool interleaved, bool turn) {
  if (any_norm) {
    T ss = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const T r = inv_sqrt(ss * (T)(1.0 / (8 * kLanes)) + (T)eps);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if (norm)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * r * (T)(e % 2 ? bf16_hi_f32(u[e / 2]) : bf16_lo_f32(u[e / 2]));
  }
  if (!rope.any) return;
  T other[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) other[e] = interleaved ? v[e ^ 1] : __shfl_sync(0xffffffffu, v[e], rope.partner);
  if (turn)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * (T)rope.c[e] + other[e] * (T)rope.s[e];
}

// The q4nx group rule in 64 bits: {scale, min} of a group from its extremes.  False when it has no finite form.
__device__ __forceinline__ bool group_scale(double lo, double hi, float &sc, float &mn) {
  mn = bf16_floor_f32(__double2float_rd(lo));
  const double base = (double)mn, span = hi - base;
  // The smallest bf16 that is at least span / 15: a candidate that may be one step low, then the exact comparison.
  // The span itself may pass the largest 32-bit number, a 15th of it does not.
  sc = bf16_ceil_f32(__double2float_rn(span * (0.999999 / 15.0)));
  if (15.0 * (double)sc < span) sc = bf16_next_up(sc);
  if (base + 15.0 * (double)sc < hi) sc = bf16_next_up(sc);   // one step covers the rounding of the sum
  if (span == 0.0) sc = 0.f;
  return isfinite(sc) && isfinite(mn);
}
__device__ __noinline__ uint32_t group_code(double v, float mn, float sc) {
  const double q = sc > 0.f ? rint((v - (double)mn) / (double)sc) : 0.0;
  return (uint32_t)(q < 0.0 ? 0.0 : q > 15.0 ? 15.0 : q);
}

// The lane's 8 codes (value e at bits 4e) and the group's {scale, min}, over the 4 lanes of a group; a group without a
// finite form becomes {0, NaN} (and false is returned).  The quotient is good to 15 * 2^-22 in 32 bits: within 1e-5 of
// a boundary, or where the numbers are extreme, the 64-bit one decides.
template <typename T>
__device__ __forceinline__ bool quantise_group(const T (&v)[8], uint32_t &codes, uint32_t &param) {
  bool fine = true;
  T lo = v[0], hi = v[0];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    fine = fine && isfinite(v[e]);
    lo = v[e] < lo ? v[e] : lo;
    hi = v[e] > hi ? v[e] : hi;
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const T a = __shfl_xor_sync(0xffffffffu, lo, o), b = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  const unsigned mine = 0xFu << (threadIdx.x & 28);
  fine = (__ballot_sync(0xffffffffu, fine) & mine) == mine;
  float sc, mn;
  fine = group_scale((double)lo, (double)hi, sc, mn) && fine;
  const float inv = sc > 0.f ? __frcp_rn(sc) : 0.f;
  const bool plain = fabs(hi) < (T)1e37 && fabs(lo) < (T)1e37 && sc > 1e-30f;
  codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (float)(v[e] - (T)mn) * inv, q = rintf(t);
    uint32_t c = (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
    if (!plain || fabsf(fabsf(t - q) - 0.5f) < 1e-5f) c = group_code((double)v[e], mn, sc);
    codes |= c << (4 * e);
  }
  if (!fine) codes = 0;
  param = fine ? (__float_as_uint(sc) >> 16) | (__float_as_uint(mn) & 0xFFFF0000u) : 0x7FC00000u;
  return fine;
}

template <int NJ, bool F32>
__global__ void __launch_bounds__(32, kAppendCtas) rc_kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int D = 32 * NJ, kLanes = D / 8, kHeads = 32 / kLanes;   // of a head; of a unit
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x, d0 = lane % kLanes * 8;
  const int r = (int)(blockIdx.x / (unsigned)p.parts), part = (int)(blockIdx.x % (unsigned)p.parts);
  const bool is_q = part < p.parts_q;
  const int end = is_q ? p.q_heads : p.q_heads + 2 * p.g.heads;                      // past the last head of the kind
  const int per = is_q ? p.units_q : p.units_kv;
  const int h0 = (is_q ? part : part - p.parts_q) * per * kHeads + (is_q ? 0 : p.q_heads);
  const int units = min(per, (end - h0 + kHeads - 1) / kHeads);
  // a lane past the last head works on that one and stores nothing
  Raw8<F32> raw[kAppendUnits];
#pragma unroll
  for (int u = 0; u < kAppendUnits; ++u)
    if (u < units) raw[u].load(p.x, (size_t)r * p.ldx + (size_t)min(h0 + u * kHeads + lane / kLanes, end - 1) * D + d0);
  const uint16_t *norm = is_q ? p.q_norm : p.k_norm;
  uint4 w = {};
  if (norm) w = __ldcg(reinterpret_cast<const uint4 *>(norm + d0));
  int seq, pos;
  if (!kv_find_row(p.b, r, lane, seq, pos)) return;
  RopeLane rope;
  rope.any = false;
  if (p.rope && pos >= 0 && h0 < p.q_heads + p.g.heads) {
    if (pos >= p.rope_rows) {
      if (lane == 0) atomicCAS(p.err, 0, kErrKvRange);
      return;
    }
    rope.load(p.rope + (size_t)pos * p.rope_dim, p.rope_dim, p.interleaved, lane, d0);
  }
  if (is_q) {
#pragma unroll
    for (int u = 0; u < kAppendUnits; ++u) {
      if (u >= units) break;
      float v[8];
      raw[u].get(v);
      norm_rope<kLanes, float>(v, true, norm != nullptr, w, p.eps, rope, p.interleaved, true);
      const int h = h0 + u * kHeads + lane / kLanes;
      if (h < end) *reinterpret_cast<uint4 *>(p.q_out + (size_t)r * p.ldq + h * D + d0) = bf16x8_rn(v);
    }
    return;
  }
  uint8_t *page = pos >= 0 ? kv_head_block(p.g, p.b, seq, pos, 0, p.err) : nullptr;
  if (!page) return;
  const int t = pos & (p.g.page - 1), j = d0 / 32, first_v = p.q_heads + p.g.heads;
#pragma unroll 1
  for (int u = 0; u < units; ++u) {
    const int h = h0 + u * kHeads + lane / kLanes;
    const bool is_v = h >= first_v;
    float v[8];
    raw[0].get(v);
#pragma unroll
    for (int i = 0; i + 1 < kAppendUnits; ++i) raw[i] = raw[i + 1];
    uint32_t codes, param;
    bool fine;
    if (h0 + u * kHeads >= first_v) {                     // values only
      fine = quantise_group<float>(v, codes, param);
    } else {
      double k[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = v[e];
      norm_rope<kLanes, double>(k, !is_v, norm != nullptr, w, p.eps, rope, p.interleaved, !is_v);
      fine = quantise_group<double>(k, codes, param);
    }
    if (h >= end) continue;
    if (!fine) atomicCAS(p.err, 0, kErrKvNonFinite);
    uint8_t *blk = page + (size_t)(h - (is_v ? first_v : p.q_heads)) * p.g.head_bytes;
    uint8_t *to = blk + (is_v ? p.g.vc_off : 0) + t * (D / 2) + (is_v ? kv_v_byte(d0, NJ) : kv_k_byte(d0, NJ));
    if (is_v) {
      *reinterpret_cast<uint16_t *>(to) = (uint16_t)codes;
      *reinterpret_cast<uint16_t *>(to + 2 * NJ) = (uint16_t)(codes >> 16);
    } else {
      *reinterpret_cast<uint32_t *>(to) = codes;
    }
    if (d0 % kKvGroup == 0) reinterpret_cast<uint32_t *>(blk + (is_v ? p.g.vp_off : p.g.kp_off))[t * NJ + j] = param;
  }
}

// ------------------------------------------------------------------- read --
// One warp per (row, 256 / D kv heads), K and V, 8 values a lane: min + scale *
// code in 32 bits (one rounding: scale * code is exact), rounded to bf16.  4096
// rows of 4 + 4 heads of 128 take 10 us (10.5 MB), most of it the launch and three
// loads that depend on one another; with a warp each for K and V it took 12, with
// blocks of one warp 19.
constexpr int kKvWarps = 8;

template <int NJ>
__global__ void __launch_bounds__(32 * kKvWarps)
    rc_kv_read_kernel(const __grid_constant__ KvGeom g, const __grid_constant__ KvBatchDev b, int parts, uint16_t *k_out,
                      uint16_t *v_out, int *err) {
  constexpr int D = 32 * NJ, kLanes = D / 8, kHeads = 32 / kLanes;
  pdl_launch_dependents();
  pdl_wait_prior();
  const int lane = threadIdx.x & 31, d0 = lane % kLanes * 8;
  const long long item = (long long)blockIdx.x * kKvWarps + (threadIdx.x >> 5);
  const int r = (int)(item / parts), h = (int)(item - (long long)r * parts) * kHeads + lane / kLanes;
  if (r >= b.n_rows) return;
  int seq, pos;
  if (!kv_find_row(b, r, lane, seq, pos) || h >= g.heads) return;
  const uint8_t *blk = pos >= 0 ? kv_head_block(g, b, seq, pos, h, err) : nullptr;
  const int t = pos & (g.page - 1);
  uint32_t par[2] = {0, 0}, codes[2] = {0, 0};   // zeros for a row that is empty or outside
  if (blk) {
    const uint8_t *k = blk + t * (D / 2) + kv_k_byte(d0, NJ), *v = blk + g.vc_off + t * (D / 2) + kv_v_byte(d0, NJ);
    const int at = t * NJ + d0 / kKvGroup;
    par[0] = __ldcg(reinterpret_cast<const uint32_t *>(blk + g.kp_off) + at);
    par[1] = __ldcg(reinterpret_cast<const uint32_t *>(blk + g.vp_off) + at);
    codes[0] = __ldcg(reinterpret_cast<const uint32_t *>(k));
    codes[1] = __ldcg(reinterpret_cast<const uint16_t *>(v)) | (uint32_t)__ldcg(reinterpret_cast<const uint16_t *>(v + 2 * NJ)) << 16;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float sc = bf16_lo_f32(par[i]), mn = bf16_hi_f32(par[i]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(sc, (float)(codes[i] >> (4 * e) & 15), mn);
    *reinterpret_cast<uint4 *>((i ? v_out : k_out) + ((size_t)r * g.heads + h) * D + d0) = bf16x8_rn(x);
  }
}

// ------------------------------------------------------------- page moves --
// Copy blocks move kMoveChunk bytes of one page of one layer; table blocks
// rewrite table entries through a hash of the moves in shared memory, built
// kMoveHash moves at a time (a destination is never a source, so one pass's
// new entries are left alone by the next).  Bound by memory: 96 pages of 64 tokens
// in 48 layers (378 MB) move in 67 us, 5.6 TB/s or 88% of the copy rate; 7 pages
// (27.5 MB) in 7 us.
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
  RC_CHECK_ARG(n_seqs == 0 || (table && kv_len), "%s: NULL table or kv_len", what);
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
  RC_CHECK_ARG(kv && (x_dev || n_rows == 0), "rc_kv_append: NULL argument");
  int rc = kv_check_batch("rc_kv_append", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(x_dtype == RC_DTYPE_BF16 || x_dtype == RC_DTYPE_F32, "rc_kv_append: unknown dtype %d", x_dtype);
  RC_CHECK_ARG(q_heads >= 0 && q_heads <= 4096, "rc_kv_append: %d query heads", q_heads);
  RC_CHECK_ARG(q_heads == 0 || n_rows == 0 || q_out_dev, "rc_kv_append: q_out is NULL");
  const long long width = (long long)(q_heads + 2 * kv->heads) * kv->dim;
  RC_CHECK_ARG(ldx >= width, "rc_kv_append: rows of %d values, %lld are needed", ldx, width);
  RC_CHECK_ARG(q_heads == 0 || ldq >= q_heads * kv->dim, "rc_kv_append: q_out rows of %d values, %d are needed", ldq,
               q_heads * kv->dim);
  RC_CHECK_ARG(ldx % 8 == 0 && ldq % 8 == 0 && aligned16(x_dev) && aligned16(q_out_dev),
               "rc_kv_append: rows must start on 16-byte boundaries");
  RC_CHECK_ARG(!rope_dev || (rope_rows >= 1 && rope_dim >= 16 && rope_dim <= kv->dim && rope_dim % 16 == 0),
               "rc_kv_append: rope_dim %d must be a multiple of 16 up to head_dim (and rope_rows, %d, positive)", rope_dim,
               rope_rows);
  RC_CHECK_ARG(aligned16(rope_dev), "rc_kv_append: the rotation table must be 16-byte aligned");
  RC_CHECK_ARG(aligned16(q_norm_dev) && aligned16(k_norm_dev), "rc_kv_append: norm weights must be 16-byte aligned");
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
  // As many units of queries a warp (4, 2 or 1) as leave 16 warps an SM, and half as many of keys and values, which take
  // longer.  4096 rows of 20 units (and their read-back): 47 us with 4, 57 with 2, 97 with 1; 859 rows of 8 units: 15.0,
  // 11.5 and 12.7; 16 rows of 20 units: 9.2, 6.6 and 5.2.  The halves took 1.7, 0.7 and 0 us off.
  const int unit = 256 / kv->dim, units_q = (q_heads + unit - 1) / unit, units_kv = (2 * kv->heads + unit - 1) / unit;
  for (p.units_q = kAppendUnits; p.units_q > 1 && (long long)n_rows * (units_q + units_kv) < 16ll * p.units_q * kv->ctx->sm_count;)
    p.units_q /= 2;
  p.units_kv = p.units_q > 1 ? p.units_q / 2 : 1;
  p.parts_q = (units_q + p.units_q - 1) / p.units_q;
  p.parts = p.parts_q + (units_kv + p.units_kv - 1) / p.units_kv;
  const long long blocks = (long long)n_rows * p.parts;
  RC_CHECK_ARG(blocks <= INT_MAX, "rc_kv_append: too many rows (%d)", n_rows);
  const dim3 grid((unsigned)blocks), block(32);
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  const bool f32 = x_dtype == RC_DTYPE_F32;
  if (kv->dim == 128)
    return f32 ? launch(rc_kv_append_kernel<4, true>, grid, block, s, p) : launch(rc_kv_append_kernel<4, false>, grid, block, s, p);
  return f32 ? launch(rc_kv_append_kernel<2, true>, grid, block, s, p) : launch(rc_kv_append_kernel<2, false>, grid, block, s, p);
}

int rc_kv_read(rc_kv *kv, int layer, int n_rows, const int32_t *table_dev, int cols, int ld_table,
               const int32_t *kv_len_dev, const int32_t *q_off_dev, int n_seqs, uint16_t *k_out_dev, uint16_t *v_out_dev, void *stream) {
  RC_CHECK_ARG(kv && ((k_out_dev && v_out_dev) || n_rows == 0), "rc_kv_read: NULL argument");
  int rc = kv_check_batch("rc_kv_read", kv, layer, n_rows, table_dev, cols, ld_table, kv_len_dev, q_off_dev, n_seqs);
  if (rc) return rc;
  RC_CHECK_ARG(aligned16(k_out_dev) && aligned16(v_out_dev), "rc_kv_read: buffers must be 16-byte aligned");
  if (n_rows == 0 || n_seqs == 0) return RC_OK;
  RC_CUDA_TRY(cudaSetDevice(kv->ctx->device));
  const KvGeom g = kv_geom(kv, layer);
  const KvBatchDev b{table_dev, kv_len_dev, q_off_dev, cols, ld_table, n_seqs, n_rows};
  const int unit = 256 / kv->dim, parts = (kv->heads + unit - 1) / unit;
  const long long blocks = ((long long)n_rows * parts + kKvWarps - 1) / kKvWarps;
  RC_CHECK_ARG(blocks <= INT_MAX, "rc_kv_read: too many rows (%d)", n_rows);
  const dim3 grid((unsigned)blocks), block(32 * kKvWarps);
  const cudaStream_t s = pick_stream(kv->ctx, stream);
  return kv->dim == 128 ? launch(rc_kv_read_kernel<4>, grid, block, s, g, b, parts, k_out_dev, v_out_dev, kv->ctx->err)
                        : launch(rc_kv_read_kernel<2>, grid, block, s, g, b, parts, k_out_dev, v_out_dev, kv->ctx->err);
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

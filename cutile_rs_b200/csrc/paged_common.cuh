// Pieces shared by the paged-cache kernels: the batch as the kernels see it, the range of keys a sequence or a block
// of query rows looks at, and the scores.
#pragma once
#include <math_constants.h>
#include <stdint.h>

#include "../../include/b200tile.h"
#include "host_common.h"
#include "sm100_ptx.cuh"

namespace b200 {

constexpr uint32_t ST_BAD_PAGE = 4;   // a page number outside the pool was met: zeros read, nothing written

// The batch's description lives on the device and can hold anything: everything the kernels derive from it is
// clamped to the tensors' extents before it becomes an address.
struct PagedBatch {
  const int32_t* table;      // [batch, max_pages]
  const int32_t* cu_q;       // [batch + 1]
  const int32_t* kv_lens;    // [batch], the new tokens included
  long long table_pitch;
  int batch, max_pages, num_pages, page_shift;
  int tokens, max_q;
};

struct SeqView {
  int q0, n;       // first token row and number of token rows
  int pos0;        // position of the first token
  int len;         // cached rows that may be read
};

__device__ __forceinline__ SeqView seq_view(const PagedBatch& p, int b) {
  const int c0 = __ldg(p.cu_q + b), c1 = __ldg(p.cu_q + b + 1), kv = __ldg(p.kv_lens + b);
  SeqView s;
  s.q0 = min(max(c0, 0), p.tokens);
  const int q1 = min(max(c1, s.q0), p.tokens);
  s.n = min(q1 - s.q0, p.max_q);
  s.len = min(max(kv, 0), p.max_pages << p.page_shift);
  s.pos0 = kv - (c1 - c0);
  return s;
}

// First key of the window of the token at position pos (which may be negative, and the window longer than anything).
__device__ __forceinline__ int window_start(int pos, int window) { return pos >= window ? pos - window + 1 : 0; }

// Page of key position `key` of sequence b, or num_pages (just outside the pool, where TMA reads zeros) with the
// status record set.  Called for positions inside [0, len) only.
__device__ __forceinline__ int page_of(const PagedBatch& p, int b, int key, uint32_t* status) {
  const int pg = __ldg(p.table + (long long)b * p.table_pitch + (key >> p.page_shift));
  if ((unsigned)pg < (unsigned)p.num_pages) return pg;
  if (atomicCAS(status, 0u, ST_BAD_PAGE) == 0u) {
    status[1] = blockIdx.x;
    status[2] = (uint32_t)b;
    status[3] = (uint32_t)pg;
  }
  return p.num_pages;
}

// Scores in the log2 domain: x = s * scale_log2, or with a cap c on the natural-log score z = s * scale
//   c log2e tanh(z / c) = c log2e (1 - 2 / (1 + exp2(2 log2e z / c)))
// which saturates cleanly at both ends (exp2 -> inf or 0).  ex2.approx and rcp.approx leave an absolute error of about
// c * 2^-22 in the score, well under the rounding of the probabilities to 16 bits for any cap up to a thousand.
struct ScoreParams {
  float scale_log2;            // scale * log2e
  float cap_arg;               // 2 * log2e * scale / c
  float cap_out;               // c * log2e
};
__device__ __forceinline__ float paged_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float paged_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool CAP>
__device__ __forceinline__ float paged_score(const ScoreParams& sp, float s) {
  if (!CAP) return s * sp.scale_log2;
  return fmaf(-2.0f * sp.cap_out, paged_rcp(1.0f + paged_ex2(s * sp.cap_arg)), sp.cap_out);
}

template <bool F16>
__device__ __forceinline__ uint32_t paged_pack16(float lo, float hi) {
  return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}
template <bool F16>
__device__ __forceinline__ float2 paged_unpack16(uint32_t w) {
  if (F16) {
    float2 f;
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(f.x), "=f"(f.y) : "r"(w));
    return f;
  }
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

}  // namespace b200

// Host side: the checked argument block that the entry points hand to the dispatchers.
struct PagedAttnArgs {
  int dtype;                         // 0 = bf16, 1 = f16
  const b200tile_paged_cache* cache;
  b200::PagedBatch batch;
  const void* q;
  void* out;
  int q_heads;
  long long q_ts, q_hs, o_ts, o_hs;  // token and head strides in elements
  b200::ScoreParams score;
  bool capped;
  int causal, window;
  int row_limit;                     // sequences with more query rows per K/V head are another kernel's
  void* workspace;
  size_t tile_off;                   // the tile kernel's part of the workspace
  cudaStream_t stream;
};

// Geometry of the row-block kernel (fmha_paged.cu) for a problem: what the workspace holds.
struct PagedSplitPlan {
  int rows_per_block;     // 8 or 16 query rows of one K/V head
  int ctas, workers;      // one worker = one warp
  long long items;        // (sequence, row block, K/V head) at most
  int coop;               // CTAs per item (no workspace needed), or 0: runs of the whole line
  int heads_abreast;      // heads that neighbouring workers take side by side, a divisor of kv_heads
  bool by_item;           // descriptors indexed by item (few items) or by worker
  size_t part_floats;     // floats per partial-result slot
  size_t desc_off, bytes;
};
PagedSplitPlan b200_paged_split_plan(int format, int head_dim, int kv_heads, int batch, long long rows,
                                     long long max_keys);
int b200_paged_split_dispatch(const PagedAttnArgs& a);
struct PagedTilePlan {
  int ctas;
  size_t desc_off, bytes;
};
PagedTilePlan b200_paged_tile_plan(int head_dim);
// Takes the sequences with more than row_limit rows; with row_limit > 0 launched right behind the row-block kernel, whose
// rows it leaves alone, and beside it.
int b200_paged_tile_dispatch(const PagedAttnArgs& a);

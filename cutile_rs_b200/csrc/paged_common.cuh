// Pieces shared by the paged-cache kernels: the batch as the kernels see it, the range of keys a sequence or a block
// of query rows looks at, and the scores.
#pragma once
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/b200tile.h"
#include "fmha_common.cuh"
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

// Scores in the log2 domain: x = s * scale_log2, or with a cap c on the natural-log score y = s * scale
//   c log2e tanh(y / c) = c log2e (1 - 2 / (1 + exp2(z))),  z = 2 log2e y / c
// which saturates cleanly at both ends (exp2 -> inf or 0), but is off by about c * 2^-22.  That is 2^-16 for a cap of 64,
// under the rounding of the probabilities; with larger caps scores |y| <= 0.4 c take an odd polynomial instead,
//   tanh(t) = t P(t^2):  the Chebyshev interpolant of tanh(sqrt u) / sqrt u on [0, 0.4^2], off by at most 4.5e-8,
// so that the score is right to 2^-20 of itself however large the cap is; far above every score it changes nothing.
// (Both forms for every cap: 32 steps over 16384 NVFP4 keys 78 us instead of 73, prompt chunks with scores near the cap 253
// instead of 211.)
struct ScoreParams {
  float scale_log2;            // scale * log2e
  float cap_arg;               // 2 * log2e * scale / c
  float cap_out;               // c * log2e
};
constexpr float CAP_POLY_MAX = 0.4f;
constexpr int CAP_POLY_N = 4;
__host__ __device__ constexpr float cap_poly(int i) {
  return i == 0 ? 0.9999998807907104f : i == 1 ? -0.33331355452537537f : i == 2 ? 0.13270874321460724f : -0.04754934832453728f;
}
constexpr float CAP_SMALL_OUT = 64.0f * 1.4426950408889634f;    // cap_out up to which one form serves
constexpr float CAP_HALF_ARG = 0.5f / 1.4426950408889634f;     // t = z * this
// A factor that underflows to 0 or overflows would make NaN of scores that are infinite, masked ones too, or 0.
__host__ __device__ __forceinline__ float factor_in_range(float x) { return fminf(fmaxf(x, 0x1p-126f), 0x1p126f); }
__device__ __forceinline__ float paged_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// z small enough for the polynomial; false for NaN
__device__ __forceinline__ bool cap_is_far(float z) { return fabsf(z) <= CAP_POLY_MAX / CAP_HALF_ARG; }
__device__ __forceinline__ float paged_score_far(const ScoreParams& sp, float s) {     // from the cap
  constexpr float w = CAP_HALF_ARG * CAP_HALF_ARG;
  const float z = s * sp.cap_arg, u = z * z;
  float h = fmaf(cap_poly(3) * w * w * w, u, cap_poly(2) * w * w);
  h = fmaf(h, u, cap_poly(1) * w);
  return s * sp.scale_log2 * fmaf(h, u, cap_poly(0));
}
__device__ __forceinline__ float paged_score_near(const ScoreParams& sp, float s) {
  return fmaf(-2.0f * sp.cap_out, paged_rcp(1.0f + ex2_approx(s * sp.cap_arg)), sp.cap_out);
}
template <bool CAP>
__device__ __forceinline__ float paged_score(const ScoreParams& sp, float s) {
  if (!CAP) return s * sp.scale_log2;
  const float a = paged_score_far(sp, s), b = paged_score_near(sp, s);
  return cap_is_far(s * sp.cap_arg) ? a : b;
}

// Probabilities are handed to the second product as 16-bit values.  f16 has nothing between 0 and 2^-24: behind a key that
// holds most of a row's weight with little of its value, 2^18 keys of 2^-19.6 each came out 2 % too small.  So they are
// exp2(x - m + 7), with the running reference m at most 8 below the maximum: up to 2^15, and down to 2^-31 of the largest,
// which is below what sums in 32 bits hold.  bf16 has f32's range.
template <bool F16>
__device__ constexpr float p_shift() { return F16 ? 7.0f : 0.0f; }

// The four bytes of w, two e2m1 codes each, as f16 pairs (low nibble in the low half).  One conversion instruction per
// pair runs at 50 pairs per clock and SM against 22 for shifting the bits into place.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{.reg .b8 a, b, c, d; mov.b32 {a, b, c, d}, %4;"
      " cvt.rn.f16x2.e2m1x2 %0, a; cvt.rn.f16x2.e2m1x2 %1, b; cvt.rn.f16x2.e2m1x2 %2, c; cvt.rn.f16x2.e2m1x2 %3, d;}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(w));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_bytes) {
  uint32_t r;
  asm("{.reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(r) : "r"(two_bytes));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A box of a page pool: {dimension, slot, head, page}.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* desc, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(desc), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
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
  double qk_scale, softcap;
  bool capped;
  int causal, window;
  int row_limit;                     // sequences with more query rows per K/V head are another kernel's
  void* workspace;
  size_t tile_off;                   // the tile kernel's part of the workspace
  cudaStream_t stream;
};

// The kernels' factors, from one over all of them: `factor` is what the cached keys have to be multiplied with.
inline b200::ScoreParams paged_score_params(const PagedAttnArgs& a, float factor) {
  const double log2e = 1.4426950408889634, scale = a.qk_scale * factor;
  b200::ScoreParams p;
  p.scale_log2 = b200::factor_in_range((float)(scale * log2e));
  p.cap_arg = a.capped ? b200::factor_in_range((float)(2.0 * log2e * scale / a.softcap)) : 0.0f;
  p.cap_out = (float)std::min(a.softcap * log2e, 1e38);      // twice it is still a number
  return p;
}

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

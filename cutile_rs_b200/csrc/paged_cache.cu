// Writing new tokens into a paged key/value cache, with the rotary embedding on the way, and reading rows back.
//
//   p = kv_lens[b] - (cu_q[b+1] - cu_q[b]) + i           position of token i of sequence b
//   y_i = x_i cos(p f_i) - x_{i+r/2} sin(p f_i),  y_{i+r/2} = x_{i+r/2} cos(p f_i) + x_i sin(p f_i)   for i < r/2
// for every head of Q (to q_out) and K (to its slot); V and the dimensions from r on are copied.  An NVFP4 cache takes
// blocks of 16: scale = e4m3(max |y| / (6 g)), code = e2m1(y / (scale g)) with g the pool's factor.
//
// HBM-bound in 16 bits (8192 tokens, 32 + 8 heads of 128: 46 us, 5.5 TB/s).  With FP4 blocks 6691 tokens take 34 us against
// 22 of traffic, 31 with angles, maxima and quotients left out: 16 warps an SM (126 registers) issue in 59 % of the cycles
// and wait for fixed latencies and loads in the rest, DRAM 38 % busy; codes and scales leave in pieces of 4 and 1 bytes.
// Reading 6691 tokens back takes 10 to 11 us against 5.4 of traffic: 55 % of the issue slots, the conversion pipe at 40 %.
// Each value is read once and written once.  A warp takes a token (or a share of its heads): lane l always holds the same
// D/16-th of a head, so its 8 cosines and sines stay in registers for all heads, and nothing but loads, 32 products and 16
// sums (each rounded by itself, see the rotation) and stores is left in the loop.  Angles: p * f_i reaches 1e5 and more,
// where a product rounded to 32 bits is off by 1e-2 radians; angle, sine and cosine are taken in 64 bits and rounded to 32
// once (64 of them per token against 10^4 values moved), so that the rotated value, and with it every rounding to 4 bits,
// does not depend on how far the position is.
#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "paged_common.cuh"

namespace b200 {
namespace {

struct CacheView {
  uint8_t *k, *v, *ks, *vs;
  long long k_st[3], v_st[3], ks_st[3], vs_st[3];   // bytes: page, head, slot
  float k_global, v_global;
  int kv_heads;
};
struct AppendParams {
  PagedBatch batch;
  CacheView c;
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  const float* inv_freq;
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
  int q_heads, rot;        // rot: dimensions that are rotated
  int shares;              // warps per token
  float k_six, k_inv_six, v_six, v_inv_six;   // FP4: 6 * global and its reciprocal
  bool k_tame, v_tame;                        // and whether that is far from the ends of f32
};
struct GatherParams {
  PagedBatch batch;
  CacheView c;
  uint16_t *k_out, *v_out;
  long long k_ts, k_hs, v_ts, v_hs;
  int shares;
};

// The sequence that holds token t (the last b with cu_q[b] <= t), found by the warp with 32 probes a round; -1 for
// tokens outside [cu_q[0], cu_q[batch]).
__device__ __forceinline__ int seq_of_token(const PagedBatch& p, int t, int lane) {
  if (t >= __ldg(p.cu_q + p.batch)) return -1;
  int lo = 0, n = p.batch;
  do {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool le = at < n && __ldg(p.cu_q + lo + at) <= t;
    const uint32_t mask = __ballot_sync(0xffffffffu, le);
    if (mask == 0) return -1;
    const int k = 31 - __clz(mask);
    lo += k * step;
    n = min(step, n - k * step);
  } while (n > 1);
  return lo;
}

struct TokenPlace {
  int pos, slot;
  long long page;          // -1: outside the cache
};
__device__ __forceinline__ TokenPlace place_of(const PagedBatch& p, int b, int t, uint32_t* status) {
  const int c1 = __ldg(p.cu_q + b + 1), kv = __ldg(p.kv_lens + b);
  TokenPlace x;
  x.pos = kv - c1 + t;
  x.page = -1;
  x.slot = x.pos & ((1 << p.page_shift) - 1);
  if (x.pos >= 0 && x.pos < (p.max_pages << p.page_shift)) {
    const int pg = page_of(p, b, x.pos, status);
    if (pg < p.num_pages) x.page = pg;
  }
  return x;
}

template <bool F16>
__device__ __forceinline__ uint32_t pack_pair(uint64_t x) {
  float lo, hi;
  unpack2(x, lo, hi);
  return paged_pack16<F16>(lo, hi);
}

// Out of line: the argument reduction's registers stay out of the streaming loop.
__device__ __noinline__ void angle_64(int pos, float inv_freq, double* s, double* c) {
  sincos((double)pos * (double)inv_freq, s, c);
}

// Quotients a / b from inv close to 1 / b by Markstein's correction: q = a inv, then q + (a - q b) inv with the exact
// remainder, which leaves half a step and a few millionths of one.  16-bit values meet the rounding borders of e2m1 and e4m3 exactly, where a plain product
// with the reciprocal would miss the tie; the correction hits a quotient that 32 bits hold.  For b and a / b well inside
// the range of f32.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
  const float q = __fmul_rn(a, inv);
  return __fmaf_rn(__fmaf_rn(-q, b, a), inv, q);
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t quotient2(uint64_t a, uint64_t neg_b, uint64_t inv) {
  const uint64_t q = mul2(a, inv);
  return fma2(fma2(q, neg_b, a), inv, q);
}
// The largest magnitude, NaN if one is NaN: the block's scale then is NaN too, and all of it reads back as NaN.  A maximum
// that passes over NaN would store it as the block's largest code, which is 0 among zeros.
__device__ __forceinline__ float absmax_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A block's scale e4m3(amax / (6 g)) and 8 of its values -> codes of 4 bits, first value lowest.
struct BlockScale {
  uint32_t byte;
  float s;
  bool plain;              // the quotients need the general division: s far out of range, an infinity or a NaN in the block
};
__device__ __forceinline__ BlockScale block_scale(float amax, float glob, float six_g, float inv_six_g, bool tame_g) {
  BlockScale x;
  x.plain = !(tame_g && amax < 0x1p90f && (amax > 0x1p-90f || amax == 0.0f));
  float q = quotient(amax, six_g, inv_six_g);
  if (x.plain) q = __fdiv_rn(amax, six_g);
  uint32_t f16x2;
  asm("{.reg .b16 h; cvt.rn.satfinite.e4m3x2.f32 h, 0f00000000, %2; cvt.u32.u16 %0, h; cvt.rn.f16x2.e4m3x2 %1, h;}"
      : "=r"(x.byte), "=r"(f16x2) : "f"(q));
  x.s = __low2float(*reinterpret_cast<__half2*>(&f16x2)) * glob;
  return x;
}
__device__ __forceinline__ uint32_t e2m1x8(const float (&y)[8]) {
  uint32_t w;
  asm("{.reg .b8 a, b, c, d;"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1; cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5; cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;"
      " mov.b32 %0, {a, b, c, d};}"
      : "=r"(w) : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return w;
}
__device__ __noinline__ uint32_t e2m1_codes_plain(uint64_t a, uint64_t b, uint64_t c, uint64_t d, float s) {
  float y[8];
  unpack2(a, y[0], y[1]);
  unpack2(b, y[2], y[3]);
  unpack2(c, y[4], y[5]);
  unpack2(d, y[6], y[7]);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(y[i], s);
  return s > 0.0f ? e2m1x8(y) : 0u;
}
__device__ __forceinline__ uint32_t e2m1_codes(const uint64_t (&y)[4], float s) {
  const float r = paged_rcp(s);
  const uint64_t neg_b = pack2(-s, -s), inv = pack2(r, r);
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2(quotient2(y[i], neg_b, inv), f[2 * i], f[2 * i + 1]);
  return s > 0.0f ? e2m1x8(f) : 0u;
}

template <int D, bool F16, bool FP4>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ AppendParams p, uint32_t* status) {
  constexpr int LPH = D / 16;                 // lanes per head: each holds 8 values of both halves
  constexpr int HPW = 32 / LPH;               // heads per warp and round
  const int lane = threadIdx.x & 31;
  const long long warp_id = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int t = (int)(warp_id / p.shares), share = (int)(warp_id - (long long)t * p.shares);
  if (t >= p.batch.tokens) return;
  const int sub = lane % LPH;
  const int total = p.q_heads + 2 * p.c.kv_heads;
  const int stride = HPW * p.shares;
  // lane's two vectors of a head: the two members of its rotated pairs, or 16 neighbours behind them
  const bool rotates = sub * 16 < p.rot;
  const int lo_at = rotates ? sub * 8 : sub * 16;
  const int hi_at = rotates ? p.rot / 2 + sub * 8 : sub * 16 + 8;
  const int v_lo = FP4 ? sub * 8 : sub * 16, v_hi = FP4 ? D / 2 + sub * 8 : sub * 16 + 8;   // V: any pairing serves

  auto load = [&](int i, uint4& lo, uint4& hi) {
    if (i >= total) return;
    const uint16_t* x;
    int a = lo_at, c = hi_at;
    if (i < p.q_heads) x = p.q + (long long)t * p.q_ts + (long long)i * p.q_hs;
    else if (i < p.q_heads + p.c.kv_heads) x = p.k + (long long)t * p.k_ts + (long long)(i - p.q_heads) * p.k_hs;
    else {
      x = p.v + (long long)t * p.v_ts + (long long)(i - p.q_heads - p.c.kv_heads) * p.v_hs;
      a = v_lo;
      c = v_hi;
    }
    lo = *reinterpret_cast<const uint4*>(x + a);             // not as read-only data: q may be q_out
    hi = *reinterpret_cast<const uint4*>(x + c);
  };
  constexpr int U = 3;                        // rounds in flight: 3 x 32 bytes a lane
  uint4 lo[U], hi[U];
  const int first = share * HPW + lane / LPH;
#pragma unroll
  for (int j = 0; j < U; ++j) {
    lo[j] = hi[j] = make_uint4(0, 0, 0, 0);
    load(first + j * stride, lo[j], hi[j]);
  }
  // the rows are on their way (they do not depend on the sequence) while the token's place is looked up
  const int b = seq_of_token(p.batch, t, lane);
  if (b < 0) return;
  const TokenPlace at = place_of(p.batch, b, t, status);

  // cos and sin of this lane's 8 pairs: every lane evaluates LPH / 4 of them, the others come by shuffle
  float cs[8], sn[8];
  {
    constexpr int PER = D / 2 / 32 > 0 ? D / 2 / 32 : 1;      // angles per lane (1 or 2)
    float c[PER], s[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = lane * PER + j;
      c[j] = 1.0f;
      s[j] = 0.0f;
      if (i < p.rot / 2) {
        double sd, cd;
        angle_64(at.pos, __ldg(p.inv_freq + i), &sd, &cd);
        s[j] = (float)sd;
        c[j] = (float)cd;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = (rotates ? sub * 8 : 0) + j;              // angle index
      cs[j] = __shfl_sync(0xffffffffu, c[j % PER], i / PER);
      sn[j] = __shfl_sync(0xffffffffu, s[j % PER], i / PER);
    }
  }

  for (int i0 = first; i0 - lane / LPH < total; i0 += U * stride) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * stride;
      const uint4 xl = lo[j], xh = hi[j];
      load(i + U * stride, lo[j], hi[j]);
      if (i - lane / LPH >= total) continue;                  // warp-uniform: nothing left in this round
      const bool is_v = i >= p.q_heads + p.c.kv_heads, is_q = i < p.q_heads;
      const bool turn = rotates && !is_v;
      const uint32_t wl[4] = {xl.x, xl.y, xl.z, xl.w}, wh[4] = {xh.x, xh.y, xh.z, xh.w};
      uint64_t a[4], c[4];                                    // pairs of neighbours
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 f = paged_unpack16<F16>(wl[e]), h = paged_unpack16<F16>(wh[e]);
        if (turn) {
          // the roundings of b200tile_rope_seq; in scalars, since the paired products and sums get fused
          const float2 x = f, y = h;
          f.x = __fsub_rn(__fmul_rn(x.x, cs[2 * e]), __fmul_rn(y.x, sn[2 * e]));
          f.y = __fsub_rn(__fmul_rn(x.y, cs[2 * e + 1]), __fmul_rn(y.y, sn[2 * e + 1]));
          h.x = __fadd_rn(__fmul_rn(y.x, cs[2 * e]), __fmul_rn(x.x, sn[2 * e]));
          h.y = __fadd_rn(__fmul_rn(y.y, cs[2 * e + 1]), __fmul_rn(x.y, sn[2 * e + 1]));
        }
        a[e] = pack2(f.x, f.y);
        c[e] = pack2(h.x, h.y);
      }
      if (!FP4 || is_q) {
        if (i < total) {
          uint16_t* dst = nullptr;
          if (is_q) dst = p.q_out + (long long)t * p.qo_ts + (long long)i * p.qo_hs;
          else if (at.page >= 0) {
            const long long h = is_v ? i - p.q_heads - p.c.kv_heads : i - p.q_heads;
            const long long* st = is_v ? p.c.v_st : p.c.k_st;
            dst = reinterpret_cast<uint16_t*>((is_v ? p.c.v : p.c.k) + at.page * st[0] + h * st[1] + at.slot * st[2]);
          }
          if (dst) {
            const int da = is_v ? v_lo : lo_at, dc = is_v ? v_hi : hi_at;
            uint4 yl = xl, yh = xh;                           // copies stay the bits they were
            if (turn) {
              yl = make_uint4(pack_pair<F16>(a[0]), pack_pair<F16>(a[1]), pack_pair<F16>(a[2]), pack_pair<F16>(a[3]));
              yh = make_uint4(pack_pair<F16>(c[0]), pack_pair<F16>(c[1]), pack_pair<F16>(c[2]), pack_pair<F16>(c[3]));
            }
            *reinterpret_cast<uint4*>(dst + da) = yl;
            *reinterpret_cast<uint4*>(dst + dc) = yh;
          }
        }
      }
      if (FP4 && i - lane / LPH + HPW > p.q_heads) {           // warp-uniform: some head of this round is K's or V's
        // a block of 16 is this vector and its neighbour lane's (rotated pairs, V) or this lane's two (the rest)
        float ma = 0.0f, mc = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x, y;
          unpack2(a[e], x, y);
          ma = absmax_nan(ma, x, y);
          unpack2(c[e], x, y);
          mc = absmax_nan(mc, x, y);
        }
        const float na = __shfl_xor_sync(0xffffffffu, ma, 1), nc = __shfl_xor_sync(0xffffffffu, mc, 1);
        if (!is_q && i < total && at.page >= 0) {
          const bool halves = is_v || rotates;
          const float both = absmax_nan(ma, mc, mc);
          const float gl = is_v ? p.c.v_global : p.c.k_global, six = is_v ? p.v_six : p.k_six,
                      inv = is_v ? p.v_inv_six : p.k_inv_six;
          const bool tame = is_v ? p.v_tame : p.k_tame;
          const BlockScale sa = block_scale(halves ? absmax_nan(ma, na, na) : both, gl, six, inv, tame);
          const BlockScale sc = block_scale(halves ? absmax_nan(mc, nc, nc) : both, gl, six, inv, tame);
          uint32_t wa = e2m1_codes(a, sa.s), wc = e2m1_codes(c, sc.s);
          if (sa.plain || sc.plain) {
            wa = e2m1_codes_plain(a[0], a[1], a[2], a[3], sa.s);
            wc = e2m1_codes_plain(c[0], c[1], c[2], c[3], sc.s);
          }
          const long long h = is_v ? i - p.q_heads - p.c.kv_heads : i - p.q_heads;
          const long long* st = is_v ? p.c.v_st : p.c.k_st;
          const long long* sst = is_v ? p.c.vs_st : p.c.ks_st;
          uint8_t* row = (is_v ? p.c.v : p.c.k) + at.page * st[0] + h * st[1] + at.slot * st[2];
          uint8_t* srow = (is_v ? p.c.vs : p.c.ks) + at.page * sst[0] + h * sst[1] + at.slot * sst[2];
          const int da = is_v ? v_lo : lo_at, dc = is_v ? v_hi : hi_at;
          *reinterpret_cast<uint32_t*>(row + da / 2) = wa;
          *reinterpret_cast<uint32_t*>(row + dc / 2) = wc;
          if (!halves || (sub & 1) == 0) srow[da / 16] = (uint8_t)sa.byte;
          if (halves && (sub & 1) == 0) srow[dc / 16] = (uint8_t)sc.byte;
        }
      }
    }
  }
}

// Rows of the batch's positions back into [tokens, kv_heads, D]; positions outside the cache read as zero.
template <int D, bool F16, bool FP4>
__global__ void __launch_bounds__(128) paged_gather_kernel(const __grid_constant__ GatherParams p, uint32_t* status) {
  constexpr int LPH = D / 16, HPW = 32 / LPH;
  const int lane = threadIdx.x & 31;
  const long long warp_id = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int t = (int)(warp_id / p.shares), share = (int)(warp_id - (long long)t * p.shares);
  if (t >= p.batch.tokens) return;
  const int b = seq_of_token(p.batch, t, lane);
  if (b < 0) return;
  const TokenPlace at = place_of(p.batch, b, t, status);
  const int sub = lane % LPH, total = 2 * p.c.kv_heads, stride = HPW * p.shares;
  constexpr int U = 4;                        // rounds whose loads are in flight together
  for (int i0 = share * HPW + lane / LPH; i0 - lane / LPH < total; i0 += U * stride) {
    uint4 y0[U], y1[U];                       // FP4: y0.x, y0.y the codes, y0.z the scale
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * stride;
      y0[j] = y1[j] = make_uint4(0, 0, 0, 0);
      if (i >= total || at.page < 0) continue;
      const bool is_v = i >= p.c.kv_heads;
      const long long h = is_v ? i - p.c.kv_heads : i;
      const long long* st = is_v ? p.c.v_st : p.c.k_st;
      const uint8_t* row = (is_v ? p.c.v : p.c.k) + at.page * st[0] + h * st[1] + at.slot * st[2];
      if constexpr (!FP4) {
        y0[j] = __ldg(reinterpret_cast<const uint4*>(row) + sub * 2);
        y1[j] = __ldg(reinterpret_cast<const uint4*>(row) + sub * 2 + 1);
      } else {
        const long long* sst = is_v ? p.c.vs_st : p.c.ks_st;
        const uint8_t* srow = (is_v ? p.c.vs : p.c.ks) + at.page * sst[0] + h * sst[1] + at.slot * sst[2];
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(row) + sub);
        y0[j] = make_uint4(w.x, w.y, __ldg(srow + sub), 0);
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * stride;
      if (i >= total) continue;
      const bool is_v = i >= p.c.kv_heads;
      const long long h = is_v ? i - p.c.kv_heads : i;
      if constexpr (FP4) {
        const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)y0[j].z, __NV_E4M3))) *
                        (is_v ? p.c.v_global : p.c.k_global);
        const uint32_t w[2] = {y0[j].x, y0[j].y};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const __half2_raw c = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)(w[k >> 2] >> (8 * (k & 3))), __NV_E2M1);
          const float2 f = __half22float2(__half2(c));
          o[k] = paged_pack16<F16>(f.x * s, f.y * s);
        }
        y0[j] = make_uint4(o[0], o[1], o[2], o[3]);
        y1[j] = make_uint4(o[4], o[5], o[6], o[7]);
      }
      uint16_t* dst = is_v ? p.v_out + (long long)t * p.v_ts + h * p.v_hs : p.k_out + (long long)t * p.k_ts + h * p.k_hs;
      reinterpret_cast<uint4*>(dst)[sub * 2] = y0[j];
      reinterpret_cast<uint4*>(dst)[sub * 2 + 1] = y1[j];
    }
  }
}

CacheView cache_view(const b200tile_paged_cache& c) {
  CacheView v;
  v.k = static_cast<uint8_t*>(c.k);
  v.v = static_cast<uint8_t*>(c.v);
  v.ks = static_cast<uint8_t*>(c.k_scales);
  v.vs = static_cast<uint8_t*>(c.v_scales);
  const int unit = c.format ? 1 : 2;
  for (int i = 0; i < 3; ++i) {
    v.k_st[i] = c.k_strides[i] * unit;
    v.v_st[i] = c.v_strides[i] * unit;
    v.ks_st[i] = c.k_scale_strides[i];
    v.vs_st[i] = c.v_scale_strides[i];
  }
  v.k_global = c.k_global;
  v.v_global = c.v_global;
  v.kv_heads = c.kv_heads;
  return v;
}

// Warps per token: one when the tokens alone fill the machine with `warps`, else as many as there are rounds to share out.
// Every warp looks its token up, and append's takes the angles: at 6700 tokens two warps instead of one cost append 4 us of
// 37 (FP4) and save gather 1 of 11.
int shares_for(int tokens, int rounds, int warps) {
  return std::max(1, std::min(rounds, (warps + tokens - 1) / tokens));
}

}  // namespace
}  // namespace b200

int b200_paged_append_dispatch(int dtype, const b200tile_paged_cache& c, const b200::PagedBatch& batch, const void* q,
                               const void* k, const void* v, void* q_out, const float* inv_freq, int q_heads, int rot,
                               const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* qos,
                               cudaStream_t stream) {
  using namespace b200;
  const b200h::DeviceInfo* di = b200h::device_info();
  if (!di) return B200_ERR_CUDA;
  AppendParams p;
  p.batch = batch;
  p.c = cache_view(c);
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_out = static_cast<uint16_t*>(q_out);
  p.inv_freq = inv_freq;
  p.q_ts = qs ? qs[0] : 0; p.q_hs = qs ? qs[1] : 0;
  p.k_ts = ks[0]; p.k_hs = ks[1];
  p.v_ts = vs[0]; p.v_hs = vs[1];
  p.qo_ts = qos ? qos[0] : 0; p.qo_hs = qos ? qos[1] : 0;
  p.q_heads = q ? q_heads : 0;
  p.rot = rot;
  p.k_six = 6.0f * c.k_global; p.k_inv_six = 1.0f / p.k_six;
  p.v_six = 6.0f * c.v_global; p.v_inv_six = 1.0f / p.v_six;
  p.k_tame = p.k_six > 0x1p-20f && p.k_six < 0x1p20f;
  p.v_tame = p.v_six > 0x1p-20f && p.v_six < 0x1p20f;
  const int hpw = 32 / (c.head_dim / 16);
  p.shares = shares_for(batch.tokens, (p.q_heads + 2 * c.kv_heads + hpw - 1) / hpw, di->sm_count * 16);
  const long long warps = (long long)batch.tokens * p.shares;
  const unsigned grid = (unsigned)((warps + 3) / 4);
#define B200_PA(D_, F_, Q_) paged_append_kernel<D_, F_, Q_><<<grid, 128, 0, stream>>>(p, di->status)
#define B200_PA_F(D_, Q_) do { if (dtype) B200_PA(D_, true, Q_); else B200_PA(D_, false, Q_); } while (0)
  if (c.head_dim == 128) { if (c.format) B200_PA_F(128, true); else B200_PA_F(128, false); }
  else { if (c.format) B200_PA_F(64, true); else B200_PA_F(64, false); }
#undef B200_PA_F
#undef B200_PA
  B200_CUDA_CHECK(cudaGetLastError());
  return B200_OK;
}

int b200_paged_gather_dispatch(int dtype, const b200tile_paged_cache& c, const b200::PagedBatch& batch, void* k_out,
                               void* v_out, const int64_t* ks, const int64_t* vs, cudaStream_t stream) {
  using namespace b200;
  const b200h::DeviceInfo* di = b200h::device_info();
  if (!di) return B200_ERR_CUDA;
  GatherParams p;
  p.batch = batch;
  p.c = cache_view(c);
  p.k_out = static_cast<uint16_t*>(k_out);
  p.v_out = static_cast<uint16_t*>(v_out);
  p.k_ts = ks[0]; p.k_hs = ks[1];
  p.v_ts = vs[0]; p.v_hs = vs[1];
  const int hpw = 32 / (c.head_dim / 16);
  p.shares = shares_for(batch.tokens, (2 * c.kv_heads + hpw - 1) / hpw, di->sm_count * 64);
  const unsigned grid = (unsigned)(((long long)batch.tokens * p.shares + 3) / 4);
#define B200_PG(D_, F_, Q_) paged_gather_kernel<D_, F_, Q_><<<grid, 128, 0, stream>>>(p, di->status)
#define B200_PG_F(D_, Q_) do { if (dtype) B200_PG(D_, true, Q_); else B200_PG(D_, false, Q_); } while (0)
  if (c.head_dim == 128) { if (c.format) B200_PG_F(128, true); else B200_PG_F(128, false); }
  else { if (c.format) B200_PG_F(64, true); else B200_PG_F(64, false); }
#undef B200_PG_F
#undef B200_PG
  B200_CUDA_CHECK(cudaGetLastError());
  return B200_OK;
}

// Attention of many query rows (prompts and prompt chunks) over a paged key/value cache on the 5th-generation tensor
// cores.  The mathematics is fmha_paged.cu's; the machine is fmha_fwd.cu's: one CTA owns two tiles of 128 query rows
// and walks the keys once for both, S = Q K^T and O += P V by tcgen05 with S, P and O in Tensor Memory, one softmax
// thread per row, O rescaled only when a row's maximum grew by more than 2^8.  What differs:
//
//   - a tile's rows are (token, head of the group) pairs of ONE K/V head, 128 / group tokens at a time, so that K and V
//     pass through a CTA once for all heads that share them (one TMA box {64, group, tokens} brings them in that order);
//   - the 128 keys of a step come from 128 / page_size pages, one TMA box each; a page that no row of the CTA looks at
//     gets the page number just outside the pool, where TMA fills in zeros without touching memory;
//   - V rows of a step that no row looks at (behind the length, before the window) are cleared in shared memory by the
//     MMA warp: their probability is 0, but 0 times whatever a free slot holds need not be;
//   - an NVFP4 cache takes four more warps: thread r expands key r of the step (64 bytes and 8 scales for D = 128) to 16
//     bits straight into the swizzled operand tile, K and V in turn, with the next row's bytes already in registers;
//   - which (sequence, pair of tiles) a CTA works on follows from the lengths on the device; CTAs without work leave.
//
// What bounds it: as fmha_fwd.cu, the softmax threads and the tensor pipe together.
#include <math_constants.h>

#include <algorithm>

#include "fmha_common.cuh"
#include "paged_common.cuh"

namespace b200 {
namespace {

struct TileParams {
  PagedBatch batch;
  ScoreParams score;
  int kv_heads, group, tpt;          // tpt: tokens per tile
  int causal, window, row_limit;
  int box_rows;                      // keys per K/V box
  uint16_t* out;
  long long o_ts, o_hs;
  float out_scale;
  // FP4 operands: byte strides
  const uint8_t *k, *v, *ks, *vs;
  long long k_st[3], v_st[3], ks_st[3], vs_st[3];
};

template <int D, bool FP4>
struct TileSmem {
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;
  static constexpr int KV_STAGES = (D == 128) ? 2 : 4;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * TILE_BYTES;
  static constexpr int OFF_V = OFF_K + KV_STAGES * TILE_BYTES;
  static constexpr int OFF_BAR = OFF_V + KV_STAGES * TILE_BYTES;
  // barriers: q_full[2], k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2], p_full[2], o_done[2]
  static constexpr int NUM_BARS = 2 + 4 * KV_STAGES + 6;
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int TOTAL = OFF_MISC + 16 + 1024;
  static constexpr int THREADS = FP4 ? 512 : 384;
};

__device__ __forceinline__ void tma_load_4d_tile(uint32_t dst, const void* desc, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(desc), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void st_shared_v4(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Pairs of tiles that sequence b has here: none when its rows are few enough for the row-block kernel.
__device__ __forceinline__ int seq_pairs(const TileParams& p, const SeqView& s) {
  if ((long long)s.n * p.group <= p.row_limit) return 0;
  return (s.n + 2 * p.tpt - 1) / (2 * p.tpt);
}

// 8 codes of a word and their scale (16 bits, twice; times 2^7, for bf16 2^119) -> 8 values * 2^-7 in order.
// The codes' bits are put where the 16-bit type reads them as e2m1 * 2^-14 (bf16: 2^-126), subnormals included; the
// product with the scale is exact (two bits times four).
template <bool F16>
__device__ __forceinline__ void expand8(uint32_t w, uint32_t scale, uint32_t (&o)[4]) {
  uint32_t pr[4];                                   // (nibble i, nibble i + 4)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t sgn = i == 3 ? w : w << (12 - 4 * i);
    uint32_t mag;
    if (F16) mag = (i == 3 ? w >> 3 : w << (9 - 4 * i)) & 0x0E000E00u;
    else mag = (i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6)) & 0x01C001C0u;
    const uint32_t x = (sgn & 0x80008000u) | mag;
    if (F16) asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(pr[i]) : "r"(x), "r"(scale));
    else asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(pr[i]) : "r"(x), "r"(scale));
  }
  o[0] = __byte_perm(pr[0], pr[1], 0x5410);
  o[1] = __byte_perm(pr[2], pr[3], 0x5410);
  o[2] = __byte_perm(pr[0], pr[1], 0x7632);
  o[3] = __byte_perm(pr[2], pr[3], 0x7632);
}
// e4m3 byte -> the scale operand of expand8
template <bool F16>
__device__ __forceinline__ uint32_t expand_scale(uint32_t byte) {
  uint32_t h;
  asm("{.reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(h) : "r"(byte & 0xffu));
  if (F16) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x58005800u));
    return __byte_perm(r, r, 0x1010);
  }
  float f;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, a;}" : "=f"(f) : "r"(h));
  const uint32_t r = __float_as_uint(f * 6.64613997892457936e+35f);   // 2^119; four significant bits: exact in bf16
  return __byte_perm(r, r, 0x3232);
}

template <int D, bool F16, bool CAP, bool FP4>
__global__ void __launch_bounds__(FP4 ? 512 : 384, 1)
fmha_paged_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TileParams p, uint32_t* status) {
  using L = TileSmem<D, FP4>;
  constexpr int STAGES = L::KV_STAGES, HALVES = L::HALVES, THREADS = L::THREADS;
  constexpr uint32_t HALF = L::HALF_BYTES, TILE = L::TILE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_first[THREADS], s_warp[THREADS / 32];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- this CTA's work: pair `rank` of all sequences' pairs, one K/V head ----
  // (launched while the row-block kernel's merge may still run: see the end of the kernel)
  const int rank = blockIdx.x / p.kv_heads, head = blockIdx.x - rank * p.kv_heads;
  int b, pair;
  SeqView sv;
  {
    const int per = (p.batch.batch + THREADS - 1) / THREADS;
    int mine = 0;
    for (int i = threadIdx.x * per; i < min(p.batch.batch, (int)(threadIdx.x + 1) * per); ++i)
      mine += seq_pairs(p, seq_view(p.batch, i));
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      before += w < warp ? s_warp[w] : 0;
      total += s_warp[w];
    }
    s_first[threadIdx.x] = before + inc - mine;
    __syncthreads();
    if (rank >= total) {
      grid_dep_wait();
      return;
    }
    int lo = 0, hi = THREADS - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= rank) lo = mid;
      else hi = mid - 1;
    }
    b = lo * per;
    int at = s_first[lo];
    sv = seq_view(p.batch, b);
    int n = seq_pairs(p, sv);
    while (at + n <= rank) {
      at += n;
      if (++b >= p.batch.batch) {
        grid_dep_wait();
        return;
      }
      sv = seq_view(p.batch, b);
      n = seq_pairs(p, sv);
    }
    pair = rank - at;
    if (p.causal) pair = n - 1 - pair;             // the longest first
  }
  // tokens and keys of the two tiles; steps of 128 keys from step j0
  int tok0[2], ntok[2], hi_key[2], n_kv[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    tok0[t] = (pair * 2 + t) * p.tpt;
    ntok[t] = min(max(sv.n - tok0[t], 0), p.tpt);
    hi_key[t] = ntok[t] == 0 ? 0 : p.causal ? min(sv.len, sv.pos0 + tok0[t] + ntok[t]) : sv.len;
  }
  const int lo_key = p.causal && p.window > 0 ? max(0, sv.pos0 + tok0[0] - p.window + 1) : 0;
  const int hi_all = max(hi_key[0], hi_key[1]);
  const int j0 = lo_key / FA_BN;
#pragma unroll
  for (int t = 0; t < 2; ++t) n_kv[t] = max(0, (hi_key[t] + FA_BN - 1) / FA_BN - j0);
  const int n_max = max(n_kv[0], n_kv[1]);

  const uint32_t sQ = base + L::OFF_Q, sK = base + L::OFF_K, sV = base + L::OFF_V;
  const uint32_t bar_q_full = base + L::OFF_BAR;
  const uint32_t bar_k_full = bar_q_full + 2 * 8;
  const uint32_t bar_k_empty = bar_k_full + STAGES * 8;
  const uint32_t bar_v_full = bar_k_empty + STAGES * 8;
  const uint32_t bar_v_empty = bar_v_full + STAGES * 8;
  const uint32_t bar_s_full = bar_v_empty + STAGES * 8;
  const uint32_t bar_p_full = bar_s_full + 2 * 8;
  const uint32_t bar_o_done = bar_p_full + 2 * 8;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gen_base + L::OFF_MISC);
  WaitCtx wctx{misc + 1, status};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q_full + i * 8, 1);
      mbar_init(bar_s_full + i * 8, 1);
      mbar_init(bar_p_full + i * 8, 4);
      mbar_init(bar_o_done + i * 8, 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_k_full + s * 8, FP4 ? 4 : 1);
      mbar_init(bar_k_empty + s * 8, 1);
      mbar_init(bar_v_full + s * 8, FP4 ? 4 : 1);
      mbar_init(bar_v_empty + s * 8, 1);
    }
    misc[1] = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    if (!FP4) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(misc)), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = misc[0];
  auto S_COL = [](int t) { return (uint32_t)(t * 128); };
  auto O_COL = [](int t) { return (uint32_t)(256 + t * 128); };

  if (warp < 4) reg_dealloc<FP4 ? 40 : FA_OTHER_REGS>();
  if (warp == 0) {
    // ------------------------------- loader -------------------------------
    if (lane == 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (n_kv[t] == 0) continue;
        mbar_expect_tx(bar_q_full + t * 8, (uint32_t)(HALVES * 128 * p.tpt * p.group));
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          tma_load_3d(sQ + t * TILE + h * HALF, &tmQ, bar_q_full + t * 8, h * 64, head * p.group, sv.q0 + tok0[t]);
      }
    }
    if (!FP4) {
      const int boxes = FA_BN / p.box_rows;
      const int slot_mask = (1 << p.batch.page_shift) - 1;
      // lane i < boxes: page of box i; lane i < boxes * HALVES issues box i % boxes of half i / boxes
      auto page_for = [&](int j) {
        const int key = (j0 + j) * FA_BN + lane * p.box_rows;
        const bool used = j < n_max && lane < boxes && key < hi_all && key + p.box_rows > lo_key;
        return used ? page_of(p.batch, b, key, status) : p.batch.num_pages;
      };
      uint32_t stage = 0, phase = 0;
      int pages = page_for(0), k_armed = 0, v_armed = 0;
      for (int j = 0; j < n_max; ++j) {
        const int next = page_for(j + 1);
        const int box = lane % boxes, half = lane / boxes;
        const int pg = __shfl_sync(0xffffffffu, pages, box);
        const int slot = ((j0 + j) * FA_BN + box * p.box_rows) & slot_mask;
        const uint32_t off = stage * TILE + half * HALF + box * p.box_rows * 128;
        if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_k_empty + stage * 8, phase ^ 1, 10))) break;
        if (lane == 0) mbar_expect_tx(bar_k_full + stage * 8, TILE);
        __syncwarp();
        if (half < HALVES) tma_load_4d_tile(sK + off, &tmK, bar_k_full + stage * 8, half * 64, slot, head, pg);
        ++k_armed;
        if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_v_empty + stage * 8, phase ^ 1, 11))) break;
        if (lane == 0) mbar_expect_tx(bar_v_full + stage * 8, TILE);
        __syncwarp();
        if (half < HALVES) tma_load_4d_tile(sV + off, &tmV, bar_v_full + stage * 8, half * 64, slot, head, pg);
        ++v_armed;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
        pages = next;
      }
      if (v_armed < n_max) {
        // a wait gave up: the copies still in flight get their (bounded) time before the shared memory goes
        for (int i = max(0, k_armed - STAGES); i < k_armed; ++i)
          mbar_wait(wctx, bar_k_full + (i % STAGES) * 8, (i / STAGES) & 1, 12);
        for (int i = max(0, v_armed - STAGES); i < v_armed; ++i)
          mbar_wait(wctx, bar_v_full + (i % STAGES) * 8, (i / STAGES) & 1, 13);
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer --------------------------------
    // the whole warp runs the control flow, one elected lane issues (fmha_fwd.cu says why)
    if (n_max > 0) {
      const bool me = elect_one() != 0;
      constexpr uint32_t fmt = F16 ? FMT_F16 : FMT_BF16;
      constexpr uint32_t idesc_qk = make_idesc(fmt, fmt, 0, 0, FA_BM, FA_BN);
      constexpr uint32_t idesc_pv = make_idesc(fmt, fmt, 0, 1, FA_BM, D);
      auto issue_qk = [&](int t, uint32_t k_addr) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk / 4) * HALF + (kk % 4) * 32;
          const uint64_t a = make_smem_desc(sQ + t * TILE + off, 16, 1024, SWZ_128B);
          const uint64_t bd = make_smem_desc(k_addr + off, 16, 1024, SWZ_128B);
          if (me) umma_f16_ss(tmem_base + S_COL(t), a, bd, idesc_qk, kk != 0);
        }
      };
      auto issue_pv = [&](int t, uint32_t v_addr, bool acc) {
#pragma unroll
        for (int kk = 0; kk < FA_BN / 16; ++kk) {
          const uint64_t bd = make_smem_desc(v_addr + kk * 2048, HALF, 1024, SWZ_128B);
          if (me) umma_f16_ts(tmem_base + O_COL(t), tmem_base + S_COL(t) + kk * 8, bd, idesc_pv, acc || kk != 0);
        }
      };
      // V rows of the step that no row of the CTA sees
      auto clear_v = [&](int j, uint32_t v_addr) {
        const int key0 = (j0 + j) * FA_BN;
        const int from = max(lo_key - key0, 0), to = min(hi_all - key0, FA_BN);
        if (from <= 0 && to >= FA_BN) return;
        for (int i = lane; i < FA_BN * HALVES * 8; i += 32) {
          const int r = i / (HALVES * 8), c = i % (HALVES * 8);
          if (r < from || r >= to) st_shared_v4(v_addr + (c >> 3) * HALF + r * 128 + (c & 7) * 16, 0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(wctx, bar_k_full + 0, 0, 20));
#pragma unroll
      for (int t = 0; t < 2 && ok; ++t) {
        if (n_kv[t] == 0) continue;
        if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_q_full + t * 8, 0, 21))) { ok = false; break; }
        tc_fence_after_sync();
        issue_qk(t, sK);
        if (me) umma_commit(bar_s_full + t * 8);
      }
      if (ok && me) umma_commit(bar_k_empty + 0);
      for (int j = 0; j < n_max && ok; ++j) {
        const uint32_t vs = j % STAGES, vph = (j / STAGES) & 1;
        const uint32_t ks = (j + 1) % STAGES, kph = ((j + 1) / STAGES) & 1;
        const bool have_next = j + 1 < n_max;
        if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_v_full + vs * 8, vph, 22))) { ok = false; break; }
        if constexpr (!FP4) clear_v(j, sV + vs * TILE);
        if (have_next && !__all_sync(0xffffffffu, mbar_wait(wctx, bar_k_full + ks * 8, kph, 23))) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j < n_kv[t]) {
            if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_p_full + t * 8, j & 1, 24))) { ok = false; break; }
            tc_fence_after_sync();
            issue_pv(t, sV + vs * TILE, j > 0);
            if (j == n_kv[t] - 1 && me) umma_commit(bar_o_done + t * 8);
          }
          if (j + 1 < n_kv[t]) {
            issue_qk(t, sK + ks * TILE);
            if (me) umma_commit(bar_s_full + t * 8);
          }
        }
        if (!ok) break;
        if (me) umma_commit(bar_v_empty + vs * 8);
        if (have_next && me) umma_commit(bar_k_empty + ks * 8);
      }
    }
  } else if (warp >= 4 && warp < 12) {
    // -------------------------------- softmax ----------------------------------
    reg_alloc<FA_SOFTMAX_REGS>();
    const int t = (warp - 4) >> 2;
    const int q = warp & 3;
    const int row = q * 32 + lane;          // row inside the tile == TMEM lane
    const int tok = row / p.group;
    const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
    const uint32_t tS = lane_base + S_COL(t);
    const uint32_t tO = lane_base + O_COL(t);
    const int n_mine = n_kv[t];
    // keys this row sees (rows that are no token's see none)
    int row_lo = 0, row_hi = 0;
    if (tok < ntok[t]) {
      const int pos = sv.pos0 + tok0[t] + tok;
      row_hi = p.causal ? min(sv.len, pos + 1) : sv.len;
      if (p.causal && p.window > 0) row_lo = max(0, pos - p.window + 1);
    }
    float m_run = -CUDART_INF_F, l_run = 0.0f;
    bool ok = true;
    for (int j = 0; j < n_mine && ok; ++j) {
      if (!mbar_wait(wctx, bar_s_full + t * 8, j & 1, 30)) { ok = false; break; }
      tc_fence_after_sync();
      uint32_t v[FA_BN];
#pragma unroll
      for (int c = 0; c < FA_BN / 32; ++c)
        tmem_ld_32x32b_x32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
      const int key0 = (j0 + j) * FA_BN;
      const int c_hi = row_hi - 1 - key0, c_lo = row_lo - key0;    // first and last column seen
      const bool masked_tile = __any_sync(0xffffffffu, c_hi < FA_BN - 1 || c_lo > 0);
      tmem_wait_ld();
      if (masked_tile) {
#pragma unroll
        for (int i = 0; i < FA_BN; ++i)
          if (i > c_hi || i < c_lo) v[i] = 0xff800000u;  // -inf
      }
      float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
      for (int i = 0; i < FA_BN; i += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          mx[u] = max3(mx[u], __uint_as_float(v[i + 2 * u]), __uint_as_float(v[i + 2 * u + 1]));
      }
      const float rmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      // the score grows with s: the largest s has the largest score (the cap maps -inf to -cap: kept apart)
      const float m_tile = rmax == -CUDART_INF_F ? rmax : paged_score<CAP>(p.score, rmax);
      const float m_new = fmaxf(m_run, m_tile);
      bool need = false;
      float alpha = 1.0f;
      if (m_run == -CUDART_INF_F) {
        m_run = m_new;                       // nothing seen before: O and l are zero
      } else if (m_new - m_run > FA_RESCALE_THRESHOLD) {
        need = true;
        alpha = ex2_approx(m_run - m_new);
        l_run *= alpha;
        m_run = m_new;
      }
      if (__any_sync(0xffffffffu, need)) {
        // S_t(j) complete implies O_t += P_t(j-1) V(j-1) complete (MMAs retire in issue order)
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(tO + c * 32, o);
        }
      }
      const float neg_m = m_run == -CUDART_INF_F ? 0.0f : -m_run;
      uint64_t ls2[4] = {0ull, 0ull, 0ull, 0ull};
      const uint64_t scale2 = CAP ? pack2(p.score.cap_arg, p.score.cap_arg) : pack2(p.score.scale_log2, p.score.scale_log2);
      const uint64_t negm2 = pack2(neg_m, neg_m);
#pragma unroll
      for (int c = 0; c < FA_BN / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a, d;
          const float sa = __uint_as_float(v[c * 32 + 2 * i]), sd = __uint_as_float(v[c * 32 + 2 * i + 1]);
          if (CAP) {
            // a masked entry keeps its -inf through the cap
            float xa, xd;
            unpack2(fma2(pack2(sa, sd), scale2, 0ull), xa, xd);
            const float off = p.score.cap_out + neg_m;
            a = ex2_approx(fmaf(-2.0f * p.score.cap_out, paged_rcp(1.0f + ex2_approx(xa)), off));
            d = ex2_approx(fmaf(-2.0f * p.score.cap_out, paged_rcp(1.0f + ex2_approx(xd)), off));
            if (masked_tile) {
              a = sa == -CUDART_INF_F ? 0.0f : a;
              d = sd == -CUDART_INF_F ? 0.0f : d;
            }
          } else {
            float xa, xd;
            unpack2(fma2(pack2(sa, sd), scale2, negm2), xa, xd);
            a = ex2_approx(xa);
            d = ex2_approx(xd);
          }
          ls2[i & 3] = add2(ls2[i & 3], pack2(a, d));
          pk[i] = F16 ? pack_f16x2(a, d) : pack_bf16x2(a, d);
        }
        tmem_st_32x32b_x16(tS + c * 16, pk);
      }
      float ls[4];
      {
        const uint64_t s01 = add2(ls2[0], ls2[1]), s23 = add2(ls2[2], ls2[3]);
        unpack2(s01, ls[0], ls[1]);
        unpack2(s23, ls[2], ls[3]);
      }
      l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
      tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_p_full + t * 8);
    }
    // ------------------------------- epilogue ----------------------------------
    // rows of this warp that are tokens, staged in Q_t's shared memory (free: all S_t MMAs retired) and copied out
    // 16 lanes (D = 64: 8) to a row
    if (ok && n_mine > 0) ok = mbar_wait(wctx, bar_o_done + t * 8, 0, 31);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after_sync();
      const float inv_l = l_run == 0.0f ? 0.0f : (FP4 ? p.out_scale : 1.0f) / l_run;
      const uint32_t stage_row = sQ + t * TILE + (uint32_t)row * 128;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n_mine > 0) {
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float lo = __uint_as_float(o[e * 8 + 2 * x]) * inv_l;
            const float hi = __uint_as_float(o[e * 8 + 2 * x + 1]) * inv_l;
            w[x] = F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
          }
          const uint32_t chunk = (uint32_t)((c & 1) * 4 + e);
          st_shared_v4(stage_row + (c >> 1) * HALF + ((chunk ^ (uint32_t)(lane & 7)) << 4), w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      constexpr int LPR = D / 8;                    // lanes per row
      for (int i = lane / LPR; i < 32; i += 32 / LPR) {
        const int r = q * 32 + i, rt = r / p.group;
        if (rt >= ntok[t]) break;
        const int c = lane % LPR;
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(sQ + t * TILE + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)));
        uint16_t* dst = p.out + (long long)(sv.q0 + tok0[t] + rt) * p.o_ts +
                        (long long)(head * p.group + r - rt * p.group) * p.o_hs + c * 8;
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  } else if (FP4 && warp >= 12) {
    // ---------------------- NVFP4 rows to 16-bit operand tiles ----------------------
    reg_dealloc<56>();
    const int r = threadIdx.x - 384;                // key of the step
    constexpr int WORDS = D / 8;                    // packed words per row
    uint32_t wk[WORDS], wv[WORDS], sk[D / 64], sw[D / 64];
    const int slot_mask = (1 << p.batch.page_shift) - 1;
    auto fetch = [&](int j, const uint8_t* pool, const long long (&st)[3], const uint8_t* spool, const long long (&sst)[3],
                     uint32_t (&w)[WORDS], uint32_t (&s)[D / 64]) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) s[i] = 0;
      const int key = (j0 + j) * FA_BN + r;
      if (j >= n_max || key < lo_key || key >= hi_all) return;    // unseen: zeros
      const int pg = page_of(p.batch, b, key, status);
      if (pg >= p.batch.num_pages) return;
      const uint8_t* row = pool + pg * st[0] + head * st[1] + (key & slot_mask) * st[2];
      const uint8_t* srow = spool + pg * sst[0] + head * sst[1] + (key & slot_mask) * sst[2];
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(row) + i);
        w[4 * i] = x.x;
        w[4 * i + 1] = x.y;
        w[4 * i + 2] = x.z;
        w[4 * i + 3] = x.w;
      }
#pragma unroll
      for (int i = 0; i < D / 64; ++i) s[i] = __ldg(reinterpret_cast<const uint32_t*>(srow) + i);
    };
    auto expand = [&](uint32_t dst, const uint32_t (&w)[WORDS], const uint32_t (&s)[D / 64]) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const uint32_t sc = expand_scale<F16>(s[i / 8] >> (8 * ((i / 2) & 3)));
        uint32_t o[4];
        expand8<F16>(w[i], sc, o);
        st_shared_v4(dst + (i >> 3) * HALF + r * 128 + (((i & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    fetch(0, p.k, p.k_st, p.ks, p.ks_st, wk, sk);
    fetch(0, p.v, p.v_st, p.vs, p.vs_st, wv, sw);
    uint32_t stage = 0, phase = 0;
    for (int j = 0; j < n_max; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_k_empty + stage * 8, phase ^ 1, 10))) break;
      expand(sK + stage * TILE, wk, sk);
      if (lane == 0) mbar_arrive(bar_k_full + stage * 8);
      fetch(j + 1, p.k, p.k_st, p.ks, p.ks_st, wk, sk);
      if (!__all_sync(0xffffffffu, mbar_wait(wctx, bar_v_empty + stage * 8, phase ^ 1, 11))) break;
      expand(sV + stage * TILE, wv, sw);
      if (lane == 0) mbar_arrive(bar_v_full + stage * 8);
      fetch(j + 1, p.v, p.v_st, p.vs, p.vs_st, wv, sw);
      if (++stage == STAGES) { stage = 0; phase ^= 1; }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
  // The row-block kernel of the same call runs beside this one and writes other rows.  Whatever follows in the stream
  // waits for this kernel only, so no CTA of it ends before that one has.
  grid_dep_wait();
}

template <int D, bool F16, bool CAP, bool FP4>
int launch_tile(const PagedAttnArgs& a) {
  using L = TileSmem<D, FP4>;
  const b200h::DeviceInfo* di = b200h::device_info();
  if (!di) return B200_ERR_CUDA;
  const b200tile_paged_cache& c = *a.cache;
  TileParams p = {};
  p.batch = a.batch;
  p.score = a.score;
  p.kv_heads = c.kv_heads;
  p.group = a.q_heads / c.kv_heads;
  p.tpt = FA_BM / p.group;
  p.causal = a.causal;
  p.window = a.window;
  p.row_limit = a.row_limit;
  p.box_rows = std::min(c.page_size, FA_BN);
  p.out = static_cast<uint16_t*>(a.out);
  p.o_ts = a.o_ts;
  p.o_hs = a.o_hs;
  const CUtensorMapDataType dt = F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tmQ, tmK = {}, tmV = {};
  const uint64_t row = (uint64_t)D * 2;
  if (int rc = b200h::encode_tmap_3d(&tmQ, dt, 2, a.q, D, a.q_heads, a.batch.tokens,
                                     a.q_heads > 1 ? (uint64_t)a.q_hs * 2 : row,
                                     a.batch.tokens > 1 ? (uint64_t)a.q_ts * 2 : row, 64, p.group, p.tpt,
                                     CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if constexpr (FP4) {
    p.score.scale_log2 *= c.k_global * 128.0f;      // the expanded operands are value * 2^-7
    p.score.cap_arg *= c.k_global * 128.0f;
    p.out_scale = c.v_global * 128.0f;
    p.k = static_cast<const uint8_t*>(c.k);
    p.v = static_cast<const uint8_t*>(c.v);
    p.ks = static_cast<const uint8_t*>(c.k_scales);
    p.vs = static_cast<const uint8_t*>(c.v_scales);
    for (int i = 0; i < 3; ++i) {
      p.k_st[i] = c.k_strides[i]; p.v_st[i] = c.v_strides[i];
      p.ks_st[i] = c.k_scale_strides[i]; p.vs_st[i] = c.v_scale_strides[i];
    }
  } else {
    if (int rc = b200h::encode_tmap_pages(&tmK, dt, c.k, D, c.page_size, c.kv_heads, c.num_pages, c.k_strides, 64, p.box_rows))
      return rc;
    if (int rc = b200h::encode_tmap_pages(&tmV, dt, c.v, D, c.page_size, c.kv_heads, c.num_pages, c.v_strides, 64, p.box_rows))
      return rc;
  }
  auto kern = fmha_paged_tile_kernel<D, F16, CAP, FP4>;
  static b200h::DeviceOnce attr_done;
  if (!attr_done.test(di->ordinal)) {
    B200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
    attr_done.set(di->ordinal);
  }
  // at most one partly filled pair per sequence that has rows for this kernel
  const long long tokens = a.batch.tokens;
  const long long some = std::min<long long>(a.batch.batch, tokens * p.group / (a.row_limit + 1LL));
  const long long ctas = (tokens / (2 * p.tpt) + some) * p.kv_heads;
  if (ctas > 0x7fffffffLL) return b200h::set_error(B200_ERR_INVALID, "paged_attention: grid too large");
  if (ctas == 0) return B200_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::TOTAL;
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tmQ, tmK, tmV, p, di->status));
  return B200_OK;
}

}  // namespace
}  // namespace b200

int b200_paged_tile_dispatch(const PagedAttnArgs& a) {
  using namespace b200;
  const b200tile_paged_cache& c = *a.cache;
#define B200_PT(D_, F_, C_, Q_) return launch_tile<D_, F_, C_, Q_>(a)
#define B200_PT_CAP(D_, F_, Q_) do { if (a.capped) B200_PT(D_, F_, true, Q_); B200_PT(D_, F_, false, Q_); } while (0)
#define B200_PT_FMT(D_, F_) do { if (c.format) B200_PT_CAP(D_, F_, true); B200_PT_CAP(D_, F_, false); } while (0)
  if (c.head_dim == 128 && a.dtype == 0) B200_PT_FMT(128, false);
  if (c.head_dim == 128 && a.dtype == 1) B200_PT_FMT(128, true);
  if (c.head_dim == 64 && a.dtype == 0) B200_PT_FMT(64, false);
  if (c.head_dim == 64 && a.dtype == 1) B200_PT_FMT(64, true);
#undef B200_PT_FMT
#undef B200_PT_CAP
#undef B200_PT
  return b200h::set_error(B200_ERR_UNSUPPORTED, "paged_attention: no kernel for head_dim %d (64 and 128 are provided)",
                          c.head_dim);
}

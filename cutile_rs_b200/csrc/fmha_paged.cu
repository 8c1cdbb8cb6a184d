// Attention of few query rows over a paged key/value cache, 16-bit or NVFP4 (every length, mask and row count is
// handled here; sequences with many rows go to fmha_paged_tile.cu).
//
//   o_i = sum_j softmax_j(score(q_i . k_j)) v_j      over the keys j < len that the masks of row i leave
//
// Query rows are packed per K/V head (row = token * group + head of the group) in blocks of 8 or 16, so that a K/V row
// is read once for all heads that share it.  What bounds it is HBM: each cached byte is used for `group` rows only.
// 8 x 65536 keys of 8 x 128: 333 us, 6.4 TB/s; 64 sequences to 8192 keys 157 us, 6.0 TB/s; launch, first copies and merge take
// about 9 us of any call.  NVFP4, 32 sequences to 16384 keys: 69 us, 3.9 TB/s, of 41 at the copy rate.  57 of them remain
// without the arithmetic: 9 to start and merge, and copies of 16 bytes a lane that reach 5.6 TB/s; the arithmetic adds 12.
// 327 instructions a step of 16 keys, 128 of them conversions and scale products, fill 59 % of the issue slots; three warps
// a scheduler, what the registers allow, wait for one another's fixed latencies in the rest.
//
// Work split.  One worker is ONE WARP.  Sequence b has steps(b) steps of 16 keys, an item is (sequence, row block, K/V
// head), and the steps of all items form one line that is cut into equal runs, one per worker.  Lengths may be as
// uneven as they like: every warp of the machine reads the same number of bytes, whatever the batch looks like, and
// nothing about the lengths has to be known on the host (a captured graph may be replayed with other lengths).  A run
// that holds whole items writes their output; a run that holds part of an item writes (m, l, O) in 32 bits, at most
// two such parts per worker, and the merge kernel adds the parts of an item in the order of the workers.  No result
// depends on an atomic (only the status record of a bad page does) or on an earlier launch: the same call gives the same
// bits.  (A run is taken by a few workers, one per head of `heads_abreast`: the line counts groups of heads.)
//
// Inside a worker the products are transposed, S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16): the 16 rows of the
// instruction are keys (or head dimensions) and its 8 columns the query rows, so 8 rows fill it; the usual orientation
// would multiply a block half full of zeros and hold twice the accumulators.  P^T comes from S^T by movmatrix.
#include <math_constants.h>

#include <algorithm>

#include "paged_common.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ void ldm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t mat_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(ok ? BYTES : 0)
               : "memory");
}
constexpr int STEP = 16;             // keys per step
// Warps per CTA, one CTA per SM.  16-bit, D = 128: 8 rings of 3 x 8 KB fill the shared memory; D = 64 halves the step and
// takes half again as many warps.  NVFP4: what the registers allow (16 rows of 128: 8 warps 97, 12 that spill 108 us for 32 x
// 16384 keys and four tokens).
constexpr int split_warps(bool fp4, int d, int nt) { return fp4 ? (d == 128 && nt == 2 ? 8 : 12) : d == 64 ? 12 : 8; }
constexpr float LAZY = 8.0f;         // the running reference of the exponents may lag behind the maximum by this

struct SplitParams {
  PagedBatch batch;
  const uint16_t* q;
  uint16_t* out;
  long long q_ts, q_hs, o_ts, o_hs;
  ScoreParams score;
  int kv_heads, group, causal, window, row_limit;
  float out_scale;                   // FP4: v_global (the score carries k_global)
  float* part;
  int4* desc;
  long long part_floats;
  int workers, by_item, rb_max;
  int heads_abreast, head_groups;    // neighbouring workers take these many heads of the same keys; kv_heads / that
  int coop;                          // CTAs per item (a cluster), whose warps share its steps: no parts, no merge kernel; or 0
  int min_steps;
  // FP4 operands, strides in bytes: those that are multiplied in every step fit in 32 bits
  const uint8_t *k, *v, *ks, *vs;
  long long k_head, v_head, ks_head, vs_head;
  uint32_t k_page, v_page, ks_page, vs_page, k_slot, v_slot, ks_slot, vs_slot;
};

// Steps of one item of the sequence, from key step `base`; 0 for a sequence without rows here, and at least 1 for one
// with rows (a row that sees no key still has to be written).
struct SeqWork {
  SeqView s;
  int base, steps, rbs;
};
template <int RB>
__device__ __forceinline__ SeqWork seq_work(const SplitParams& p, int b) {
  SeqWork w;
  w.s = seq_view(p.batch, b);
  const int rows = w.s.n * p.group;
  w.rbs = rows > p.row_limit ? 0 : (rows + RB - 1) / RB;
  int lo = 0, hi = w.s.len;
  if (p.causal) {
    hi = min(hi, w.s.pos0 + w.s.n);
    if (p.window > 0) lo = window_start(w.s.pos0, p.window);
  }
  w.base = hi > lo ? lo / STEP : 0;
  w.steps = hi > lo ? (hi + STEP - 1) / STEP - w.base : 1;
  return w;
}

// Per-warp state of one part of an item: the block's rows as this lane sees them.
template <int NT>
struct RowMask {
  int lo[NT][2], hi[NT][2];          // visible keys of query rows 8 nt + 2t and + 1
  int lo_min, hi_max;                // over the block
  int lo_max, hi_min;                // a step inside [lo_max, hi_min) needs no mask
};
template <int NT>
__device__ __forceinline__ RowMask<NT> row_mask(const SplitParams& p, const SeqView& s, int rb, int lane) {
  RowMask<NT> m;
  const int rows = s.n * p.group, first = rb * 8 * NT;
  auto range = [&](int row, int& lo, int& hi) {
    lo = 0;
    hi = s.len;
    if (p.causal) {
      const int pos = s.pos0 + row / p.group;
      hi = min(hi, pos + 1);
      if (p.window > 0) lo = window_start(pos, p.window);
    }
  };
  int l0, h0, l1, h1;
  range(first, l0, h0);
  range(min(rows, first + 8 * NT) - 1, l1, h1);
  m.lo_min = l0;
  m.lo_max = l1;
  m.hi_min = h0;
  m.hi_max = h1;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = first + nt * 8 + (lane & 3) * 2 + j;
      if (row < rows) range(row, m.lo[nt][j], m.hi[nt][j]);
      else { m.lo[nt][j] = 0; m.hi[nt][j] = 0; }
    }
  return m;
}

// The online softmax of one step: s[nt] holds S^T (keys g and g + 8, rows 2t and 2t + 1 of block nt) and becomes the
// B operand of O^T += V^T P^T.  Statistics in 32 bits.  The reference m that is subtracted from the exponents is the
// same for all lanes of a row and moves only when some score exceeds it by more than 2^8: one vote per step instead of
// a maximum over eight lanes.  P <= 2^(8 + p_shift) then, and l >= 1 for any row that saw a key.  P is handed over as a
// 16-bit value plus the 16-bit rest of it (HILO): the rounding of P alone would put an error as large as the output's own
// rounding beside it, and the second product costs nothing next to the loads.
template <bool F16, int KS, int NT, int DT, bool CAP, bool HILO>
__device__ __forceinline__ void softmax_step(const ScoreParams (&sp)[NT][2], const RowMask<NT>& rm, int key0, int lane,
                                             bool ragged, float (&s)[KS][NT][4], float (&m_run)[NT][2],
                                             float (&l_run)[NT][2], float (&o)[DT][NT][4], uint32_t (&pb)[KS][NT][2],
                                             uint32_t (&pl)[KS][NT][2]) {
  const int g = lane >> 2;
  bool over = false;
  if (CAP) {
    auto capped = [&](auto&& score) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[ks][nt][e] = score(sp[nt][e & 1], s[ks][nt][e]);
    };
    if (sp[0][0].cap_out <= CAP_SMALL_OUT) capped([](const ScoreParams& a, float x) { return paged_score_near(a, x); });
    else capped([](const ScoreParams& a, float x) { return paged_score<true>(a, x); });
  }
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = CAP ? s[ks][nt][e] : paged_score<false>(sp[nt][e & 1], s[ks][nt][e]);
        if (ragged) {
          const int key = key0 + ks * STEP + g + (e >> 1) * 8;
          if (key < rm.lo[nt][e & 1] || key >= rm.hi[nt][e & 1]) x = -CUDART_INF_F;
        }
        s[ks][nt][e] = x;
        over |= x > m_run[nt][e & 1] + LAZY;
      }
  if (__any_sync(0xffffffffu, over)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = fmaxf(s[0][nt][j], s[0][nt][2 + j]);
#pragma unroll
        for (int ks = 1; ks < KS; ++ks) mx = fmaxf(mx, fmaxf(s[ks][nt][j], s[ks][nt][2 + j]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(m_run[nt][j], mx);
        const float alpha = m_new == m_run[nt][j] ? 1.0f : ex2_approx(m_run[nt][j] - m_new);
        m_run[nt][j] = m_new;
        l_run[nt][j] *= alpha;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          o[i][nt][j] *= alpha;
          o[i][nt][2 + j] *= alpha;
        }
      }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float m_use[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)                        // -inf: nothing seen yet
      m_use[j] = m_run[nt][j] == -CUDART_INF_F ? 0.0f : m_run[nt][j] - p_shift<F16>();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[ks][nt][j] = ex2_approx(s[ks][nt][j] - m_use[j]);
        s[ks][nt][2 + j] = ex2_approx(s[ks][nt][2 + j] - m_use[j]);
        l_run[nt][j] += s[ks][nt][j] + s[ks][nt][2 + j];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t hi = paged_pack16<F16>(s[ks][nt][2 * h], s[ks][nt][2 * h + 1]);
        pb[ks][nt][h] = mat_trans(hi);
        if (HILO) {
          const float2 f = paged_unpack16<F16>(hi);
          pl[ks][nt][h] = mat_trans(paged_pack16<F16>(s[ks][nt][2 * h] - f.x, s[ks][nt][2 * h + 1] - f.y));
        }
      }
    }
  }
}

// One 16-bit K/V step: TMA boxes of 16 keys x 64 elements with the 128-byte swizzle, in a ring of the warp's own.
template <int D, int NT>
struct Core16 {
  static constexpr int WARPS = split_warps(false, D, NT), STAGES = D == 64 ? 4 : 3;
  static constexpr int KS = D == 64 ? 2 : 1;           // steps per iteration
  static constexpr int HALVES = D / 64, BOX = STEP * 128, TILE = HALVES * BOX, STAGE = 2 * TILE;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int SMEM = 1024 + RING + WARPS * STAGES * 8 + 16;
};
// One FP4 step: 16 keys of packed values and scales copied with cp.async into a ring of the warp's own.
template <int D, int NT>
struct Core4 {
  static constexpr int WARPS = split_warps(true, D, NT), STAGES = 6;
  static constexpr int KS = 2;
  static constexpr int ROW = D / 2, SROW = D / 16;
  static constexpr int STAGE = 2 * STEP * (ROW + SROW);
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int SMEM = RING;
};

// One 16 x 8 tile of O^T (numerators and their sums) to the output rows of block nt.
template <int D, bool F16, bool FP4, int NT>
__device__ __forceinline__ void write_tile(const SplitParams& p, const SeqView& sv, int rb, int h, int nt, int c, int lane,
                                           const float (&o)[4], const float (&l)[2]) {
  const int g = lane >> 2, t = lane & 3;
  // a row that saw nothing is 0; NaN stays NaN
  const float i0 = l[0] == 0.0f ? 0.0f : (FP4 ? p.out_scale : 1.0f) / l[0];
  const float i1 = l[1] == 0.0f ? 0.0f : (FP4 ? p.out_scale : 1.0f) / l[1];
  // (dimension, rows 2t, 2t + 1) -> (row g, dimensions 2t, 2t + 1 of the tile's eight)
  const uint32_t a = mat_trans(paged_pack16<F16>(o[0] * i0, o[1] * i1));
  const uint32_t d2 = mat_trans(paged_pack16<F16>(o[2] * i0, o[3] * i1));
  const int row = rb * 8 * NT + nt * 8 + g;
  const int tok = row / p.group;
  if (tok >= sv.n) return;
  uint16_t* orow = p.out + (long long)(sv.q0 + tok) * p.o_ts + (long long)(h * p.group + row - tok * p.group) * p.o_hs;
  if constexpr (!FP4) {
    *reinterpret_cast<uint32_t*>(orow + c * 16 + 2 * t) = a;
    *reinterpret_cast<uint32_t*>(orow + c * 16 + 8 + 2 * t) = d2;
  } else {
    // tile row m stands for dimension D/8 m + 2c, row m + 8 for the next one
    *reinterpret_cast<uint32_t*>(orow + (D / 8) * (2 * t) + 2 * c) = __byte_perm(a, d2, 0x5410);
    *reinterpret_cast<uint32_t*>(orow + (D / 8) * (2 * t + 1) + 2 * c) = __byte_perm(a, d2, 0x7632);
  }
}

// Finds the first piece of work of every worker of the CTA.  s_sum[i] = steps of the sequences before chunk i.
template <int RB, int THREADS>
__device__ __forceinline__ long long block_line(const SplitParams& p, long long* s_sum) {
  const int per = (p.batch.batch + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int b = threadIdx.x * per; b < min(p.batch.batch, (int)(threadIdx.x + 1) * per); ++b) {
    const SeqWork w = seq_work<RB>(p, b);
    mine += (long long)w.rbs * p.head_groups * w.steps;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  __shared__ long long s_warp[32];
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  long long before = 0, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  s_sum[threadIdx.x] = before + inc - mine;
  __syncthreads();
  return total;
}

template <int D, bool F16, int NT, bool CAP, bool FP4>
__global__ void __launch_bounds__((FP4 ? Core4<D, NT>::WARPS : Core16<D, NT>::WARPS) * 32, 1)
fmha_paged_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ SplitParams p, uint32_t* status) {
  using C16 = Core16<D, NT>;
  using C4 = Core4<D, NT>;
  constexpr int WARPS = FP4 ? C4::WARPS : C16::WARPS, THREADS = WARPS * 32;
  constexpr int STAGES = FP4 ? C4::STAGES : C16::STAGES;
  constexpr int KS = FP4 ? C4::KS : C16::KS;
  static_assert(!FP4 || STAGES % KS == 0, "a group of copies is KS steps");
  constexpr int DT = D / 16, RB = 8 * NT;
  constexpr bool HILO = !FP4 || F16;         // bf16 output over f16 probabilities needs no second product
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long s_sum[THREADS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  // the merge kernel may be scheduled now; it waits for this grid before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const uint32_t base = FP4 ? smem_u32(smem_raw) : (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint32_t ring, bars = 0;
  WaitCtx wctx{nullptr, status};
  if constexpr (!FP4) {
    ring = base + warp * (STAGES * C16::STAGE);
    bars = base + C16::RING + warp * STAGES * 8;
    volatile uint32_t* abort_flag =
        reinterpret_cast<volatile uint32_t*>(smem_raw + (base - smem_u32(smem_raw)) + C16::RING + WARPS * STAGES * 8);
    wctx.abort_flag = abort_flag;
    if (threadIdx.x == 0) *abort_flag = 0;
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      for (int s = 0; s < STAGES; ++s) mbar_init(bars + s * 8, 1);
      fence_mbar_init();
    }
  } else {
    ring = base + warp * (STAGES * C4::STAGE);
  }
  long long per = 0, u = 0, u_end = 0, line = 0;
  int b, wid = 0, coop_rb = 0, coop_h = 0;
  SeqWork sw;
  if (p.coop) {
    const int item = blockIdx.x / p.coop;               // (sequence * rb_max + row block) * kv_heads + head
    b = item / (p.rb_max * p.kv_heads);
    coop_rb = item / p.kv_heads % p.rb_max;
    coop_h = item % p.kv_heads;
    sw = seq_work<RB>(p, b);
    if (coop_rb >= sw.rbs) return;                      // the whole cluster
    __syncthreads();
    u_end = 1;
  } else {
    const long long total = block_line<RB, THREADS>(p, s_sum);
    wid = warp * gridDim.x + blockIdx.x;                // neighbouring runs on different SMs
    const int runs = p.workers / p.heads_abreast;
    per = (total + runs - 1) / runs;
    if (per < p.min_steps) per = p.min_steps;
    u = (long long)(wid / p.heads_abreast) * per;
    u_end = min(total, u + per);
    if (!p.by_item) {
      if (lane == 0) p.desc[wid] = make_int4(0, 0, 0, 0);
    } else {
      // items that do not exist in this launch: nobody else writes their descriptors
      for (int i = blockIdx.x * THREADS + threadIdx.x; i < p.batch.batch * p.rb_max * p.kv_heads; i += gridDim.x * THREADS)
        if (i / p.kv_heads % p.rb_max >= seq_work<RB>(p, i / (p.rb_max * p.kv_heads)).rbs) p.desc[i] = make_int4(0, 0, 0, 0);
    }
    if (u >= u_end) return;

    // the sequence that holds step u: binary search over the chunks, then along the chunk
    int c_lo = 0, c_hi = THREADS - 1;
    while (c_lo < c_hi) {
      const int mid = (c_lo + c_hi + 1) >> 1;
      if (s_sum[mid] <= u) c_lo = mid;
      else c_hi = mid - 1;
    }
    b = c_lo * ((p.batch.batch + THREADS - 1) / THREADS);
    line = s_sum[c_lo];                                 // first step of sequence b
    sw = seq_work<RB>(p, b);
    while (line + (long long)sw.rbs * p.head_groups * sw.steps <= u) {
      line += (long long)sw.rbs * p.head_groups * sw.steps;
      if (++b >= p.batch.batch) return;
      sw = seq_work<RB>(p, b);
    }
  }

  uint32_t ring_at = 0;        // steps taken through the ring since the kernel began (stage and phase of the next)
  const int rowk = ((lane >> 3) & 1) * 8 + (lane & 7), rowv = (lane >> 4) * 8 + (lane & 7);
  const int ck = lane >> 4, cv = (lane >> 3) & 1;

  while (u < u_end) {
    int item = 0, st0, st1, rb, h;
    if (p.coop) {
      const int share = (sw.steps + p.coop * WARPS - 1) / (p.coop * WARPS);
      st0 = min(sw.steps, ((int)blockIdx.x % p.coop * WARPS + warp) * share);
      st1 = min(sw.steps, st0 + share);
      rb = coop_rb;
      h = coop_h;
    } else {
      const long long rel = u - line;
      item = (int)(rel / sw.steps);
      st0 = (int)(rel - (long long)item * sw.steps);
      st1 = (int)min((long long)sw.steps, st0 + (u_end - u));
      rb = item / p.head_groups;
      h = (item - rb * p.head_groups) * p.heads_abreast + wid % p.heads_abreast;
    }
    const SeqView& sv = sw.s;
    RowMask<NT> rm = row_mask<NT>(p, sv, rb, lane);
    // the part's key steps, cut to what the block's rows can see
    const int k0 = max(sw.base + st0, rm.lo_min / STEP);
    const int k1 = rm.hi_max > rm.lo_min ? min(sw.base + st1, (rm.hi_max + STEP - 1) / STEP) : 0;
    const int nk = k1 - k0;
    // with two steps per iteration an odd number leaves the last one without a partner: what stands in its place is
    // another worker's or nobody's, and lies behind every row's range
    if (KS > 1 && nk > 0) {
      rm.hi_max = min(rm.hi_max, k1 * STEP);
      rm.hi_min = min(rm.hi_min, k1 * STEP);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) rm.hi[nt][j] = min(rm.hi[nt][j], k1 * STEP);
    }

    // page numbers of 32 steps at a time, one per lane; with FP4's shorter steps the next 32 are on their way
    int pages = 0, pages_ahead = 0, pages_at = 0;
    auto fetch_pages = [&](int i) { return i + lane < nk ? page_of(p.batch, b, (k0 + i + lane) * STEP, status) : 0; };
    auto page_at = [&](int i) {                       // of step i, for steps in rising order
      while (i - pages_at >= 32) {
        pages_at += 32;
        pages = FP4 ? pages_ahead : fetch_pages(pages_at);
        if (FP4) pages_ahead = fetch_pages(pages_at + 32);
      }
      return __shfl_sync(0xffffffffu, pages, i - pages_at);
    };
    const int slot_mask = (1 << p.batch.page_shift) - 1;
    // FP4: where this lane's pieces of a step lie in the pools, for page 0 and slot 0 of this head
    const uint8_t *k_lane = nullptr, *v_lane = nullptr, *s_lane = nullptr;
    uint32_t s_page = 0, s_slot = 0;
    if constexpr (FP4) {
      constexpr int CH = C4::ROW / 16;
      k_lane = p.k + (long long)h * p.k_head + (long long)(lane / CH) * p.k_slot + (lane % CH) * 16;
      v_lane = p.v + (long long)h * p.v_head + (long long)(lane / CH) * p.v_slot + (lane % CH) * 16;
      const bool is_v = lane >= 16;                   // scales: K's rows in the first half of the lanes, V's in the second
      s_page = is_v ? p.vs_page : p.ks_page;
      s_slot = is_v ? p.vs_slot : p.ks_slot;
      s_lane = (is_v ? p.vs : p.ks) + (long long)h * (is_v ? p.vs_head : p.ks_head) + (long long)(lane & 15) * s_slot;
    }
    // FP4: this lane's pieces of the step issued last; the next step of the same page is one addition away
    const uint8_t *k_from = nullptr, *v_from = nullptr, *s_from = nullptr;
    bool page_ok = false;
    auto issue = [&](int i, uint32_t dst) {
      if (i >= nk) return;                            // warp-uniform
      const int slot = ((k0 + i) * STEP) & slot_mask;
      if constexpr (!FP4) {
        const int pg = page_at(i);
        const uint32_t bar = bars + ((ring_at + i) % STAGES) * 8;
        if (lane == 0) {
          mbar_expect_tx(bar, C16::STAGE);
#pragma unroll
          for (int x = 0; x < C16::HALVES; ++x) {
            tma_load_4d(dst + x * C16::BOX, &tmK, bar, x * 64, slot, h, pg);
            tma_load_4d(dst + C16::TILE + x * C16::BOX, &tmV, bar, x * 64, slot, h, pg);
          }
        }
      } else {
        if (i == 0 || slot == 0) {
          const int pg = page_at(i);
          page_ok = pg < p.batch.num_pages;
          const uint32_t pgc = page_ok ? pg : 0;      // a valid address for the copies that read nothing
          k_from = k_lane + (uint64_t)pgc * p.k_page + (uint64_t)(uint32_t)slot * p.k_slot;
          v_from = v_lane + (uint64_t)pgc * p.v_page + (uint64_t)(uint32_t)slot * p.v_slot;
          s_from = s_lane + (uint64_t)pgc * s_page + (uint64_t)(uint32_t)slot * s_slot;
        } else {
          k_from += (uint64_t)STEP * p.k_slot;
          v_from += (uint64_t)STEP * p.v_slot;
          s_from += (uint64_t)STEP * s_slot;
        }
        constexpr int CH = C4::ROW / 16, ROWS = 32 / CH;   // 16-byte chunks per row; rows a pass of the warp covers
#pragma unroll
        for (int c = 0; c < STEP / ROWS; ++c) {
          cp_async_16(dst + c * 512 + lane * 16, k_from + (uint64_t)(c * ROWS) * p.k_slot, page_ok);
          cp_async_16(dst + STEP * C4::ROW + c * 512 + lane * 16, v_from + (uint64_t)(c * ROWS) * p.v_slot, page_ok);
        }
        cp_async_small<C4::SROW>(dst + 2 * STEP * C4::ROW + lane * C4::SROW, s_from, page_ok);
      }
    };
    constexpr uint32_t STAGE_BYTES = FP4 ? C4::STAGE : C16::STAGE;
    // FP4: an iteration's KS slots lie side by side; those being worked on, and those the next copies go to
    uint32_t group_at = ring, group_to = ring + (STAGES - KS) * STAGE_BYTES;
    if (nk > 0) {
      pages = fetch_pages(0);
      if (FP4) pages_ahead = fetch_pages(32);
#pragma unroll
      for (int s = 0; s < STAGES - (FP4 ? KS : 0); ++s) {
        issue(s, ring + (FP4 ? s : (ring_at + s) % STAGES) * STAGE_BYTES);
        if (FP4 && s % KS == KS - 1) asm volatile("cp.async.commit_group;" ::: "memory");
      }
    }

    // Q^T as the B operand: query row 8 nt + g, two adjacent dimensions per register (FP4: the pairs that the K words
    // unpack to, see below; the row is brought to a power of two near 1 first, so that f16 holds it whatever its size)
    uint32_t qb[NT][DT][2];
    ScoreParams sp[NT][2];                            // of the rows 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      sp[nt][0] = sp[nt][1] = p.score;
      const int row = rb * RB + nt * 8 + g;
      const int tok = row / p.group;
      const bool ok = tok < sv.n;
      const uint16_t* qr = p.q + (long long)(sv.q0 + (ok ? tok : 0)) * p.q_ts +
                           (long long)(h * p.group + (ok ? row - tok * p.group : 0)) * p.q_hs;
      if constexpr (!FP4) {
#pragma unroll
        for (int ks = 0; ks < DT; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qb[nt][ks][x] = ok ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + x * 8 + 2 * t) : 0u;
      } else {
        // lane t holds dimensions [D/4 t, D/4 (t + 1)); word w of 8 of them gives k-steps 2w and 2w + 1
        float f[D / 4];
        float mx = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t w = ok ? *reinterpret_cast<const uint32_t*>(qr + t * (D / 4) + 2 * i) : 0u;
          const float2 v = paged_unpack16<F16>(w);
          f[2 * i] = v.x;
          f[2 * i + 1] = v.y;
          mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // power of two with mx * inv in [1, 2); rows that are zero, infinite or NaN keep factor 1
        const uint32_t e = __float_as_uint(mx) & 0x7f800000u;
        const bool scaled = e > (27u << 23) && e < (227u << 23);
        const float inv = scaled ? __uint_as_float((254u << 23) - e) : 1.0f;
        const float unit = scaled ? __uint_as_float(e) : 1.0f;
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int x = 0; x < 4; ++x)                 // byte x of the word
            qb[nt][2 * w + (x >> 1)][x & 1] = pack_f16x2(f[w * 8 + 2 * x] * inv, f[w * 8 + 2 * x + 1] * inv);
        // rows 2t and 2t + 1 sit in the lanes with g = 2t, 2t + 1
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float f = __shfl_sync(0xffffffffu, unit, 8 * t + 4 * j);
          sp[nt][j].scale_log2 = factor_in_range(sp[nt][j].scale_log2 * f);
          sp[nt][j].cap_arg = factor_in_range(sp[nt][j].cap_arg * f);
        }
      }
    }

    float m_run[NT][2], l_run[NT][2], o[DT][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt][0] = m_run[nt][1] = -CUDART_INF_F;
      l_run[nt][0] = l_run[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;
    }

    for (int i = 0; i < nk; i += KS) {
      const int key0 = (k0 + i) * STEP;
      const bool ragged = key0 < rm.lo_max || key0 + KS * STEP > rm.hi_min;
      const bool clear = key0 < rm.lo_min || key0 + KS * STEP > rm.hi_max;
      // keys of this lane's V operand that no row of the block sees hold anything at all: cleared bit by bit
      auto v_mask = [&](int ks, uint32_t& vm0, uint32_t& vm1) {
        auto seen = [&](int key) { return key >= rm.lo_min && key < rm.hi_max; };
        const int ka = key0 + ks * STEP + 2 * t;
        vm0 = (seen(ka) ? 0xffffu : 0u) | (seen(ka + 1) ? 0xffff0000u : 0u);
        vm1 = (seen(ka + 8) ? 0xffffu : 0u) | (seen(ka + 9) ? 0xffff0000u : 0u);
      };
      float s[KS][NT][4];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[ks][nt][0] = s[ks][nt][1] = s[ks][nt][2] = s[ks][nt][3] = 0.0f;
      uint32_t pb[KS][NT][2], pl[KS][NT][2];
      if constexpr (!FP4) {
        uint32_t at[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t slot_at = (ring_at + i + ks) % STAGES;
          at[ks] = ring + slot_at * C16::STAGE;
          if (i + ks < nk &&
              !__all_sync(0xffffffffu, mbar_wait(wctx, bars + slot_at * 8, ((ring_at + i + ks) / STAGES) & 1u, 90u + slot_at))) {
            // gave up: the copies still in flight get their (bounded) time before the shared memory goes
            for (int x = ks + 1; x < STAGES && i + x < nk; ++x)
              mbar_wait(wctx, bars + ((ring_at + i + x) % STAGES) * 8, ((ring_at + i + x) / STAGES) & 1u, 99u);
            return;
          }
#pragma unroll
          for (int c = 0; c < DT; ++c) {
            uint32_t a[4];
            ldm_x4(at[ks] + (c >> 2) * C16::BOX + rowk * 128 + ((((c & 3) * 2 + ck) ^ (lane & 7)) << 4), a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<F16>(s[ks][nt], a, qb[nt][c][0], qb[nt][c][1]);
          }
        }
        softmax_step<F16, KS, NT, DT, CAP, HILO>(sp, rm, key0, lane, ragged, s, m_run, l_run, o, pb, pl);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t vm0 = ~0u, vm1 = ~0u;
          if (clear) v_mask(ks, vm0, vm1);
#pragma unroll
          for (int c = 0; c < DT; ++c) {
            uint32_t a[4];
            ldm_x4_trans(at[ks] + C16::TILE + (c >> 2) * C16::BOX + rowv * 128 + ((((c & 3) * 2 + cv) ^ (lane & 7)) << 4), a);
            if (clear) {
              a[0] &= vm0;
              a[1] &= vm0;
              a[2] &= vm1;
              a[3] &= vm1;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<F16>(o[c][nt], a, pb[ks][nt][0], pb[ks][nt][1]);
              mma_16816<F16>(o[c][nt], a, pl[ks][nt][0], pl[ks][nt][1]);
            }
          }
        }
        __syncwarp();                                 // every lane is done with the slots before they are filled again
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) issue(i + STAGES + ks, at[ks]);
      } else {
        // one group per iteration: KS steps
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES / KS - 2) : "memory");
        __syncwarp();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) issue(i + STAGES - KS + ks, group_to + ks * STAGE_BYTES);   // the last iteration is done with those
        asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t sK = group_at + ks * C4::STAGE;
          const uint32_t sKs = sK + 2 * STEP * C4::ROW;
          // K: keys g and g + 8, D/4 dimensions of each (D/8 bytes), one scale per two words
          constexpr int WORDS = D / 32;
          uint32_t wk[2][WORDS];
          uint32_t sc[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t at = sK + (g + 8 * x) * C4::ROW + t * (D / 8);
            uint32_t two;                               // scales of this lane's dimensions
            if constexpr (WORDS == 4) {
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(wk[x][0]), "=r"(wk[x][1]), "=r"(wk[x][2]), "=r"(wk[x][3]) : "r"(at));
              asm volatile("{.reg .b16 h; ld.shared.b16 h, [%1]; cvt.u32.u16 %0, h;}"
                           : "=r"(two) : "r"(sKs + (g + 8 * x) * C4::SROW + t * 2));
            } else {
              asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wk[x][0]), "=r"(wk[x][1]) : "r"(at));
              asm volatile("{.reg .b16 h; ld.shared.u8 h, [%1]; cvt.u32.u16 %0, h;}"
                           : "=r"(two) : "r"(sKs + (g + 8 * x) * C4::SROW + t));
            }
            sc[x] = e4m3x2_to_f16x2(two);
          }
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            uint32_t f0[4], f1[4];
            const uint32_t s0 = __byte_perm(sc[0], sc[0], w >= 2 ? 0x3232 : 0x1010);
            const uint32_t s1 = __byte_perm(sc[1], sc[1], w >= 2 ? 0x3232 : 0x1010);
            e2m1x8_to_f16(wk[0][w], f0);
            e2m1x8_to_f16(wk[1][w], f1);
#pragma unroll
            for (int x = 0; x < 4; ++x) {               // exact: two significant bits times four
              f0[x] = hmul2(f0[x], s0);
              f1[x] = hmul2(f1[x], s1);
            }
            const uint32_t a0[4] = {f0[0], f1[0], f0[1], f1[1]}, a1[4] = {f0[2], f1[2], f0[3], f1[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<true>(s[ks][nt], a0, qb[nt][2 * w][0], qb[nt][2 * w][1]);
              mma_16816<true>(s[ks][nt], a1, qb[nt][2 * w + 1][0], qb[nt][2 * w + 1][1]);
            }
          }
        }
        softmax_step<true, KS, NT, DT, CAP, HILO>(sp, rm, key0, lane, ragged, s, m_run, l_run, o, pb, pl);
        // V: dimensions [D/8 g, D/8 (g + 1)) of keys 2t, 2t + 1, 2t + 8, 2t + 9.  The operand wants two keys side by side
        // in a register, so the codes of two keys are put into one byte first: lo holds the even dimensions, hi the odd
        // ones.  Row m of tile c <-> dimension D/8 m + 2c, row m + 8 <-> the next one.
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t sV = group_at + ks * C4::STAGE + STEP * C4::ROW;
          const uint32_t sVs = sV + STEP * C4::ROW + STEP * C4::SROW;
          uint32_t vm0 = ~0u, vm1 = ~0u;
          if (clear) v_mask(ks, vm0, vm1);
          constexpr int VW = D / 64;                    // words per key
          uint32_t wv[4][VW], sb[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = 2 * t + (x & 1) + (x >> 1) * 8;
            const uint32_t at = sV + key * C4::ROW + g * (D / 16);
            if constexpr (VW == 2)
              asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wv[x][0]), "=r"(wv[x][1]) : "r"(at));
            else
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(wv[x][0]) : "r"(at));
            asm volatile("{.reg .b16 h; ld.shared.u8 h, [%1]; cvt.u32.u16 %0, h;}"
                         : "=r"(sb[x]) : "r"(sVs + key * C4::SROW + g * (D / 8) / 16));
          }
          // a masked key's scale may be a NaN pattern: the mask clears the product, not the factor
          const uint32_t sv0 = e4m3x2_to_f16x2(sb[0] | (sb[1] << 8)), sv1 = e4m3x2_to_f16x2(sb[2] | (sb[3] << 8));
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            constexpr uint32_t M = 0x0F0F0F0Fu;
            uint32_t f[4][4];                           // lo and hi of keys 2t, 2t + 1; of keys 2t + 8, 2t + 9
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t ka = wv[2 * x][w], kb = wv[2 * x + 1][w], sc2 = x ? sv1 : sv0;
              e2m1x8_to_f16((ka & M) | ((kb << 4) & ~M), f[2 * x]);
              e2m1x8_to_f16(((ka >> 4) & M) | (kb & ~M), f[2 * x + 1]);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                f[2 * x][k] = hmul2(f[2 * x][k], sc2);
                f[2 * x + 1][k] = hmul2(f[2 * x + 1][k], sc2);
              }
            }
            if (clear) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                f[0][k] &= vm0;
                f[1][k] &= vm0;
                f[2][k] &= vm1;
                f[3][k] &= vm1;
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a[4] = {f[0][k], f[1][k], f[2][k], f[3][k]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816<true>(o[w * 4 + k][nt], a, pb[ks][nt][0], pb[ks][nt][1]);
                if (HILO) mma_16816<true>(o[w * 4 + k][nt], a, pl[ks][nt][0], pl[ks][nt][1]);
              }
            }
          }
        }
        group_to = group_at;
        group_at = group_at == ring + (STAGES - KS) * STAGE_BYTES ? ring : group_at + KS * STAGE_BYTES;
      }
    }
    if (FP4 && nk > 0) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
    if (!FP4 && nk > 0) ring_at += nk;

    // ---- the part's result ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 4);
        l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 8);
        l_run[nt][j] += __shfl_xor_sync(0xffffffffu, l_run[nt][j], 16);
      }
    if (p.coop) {
      // the warps' parts through shared memory, each in its own ring (done with), and added tile by tile
      float* mine = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));
#pragma unroll
      for (int c = 0; c < DT; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          reinterpret_cast<float4*>(mine)[(c * NT + nt) * 32 + lane] =
              make_float4(o[c][nt][0], o[c][nt][1], o[c][nt][2], o[c][nt][3]);
      if (g == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            mine[DT * NT * 128 + nt * 8 + 2 * t + j] = m_run[nt][j];
            mine[DT * NT * 128 + RB + nt * 8 + 2 * t + j] = l_run[nt][j];
          }
      }
      __syncthreads();
      constexpr int RING_BYTES = STAGES * (FP4 ? C4::STAGE : C16::STAGE);
      constexpr int TILE_BYTES = 32 * 16 + 2 * 8 * 4;  // a tile of the CTA's sum: O, and m and l of its eight rows
      static_assert(RING_BYTES >= RB * (D + 2) * 4 && WARPS >= DT, "a part fits a ring, a warp takes a tile");
      auto add = [&](float (&m)[2], float (&l)[2], float (&x)[4], const float2& pm, const float2& pl2, const float4& v) {
        const float a[2] = {pm.x, pm.y}, q[2] = {pl2.x, pl2.y}, vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float mn = fmaxf(m[j], a[j]), mu = mn == -CUDART_INF_F ? 0.0f : mn;
          const float wa = ex2_approx(m[j] - mu), wb = ex2_approx(a[j] - mu);
          m[j] = mn;
          l[j] = l[j] * wa + q[j] * wb;
          x[j] = x[j] * wa + vv[j] * wb;
          x[2 + j] = x[2 + j] * wa + vv[2 + j] * wb;
        }
      };
      // warp c: tile c of every warp's part
      const int c = warp;
      float m[NT][2], l[NT][2], x[NT][4];
      if (c < DT) {
        const float* all = reinterpret_cast<const float*>(smem_raw + (base - smem_u32(smem_raw)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          m[nt][0] = m[nt][1] = -CUDART_INF_F;
          l[nt][0] = l[nt][1] = x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
#pragma unroll 4
          for (int w = 0; w < WARPS; ++w) {
            const float* src = all + w * (RING_BYTES / 4);
            const float* ml = src + DT * NT * 128 + nt * 8 + 2 * t;
            add(m[nt], l[nt], x[nt], *reinterpret_cast<const float2*>(ml), *reinterpret_cast<const float2*>(ml + RB),
                reinterpret_cast<const float4*>(src)[(c * NT + nt) * 32 + lane]);
          }
        }
      }
      if (p.coop == 1) {
        if (c < DT)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) write_tile<D, F16, FP4, NT>(p, sv, rb, h, nt, c, lane, x[nt], l[nt]);
        return;
      }
      // the cluster's CTAs: every one leaves its sums in its shared memory, and tile c goes to CTA c mod coop
      __syncthreads();                                 // the warps' parts have been read
      if (c < DT) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* dst = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)) + (c * NT + nt) * TILE_BYTES);
          reinterpret_cast<float4*>(dst)[lane] = make_float4(x[nt][0], x[nt][1], x[nt][2], x[nt][3]);
          if (g == 0) {
            *reinterpret_cast<float2*>(dst + 128 + 2 * t) = make_float2(m[nt][0], m[nt][1]);
            *reinterpret_cast<float2*>(dst + 136 + 2 * t) = make_float2(l[nt][0], l[nt][1]);
          }
        }
      }
      cluster_sync_all();
      if (c < DT && c % p.coop == (int)blockIdx.x % p.coop) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          m[nt][0] = m[nt][1] = -CUDART_INF_F;
          l[nt][0] = l[nt][1] = x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
          const uint32_t at = base + (c * NT + nt) * TILE_BYTES;
#pragma unroll 8
          for (int r = 0; r < p.coop; ++r) {
            const uint32_t src = mapa_u32(at, r);
            float4 v;
            float2 pm, pl2;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(src + lane * 16));
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm.x), "=f"(pm.y) : "r"(src + 512 + t * 8));
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pl2.x), "=f"(pl2.y) : "r"(src + 544 + t * 8));
            add(m[nt], l[nt], x[nt], pm, pl2, v);
          }
          write_tile<D, F16, FP4, NT>(p, sv, rb, h, nt, c, lane, x[nt], l[nt]);
        }
      }
      cluster_sync_all();                              // no CTA leaves while another reads its shared memory
      return;
    }
    const bool whole = st0 == 0 && st1 == sw.steps;
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < DT; ++c) write_tile<D, F16, FP4, NT>(p, sv, rb, h, nt, c, lane, o[c][nt], l_run[nt]);
    } else {
      const int slot = st0 == 0 ? 1 : 0;              // an item's first part, or the continuation of an earlier worker's
      float* dst = p.part + ((long long)wid * 2 + slot) * p.part_floats;
#pragma unroll
      for (int c = 0; c < DT; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          reinterpret_cast<float4*>(dst)[(c * NT + nt) * 32 + lane] =
              make_float4(o[c][nt][0], o[c][nt][1], o[c][nt][2], o[c][nt][3]);
      float* ml = dst + DT * NT * 128;
      if (g == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            ml[nt * 8 + 2 * t + j] = m_run[nt][j];
            ml[RB + nt * 8 + 2 * t + j] = l_run[nt][j];
          }
      }
    }
    if (st0 == 0 && lane == 0) {
      const long long rest = line + (long long)(item + 1) * sw.steps - u_end;    // steps left to the next workers
      const int parts = whole ? 0 : 1 + (int)((rest + per - 1) / per);
      const long long at = p.by_item ? ((long long)b * p.rb_max + rb) * p.kv_heads + h : wid;
      if (p.by_item || parts) p.desc[at] = make_int4(parts, wid, b, rb * p.kv_heads + h);
    }
    u += st1 - st0;
    if (u >= line + (long long)sw.rbs * p.head_groups * sw.steps) {
      line += (long long)sw.rbs * p.head_groups * sw.steps;
      do {
        if (++b >= p.batch.batch) return;
        sw = seq_work<RB>(p, b);
      } while (sw.rbs == 0);
    }
  }
}

// Adds the parts of the items that were cut: O = sum w_i O_i / sum w_i l_i with w_i = exp2(m_i - max m).  The parts
// are stored the way the worker held them (one float4 per lane and 16 x 8 tile), so a warp adds one tile with
// full-width loads; PW warps share the parts of a tile and are added through shared memory in a fixed order.
template <int D, bool F16, int NT, bool FP4, int PW>
__global__ void __launch_bounds__(256, NT == 1 ? 4 : 2) fmha_paged_merge_kernel(const __grid_constant__ SplitParams p) {
  constexpr int DT = D / 16, RB = 8 * NT, CT = 8 / PW;
  __shared__ float4 s_o[8][NT][32];
  __shared__ float s_ml[8][NT][2][4][2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the tile kernel of the same call, if there is one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int4 d = p.desc[blockIdx.x];
  // whatever a workspace holds that other work has written to meanwhile, nothing outside of it is touched
  if (d.x <= 0 || (unsigned)d.y >= (unsigned)p.workers || (unsigned)d.z >= (unsigned)p.batch.batch || d.w < 0 ||
      d.w >= p.rb_max * p.kv_heads)
    return;
  d.x = min(d.x, (p.workers - 1 - d.y) / p.heads_abreast + 1);
  const int pw = warp % PW, c = blockIdx.y * CT + warp / PW;
  const int b = d.z, rb = d.w / p.kv_heads, h = d.w % p.kv_heads;
  float m[NT][2], l[NT][2], o[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -CUDART_INF_F;
    l[nt][0] = l[nt][1] = 0.0f;
    o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.0f;
  }
  auto add = [&](int nt, const float (&pm)[2], const float (&plx)[2], const float4& v) {
    const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float mn = fmaxf(m[nt][j], pm[j]);
      const float mu = mn == -CUDART_INF_F ? 0.0f : mn;
      const float wa = ex2_approx(m[nt][j] - mu), wb = ex2_approx(pm[j] - mu);
      m[nt][j] = mn;
      l[nt][j] = l[nt][j] * wa + plx[j] * wb;
      o[nt][j] = o[nt][j] * wa + vv[j] * wb;
      o[nt][2 + j] = o[nt][2 + j] * wa + vv[2 + j] * wb;
    }
  };
  if (c < DT) {
    constexpr int U = 4;                             // parts whose loads are in flight together
    for (int i0 = pw; i0 < d.x; i0 += U * PW) {
      float4 v[U][NT];
      float2 pm[U][NT], pl[U][NT];
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int i = i0 + x * PW;
        const float* src = p.part + ((long long)(d.y + i * p.heads_abreast) * 2 + (i == 0 ? 1 : 0)) * p.part_floats;
        const float* ml = src + DT * NT * 128;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const bool there = i < d.x;
          v[x][nt] = there ? reinterpret_cast<const float4*>(src)[(c * NT + nt) * 32 + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          pm[x][nt] = there ? *reinterpret_cast<const float2*>(ml + nt * 8 + 2 * t) : make_float2(-CUDART_INF_F, -CUDART_INF_F);
          pl[x][nt] = there ? *reinterpret_cast<const float2*>(ml + RB + nt * 8 + 2 * t) : make_float2(0.0f, 0.0f);
        }
      }
#pragma unroll
      for (int x = 0; x < U; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float a[2] = {pm[x][nt].x, pm[x][nt].y}, q[2] = {pl[x][nt].x, pl[x][nt].y};
          add(nt, a, q, v[x][nt]);
        }
    }
  }
  if (PW > 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s_o[warp][nt][lane] = make_float4(o[nt][0], o[nt][1], o[nt][2], o[nt][3]);
      if (g == 0) {
        s_ml[warp][nt][0][t][0] = m[nt][0];
        s_ml[warp][nt][0][t][1] = m[nt][1];
        s_ml[warp][nt][1][t][0] = l[nt][0];
        s_ml[warp][nt][1][t][1] = l[nt][1];
      }
    }
    __syncthreads();
    if (pw != 0) return;
    for (int w = 1; w < PW; ++w)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float a[2] = {s_ml[warp + w][nt][0][t][0], s_ml[warp + w][nt][0][t][1]};
        const float q[2] = {s_ml[warp + w][nt][1][t][0], s_ml[warp + w][nt][1][t][1]};
        add(nt, a, q, s_o[warp + w][nt][lane]);
      }
  }
  if (c >= DT) return;
  const SeqView sv = seq_view(p.batch, b);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) write_tile<D, F16, FP4, NT>(p, sv, rb, h, nt, c, lane, o[nt], l[nt]);
}

template <int D, bool F16, int NT, bool CAP, bool FP4>
int launch_split(const PagedAttnArgs& a, const PagedSplitPlan& plan) {
  using C16 = Core16<D, NT>;
  using C4 = Core4<D, NT>;
  constexpr int SMEM = FP4 ? C4::SMEM : C16::SMEM;
  constexpr int THREADS = (FP4 ? C4::WARPS : C16::WARPS) * 32;
  const b200h::DeviceInfo* di = b200h::device_info();
  if (!di) return B200_ERR_CUDA;
  const b200tile_paged_cache& c = *a.cache;
  SplitParams p = {};
  p.batch = a.batch;
  p.q = static_cast<const uint16_t*>(a.q);
  p.out = static_cast<uint16_t*>(a.out);
  p.q_ts = a.q_ts; p.q_hs = a.q_hs; p.o_ts = a.o_ts; p.o_hs = a.o_hs;
  p.score = paged_score_params(a, FP4 ? c.k_global : 1.0f);
  p.kv_heads = c.kv_heads;
  p.group = a.q_heads / c.kv_heads;
  p.causal = a.causal;
  p.window = a.window;
  p.row_limit = a.row_limit;
  p.part = static_cast<float*>(a.workspace);
  p.part_floats = (long long)plan.part_floats;
  p.desc = reinterpret_cast<int4*>(static_cast<char*>(a.workspace) + plan.desc_off);
  p.workers = plan.workers;
  p.by_item = plan.by_item;
  p.coop = plan.coop;
  p.heads_abreast = plan.heads_abreast;
  p.head_groups = c.kv_heads / plan.heads_abreast;
  p.rb_max = (int)((std::min<long long>((long long)a.batch.max_q * p.group, a.row_limit) + 8 * NT - 1) / (8 * NT));
  p.min_steps = 2;
  CUtensorMap tmK = {}, tmV = {};
  if constexpr (FP4) {
    p.out_scale = c.v_global;
    p.k = static_cast<const uint8_t*>(c.k);
    p.v = static_cast<const uint8_t*>(c.v);
    p.ks = static_cast<const uint8_t*>(c.k_scales);
    p.vs = static_cast<const uint8_t*>(c.v_scales);
    p.k_page = (uint32_t)c.k_strides[0]; p.k_head = c.k_strides[1]; p.k_slot = (uint32_t)c.k_strides[2];
    p.v_page = (uint32_t)c.v_strides[0]; p.v_head = c.v_strides[1]; p.v_slot = (uint32_t)c.v_strides[2];
    p.ks_page = (uint32_t)c.k_scale_strides[0]; p.ks_head = c.k_scale_strides[1]; p.ks_slot = (uint32_t)c.k_scale_strides[2];
    p.vs_page = (uint32_t)c.v_scale_strides[0]; p.vs_head = c.v_scale_strides[1]; p.vs_slot = (uint32_t)c.v_scale_strides[2];
  } else {
    const CUtensorMapDataType dt = F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (int rc = b200h::encode_tmap_pages(&tmK, dt, c.k, D, c.page_size, c.kv_heads, c.num_pages, c.k_strides, 64, STEP))
      return rc;
    if (int rc = b200h::encode_tmap_pages(&tmV, dt, c.v, D, c.page_size, c.kv_heads, c.num_pages, c.v_strides, 64, STEP))
      return rc;
  }
  auto kern = fmha_paged_split_kernel<D, F16, NT, CAP, FP4>;
  static b200h::DeviceOnce attr_done;
  if (!attr_done.test(di->ordinal)) {
    B200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    attr_done.set(di->ordinal);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = a.stream;
  cfg.attrs = attr;
  if (plan.coop > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = plan.coop;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tmK, tmV, p, di->status));
  if (plan.coop) return B200_OK;
  // PW warps of a CTA share the parts of one tile, as many as an item has parts on average to keep them all in flight
  const unsigned x = (unsigned)(plan.by_item ? plan.items : plan.workers);
  const unsigned parts = plan.workers / x;
  const int pw = x * (D / 16) <= 8u * di->sm_count ? 8 : parts > 4 ? 2 : 1;
  cfg.gridDim = dim3(x, (D / 16 * pw + 7) / 8);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (pw == 8) B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fmha_paged_merge_kernel<D, F16, NT, FP4, 8>, p));
  else if (pw == 2) B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fmha_paged_merge_kernel<D, F16, NT, FP4, 2>, p));
  else B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fmha_paged_merge_kernel<D, F16, NT, FP4, 1>, p));
  return B200_OK;
}

}  // namespace
}  // namespace b200

// The plan depends on sizes the host knows; SM count 148 is the part's (fewer SMs run the same CTAs in turn).
static constexpr int COOP_STEPS = 16;

PagedSplitPlan b200_paged_split_plan(int format, int head_dim, int kv_heads, int batch, long long rows,
                                     long long max_keys) {
  PagedSplitPlan pl;
  const int warps = b200::split_warps(format != 0, head_dim, rows <= 8 ? 1 : 2);
  pl.rows_per_block = rows <= 8 ? 8 : 16;
  const long long rb_max = (rows + pl.rows_per_block - 1) / pl.rows_per_block;
  pl.items = (long long)batch * rb_max * kv_heads;
  const long long steps = pl.items * ((max_keys + 15) / 16);
  // As many CTAs per item as the machine has for it, if that leaves a warp a few steps only: 700 keys of 8 heads 6.8
  // against 8.9 us, 18 x 8 items of 700 keys 9.9 against 21, of 2048 keys 29 against 39.  With more steps the two come
  // together for equal lengths (1.03 at 18 x 32768 keys), and runs win where lengths differ, which the host does not
  // know.  Clusters of eight stop fitting side by side at 16 of them (11.5 against 6.4 us for 8).
  int per_item = 1;
  while (per_item < 8 && pl.items * per_item * 2 <= (per_item == 4 ? 96 : 148)) per_item *= 2;
  pl.coop = pl.items <= 148 && (max_keys + 15) / 16 <= (long long)per_item * warps * COOP_STEPS ? per_item : 0;
  if (pl.coop) {
    pl.ctas = (int)pl.items * pl.coop;
    pl.workers = 0;
    pl.by_item = false;
    pl.part_floats = pl.desc_off = 0;
    pl.heads_abreast = 1;
    pl.bytes = 16;
    return pl;
  }
  pl.ctas = (int)std::max<long long>(1, std::min<long long>(148, (steps + 1) / 2));
  pl.workers = pl.ctas * warps;
  pl.by_item = pl.items <= pl.workers;
  // Heads of a token lie side by side in one of the two usual orders, 64 to 256 bytes each: workers that take four of them
  // at the same keys use what DRAM has open (NVFP4 32 x 16384 keys 99 -> 73 us, 24 x 16 heads of 64 70 -> 63; more than four,
  // and the other order, change 2 % either way).  The smallest divisor from four on.
  pl.heads_abreast = std::min(kv_heads, 4);
  while (kv_heads % pl.heads_abreast) ++pl.heads_abreast;
  if (pl.heads_abreast > 32 || pl.heads_abreast > pl.workers) pl.heads_abreast = 1;
  pl.part_floats = (size_t)pl.rows_per_block * (head_dim + 2);
  pl.desc_off = (size_t)pl.workers * 2 * pl.part_floats * sizeof(float);
  pl.bytes = pl.desc_off + sizeof(int4) * (size_t)(pl.by_item ? pl.items : pl.workers);
  return pl;
}

int b200_paged_split_dispatch(const PagedAttnArgs& a) {
  using namespace b200;
  const b200tile_paged_cache& c = *a.cache;
  const PagedSplitPlan plan =
      b200_paged_split_plan(c.format, c.head_dim, c.kv_heads, a.batch.batch,
                            std::min<long long>((long long)a.batch.max_q * (a.q_heads / c.kv_heads), a.row_limit),
                            (long long)a.batch.max_pages * c.page_size);
#define B200_PS(D_, F_, N_, C_, Q_) return launch_split<D_, F_, N_, C_, Q_>(a, plan)
#define B200_PS_CAP(D_, F_, N_, Q_) do { if (a.capped) B200_PS(D_, F_, N_, true, Q_); B200_PS(D_, F_, N_, false, Q_); } while (0)
#define B200_PS_NT(D_, F_, Q_) do { if (plan.rows_per_block == 8) B200_PS_CAP(D_, F_, 1, Q_); B200_PS_CAP(D_, F_, 2, Q_); } while (0)
#define B200_PS_FMT(D_, F_) do { if (c.format) B200_PS_NT(D_, F_, true); B200_PS_NT(D_, F_, false); } while (0)
  if (c.head_dim == 128 && a.dtype == 0) B200_PS_FMT(128, false);
  if (c.head_dim == 128 && a.dtype == 1) B200_PS_FMT(128, true);
  if (c.head_dim == 64 && a.dtype == 0) B200_PS_FMT(64, false);
  if (c.head_dim == 64 && a.dtype == 1) B200_PS_FMT(64, true);
#undef B200_PS_FMT
#undef B200_PS_NT
#undef B200_PS_CAP
#undef B200_PS
  return b200h::set_error(B200_ERR_UNSUPPORTED, "paged_attention: no kernel for head_dim %d (64 and 128 are provided)",
                          c.head_dim);
}

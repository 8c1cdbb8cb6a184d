// Attention of many query rows (prompts and prompt chunks) over a paged key/value cache on the 5th-generation tensor
// cores.  The mathematics is fmha_paged.cu's; the machine is fmha_fwd.cu's: one CTA works on two tiles of 128 query rows
// and walks the keys once for both, S = Q K^T and O += P V by tcgen05 with S, P and O in Tensor Memory, one softmax
// thread per row, O rescaled only when a row's maximum grew by more than 2^8.  What differs:
//
//   - a tile's rows are (token, head of the group) pairs of ONE K/V head, 128 / group tokens at a time, so that K and V
//     pass through a CTA once for all heads that share them (one TMA box {64, group, tokens} brings them in that order);
//   - the 128 keys of a step come from 128 / page_size pages, one TMA box each; a page that no row of the pair looks at
//     gets the page number just outside the pool, where TMA fills in zeros without touching memory;
//   - V rows of a step that no row looks at (behind the length, before the window) are cleared in shared memory by the
//     MMA warp: their probability is 0, but 0 times whatever a free slot holds need not be;
//   - the grid is one CTA per SM, and the steps of all items (sequence, pair of tiles, K/V head) form one line that is cut
//     into equal runs, as in fmha_paged.cu: few long chunks and many short prompts fill the machine alike, and nothing
//     about the lengths is needed on the host.  The rings run on from item to item and the next Q is fetched while the
//     last keys of the present one are worked on.  An item that is cut leaves (m, l, O) of its parts in 32 bits for the
//     merge kernel, at most two parts per CTA;
//   - an NVFP4 cache takes four more warps: thread r expands key r of the step (64 bytes and 8 scales for D = 128) to f16
//     straight into the swizzled operand tile, K and V in turn, with the next row's bytes already in registers.  The
//     products are then f16 x f16, which holds every code * scale exactly; bf16 queries are brought to a power of two near
//     1 row by row and converted in shared memory by the softmax threads before their first scores.
//
// What bounds it: as fmha_fwd.cu, the softmax threads and the tensor pipe in turn, 2.1 us a step of 256 x 128 (2.45 with the
// cap, 2.6 over NVFP4) where the tensor pipe alone needs 1.5, and 4 to 5 us to begin and end an item.  A prompt of 4096
// tokens, 32 / 8 heads of 128: 144 us, 950 TFLOP/s, the tensor pipe 51 % active (163 us with all data from HBM); four chunks
// to 256 tokens over 5000 NVFP4 keys 51 us, 29 % active.
//
// P is handed to the second product as ONE 16-bit value (bf16 2^-9, f16 2^-12 of each weight, at random), as in fmha_fwd.cu;
// the row-block kernel's two pieces would double the second product, 0.75 us of tensor time a step.  Against 64 bits the
// output's error grows from 1.6e-3 to 2.0e-3 of its norm in bf16 and from 2.1e-4 to 2.9e-4 in f16, by about as much as the
// output's own rounding.  The sums of the weights take the values before that rounding, in 32 bits.
#include <math_constants.h>

#include <algorithm>

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
  int wide_out;                      // the output's rows lie on 32-byte boundaries
  float out_scale;
  float* part;                       // two slots per CTA
  int4* desc;                        // one per CTA
  // FP4 operands: byte strides
  const uint8_t *k, *v, *ks, *vs;
  long long k_st[3], v_st[3], ks_st[3], vs_st[3];
};

// A part: O as [2 tiles][D / 4][128 rows] float4 (lanes = rows, so that stores and loads are full lines), then
// [2][128] maxima and [2][128] sums.
__host__ __device__ constexpr int part_floats(int d) { return 2 * 128 * (d + 2); }
// Starting and ending an item costs about as much as this many keys.
constexpr int ITEM_COST = 384;
constexpr int MIN_RUN = 768;         // keys: a shorter run would be mostly start-up
constexpr int PART_RING = 4;         // parts known ahead of their turn

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
  // barriers: q_full[2], q_free[2], q_ready[2], k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2], p_full[2],
  // o_done[2], part_full[R], part_free[R]
  static constexpr int NUM_BARS = 6 + 4 * KV_STAGES + 6 + 2 * PART_RING;
  static constexpr int OFF_MISC = (OFF_BAR + NUM_BARS * 8 + 15) / 16 * 16;
  static constexpr int TOTAL = OFF_MISC + 16 + 1024;
  static constexpr int THREADS = FP4 ? 512 : 384;
};

__device__ __forceinline__ float absmax3(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {   // of a number and a NaN, the number
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void st_shared_v4(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void ld_shared_v4(uint32_t src, uint32_t (&w)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src) : "memory");
}

// Out of line, for caps beyond CAP_SMALL_OUT with scores near them, which is rare: the registers of both forms stay out of
// the softmax loop (inlined, prompt chunks with a cap of 30 took 126 us instead of 122).
__device__ __noinline__ float score_any_cap(float scale, float cap_arg, float cap_out, float s) {
  return paged_score<true>(ScoreParams{scale, cap_arg, cap_out}, s);
}

// Pairs of tiles that sequence b has here: none when its rows are few enough for the row-block kernel.
__device__ __forceinline__ int seq_pairs(const TileParams& p, const SeqView& s) {
  if ((long long)s.n * p.group <= p.row_limit) return 0;
  return (s.n + 2 * p.tpt - 1) / (2 * p.tpt);
}
// Key range and steps of a pair; a pair that sees no key still has one step, so that its rows are written.
struct PairSpan {
  int lo, hi, j0, steps;
};
__device__ __forceinline__ PairSpan pair_span(const TileParams& p, const SeqView& s, int pair) {
  PairSpan x;
  const int t0 = pair * 2 * p.tpt, n = min(s.n - t0, 2 * p.tpt);
  x.hi = p.causal ? min(s.len, s.pos0 + t0 + n) : s.len;
  x.lo = p.causal && p.window > 0 ? window_start(s.pos0 + t0, p.window) : 0;
  x.j0 = x.hi > x.lo ? x.lo / FA_BN : 0;
  x.steps = x.hi > x.lo ? (x.hi + FA_BN - 1) / FA_BN - x.j0 : 1;
  return x;
}

// The line that is cut into runs is measured in keys: an item of pair i is ITEM_COST plus the keys its rows can see at
// most, span(i) = min(base + (i + 1) tokens, top) for a causal sequence, whose sums have a closed form; so a warp finds
// any place on the line with a few divisions, whatever the number of pairs.  A part's share of the item's length is its
// share of the item's steps.
struct SeqLine {
  long long base, slope, top;        // span(i) = min(base + i slope, top)
  int pairs;
  int bend;                          // pairs below the top
};
__device__ __forceinline__ SeqLine seq_line(const TileParams& p, const SeqView& s) {
  SeqLine x;
  x.pairs = seq_pairs(p, s);
  const int tokens = 2 * p.tpt;
  x.slope = p.causal ? tokens : 0;
  x.base = p.causal ? (long long)max(0, s.pos0) + tokens : s.len;
  x.top = p.causal && p.window > 0 ? (long long)p.window + tokens : (1ll << 40);
  x.bend = x.top <= x.base ? 0 : x.slope == 0 ? x.pairs : (int)min((long long)x.pairs, (x.top - x.base) / x.slope + 1);
  return x;
}
__device__ __forceinline__ long long line_len(const SeqLine& x, int i) {    // of one item of pair i
  return ITEM_COST + (i < x.bend ? x.base + i * x.slope : x.top);
}
__device__ __forceinline__ long long line_sum(const SeqLine& x, int n) {    // of the first n pairs, one item each
  const long long k = min(n, x.bend);
  return (long long)n * ITEM_COST + k * x.base + x.slope * (k * (k - 1) / 2) + (n - k) * x.top;
}

// Place on the line.
struct Walk {
  long long u, u_end;
  long long at, len;                 // place in the item and the item's length
  int b, pair, head;
  SeqView sv;
  SeqLine line;
  PairSpan sp;
  int a0, a1;                        // steps of this part, relative to sp.j0
  __device__ __forceinline__ long long left() const { return min(len - at, u_end - u); }
  // steps of the part at `at`; false if it is an item's beginning too short for a step: the next CTA begins it then
  __device__ __forceinline__ bool cut() {
    a0 = (int)(at * sp.steps / len);
    a1 = (int)((at + left()) * sp.steps / len);
    return a1 > 0;
  }
  __device__ __forceinline__ void open(const TileParams& p) {
    sp = pair_span(p, sv, pair);
    len = line_len(line, pair);
    at = 0;
  }
  __device__ __forceinline__ void next(const TileParams& p) {
    u += left();
    if (u >= u_end) return;
    at = 0;                          // the run goes on, so the item has ended
    if (++head == p.kv_heads) {
      head = 0;
      if (++pair == line.pairs) {
        pair = 0;
        do {
          if (++b >= p.batch.batch) {
            u = u_end;
            return;
          }
          sv = seq_view(p.batch, b);
          line = seq_line(p, sv);
        } while (line.pairs == 0);
      }
      open(p);
    }
    if (!cut()) u = u_end;
  }
};

// The line's length, by one warp.
__device__ __forceinline__ long long whole_line(const TileParams& p, int lane) {
  long long mine = 0;
  for (int b = lane; b < p.batch.batch; b += 32) {
    const SeqLine x = seq_line(p, seq_view(p.batch, b));
    mine += line_sum(x, x.pairs);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine * p.kv_heads;
}
// The item at place u < u_end <= the line's length; all lanes together, the result in all of them.
__device__ __forceinline__ void find_place(const TileParams& p, int lane, Walk& w) {
  long long before = 0;                            // of the sequences already passed
  for (int b0 = 0; b0 < p.batch.batch; b0 += 32) {
    long long mine = 0;
    if (b0 + lane < p.batch.batch) {
      const SeqLine x = seq_line(p, seq_view(p.batch, b0 + lane));
      mine = line_sum(x, x.pairs) * p.kv_heads;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + inc > w.u);
    if (past) {
      const int l = __ffs(past) - 1;
      before += __shfl_sync(0xffffffffu, inc - mine, l);
      w.b = b0 + l;
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  w.sv = seq_view(p.batch, w.b);
  w.line = seq_line(p, w.sv);
  const long long rel = w.u - before;
  int lo = 0, hi = w.line.pairs - 1;               // the last pair that begins at or before rel
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (line_sum(w.line, mid) * p.kv_heads <= rel) lo = mid;
    else hi = mid - 1;
  }
  w.pair = lo;
  w.open(p);
  const long long in_pair = rel - line_sum(w.line, lo) * p.kv_heads;
  w.head = (int)(in_pair / w.len);
  w.at = in_pair - w.head * w.len;
}

// One part of an item as the roles need it.  The loader warp walks the run and hands the parts to the others through a
// ring in shared memory: the walk's divisions and loads happen once, ahead of time, instead of in every role between
// two items.
struct Part {
  int end;                           // no more parts
  int steps[2];                      // steps of either tile in this part
  int tokens[2];
  int key0, lo, hi;                  // first key of the part; keys that some row of the pair sees
  int b, pair, head;
  int row0, pos0, len;               // row and position of the pair's first token; cached rows of the sequence
  int whole, slot, parts;            // the item is not cut; which slot its part takes; parts (first one only)
};
__device__ __forceinline__ Part make_part(const TileParams& p, const Walk& w, long long per) {
  Part x;
  x.end = 0;
  x.b = w.b;
  x.pair = w.pair;
  x.head = w.head;
  x.row0 = w.sv.q0 + w.pair * 2 * p.tpt;
  x.pos0 = w.sv.pos0 + w.pair * 2 * p.tpt;
  x.len = w.sv.len;
  x.key0 = (w.sp.j0 + w.a0) * FA_BN;
  x.lo = w.sp.lo;
  x.hi = w.sp.hi;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int n = min(max(w.sv.n - (w.pair * 2 + t) * p.tpt, 0), p.tpt);
    const int hi = n == 0 ? 0 : p.causal ? min(w.sv.len, x.pos0 + t * p.tpt + n) : w.sv.len;
    x.tokens[t] = n;
    x.steps[t] = max(0, min(w.a1, (hi + FA_BN - 1) / FA_BN - w.sp.j0) - w.a0);
  }
  x.whole = w.a0 == 0 && w.a1 == w.sp.steps;
  x.slot = w.a0 == 0 ? 1 : 0;        // an item's first part, or the continuation of an earlier CTA's
  x.parts = 1 + (int)((w.len - w.at - w.left() + per - 1) / per);
  return x;
}

template <int D, bool F16, bool CAP, bool FP4>
__global__ void __launch_bounds__(FP4 ? 512 : 384, 1)
fmha_paged_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TileParams p, uint32_t* status) {
  using L = TileSmem<D, FP4>;
  constexpr int STAGES = L::KV_STAGES, HALVES = L::HALVES, THREADS = L::THREADS;
  constexpr uint32_t HALF = L::HALF_BYTES, TILE = L::TILE_BYTES;
  constexpr bool MF16 = F16 || FP4;               // element type of the products
  constexpr bool CONVERT = FP4 && !F16;           // bf16 queries for f16 products
  extern __shared__ uint8_t smem_raw[];
  __shared__ Walk s_walk;
  __shared__ Part s_part[PART_RING];
  __shared__ long long s_row_off[FA_BM];          // element offset of a tile's row in the output, from its first token
  __shared__ int s_row_tok[FA_BM];                // its token
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge, which waits for this grid

  if (threadIdx.x < FA_BM) {
    const int tok = threadIdx.x / p.group;
    s_row_tok[threadIdx.x] = tok;
    s_row_off[threadIdx.x] = tok * p.o_ts + (long long)(threadIdx.x - tok * p.group) * p.o_hs;
  }
  const uint32_t sQ = base + L::OFF_Q, sK = base + L::OFF_K, sV = base + L::OFF_V;
  const uint32_t bar_q_full = base + L::OFF_BAR;
  const uint32_t bar_q_free = bar_q_full + 2 * 8;
  const uint32_t bar_q_ready = bar_q_free + 2 * 8;
  const uint32_t bar_k_full = bar_q_ready + 2 * 8;
  const uint32_t bar_k_empty = bar_k_full + STAGES * 8;
  const uint32_t bar_v_full = bar_k_empty + STAGES * 8;
  const uint32_t bar_v_empty = bar_v_full + STAGES * 8;
  const uint32_t bar_s_full = bar_v_empty + STAGES * 8;
  const uint32_t bar_p_full = bar_s_full + 2 * 8;
  const uint32_t bar_o_done = bar_p_full + 2 * 8;
  const uint32_t bar_part_full = bar_o_done + 2 * 8;
  const uint32_t bar_part_free = bar_part_full + PART_RING * 8;
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gen_base + L::OFF_MISC);
  WaitCtx wctx{misc + 1, status};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q_full + i * 8, 1);
      mbar_init(bar_q_free + i * 8, 1);
      mbar_init(bar_q_ready + i * 8, 4);               // the tile's softmax warps
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
    for (int i = 0; i < PART_RING; ++i) {
      mbar_init(bar_part_full + i * 8, 1);
      mbar_init(bar_part_free + i * 8, THREADS / 32 - 1);    // every warp but the loader's
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
  auto wait_all = [&](uint32_t bar, uint32_t parity, uint32_t site) {
    return __all_sync(0xffffffffu, mbar_wait(wctx, bar, parity, site)) != 0;
  };

  // the i-th part, once it is there (all lanes of the warp together); false when the run has ended or a wait gave up
  auto have_part = [&](int i) {
    return wait_all(bar_part_full + (i % PART_RING) * 8, (i / PART_RING) & 1, 16) && !s_part[i % PART_RING].end;
  };
  auto done_part = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_part_free + (i % PART_RING) * 8);
  };

  // the run of this CTA, found by the loader warp before it gives up its registers
  long long per = 0;
  if (warp == 0) {
    const long long total = whole_line(p, lane);
    per = max((long long)MIN_RUN, (total + gridDim.x - 1) / gridDim.x);
    Walk first;
    first.u = blockIdx.x * per;
    first.u_end = min(total, first.u + per);
    if (first.u < first.u_end) {
      find_place(p, lane, first);
      if (!first.cut()) first.u = first.u_end;
    }
    if (lane == 0) {
      p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
      s_walk = first;
    }
    __syncwarp();
  }
  if (warp < 4) reg_dealloc<FP4 ? 40 : FA_OTHER_REGS>();
  if (warp == 0) {
    // ------------------------------- parts, K and V -------------------------------
    const int boxes = FA_BN / p.box_rows;
    const int slot_mask = (1 << p.batch.page_shift) - 1;
    int armed_k = 0, armed_v = 0;        // K and V steps fetched so far: stage and phase of the ring
    bool ok = true;
    for (int i = 0;; ++i) {
      const int at = i % PART_RING;
      if (i >= PART_RING && !wait_all(bar_part_free + at * 8, (i / PART_RING - 1) & 1, 17)) { ok = false; break; }
      if (lane == 0) {
        if (i > 0) s_walk.next(p);
        if (s_walk.u < s_walk.u_end) s_part[at] = make_part(p, s_walk, per);
        else s_part[at].end = 1;
        mbar_arrive(bar_part_full + at * 8);
      }
      __syncwarp();
      const Part& w = s_part[at];
      if (w.end) break;
      if (FP4) continue;
      // lane i < boxes: page of box i; lane i < boxes * HALVES issues box i % boxes of half i / boxes
      const int n = max(w.steps[0], w.steps[1]), key0 = w.key0, lo = w.lo, hi = w.hi, b = w.b, head = w.head;
      auto page_for = [&](int j) {
        const int key = key0 + j * FA_BN + lane * p.box_rows;
        const bool used = j < n && lane < boxes && key < hi && key + p.box_rows > lo;
        return used ? page_of(p.batch, b, key, status) : p.batch.num_pages;
      };
      int pages = n > 0 ? page_for(0) : 0;
      for (int j = 0; j < n; ++j) {
        const int next = page_for(j + 1);
        const int box = lane % boxes, half = lane / boxes;
        const int pg = __shfl_sync(0xffffffffu, pages, box);
        const int slot = (key0 + j * FA_BN + box * p.box_rows) & slot_mask;
        const uint32_t stage = armed_k % STAGES, phase = (armed_k / STAGES) & 1;
        const uint32_t off = stage * TILE + half * HALF + box * p.box_rows * 128;
        if (!wait_all(bar_k_empty + stage * 8, phase ^ 1, 10)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(bar_k_full + stage * 8, TILE);
        __syncwarp();
        if (half < HALVES) tma_load_4d(sK + off, &tmK, bar_k_full + stage * 8, half * 64, slot, head, pg);
        ++armed_k;
        if (!wait_all(bar_v_empty + stage * 8, phase ^ 1, 11)) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(bar_v_full + stage * 8, TILE);
        __syncwarp();
        if (half < HALVES) tma_load_4d(sV + off, &tmV, bar_v_full + stage * 8, half * 64, slot, head, pg);
        ++armed_v;
        pages = next;
      }
      if (!ok) break;
    }
    if (!ok) {
      // a wait gave up: the copies still in flight get their (bounded) time before the shared memory goes
      for (int i = max(0, armed_k - STAGES); i < armed_k; ++i)
        mbar_wait(wctx, bar_k_full + (i % STAGES) * 8, (i / STAGES) & 1, 12);
      for (int i = max(0, armed_v - STAGES); i < armed_v; ++i)
        mbar_wait(wctx, bar_v_full + (i % STAGES) * 8, (i / STAGES) & 1, 13);
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer --------------------------------
    // the whole warp runs the control flow, one elected lane issues (fmha_fwd.cu says why)
    const bool me = elect_one() != 0;
    constexpr uint32_t fmt = MF16 ? FMT_F16 : FMT_BF16;
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
    // V rows of a step that no row of the pair sees
    auto clear_v = [&](int key0, int lo, int hi, uint32_t v_addr) {
      const int from = max(lo - key0, 0), to = min(hi - key0, FA_BN);
      if (from <= 0 && to >= FA_BN) return;
      for (int i = lane; i < FA_BN * HALVES * 8; i += 32) {
        const int r = i / (HALVES * 8), c = i % (HALVES * 8);
        if (r < from || r >= to) st_shared_v4(v_addr + (c >> 3) * HALF + r * 128 + (c & 7) * 16, 0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    int it = 0;                          // steps through the rings so far
    uint32_t q_items[2] = {0, 0}, steps[2] = {0, 0};   // items and steps of each tile so far
    bool ok = true;
    for (int i = 0; ok && have_part(i); ++i) {
      const Part& w = s_part[i % PART_RING];
      const int cnt[2] = {w.steps[0], w.steps[1]};
      const int n = max(cnt[0], cnt[1]), key0 = w.key0, lo = w.lo, hi = w.hi;
      done_part(i);
      if (n == 0) continue;
      if (!wait_all(bar_k_full + (it % STAGES) * 8, (it / STAGES) & 1, 20)) { ok = false; break; }
#pragma unroll
      for (int t = 0; t < 2 && ok; ++t) {
        if (cnt[t] == 0) continue;
        if (!wait_all((CONVERT ? bar_q_ready : bar_q_full) + t * 8, q_items[t] & 1, 21)) { ok = false; break; }
        tc_fence_after_sync();
        issue_qk(t, sK + (it % STAGES) * TILE);
        if (me) umma_commit(bar_s_full + t * 8);
        if (cnt[t] == 1 && me) umma_commit(bar_q_free + t * 8);
        ++q_items[t];
      }
      if (ok && me) umma_commit(bar_k_empty + (it % STAGES) * 8);
      for (int j = 0; j < n && ok; ++j, ++it) {
        const uint32_t vs = it % STAGES, vph = (it / STAGES) & 1;
        const uint32_t ks = (it + 1) % STAGES, kph = ((it + 1) / STAGES) & 1;
        const bool have_next = j + 1 < n;
        if (!wait_all(bar_v_full + vs * 8, vph, 22)) { ok = false; break; }
        if constexpr (!FP4) clear_v(key0 + j * FA_BN, lo, hi, sV + vs * TILE);
        if (have_next && !wait_all(bar_k_full + ks * 8, kph, 23)) { ok = false; break; }
        tc_fence_after_sync();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j < cnt[t]) {
            if (!wait_all(bar_p_full + t * 8, steps[t] & 1, 24)) { ok = false; break; }
            tc_fence_after_sync();
            issue_pv(t, sV + vs * TILE, j > 0);
            ++steps[t];
            if (j == cnt[t] - 1 && me) umma_commit(bar_o_done + t * 8);
          }
          if (j + 1 < cnt[t]) {
            issue_qk(t, sK + ks * TILE);
            if (me) umma_commit(bar_s_full + t * 8);
            if (j + 2 == cnt[t] && me) umma_commit(bar_q_free + t * 8);
          }
        }
        if (!ok) break;
        if (me) umma_commit(bar_v_empty + vs * 8);
        if (have_next && me) umma_commit(bar_k_empty + ks * 8);
      }
    }
  } else if (warp < 4) {
    // ----------------------------- Q of tile `warp - 2` -----------------------------
    const int t = warp - 2;
    uint32_t items = 0;
    for (int i = 0; have_part(i); ++i) {
      const Part& w = s_part[i % PART_RING];
      const int n = w.steps[t], q_head = w.head * p.group, q_row = w.row0 + t * p.tpt;
      done_part(i);
      if (n == 0) continue;
      // the products of the last item with this tile's Q have been read
      if (items > 0 && !wait_all(bar_q_free + t * 8, (items - 1) & 1, 14)) break;
      if (lane == 0) {
        mbar_expect_tx(bar_q_full + t * 8, (uint32_t)(HALVES * 128 * p.tpt * p.group));
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          tma_load_3d(sQ + t * TILE + h * HALF, &tmQ, bar_q_full + t * 8, h * 64, q_head, q_row);
      }
      ++items;
    }
    if (items > 0) mbar_wait(wctx, bar_q_full + t * 8, (items - 1) & 1, 15);   // nothing in flight when this warp leaves
  } else if (warp >= 4 && warp < 12) {
    // -------------------------------- softmax ----------------------------------
    reg_alloc<FP4 ? 208 : 224>();       // 224 x 256 + 56 x 128 = 168 x 384; with NVFP4 208 x 256 + (40 + 56) x 128 = 128 x 512
    const int t = (warp - 4) >> 2;
    const int q = warp & 3;
    const int row = q * 32 + lane;          // row inside the tile == TMEM lane
    const int tok = s_row_tok[row];
    const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
    const uint32_t tS = lane_base + S_COL(t);
    const uint32_t tO = lane_base + O_COL(t);
    uint32_t steps = 0, items = 0;
    bool ok = true;
    for (int i = 0; ok && have_part(i); ++i) {
      const Part& w = s_part[i % PART_RING];
      const int n_mine = w.steps[t], key_base = w.key0;
      // keys this row sees (rows that are no token's see none)
      int row_lo = 0, row_hi = 0;
      if (tok < w.tokens[t]) {
        const int pos = w.pos0 + t * p.tpt + tok;
        row_hi = p.causal ? min(w.len, pos + 1) : w.len;
        if (p.causal && p.window > 0) row_lo = window_start(pos, p.window);
      }
      const bool blind = row_hi <= row_lo;
      float poly_max = 0.0f;
      uint64_t k2[CAP_POLY_N];             // the polynomial in s itself
      float scale = p.score.scale_log2, cap_arg = p.score.cap_arg;
      float m_run = -CUDART_INF_F, l_run = 0.0f;
      if (CONVERT && n_mine > 0) {
        // bf16 queries for f16 products: this thread's row, a power of two taken out of it and put into the scale.  (By a
        // warp per tile beside the softmax of the item before, a first item waited 10 us for it.)
        if (!wait_all(bar_q_full + t * 8, items & 1, 25)) { ok = false; break; }
        const uint32_t at = sQ + t * TILE + row * 128;
        uint32_t x[HALVES * 8][4], most = 0;
#pragma unroll
        for (int c = 0; c < HALVES * 8; ++c) ld_shared_v4(at + (c >> 3) * HALF + (((c & 7) ^ (row & 7)) << 4), x[c]);
#pragma unroll
        for (int c = 0; c < HALVES * 8; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k) most = max_bf16x2(most, x[c][k] & 0x7fff7fffu);
        const float2 m2 = paged_unpack16<false>(most);
        const uint32_t e = __float_as_uint(fmaxf(m2.x, m2.y)) & 0x7f800000u;
        const bool scaled = e > (27u << 23) && e < (227u << 23);   // not for rows of zeros, infinities or NaN
        const float inv = scaled ? __uint_as_float((254u << 23) - e) : 1.0f;
        const float unit = scaled ? __uint_as_float(e) : 1.0f;
#pragma unroll
        for (int c = 0; c < HALVES * 8; ++c) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = paged_unpack16<false>(x[c][k]);
            x[c][k] = pack_f16x2(f.x * inv, f.y * inv);
          }
          st_shared_v4(at + (c >> 3) * HALF + (((c & 7) ^ (row & 7)) << 4), x[c][0], x[c][1], x[c][2], x[c][3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q_ready + t * 8);
        scale = factor_in_range(scale * unit);
        cap_arg = factor_in_range(cap_arg * unit);
      }
      for (int j = 0; j < n_mine; ++j, ++steps) {
        if (!wait_all(bar_s_full + t * 8, steps & 1, 30)) { ok = false; break; }
        tc_fence_after_sync();
        if (CAP && j == 0) {
          // The polynomial in s itself, for rows whose scores are all a small part of the cap: c tanh(s a) log2e = s (k0 + k1 s^2
          // + ..), a = scale / c.  Up to 2^62 the powers of s are numbers; those of a may underflow, where the cap is so
          // far away that they do not matter.  With a beyond 2^14 they might overflow.
          const float a = cap_arg * CAP_HALF_ARG, aa = a * a;
          poly_max = a < 0x1p14f ? fminf(CAP_POLY_MAX / a, 0x1p62f) : -1.0f;
          float f = scale;
#pragma unroll
          for (int i = 0; i < CAP_POLY_N; ++i) {
            k2[i] = pack2(cap_poly(i) * f, cap_poly(i) * f);
            f *= aa;
          }
        }
        uint32_t v[FA_BN];
#pragma unroll
        for (int c = 0; c < FA_BN / 32; ++c)
          tmem_ld_32x32b_x32(tS + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&v[c * 32]));
        const int key0 = key_base + j * FA_BN;
        const int c_hi = row_hi - 1 - key0, c_lo = row_lo - key0;    // first and last column seen
        // rows that see nothing (no token's, mostly) hold what they like: nothing of it is written
        const bool masked_tile = __any_sync(0xffffffffu, !blind && (c_hi < FA_BN - 1 || c_lo > 0));
        tmem_wait_ld();
        bool poly = false;                    // the cap's polynomial serves every score of the warp's rows
        if (CAP) {
          float mp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < FA_BN; i += 8)
#pragma unroll
            for (int u = 0; u < 4; ++u)
              mp[u] = absmax3(mp[u], __uint_as_float(v[i + 2 * u]), __uint_as_float(v[i + 2 * u + 1]));
          const float big = fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3]));
          poly = __all_sync(0xffffffffu, blind || big <= poly_max);
        }
        // What a masked column holds: -inf, or with a cap, which makes -c of a score of -inf, a NaN of its own that no product
        // gives and the maximum passes over.
        constexpr uint32_t MASKED = CAP ? 0xffc0ffeeu : 0xff800000u;
        if (masked_tile) {
#pragma unroll
          for (int c = 0; c < FA_BN / 32; ++c) {
            // bits of the columns [c_lo, c_hi] among these 32
            const int h = c_hi - c * 32, l = c_lo - c * 32;
            uint32_t bits = h >= 31 ? ~0u : h < 0 ? 0u : (2u << h) - 1u;
            bits &= l <= 0 ? ~0u : l > 31 ? 0u : ~0u << l;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((bits >> i) & 1u)) v[c * 32 + i] = MASKED;
          }
        }
        float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int i = 0; i < FA_BN; i += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            mx[u] = max3(mx[u], __uint_as_float(v[i + 2 * u]), __uint_as_float(v[i + 2 * u + 1]));
        }
        const float rmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // the score grows with s: the largest s has the largest score (under a cap a row of -inf has -c)
        const bool none = CAP ? max(c_lo, 0) > min(c_hi, FA_BN - 1) : rmax == -CUDART_INF_F;
        const float m_tile = blind || none ? -CUDART_INF_F
                             : CAP             ? paged_score<true>(ScoreParams{scale, cap_arg, p.score.cap_out}, rmax)
                                               : rmax * scale;
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
        const float neg_m = m_run == -CUDART_INF_F ? 0.0f : p_shift<MF16>() - m_run;
        uint64_t ls2[4] = {0ull, 0ull, 0ull, 0ull};
        // P = exp2(score - m) of 32 columns at a time, to 16 bits, over S's columns
        auto probabilities = [&](auto&& score_minus_m) {
#pragma unroll
          for (int c = 0; c < FA_BN / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float xa, xd;
              unpack2(score_minus_m(pack2(__uint_as_float(v[c * 32 + 2 * i]), __uint_as_float(v[c * 32 + 2 * i + 1]))), xa, xd);
              const float a = ex2_approx(xa), d = ex2_approx(xd);
              ls2[i & 3] = add2(ls2[i & 3], pack2(a, d));
              pk[i] = MF16 ? pack_f16x2(a, d) : pack_bf16x2(a, d);
            }
            tmem_st_32x32b_x16(tS + c * 16, pk);
          }
        };
        const uint64_t negm2 = pack2(neg_m, neg_m);
        if (!CAP) {
          const uint64_t scale2 = pack2(scale, scale);
          probabilities([&](uint64_t s2) { return fma2(s2, scale2, negm2); });
        } else if (poly) {
          auto capped = [&](uint64_t s2) {
            const uint64_t y = fma2(s2, s2, 0ull);
            uint64_t h = fma2(k2[3], y, k2[2]);
            h = fma2(h, y, k2[1]);
            h = fma2(h, y, k2[0]);
            return fma2(s2, h, negm2);
          };
          if (!masked_tile) {
            probabilities(capped);
          } else {
            probabilities([&](uint64_t s2) {
              float sa, sd, xa, xd;
              unpack2(s2, sa, sd);
              unpack2(capped(s2), xa, xd);
              if (__float_as_uint(sa) == MASKED) xa = -CUDART_INF_F;
              if (__float_as_uint(sd) == MASKED) xd = -CUDART_INF_F;
              return pack2(xa, xd);
            });
          }
        } else {
          // some score of the warp's rows is near the cap
          auto each = [&](auto&& score) {
            probabilities([&](uint64_t s2) {
              float sa, sd;
              unpack2(s2, sa, sd);
              float xa = score(sa), xd = score(sd);
              if (__float_as_uint(sa) == MASKED) xa = -CUDART_INF_F;
              if (__float_as_uint(sd) == MASKED) xd = -CUDART_INF_F;
              return pack2(xa, xd);
            });
          };
          const float off = p.score.cap_out + neg_m;
          if (p.score.cap_out <= CAP_SMALL_OUT)
            each([&](float x) { return fmaf(-2.0f * p.score.cap_out, paged_rcp(1.0f + ex2_approx(x * cap_arg)), off); });
          else
            each([&](float x) { return score_any_cap(scale, cap_arg, p.score.cap_out, x) + neg_m; });
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
      // ------------------------------- the part's result ----------------------------------
      if (ok && n_mine > 0) ok = wait_all(bar_o_done + t * 8, items & 1, 31);
      if (!ok) break;
      tc_fence_after_sync();
      if (blind) {
        m_run = -CUDART_INF_F;
        l_run = 0.0f;
      }
      const bool whole = w.whole;
      const float inv_l = !whole ? 1.0f : l_run == 0.0f ? 0.0f : (FP4 ? p.out_scale : 1.0f) / l_run;
      float* part = p.part + ((long long)blockIdx.x * 2 + w.slot) * part_floats(D);
      const int ntok = w.tokens[t];
      uint16_t* out = p.out + (long long)(w.row0 + t * p.tpt) * p.o_ts + (long long)(w.head * p.group) * p.o_hs;
      uint16_t* dst = out + s_row_off[row];
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {           // 32 columns at a time: more spill the softmax loop's registers
        uint32_t o[32];
        if (n_mine > 0) {
          tmem_ld_32x32b_x32(tO + c * 32, o);
          tmem_wait_ld();
        }
        if (n_mine == 0 || l_run == 0.0f) {        // whatever stands there, a row without a key is zero
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (whole) {
          if (tok < ntok) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float lo = __uint_as_float(o[e * 16 + 2 * k]) * inv_l;
                const float hi = __uint_as_float(o[e * 16 + 2 * k + 1]) * inv_l;
                x[k] = F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
              }
              if (p.wide_out) {                    // a full 32-byte sector per lane
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                             ::"l"(dst + c * 32 + e * 16), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]),
                               "r"(x[6]), "r"(x[7]) : "memory");
              } else {
                *reinterpret_cast<uint4*>(dst + c * 32 + e * 16) = make_uint4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<uint4*>(dst + c * 32 + e * 16 + 8) = make_uint4(x[4], x[5], x[6], x[7]);
              }
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            reinterpret_cast<uint4*>(part)[(t * (D / 4) + c * 8 + e) * 128 + row] =
                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      if (!whole) {
        float* ml = part + 2 * 128 * D;
        ml[t * 128 + row] = m_run;
        ml[256 + t * 128 + row] = l_run;
        // the parts of this item: this CTA's and the next ones' first
        if (w.slot == 1 && warp == 4 && lane == 0) p.desc[blockIdx.x] = make_int4(w.parts, w.b, w.pair, w.head);
      }
      done_part(i);
      if (n_mine > 0) ++items;
      tc_fence_before_sync();
    }
  } else if (FP4 && warp >= 12) {
    // ---------------------- NVFP4 rows to f16 operand tiles ----------------------
    reg_dealloc<56>();
    const int r = threadIdx.x - 384;                // key of the step
    constexpr int WORDS = D / 8;                    // packed words per row
    uint32_t wk[WORDS], wv[WORDS], sk[D / 64], sw[D / 64];
    const int slot_mask = (1 << p.batch.page_shift) - 1;
    auto fetch = [&](const Part& w, int j, const uint8_t* pool, const long long (&st)[3], const uint8_t* spool,
                     const long long (&sst)[3], uint32_t (&x)[WORDS], uint32_t (&s)[D / 64]) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) x[i] = 0;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) s[i] = 0;
      const int key = w.key0 + j * FA_BN + r;
      if (key < w.lo || key >= w.hi) return;        // unseen: zeros
      const int pg = page_of(p.batch, w.b, key, status);
      if (pg >= p.batch.num_pages) return;
      const uint8_t* src = pool + pg * st[0] + w.head * st[1] + (key & slot_mask) * st[2];
      const uint8_t* ssrc = spool + pg * sst[0] + w.head * sst[1] + (key & slot_mask) * sst[2];
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        const uint4 y = __ldg(reinterpret_cast<const uint4*>(src) + i);
        x[4 * i] = y.x;
        x[4 * i + 1] = y.y;
        x[4 * i + 2] = y.z;
        x[4 * i + 3] = y.w;
      }
#pragma unroll
      for (int i = 0; i < D / 64; ++i) s[i] = __ldg(reinterpret_cast<const uint32_t*>(ssrc) + i);
    };
    auto expand = [&](uint32_t dst, const uint32_t (&x)[WORDS], const uint32_t (&s)[D / 64]) {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {           // two scales
        const uint32_t two = e4m3x2_to_f16x2((s[i / 8] >> (4 * (i & 4))) & 0xffffu);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t scale = __byte_perm(two, two, k < 2 ? 0x1010 : 0x3232);
          uint32_t o[4];
          e2m1x8_to_f16(x[i + k], o);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = hmul2(o[e], scale);       // exact: two bits times four
          const int c = i + k;
          st_shared_v4(dst + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4), o[0], o[1], o[2], o[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    int it = 0;
    bool ok = true;
    int i = 0, n = 0;
    auto open_part = [&]() {
      for (; have_part(i); ++i) {
        const Part& w = s_part[i % PART_RING];
        n = max(w.steps[0], w.steps[1]);
        if (n > 0) {
          fetch(w, 0, p.k, p.k_st, p.ks, p.ks_st, wk, sk);
          fetch(w, 0, p.v, p.v_st, p.vs, p.vs_st, wv, sw);
          return true;
        }
        done_part(i);
      }
      return false;
    };
    while (ok && open_part()) {
      const Part& w = s_part[i % PART_RING];
      for (int j = 0; j < n; ++j, ++it) {
        const uint32_t stage = it % STAGES, phase = (it / STAGES) & 1;
        if (!wait_all(bar_k_empty + stage * 8, phase ^ 1, 10)) { ok = false; break; }
        expand(sK + stage * TILE, wk, sk);
        if (lane == 0) mbar_arrive(bar_k_full + stage * 8);
        const bool more = j + 1 < n;
        if (more) fetch(w, j + 1, p.k, p.k_st, p.ks, p.ks_st, wk, sk);
        if (!wait_all(bar_v_empty + stage * 8, phase ^ 1, 11)) { ok = false; break; }
        expand(sV + stage * TILE, wv, sw);
        if (lane == 0) mbar_arrive(bar_v_full + stage * 8);
        if (more) fetch(w, j + 1, p.v, p.v_st, p.vs, p.vs_st, wv, sw);
      }
      done_part(i++);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
  // The row-block kernel of the same call runs beside this one and writes other rows.  Whatever follows in the stream
  // waits for the last kernel of the call only, so no CTA here ends before that one has.
  grid_dep_wait();
}

// Adds the parts of the items that were cut, as the row-block kernel's merge does.  Thread = row; blockIdx.y = tile and
// an eighth of the dimensions.
template <int D, bool F16>
__global__ void __launch_bounds__(128) fmha_paged_tile_merge_kernel(const __grid_constant__ TileParams p) {
  grid_dep_wait();
  int4 d = p.desc[blockIdx.x];
  // whatever a workspace holds that other work has written to meanwhile, nothing outside of it is touched
  if (d.x <= 0 || (unsigned)d.y >= (unsigned)p.batch.batch || d.z < 0 || (unsigned)d.w >= (unsigned)p.kv_heads) return;
  d.x = min(d.x, (int)(gridDim.x - blockIdx.x));
  const int t = blockIdx.y & 1, c0 = (blockIdx.y >> 1) * (D / 32);       // float4 columns c0 .. c0 + D / 32
  const int row = threadIdx.x, tok = row / p.group;
  const SeqView sv = seq_view(p.batch, d.y);
  const long long tok0 = (d.z * 2ll + t) * p.tpt;
  if (tok >= min(max(sv.n - tok0, 0ll), (long long)p.tpt)) return;
  float m = -CUDART_INF_F, l = 0.0f;
  float4 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < d.x; ++i) {
    const float* part = p.part + ((long long)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * part_floats(D);
    const float pm = part[2 * 128 * D + t * 128 + row], pl = part[2 * 128 * D + 256 + t * 128 + row];
    float4 v[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) v[c] = reinterpret_cast<const float4*>(part)[(t * (D / 4) + c0 + c) * 128 + row];
    const float mn = fmaxf(m, pm), mu = mn == -CUDART_INF_F ? 0.0f : mn;
    const float wa = ex2_approx(m - mu), wb = ex2_approx(pm - mu);
    m = mn;
    l = l * wa + pl * wb;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      o[c].x = o[c].x * wa + v[c].x * wb;
      o[c].y = o[c].y * wa + v[c].y * wb;
      o[c].z = o[c].z * wa + v[c].z * wb;
      o[c].w = o[c].w * wa + v[c].w * wb;
    }
  }
  const float inv = l == 0.0f ? 0.0f : p.out_scale / l;
  uint16_t* dst = p.out + (long long)(sv.q0 + tok0 + tok) * p.o_ts +
                  (long long)(d.w * p.group + row - tok * p.group) * p.o_hs + c0 * 4;
#pragma unroll
  for (int c = 0; c < D / 32; c += 2)
    *reinterpret_cast<uint4*>(dst + c * 4) =
        make_uint4(paged_pack16<F16>(o[c].x * inv, o[c].y * inv), paged_pack16<F16>(o[c].z * inv, o[c].w * inv),
                   paged_pack16<F16>(o[c + 1].x * inv, o[c + 1].y * inv), paged_pack16<F16>(o[c + 1].z * inv, o[c + 1].w * inv));
}

template <int D, bool F16, bool CAP, bool FP4>
int launch_tile(const PagedAttnArgs& a, const PagedTilePlan& plan) {
  using L = TileSmem<D, FP4>;
  const b200h::DeviceInfo* di = b200h::device_info();
  if (!di) return B200_ERR_CUDA;
  const b200tile_paged_cache& c = *a.cache;
  TileParams p = {};
  p.batch = a.batch;
  p.score = paged_score_params(a, FP4 ? c.k_global : 1.0f);
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
  p.wide_out = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.o_ts % 16 == 0 && a.o_hs % 16 == 0;
  p.out_scale = 1.0f;
  p.part = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + a.tile_off);
  p.desc = reinterpret_cast<int4*>(static_cast<char*>(a.workspace) + a.tile_off + plan.desc_off);
  const CUtensorMapDataType dt = F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tmQ, tmK = {}, tmV = {};
  const uint64_t row = (uint64_t)D * 2;
  if (int rc = b200h::encode_tmap_3d(&tmQ, dt, 2, a.q, D, a.q_heads, a.batch.tokens,
                                     a.q_heads > 1 ? (uint64_t)a.q_hs * 2 : row,
                                     a.batch.tokens > 1 ? (uint64_t)a.q_ts * 2 : row, 64, p.group, p.tpt,
                                     CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if constexpr (FP4) {
    p.out_scale = c.v_global;
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(L::THREADS);
  cfg.dynamicSmemBytes = L::TOTAL;
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.row_limit > 0 ? 1 : 0;          // beside the row-block kernel, or alone behind whatever came before
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, tmQ, tmK, tmV, p, di->status));
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(plan.ctas, 16);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  B200_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fmha_paged_tile_merge_kernel<D, F16>, p));
  return B200_OK;
}

}  // namespace
}  // namespace b200

PagedTilePlan b200_paged_tile_plan(int head_dim) {
  PagedTilePlan pl;
  pl.ctas = 148;
  pl.desc_off = (size_t)pl.ctas * 2 * b200::part_floats(head_dim) * sizeof(float);
  pl.bytes = pl.desc_off + (size_t)pl.ctas * sizeof(int4);
  return pl;
}

int b200_paged_tile_dispatch(const PagedAttnArgs& a) {
  using namespace b200;
  const b200tile_paged_cache& c = *a.cache;
  const PagedTilePlan plan = b200_paged_tile_plan(c.head_dim);
#define B200_PT(D_, F_, C_, Q_) return launch_tile<D_, F_, C_, Q_>(a, plan)
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

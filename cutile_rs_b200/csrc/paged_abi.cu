// Entry points of the paged-cache operators: argument checks, then the dispatchers.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "paged_common.cuh"

using b200h::set_error;

int b200_paged_append_dispatch(int dtype, const b200tile_paged_cache& c, const b200::PagedBatch& batch, const void* q,
                               const void* k, const void* v, void* q_out, const float* inv_freq, int q_heads, int rot,
                               const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* qos,
                               cudaStream_t stream);
int b200_paged_gather_dispatch(int dtype, const b200tile_paged_cache& c, const b200::PagedBatch& batch, void* k_out,
                               void* v_out, const int64_t* ks, const int64_t* vs, cudaStream_t stream);

namespace {

// Which kernel takes a sequence of `rows` query rows (tokens * group) per K/V head.  The row-block kernel reads the cache
// once per 16 rows, the tile kernel once per 256 but with more to start and end; it pays once the call is large enough.
// Measured (us, row blocks against tiles, 8 K/V heads of 128):
//   16-bit, 20 rows:  8 x 1024 keys 17 / 27, 8 x 2048 keys 38 / 32, 32 x 8192 keys 354 / 211
//   16-bit, 64 rows:  1 x 2048 keys 16 / 25, 8 x 1024 keys 30 / 28, 32 x 2048 keys 191 / 71
//   NVFP4,  36 rows:  8 x 1024 keys 34 / 38, 32 x 8192 keys 312 / 304;  20 rows: 32 x 8192 keys 217 / 303
//   NVFP4,  64 rows:  8 x 512 keys 32 / 36, 8 x 2048 keys 49 / 42, 32 x 8192 keys 410 / 305
int tile_rows(const b200tile_paged_cache* c) { return c->format ? 48 : 16; }
bool may_tile(const b200tile_paged_cache* c, const b200tile_paged_batch* b, int group) {
  const long long rows = (long long)b->max_q_len * group;
  if (group > 128 || rows <= tile_rows(c)) return false;
  // steps of 16 keys that the row blocks of the largest such call would take
  const long long keys = (long long)b->max_pages * c->page_size;
  const double steps = (double)b->batch * c->kv_heads * (double)((rows + 15) / 16) * (double)((keys + 15) / 16);
  return steps >= (c->format ? 16384.0 : 12288.0);
}

bool misaligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int check_dtype(const char* dtype, const char* who, int* dt) {
  if (!dtype) return set_error(B200TILE_ERR_INVALID, "%s: dtype is null", who);
  if (!strcmp(dtype, "bf16")) *dt = 0;
  else if (!strcmp(dtype, "f16")) *dt = 1;
  else return set_error(B200TILE_ERR_UNSUPPORTED, "%s: unsupported element type '%s'", who, dtype);
  return B200TILE_OK;
}

// extents of 1 put no condition on their stride
int check_pool(const char* who, const char* name, const void* p, const int64_t* st, const int extents[3], int unit,
               uintptr_t align, bool bytes) {
  if (!p) return set_error(B200TILE_ERR_INVALID, "%s: the %s pool is null", who, name);
  bool bad = misaligned(p, align);
  for (int i = 0; i < 3; ++i) {
    if (extents[i] > 1 && st[i] <= 0)
      return set_error(B200TILE_ERR_INVALID, "%s: strides of the %s pool must be positive", who, name);
    bad |= extents[i] > 1 && st[i] % unit != 0;
    if (bytes && i != 1 && extents[i] > 1 && st[i] > 0x7fffffff)
      return set_error(B200TILE_ERR_UNSUPPORTED, "%s: page and slot strides of the %s pool must be below 2^31 bytes", who, name);
  }
  if (bad)
    return set_error(B200TILE_ERR_ALIGN, "%s: the %s pool must be %d-byte aligned with strides that are multiples of %d",
                     who, name, (int)align, unit);
  return B200TILE_OK;
}

int check_cache(const char* who, const b200tile_paged_cache* c) {
  if (!c) return set_error(B200TILE_ERR_INVALID, "%s: cache is null", who);
  if (c->format != 0 && c->format != 1)
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: cache format %d (0: 16-bit, 1: NVFP4)", who, c->format);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are provided)", who, c->head_dim);
  if (c->num_pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0)
    return set_error(B200TILE_ERR_INVALID, "%s: Shape dimensions must be positive", who);
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1)))
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: page_size %d is not a power of two of at least 16", who, c->page_size);
  const int ext[3] = {c->num_pages, c->kv_heads, c->page_size};
  const int unit = c->format ? 16 : 8;
  if (int rc = check_pool(who, "K", c->k, c->k_strides, ext, unit, 16, c->format == 1)) return rc;
  if (int rc = check_pool(who, "V", c->v, c->v_strides, ext, unit, 16, c->format == 1)) return rc;
  if (c->format) {
    const int row = c->head_dim / 16;
    if (int rc = check_pool(who, "K scale", c->k_scales, c->k_scale_strides, ext, row, row, true)) return rc;
    if (int rc = check_pool(who, "V scale", c->v_scales, c->v_scale_strides, ext, row, row, true)) return rc;
    if (!(c->k_global > 0.0f && c->v_global > 0.0f) || !isfinite(c->k_global) || !isfinite(c->v_global))
      return set_error(B200TILE_ERR_INVALID, "%s: k_global and v_global must be positive and finite", who);
  }
  return B200TILE_OK;
}

int check_batch(const char* who, const b200tile_paged_cache* c, const b200tile_paged_batch* b, int tokens) {
  if (!b) return set_error(B200TILE_ERR_INVALID, "%s: batch is null", who);
  if (b->batch < 0 || tokens < 0) return set_error(B200TILE_ERR_INVALID, "%s: batch and tokens must not be negative", who);
  // without sequences or tokens there is nothing to point to, and nothing to do
  if (b->batch > 0 && tokens > 0 && (!b->block_table || !b->cu_q || !b->kv_lens))
    return set_error(B200TILE_ERR_INVALID, "%s: block_table, cu_q and kv_lens are required", who);
  if (misaligned(b->block_table, 4) || misaligned(b->cu_q, 4) || misaligned(b->kv_lens, 4))
    return set_error(B200TILE_ERR_ALIGN, "%s: block_table, cu_q and kv_lens must be 4-byte aligned", who);
  if (b->max_pages <= 0 || b->max_q_len <= 0)
    return set_error(B200TILE_ERR_INVALID, "%s: max_pages and max_q_len must be positive", who);
  if (b->block_table_pitch < b->max_pages && b->batch > 1)
    return set_error(B200TILE_ERR_INVALID, "%s: block_table_pitch is shorter than max_pages", who);
  if ((long long)b->max_pages * c->page_size > 0x7fffff00LL)
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: %d pages of %d exceed 2^31 positions", who, b->max_pages, c->page_size);
  return B200TILE_OK;
}

// Workspace of the row-block kernel for sequences of up to `rows` query rows, a multiple of 256 bytes.
size_t split_bytes(const b200tile_paged_cache* c, const b200tile_paged_batch* b, long long rows) {
  const size_t n = b200_paged_split_plan(c->format, c->head_dim, c->kv_heads, b->batch, rows,
                                         (long long)b->max_pages * c->page_size).bytes;
  return (n + 255) & ~(size_t)255;
}

b200::PagedBatch device_batch(const b200tile_paged_cache* c, const b200tile_paged_batch* b, int tokens) {
  b200::PagedBatch p;
  p.table = b->block_table;
  p.cu_q = b->cu_q;
  p.kv_lens = b->kv_lens;
  p.table_pitch = b->block_table_pitch;
  p.batch = b->batch;
  p.max_pages = b->max_pages;
  p.num_pages = c->num_pages;
  p.page_shift = __builtin_ctz((unsigned)c->page_size);
  p.tokens = tokens;
  p.max_q = std::min(b->max_q_len, tokens);
  return p;
}

int check_rows(const char* who, const char* name, const void* p, const int64_t* st, int tokens, int unit,
               uintptr_t align) {
  if ((!p && tokens > 0) || !st) return set_error(B200TILE_ERR_INVALID, "%s: %s and its strides are required", who, name);
  if (misaligned(p, align) || st[0] % unit || st[1] % unit)
    return set_error(B200TILE_ERR_ALIGN, "%s: %s must be %d-byte aligned with strides that are multiples of %d", who, name,
                     (int)align, unit);
  return B200TILE_OK;
}

// the same for rows that are written: each must have a place of its own
int check_out_rows(const char* who, const char* name, const void* p, const int64_t* st, int tokens, int heads, int unit,
                   uintptr_t align) {
  if (int rc = check_rows(who, name, p, st, tokens, unit, align)) return rc;
  if ((tokens > 1 && st[0] == 0) || (heads > 1 && st[1] == 0))
    return set_error(B200TILE_ERR_INVALID, "%s: the rows of %s must not share memory (a stride is 0)", who, name);
  return B200TILE_OK;
}

}  // namespace

extern "C" {

int b200tile_paged_kv_append(const char* dtype, const b200tile_paged_cache* cache, const b200tile_paged_batch* batch,
                             const void* q, const void* k, const void* v, void* q_out, const float* inv_freq, int tokens,
                             int q_heads, int rotary_dim, const int64_t q_strides[2], const int64_t k_strides[2],
                             const int64_t v_strides[2], const int64_t q_out_strides[2], void* cu_stream) {
  const char* who = "paged_kv_append";
  int dt;
  if (int rc = check_dtype(dtype, who, &dt)) return rc;
  if (int rc = check_cache(who, cache)) return rc;
  if (int rc = check_batch(who, cache, batch, tokens)) return rc;
  const int unit = cache->format ? 32 : 16;
  if (rotary_dim < 0 || rotary_dim > cache->head_dim || rotary_dim % unit)
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: rotary_dim %d must be a multiple of %d from 0 to head_dim %d", who,
                     rotary_dim, unit, cache->head_dim);
  if (rotary_dim > 0 && !inv_freq) return set_error(B200TILE_ERR_INVALID, "%s: inv_freq is required for a rotation", who);
  if (misaligned(inv_freq, 4)) return set_error(B200TILE_ERR_ALIGN, "%s: inv_freq must be 4-byte aligned", who);
  if ((q == nullptr) != (q_out == nullptr))
    return set_error(B200TILE_ERR_INVALID, "%s: q and q_out are given together or not at all", who);
  if (q) {
    if (q_heads <= 0) return set_error(B200TILE_ERR_INVALID, "%s: q_heads must be positive", who);
    if (int rc = check_rows(who, "q", q, q_strides, tokens, 8, 16)) return rc;
    if (int rc = check_out_rows(who, "q_out", q_out, q_out_strides, tokens, q_heads, 8, 16)) return rc;
  }
  if (int rc = check_rows(who, "k", k, k_strides, tokens, 8, 16)) return rc;
  if (int rc = check_rows(who, "v", v, v_strides, tokens, 8, 16)) return rc;
  if (tokens == 0 || batch->batch == 0) return B200TILE_OK;
  return b200_paged_append_dispatch(dt, *cache, device_batch(cache, batch, tokens), q, k, v, q_out, inv_freq, q_heads,
                                    rotary_dim, q_strides, k_strides, v_strides, q_out_strides,
                                    static_cast<cudaStream_t>(cu_stream));
}

int b200tile_paged_kv_gather(const char* dtype, const b200tile_paged_cache* cache, const b200tile_paged_batch* batch,
                             void* k_out, void* v_out, int tokens, const int64_t k_out_strides[2],
                             const int64_t v_out_strides[2], void* cu_stream) {
  const char* who = "paged_kv_gather";
  int dt;
  if (int rc = check_dtype(dtype, who, &dt)) return rc;
  if (int rc = check_cache(who, cache)) return rc;
  if (int rc = check_batch(who, cache, batch, tokens)) return rc;
  if (int rc = check_out_rows(who, "k_out", k_out, k_out_strides, tokens, cache->kv_heads, 8, 16)) return rc;
  if (int rc = check_out_rows(who, "v_out", v_out, v_out_strides, tokens, cache->kv_heads, 8, 16)) return rc;
  if (tokens == 0 || batch->batch == 0) return B200TILE_OK;
  return b200_paged_gather_dispatch(dt, *cache, device_batch(cache, batch, tokens), k_out, v_out, k_out_strides,
                                    v_out_strides, static_cast<cudaStream_t>(cu_stream));
}

uint64_t b200tile_paged_attention_workspace_bytes(const b200tile_paged_cache* cache, const b200tile_paged_batch* batch,
                                                  int q_heads) {
  if (!cache || !batch || cache->kv_heads <= 0 || q_heads <= 0 || batch->batch <= 0 || batch->max_pages <= 0 ||
      batch->max_q_len <= 0 || cache->page_size <= 0 || cache->head_dim <= 0)
    return 0;
  const int group = q_heads / cache->kv_heads;
  const size_t all = split_bytes(cache, batch, (long long)batch->max_q_len * group);
  if (!may_tile(cache, batch, group)) return all;
  // the tile kernel's part lies behind the row-block kernel's; without it (rows it cannot move) the latter takes all rows
  return std::max(all, split_bytes(cache, batch, tile_rows(cache)) + b200_paged_tile_plan(cache->head_dim).bytes);
}

int b200tile_paged_attention(const char* dtype, const b200tile_paged_cache* cache, const b200tile_paged_batch* batch,
                             const void* q, void* out, int tokens, int q_heads, const int64_t q_strides[2],
                             const int64_t out_strides[2], float qk_scale, int causal, int window, float softcap,
                             void* workspace, uint64_t workspace_bytes, void* cu_stream) {
  const char* who = "paged_attention";
  PagedAttnArgs a = {};
  if (int rc = check_dtype(dtype, who, &a.dtype)) return rc;
  if (int rc = check_cache(who, cache)) return rc;
  if (int rc = check_batch(who, cache, batch, tokens)) return rc;
  if (int rc = check_rows(who, "q", q, q_strides, tokens, 2, 4)) return rc;
  if (int rc = check_out_rows(who, "out", out, out_strides, tokens, q_heads, 2, 4)) return rc;
  if (q_heads <= 0 || q_heads % cache->kv_heads)
    return set_error(B200TILE_ERR_INVALID, "%s: q_heads %d must be a positive multiple of kv_heads %d", who, q_heads,
                     cache->kv_heads);
  const int group = q_heads / cache->kv_heads;
  if ((long long)tokens * group > 0x7fffff00LL)
    return set_error(B200TILE_ERR_UNSUPPORTED, "%s: more than 2^31 query rows per K/V head", who);
  if (!(qk_scale > 0.0f) || !isfinite(qk_scale))
    return set_error(B200TILE_ERR_INVALID, "%s: qk_scale must be positive and finite", who);
  if (!(softcap >= 0.0f) || !isfinite(softcap))
    return set_error(B200TILE_ERR_INVALID, "%s: softcap must be 0 (none) or positive and finite", who);
  if (window < 0 || (window > 0 && !causal))
    return set_error(B200TILE_ERR_INVALID, "%s: window must be 0 (none) or positive, and needs causal", who);
  if (tokens == 0 || batch->batch == 0) return B200TILE_OK;
  const uint64_t need = b200tile_paged_attention_workspace_bytes(cache, batch, q_heads);
  if (!workspace || workspace_bytes < need)
    return set_error(B200TILE_ERR_INVALID, "%s: a workspace of %llu bytes is required (got %llu)", who,
                     (unsigned long long)need, (unsigned long long)(workspace ? workspace_bytes : 0));
  if (misaligned(workspace, 16)) return set_error(B200TILE_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
  a.cache = cache;
  a.batch = device_batch(cache, batch, tokens);
  a.q = q;
  a.out = out;
  a.q_heads = q_heads;
  a.q_ts = q_strides[0];
  a.q_hs = q_strides[1];
  a.o_ts = out_strides[0];
  a.o_hs = out_strides[1];
  a.qk_scale = qk_scale;
  a.softcap = softcap;
  a.capped = softcap > 0.0f;
  a.causal = causal != 0;
  a.window = window;
  a.workspace = workspace;
  a.stream = static_cast<cudaStream_t>(cu_stream);
  // the tile kernel moves rows by TMA and in 16-byte pieces; rows that do not lie so take row blocks, whatever their number
  const bool tiles = may_tile(cache, batch, group) && (long long)a.batch.max_q * group > tile_rows(cache) && !misaligned(q, 16) && !misaligned(out, 16) && !(a.q_ts % 8) &&
                     !(a.q_hs % 8) && !(a.o_ts % 8) && !(a.o_hs % 8) && a.q_ts > 0 && a.q_hs > 0;
  a.tile_off = tiles ? split_bytes(cache, batch, tile_rows(cache)) : 0;
  // Prompts alone take one launch of the tile kernel; decode steps with prompts among them take both kernels, each its
  // own sequences.  The second kernel costs 2 to 20 us (launches, merge, its CTAs in front of the tiles'); a decode step in
  // the tile kernel costs a whole tile per 128 keys and about two more to begin and end, and its probabilities get one
  // 16-bit piece instead of two.  How many decode steps there may be follows from the sizes: as many sequences as are
  // left when the others have max_q_len tokens each; how many keys they may have, from the table's width.
  // Measured (us, one kernel against two, 8 K/V heads of 128, beside a prompt of 512 tokens; in brackets heads * (keys / 128 + 2)):
  //   NVFP4   16 steps of 1024 keys (1280) 44 / 49, 31 of 1024 (2480) 62 / 55, 16 of 4096 (4352) 96 / 67, 1 of 65536 (4112)
  //           96 / 66, 255 of 256 (8160) 197 / 90, 8 of 131072 (65664) 1115 / 407
  //   16-bit  16 steps of 4096 keys (4352) 72 / 96, 16 of 16384 (16640) 210 / 223, 31 of 16384 (32240) 384 / 365, 8 of
  //           131072 (65664) 766 / 726; by their number: 31 of 256 37 / 40, 64 of 256 53 / 52, 127 of 256 87 / 72
  //   prompts alone, their lengths so uneven that some could be steps: 35 / 37 to 182 / 187, NVFP4 40 / 41 to 135 / 142
  const long long full = (tokens + (long long)batch->max_q_len - 1) / batch->max_q_len;
  const long long steps = (batch->batch - full) * cache->kv_heads;
  const long long each = (long long)batch->max_pages * cache->page_size / 128 + 2;
  const bool only_tiles = tiles && (cache->format ? steps * each <= 1536 : steps <= 256 && steps * each <= 20480);
  a.row_limit = only_tiles ? 0 : tiles ? tile_rows(cache) : 0x7fffffff;
  if (!only_tiles)
    if (int rc = b200_paged_split_dispatch(a)) return rc;
  return tiles ? b200_paged_tile_dispatch(a) : B200TILE_OK;
}

}  // extern "C"

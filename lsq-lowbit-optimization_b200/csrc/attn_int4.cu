// Entry points of the attention over the 4-bit cache: checks, the plan of a call, dispatch.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "attn_int4_host.cuh"
#include "prefill_int4.cuh"

namespace {

using namespace w4a8;

struct Plan {
  int n_tiles, row_tiles, splits, chunk;
  long long tiles;  // (sequence, key head, row tile)
};

// How a call is split. One sequence goes to as many blocks as the GPU holds at once. Several may have
// unequal lengths: their blocks are short enough to fill the GPU kWaves times over. A block has at least
// kMinChunk tokens, twice as many in a batch: below that its start and the join cost more than the tokens (1024 tokens
// of one sequence: 7.4 us with 128, 8.0 with 256; 7 sequences of up to 2011: 16.4 and 13.1).
constexpr int kWaves = 6, kMinChunk = kAttnWarps * kTile, kPreMinChunk = 4 * kPreTile;
// From this many query rows a key head on, the tensor cores' tiles of 128 rows pay. 8192 tokens, 8 heads of 128 channels, few-row
// kernel and prompt kernel, us: 16 sequences of 48 rows 194 and 203, of 64 rows 250 and 200, of 128 rows 447 and 165. One
// sequence alone, which few rows split finer: 64 rows 25 and 32, 96 rows 30 and 33, 128 rows 39 and 33. 64 channels alike.
constexpr int kPrefillRows = 64;

// Tensor maps of the codes, for boxes of 32 or 16 rows of a page; the rows of a box, or 0 where pages are
// not whole boxes or a stride cannot be mapped.
int code_maps(const w4a8_kv_cache* c, AttnParams* p) {
  const int box = c->page_size % 32 == 0 ? 32 : c->page_size % 16 == 0 ? 16 : 0;
  const uint64_t strides[3] = {uint64_t(c->code_tok), uint64_t(c->code_head), uint64_t(c->code_page)};
  std::memset(&p->k_map, 0, sizeof(p->k_map));
  std::memset(&p->v_map, 0, sizeof(p->v_map));
  if (!box || !c->pages) return 0;
  for (const uint64_t s : strides)
    if (s == 0 || s >= (1ull << 40)) return 0;
  const uint64_t dims[4] = {uint64_t(c->head_dim / 2), uint64_t(c->page_size), uint64_t(c->heads), uint64_t(c->pages)};
  const uint32_t extent[4] = {uint32_t(c->head_dim / 2), uint32_t(box), 1, 1};
  const CUtensorMapSwizzle swizzle = c->head_dim == 64    ? CU_TENSOR_MAP_SWIZZLE_32B
                                     : c->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B
                                     : c->head_dim == 256 ? CU_TENSOR_MAP_SWIZZLE_128B
                                                          : CU_TENSOR_MAP_SWIZZLE_NONE;
  if (encode_u8(&p->k_map, c->k_codes, 4, dims, strides, extent, swizzle) != W4A8_OK ||
      encode_u8(&p->v_map, c->v_codes, 4, dims, strides, extent, swizzle) != W4A8_OK)
    return 0;
  return box;
}

int make_plan(const w4a8_kv_cache* c, int q_heads, int dtype, int max_q, int max_len, int window, Plan* p) {
  const long long rows = (long long)max_q * (q_heads / c->heads);
  if (rows > 0x7fffffff) return W4A8_ERR_UNSUPPORTED;
  const bool f32 = dtype == W4A8_F32;
  p->n_tiles = rows >= kPrefillRows && prefill_ok(c->head_dim, f32) ? 0
               : rows > 8 && attn_wide_ok(c->head_dim, f32)         ? 2
                                                                    : 1;
  const int tile_rows = p->n_tiles ? 8 * p->n_tiles : kPreRows, tile_tokens = p->n_tiles ? kTile : kPreTile;
  const int least = !p->n_tiles ? kPreMinChunk : c->batch > 1 || max_len <= 2 * kMinChunk ? 2 * kMinChunk : kMinChunk;
  p->row_tiles = int((rows + tile_rows - 1) / tile_rows);
  p->tiles = (long long)c->batch * c->heads * p->row_tiles;
  long long tokens = std::min((long long)max_len, std::max(0ll, (long long)c->table_cols * c->page_size));
  if (window > 0) tokens = std::min(tokens, (long long)window + tile_rows + tile_tokens);
  const long long blocks = (long long)device_sms() *
                           (p->n_tiles ? attn_blocks_sm(c->head_dim, p->n_tiles, f32) * (c->batch > 1 ? kWaves : 1) : 1);
  const long long want = std::max(1ll, blocks / std::max(1ll, p->tiles));
  long long chunk = std::max<long long>(least, (tokens + want - 1) / want);
  chunk = (chunk + least - 1) / least * least;
  p->chunk = int(std::min<long long>(chunk, 0x7fffffff / least * least));
  p->splits = int(std::max(1ll, (tokens + chunk - 1) / chunk));
  if (p->tiles * (p->n_tiles ? p->splits : std::max(p->splits, kRedoParts)) > 0x7fffffff) return W4A8_ERR_UNSUPPORTED;
  return W4A8_OK;
}

// Partial results of calls that are split, then a word for each block of many rows.
size_t parts_of(const w4a8_kv_cache* c, int q_heads, const Plan& p) {
  if (p.splits == 1) return 0;
  return size_t(c->rows) * q_heads * p.splits * (size_t(c->head_dim) + 2) * 4;
}
size_t workspace_of(const w4a8_kv_cache* c, int q_heads, const Plan& p) {
  return parts_of(c, q_heads, p) + (p.n_tiles ? 0 : size_t(p.tiles) * p.splits * 4);
}

int check(const w4a8_kv_cache* c, int q_heads, int dtype, int max_q, int max_len, int window) {
  if (!c || c->pages < 0 || c->page_size < 1 || c->batch < 0 || c->rows < 0 || c->table_cols < 0) return W4A8_ERR_ARG;
  if (dtype < W4A8_F32 || dtype > W4A8_BF16 || c->heads < 1 || q_heads < 1 || q_heads % c->heads || max_q < 0 ||
      max_len < 0 || window < 0)
    return W4A8_ERR_ARG;
  if ((long long)c->table_cols * c->page_size > kKvMostTokens) return W4A8_ERR_UNSUPPORTED;
  if (!kv_head_dim_ok(c->head_dim)) return W4A8_ERR_UNSUPPORTED;
  return W4A8_OK;
}

}  // namespace

extern "C" int w4a8_attention_int4_workspace(const w4a8_kv_cache* cache, int q_heads, int dtype, int max_q, int max_len,
                                             int window, size_t* bytes) {
  if (!bytes) return W4A8_ERR_ARG;
  *bytes = 0;
  int rc = check(cache, q_heads, dtype, max_q, max_len, window);
  if (rc != W4A8_OK) return rc;
  if (cache->rows == 0 || cache->batch == 0 || max_q == 0) return W4A8_OK;
  Plan plan;
  rc = make_plan(cache, q_heads, dtype, max_q, max_len, window, &plan);
  if (rc == W4A8_OK) *bytes = workspace_of(cache, q_heads, plan);
  return rc;
}

extern "C" int w4a8_attention_int4(const w4a8_kv_cache* cache, const void* q, int64_t q_row, int64_t q_head,
                                   int q_heads, int dtype, void* out, float* lse, float scale, int causal, int window,
                                   int max_q, int max_len, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(cache, q_heads, dtype, max_q, max_len, window);
  if (rc != W4A8_OK) return rc;
  AttnParams p;
  rc = kv_view(cache, &p.view);
  if (rc != W4A8_OK) return rc;
  if (cache->rows == 0) return W4A8_OK;
  if (cache->batch == 0 || max_q == 0) return W4A8_ERR_ARG;
  if (!q || !out || !std::isfinite(scale)) return W4A8_ERR_ARG;
  const int size = dtype == W4A8_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(q) % size || reinterpret_cast<uintptr_t>(out) % 16) return W4A8_ERR_ALIGN;
  Plan plan;
  rc = make_plan(cache, q_heads, dtype, max_q, max_len, window, &plan);
  if (rc != W4A8_OK) return rc;
  const size_t need = workspace_of(cache, q_heads, plan), parts = parts_of(cache, q_heads, plan);
  if (need > workspace_bytes || (need && !workspace)) return W4A8_ERR_ARG;
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16) return W4A8_ERR_ALIGN;
  p.q = q;
  p.q_row = q_row;
  p.q_head = q_head;
  p.q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_row * size % 16 == 0 && q_head * size % 16 == 0;
  p.out = out;
  p.lse = lse;
  p.q_heads = q_heads;
  p.ratio = q_heads / cache->heads;
  p.by_ratio = fast_div(unsigned(p.ratio));
  // The kernels multiply by a positive factor and give the query the scale's sign (or zeros for 0).
  p.scale_log2 = scale == 0.0f ? 1.0f : std::max(float(std::fabs(double(scale)) * 1.4426950408889634), 1.2e-38f);
  p.sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
  p.box_rows = code_maps(cache, &p);
  p.causal = causal != 0;
  p.window = window;
  p.max_q = max_q;
  p.row_tiles = plan.row_tiles;
  p.splits = plan.splits;
  p.by_splits = fast_div(unsigned(plan.splits));
  p.by_row_tiles = fast_div(unsigned(plan.row_tiles));
  p.by_heads = fast_div(unsigned(cache->heads));
  p.chunk = plan.chunk;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (parts ? size_t(cache->rows) * q_heads * plan.splits * cache->head_dim : 0));
  p.handover = plan.n_tiles ? nullptr : reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + parts);
  const unsigned grid = unsigned(plan.tiles * plan.splits);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->head_dim) {
    case 64: return launch_attn_int4_d64(p, dtype, plan.n_tiles, grid, st);
    case 96: return launch_attn_int4_d96(p, dtype, plan.n_tiles, grid, st);
    case 128: return launch_attn_int4_d128(p, dtype, plan.n_tiles, grid, st);
    case 192: return launch_attn_int4_d192(p, dtype, plan.n_tiles, grid, st);
    default: return launch_attn_int4_d256(p, dtype, plan.n_tiles, grid, st);
  }
}

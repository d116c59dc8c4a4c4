// C entry of paged attention: checks, workspace layout, launches.
#include <algorithm>

#include "paged_attention.cuh"

namespace sunshape {
namespace {


int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  int64_t slots, desc, pieces, prefix, prefix_slots, total;
};

// Query rows of a KV head from which on the prefix goes to the tensor-core kernel: it rebuilds a key once for 256 rows
// where the memory-bound kernel reads it again for every 16.  The whole call in us, 8 heads, 100 to 500 own tokens a sequence,
// prefixes of 100, 1000, 10000 and 40000 tokens:
//   rows   tensor cores        memory-bound
//    16    23  27  38  71      35  36  41   71
//    20    27  30  41  71      34  36  44   79
//    64    31  34  46  80      36  38  54  113
//   128    36  40  52  88      39  43  72  175
// With one head, whose tiles spread over all blocks, the memory-bound kernel is ahead from about 8000 tokens on (40 rows, 10000
// tokens: 53 against 41).
constexpr int64_t kPrefixRows = 17;

constexpr int64_t kOverlapTiles = kWaitLimitNs / 2500 / 8;

// item_rows: of the memory-bound kernel's calls; tensor: the prefix goes to the tensor-core kernel
Layout layout(int grid, int64_t rows, int64_t item_rows, int dv, bool prefix, bool tensor) {
  const int64_t row = row_floats(dv) * 4;
  Layout l;
  l.slots = 0;
  l.desc = round256(2 * grid * kItemRows * row);
  l.pieces = l.desc + round256((int64_t)grid * 16);
  l.prefix = l.pieces + round256((int64_t)grid * kPairs * 2 * item_rows * row);
  l.prefix_slots = l.prefix + (prefix ? round256(rows * row) : 0);
  l.total = l.prefix_slots + (tensor ? round256(2 * (int64_t)grid * 256 * row) : 0);
  return l;
}

// 8 or 16 query rows an item
int item_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }

// Stages of the rings: what is left beside the codebook and the plan, at least two for each pair of warps that works.
bool plan(AttnParams& p, int d, int dv, int bd) {
  p.item_rows = item_rows((p.prefix_mode ? (int64_t)p.B : 1) * p.G * p.L);
  p.off_idx = kTile * dv * 2;
  p.off_heavy = p.off_idx + kTile * p.nb;
  p.stage_bytes = (p.off_heavy + kTile * p.n_heavy * bd * 2 + 1023) / 1024 * 1024;
  // alignment, codebook, permutation, plan, codebook barrier, pieces' descriptions, dense slots
  const int fixed = 1024 + d * 512 + d * 4 + (2 * kPlanChunks + 2) * 4 + 8 + 16 + kPairs * 32 + p.nb;
  const int left = kSmemMax - fixed;
  p.stages = std::min(6, left / (kPairs * (p.stage_bytes + 20)));
  p.pairs = kPairs;
  if (p.stages < 2) {
    p.stages = 2;
    p.pairs = (left - kPairs * 2 * 20) / (2 * p.stage_bytes);
  }
  p.smem = fixed + p.pairs * p.stages * p.stage_bytes + kPairs * p.stages * 20;
  return p.pairs >= 1;
}

template <typename T, bool PREFIX>
int launch(const AttnParams& p, const CUtensorMap& vmap, int d, int dv, int bd, int grid, cudaStream_t st) {
#define SUNSHAPE_PAGED_CASE(D, DV, BD)                       \
  if (d == D && dv == DV && bd == BD) {                      \
    if constexpr (PREFIX) return launch_paged_prefix<D, DV, BD, T>(p, vmap, grid, st); \
    else return launch_paged_attention<D, DV, BD, T>(p, vmap, grid, st); \
  }
  SUNSHAPE_PAGED_CASE(64, 64, 2) SUNSHAPE_PAGED_CASE(64, 64, 4) SUNSHAPE_PAGED_CASE(64, 64, 8)
  SUNSHAPE_PAGED_CASE(64, 128, 2) SUNSHAPE_PAGED_CASE(64, 128, 4) SUNSHAPE_PAGED_CASE(64, 128, 8)
  SUNSHAPE_PAGED_CASE(128, 64, 2) SUNSHAPE_PAGED_CASE(128, 64, 4) SUNSHAPE_PAGED_CASE(128, 64, 8)
  SUNSHAPE_PAGED_CASE(128, 128, 2) SUNSHAPE_PAGED_CASE(128, 128, 4) SUNSHAPE_PAGED_CASE(128, 128, 8)
#undef SUNSHAPE_PAGED_CASE
  return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention: no kernel for these dimensions.");
}

}  // namespace
}  // namespace sunshape

using namespace sunshape;

extern "C" {

int64_t sunshape_paged_attention_workspace_bytes(int32_t batch, int32_t q_heads, int32_t kv_heads, int32_t query_len,
                                                 int32_t value_dim, int32_t table_cols, int32_t page_size,
                                                 int32_t prefix_len) {
  (void)table_cols;
  (void)page_size;
  const int64_t rows = (int64_t)batch * q_heads * query_len;
  const int64_t own = kv_heads > 0 ? (int64_t)q_heads / kv_heads * query_len : 0;
  const bool tensor = prefix_len > 0 && own * batch >= kPrefixRows;
  return layout(paged_sm_count(), rows, item_rows(prefix_len > 0 && !tensor ? own * batch : own), value_dim, prefix_len > 0, tensor).total;
}

int sunshape_paged_attention(const sunshape_codec_t* codec, const void* tables, const sunshape_pages_t* pages,
                             const sunshape_rows_t* query, int32_t batch, int32_t query_len,
                             const int32_t* page_table, int64_t table_stride, int32_t table_cols,
                             const int32_t* seq_lens, const int32_t* prefix_table, int32_t prefix_len, float scale,
                             int32_t causal, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_pages(codec, pages)) return rc;
  if (!query) return set_last_error(SUNSHAPE_E_INVALID, "query rows descriptor is NULL.");
  if (codec->head_dim != 64 && codec->head_dim != 128)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention takes head_dim 64 or 128.");
  if (pages->value_dim != 64 && pages->value_dim != 128)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention takes value_dim 64 or 128.");
  if (batch < 0 || query_len < 0 || query->heads < 0 || table_cols < 0 || prefix_len < 0)
    return set_last_error(SUNSHAPE_E_INVALID, "negative size.");
  if (query->heads % pages->kv_heads)
    return set_last_error(SUNSHAPE_E_INVALID, "Query head count must be divisible by kv-head count.");
  if ((int64_t)table_cols * pages->page_size > (int64_t)1 << 30 || prefix_len > 1 << 30)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 2^30 tokens a sequence.");
  const int64_t rows = (int64_t)batch * query->heads * query_len;
  if (rows == 0) return SUNSHAPE_OK;
  if (batch > 65535 || rows > (int64_t)1 << 30)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 65535 sequences and 2^30 query rows a call.");
  if (!query->data || !out || !seq_lens || (table_cols && !page_table) || (prefix_len && !prefix_table) || !tables)
    return set_last_error(SUNSHAPE_E_INVALID, "query / out / seq_lens / page table / tables pointer is NULL.");
  if ((uintptr_t)out % 8) return set_last_error(SUNSHAPE_E_INVALID, "paged attention: out must be 8-byte aligned.");
  if (!workspace || (uintptr_t)workspace % 256 ||
      workspace_bytes < sunshape_paged_attention_workspace_bytes(batch, query->heads, pages->kv_heads, query_len,
                                                                 pages->value_dim, table_cols, pages->page_size,
                                                                 prefix_len))
    return set_last_error(SUNSHAPE_E_WORKSPACE, "paged attention: workspace missing, misaligned or too small.");
  AttnParams p{};
  p.q = query->data;
  p.qs[0] = query->stride_b;
  p.qs[1] = query->stride_h;
  p.qs[2] = query->stride_l;
  p.B = batch;
  p.Hq = query->heads;
  p.H = pages->kv_heads;
  p.L = query_len;
  p.G = p.Hq / p.H;
  const int d = codec->head_dim, dv = pages->value_dim, bd = codec->block_dim;
  p.nb = d / bd;
  p.n_cb = codec->n_cb;
  p.ps = pages->page_size;
  p.n_heavy = codec->heavy_mask ? codec->n_heavy : 0;
  p.cols = table_cols;
  p.causal = causal;
  p.chunk = p.ps % kTile ? 16 : kTile;
  p.num_pages = pages->num_pages;
  p.table_stride = table_stride;
  p.scale_log2 = scale * kLog2e;
  p.table = page_table;
  p.lens = seq_lens;
  p.perm = codec->permutation;
  p.heavy_mask = p.n_heavy ? codec->heavy_mask : nullptr;
  p.idx = pages->indices;
  p.heavy = pages->heavy;
  const Tables tab(p.n_cb, p.nb, d);
  p.image = tables;
  p.image_scale = reinterpret_cast<const float*>(static_cast<const uint8_t*>(tables) + tab.iscale);
  p.out = out;
  const int grid = paged_sm_count();
  const int64_t own = (int64_t)p.G * p.L;
  const bool tensor = prefix_len > 0 && own * batch >= kPrefixRows;
  const Layout at = layout(grid, rows, item_rows(prefix_len && !tensor ? own * batch : own), dv, prefix_len > 0, tensor);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  p.slots = reinterpret_cast<float*>(ws + at.slots);
  p.desc = reinterpret_cast<int4*>(ws + at.desc);
  p.pieces = reinterpret_cast<float*>(ws + at.pieces);
  p.prefix_part = reinterpret_cast<float*>(ws + at.prefix);
  p.prefix_slots = reinterpret_cast<float*>(ws + at.prefix_slots);
  const int64_t pool_rows = p.num_pages * p.H * p.ps;
  if (pool_rows > 0x7fffffff) return set_last_error(SUNSHAPE_E_UNSUPPORTED, "at most 2^31 - 1 page rows in a pool.");
  // the kernels count tiles, and the gaps between heads, in 31 bits
  const int64_t most = (int64_t)std::max(batch, 1) * (((int64_t)table_cols * p.ps + kTile - 1) / kTile + 1 + kItemTiles) *
                       ((p.G * (int64_t)p.L + 7) / 8);
  const int64_t most_prefix = (prefix_len / kTile + 1 + kItemTiles) * ((rows / p.H + 7) / 8);
  if ((std::max(most, most_prefix) + kHeadTiles) * p.H > 0x7fffffff)
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention: more than 2^31 tiles of 32 tokens in a call.");
  CUtensorMap vmap{};
  if (pool_rows)
    if (int rc = make_rows_map(&vmap, pages->value, pages->dtype == SUNSHAPE_BF16, dv, pool_rows, p.chunk)) return rc;
  p.err = paged_error_word();
  if (!p.err) return set_last_error(SUNSHAPE_E_CUDA, "the paged error word is unavailable on this device.");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf16 = pages->dtype == SUNSHAPE_BF16;
  AttnParams f = p;
  f.prefix_mode = 1;
  f.prefix_len = prefix_len;
  if (!plan(p, d, dv, bd) || !plan(f, d, dv, bd))
    return set_last_error(SUNSHAPE_E_UNSUPPORTED, "paged attention: too little shared memory.");
  if (prefix_len) {
    f.table = prefix_table;
    f.table_stride = 0;
    int rc;
    if (tensor) rc = bf16 ? launch<__nv_bfloat16, true>(f, vmap, d, dv, bd, grid, st) : launch<__half, true>(f, vmap, d, dv, bd, grid, st);
    else rc = bf16 ? launch<__nv_bfloat16, false>(f, vmap, d, dv, bd, grid, st) : launch<__half, false>(f, vmap, d, dv, bd, grid, st);
    if (rc) return rc;
    p.prefix_parts = 1;
    // else both use the same slots of the workspace.  Producers that run ahead wait for the prefix's end with their rings full,
    // and give up after kWaitLimitNs: not beside a prefix of more than kOverlapTiles tiles of 2.5 us a thread block
    const int64_t tiles = ((prefix_len + 127) / 128) * ((own * batch + 255) / 256) * p.H / grid;
    p.overlap = tensor && tiles <= kOverlapTiles;
  }
  return bf16 ? launch<__nv_bfloat16, false>(p, vmap, d, dv, bd, grid, st)
              : launch<__half, false>(p, vmap, d, dv, bd, grid, st);
}

}  // extern "C"

// drift_attention_chunks: the choice of kernel and of splits, and the checks.
// (The window, causality, softcap and sinks are Ops.attention's,
// ops/AttentionOps.scala:113-121.)
#include <cuda_runtime.h>

#include <algorithm>

#include "chunks.cuh"
#include "common.cuh"

namespace drift {

namespace {

struct Plan {
  int columns;          // attention_rows' column tiles
  int rows_per_unit;    // rows of a key head that a CTA takes
  int keys_per_tile;
  int splits, tiles_per_split;
};

// The most key tiles of `width` that a unit of a chunk can see
// (SeenTiles::count's bound).
long long tiles_bound(int longest, int max_key_count, int window, int first, int width) {
  const long long all = ((long long)max_key_count + width - 1) / width;
  if (window <= 0) return all;
  const long long seen = ((long long)window + longest) / width + 2 + ((long long)first + width - 1) / width;
  return std::min(all, seen);
}

Plan plan_rows(int batch, int longest, int group, int kv_heads, int head_dim, bool codes, int max_key_count,
               int window, int first) {
  Plan p;
  const long long rows = (long long)longest * group;
  p.columns = head_dim > 128 || rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  p.rows_per_unit = 8 * p.columns;
  p.keys_per_tile = attention_rows_tile(head_dim, codes, p.columns);
  const long long units = (rows + p.rows_per_unit - 1) / p.rows_per_unit * batch * kv_heads;
  const long long tiles = std::max(1LL, tiles_bound(longest, max_key_count, window, first, p.keys_per_tile));
  // CTAs for every SM twice over, of a tile a warp at least
  const long long wanted = std::max(1LL, 4LL * sm_count() / std::max(1LL, units));
  const long long splits = std::min(wanted, (tiles + 7) / 8);
  const long long each = (tiles + splits - 1) / splits;
  p.tiles_per_split = int((each + 7) / 8 * 8);
  p.splits = int((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  return p;
}

int check_shape(int q_heads, int kv_heads, int max_key_count, int table_stride, int page_size, int longest,
                int window, int first) {
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0)
    return invalid("attention: %d query heads over %d key heads", q_heads, kv_heads);
  if (q_heads / kv_heads > 16) return invalid("attention: %d query heads per key head (at most 16)", q_heads / kv_heads);
  if (max_key_count < longest || max_key_count > (long long)table_stride * page_size)
    return invalid("attention: %d keys in a page table of %d pages, chunks of %d", max_key_count, table_stride, longest);
  if (window < 0 || first < 0) return invalid("attention: a window of %d with %d first keys", window, first);
  if (first > 0 && window == 0) return invalid("attention: first keys without a window");
  return 0;
}

size_t parts_bytes(const Plan& p, long long tokens, int q_heads, int head_dim) {
  return p.splits > 1 ? size_t(tokens) * q_heads * p.splits * (head_dim + 2) * sizeof(float) : 0;
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" {

size_t drift_attention_chunks_workspace_bytes(int x_dtype, int64_t tokens, int q_heads, int kv_heads, int head_dim,
                                              int cache_dtype, int batch, int longest, int max_key_count, int window,
                                              int first) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || batch <= 0 || longest <= 0 || max_key_count <= 0)
    return 0;
  (void)x_dtype;
  const Plan p = plan_rows(batch, longest, q_heads / kv_heads, kv_heads, head_dim, cache_dtype == DRIFT_I8, max_key_count,
                           window, first);
  return parts_bytes(p, tokens, q_heads, head_dim);
}

int drift_attention_chunks(int x_dtype, const void* q, int64_t tokens, int q_heads, int kv_heads, int head_dim,
                           int cache_dtype, const void* keys, const void* values, const float* key_scales,
                           const float* value_scales, int pages, int page_size, const int32_t* page_tables,
                           int table_stride, const int32_t* starts, const int32_t* positions, int batch, int longest,
                           int max_key_count, float scale, int causal, int window, int first, float softcap,
                           const float* sinks, void* out, void* workspace, size_t workspace_bytes,
                           drift_stream_t stream) {
  DRIFT_TRY(check_chunks("attention", x_dtype, tokens, kv_heads, head_dim, cache_dtype, keys, values, key_scales,
                         value_scales, pages, page_size, page_tables, table_stride, starts, positions, batch, longest));
  DRIFT_TRY(check_shape(q_heads, kv_heads, max_key_count, table_stride, page_size, longest, window, first));
  if (tokens == 0 || batch == 0 || longest == 0) return 0;
  DRIFT_TRY(check_rows_aligned("attention", q, out));
  const int group = q_heads / kv_heads;
  const Plan p = plan_rows(batch, longest, group, kv_heads, head_dim, cache_dtype == DRIFT_I8, max_key_count, window, first);
  const long long units = ((long long)longest * group + p.rows_per_unit - 1) / p.rows_per_unit;
  if (units * p.splits > 0x7fffffffll || (long long)longest * q_heads > 0x7fffffffll)
    return invalid("attention: chunks of %d tokens of %d heads", longest, q_heads);
  const size_t needed = parts_bytes(p, tokens, q_heads, head_dim);
  if (needed > workspace_bytes || (needed && !workspace))
    return invalid("attention: a workspace of %zu bytes, %zu needed", workspace_bytes, needed);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return invalid("attention: the workspace does not start on a 16-byte boundary");
  AttentionChunksArgs a;
  a.at = {starts, positions, page_tables, tokens, table_stride, pages, page_size, batch, longest, max_key_count};
  a.q = q;
  a.out = out;
  a.keys = keys;
  a.values = values;
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.sinks = sinks;
  a.part_o = needed ? static_cast<float*>(workspace) : nullptr;
  a.part_ml = needed ? a.part_o + size_t(tokens) * q_heads * p.splits * head_dim : nullptr;
  a.error = device_error_word();
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = group;
  a.causal = causal;
  a.window = window;
  a.first = first;
  a.splits = p.splits;
  a.tiles_per_split = p.tiles_per_split;
  a.scale = scale;
  a.softcap = softcap;
  const cudaStream_t s = cudaStream_t(stream);
  DRIFT_TRY(launch_attention_rows(a, x_dtype, cache_dtype, head_dim, p.columns, s));
  if (!needed) return 0;
  return launch_attention_join(a, x_dtype, head_dim, p.rows_per_unit, p.keys_per_tile, s);
}

}  // extern "C"

// What the operators over a batch of sequences' new tokens share (chunks.cu,
// attention_rows.cu, attention_tiles.cu): where a sequence's rows and
// positions are, which keys a token sees, and the split attention's partials.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace drift {

int* device_error_word();

// Sequence z's new tokens are rows [starts[z], starts[z + 1]) of q, k, v and
// out, at positions positions[z], positions[z] + 1, ... of the pages in row z
// of `tables`.
struct ChunkLayout {
  const int* starts;
  const int* positions;
  const int* tables;
  long long tokens;  // rows of q, k, v, out
  int table_stride, pages, page_size, batch, longest, max_keys;
};

// One sequence's chunk. Starts that are not ascending rows, a chunk longer
// than `longest`, or positions outside its page table (or past `max_keys`) make
// it not `ok`: the
// sequence is left out (its rows are not written) and the caller sets the
// device error word.
struct Chunk {
  long long row;  // its first row
  int tokens, position;
  const int* table;
  bool ok;
  __device__ Chunk(const ChunkLayout& a, int z) {
    const int begin = a.starts[z], end = a.starts[z + 1];
    position = a.positions[z];
    row = begin;
    tokens = end - begin;
    table = a.tables + (long long)z * a.table_stride;
    ok = begin >= 0 && end >= begin && end <= a.tokens && end - begin <= a.longest && position >= 0 &&
         position <= a.max_keys - (end - begin);
    if (!ok) tokens = 0;
  }
};

__device__ __forceinline__ void chunk_error(int* error) {
  if (error) atomicCAS(error, 0, 1);
}

struct AttentionChunksArgs {
  ChunkLayout at;
  const void* q;
  void* out;
  const void* keys;
  const void* values;
  const float* key_scales;    // 8-bit caches (expanded: [batch][kv_heads][positions])
  const float* value_scales;
  const float4* units;        // [batch][kv_heads], of expanded codes (attention_expand): what values are over, what
                              // keys are over, whether scales are by key; or null
  const float* sinks;
  float* part_o;   // [token row][q_heads][splits][D], or null for one split
  float* part_ml;  // [token row][q_heads][splits][2]: largest, sum
  int* error;
  int q_heads, kv_heads, group;
  int causal, window, first;
  int splits, tiles_per_split;  // key tiles a split takes, of the tiles its rows see
  float scale, softcap;
};

constexpr float LOG2E = 1.4426950408889634f;

// e^(score - base), 0 for a score that is not seen.
__device__ __forceinline__ float weight_of(float score, float base) {
  return score == -INFINITY ? 0.0f : exp2f((score - base) * LOG2E);
}

__device__ __forceinline__ uint32_t half_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A power of two at or above x whose inverse is normal.
__device__ __forceinline__ float power_over(float x) {
  const uint32_t bits = __float_as_uint(x);
  const uint32_t up = min((bits & 0x7f800000u) + ((bits & 0x7fffffu) ? 0x800000u : 0u), 0x7e800000u);
  return __uint_as_float(max(up, 0x01000000u));
}

// A value's scale (over a power of two, 1 at most) to base 2, as it moves a
// row's base: 2^-80 at least, so that no weight is past F32's range because its
// value has none.
__device__ __forceinline__ float logarithm(float scale) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(scale));
  return scale > 0.0f ? fminf(fmaxf(y, -80.0f), 0.0f) : -80.0f;
}

// The keys some row among the chunk's tokens [token0, token1) sees, as key
// tiles of `keys_per_tile`: the first `head` tiles hold the first positions
// that stay visible under the window, the others run from tile `low` on.
// Tile j of `count` covers keys from key_of(j).
struct SeenTiles {
  int head, low, count, keys_per_tile, end;  // end: past the last key any of the rows sees
  __device__ SeenTiles(const AttentionChunksArgs& a, const Chunk& c, int token0, int token1, int width) {
    keys_per_tile = width;
    end = c.position + (a.causal ? token1 : c.tokens);
    const int lowest = a.window > 0 ? c.position + token0 - a.window + 1 : 0;
    low = lowest > 0 ? lowest / width : 0;
    head = a.window > 0 ? (min(a.first, end) + width - 1) / width : 0;
    if (head > low) head = low;
    count = token1 > token0 ? head + (end + width - 1) / width - low : 0;
  }
  __device__ int key_of(int j) const { return (j < head ? j : low + j - head) * keys_per_tile; }
  __device__ int splits(int tiles_per_split) const { return (count + tiles_per_split - 1) / tiles_per_split; }
};

// What a row that sees the keys in [key0, end) that are `lowest` or later or
// below `first` gets of their values that are not finite, in dimensions d .. d
// + 3: such values were left out of the products in which they would have met
// the zero weights of rows that do not see them. `values`: dimension d of the
// key head in page 0; pages are `page_stride` values apart.
static __device__ __noinline__ float4 not_finite(const __half* values, long long page_stride, const int* table,
                                                 int pages, int page_size, int key0, int end, int lowest, int first) {
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int key = key0; key < end; ++key) {
    if (key < lowest && key >= first) continue;
    const int page = table[key / page_size];
    if (page < 0 || page >= pages) continue;
    const __half* at = values + page * page_stride + key % page_size;
    const float v[4] = {float(at[0]), float(at[page_size]), float(at[2 * page_size]), float(at[3 * page_size])};
    if (!isfinite(v[0])) x.x += v[0];
    if (!isfinite(v[1])) x.y += v[1];
    if (!isfinite(v[2])) x.z += v[2];
    if (!isfinite(v[3])) x.w += v[3];
  }
  return x;
}

// The checks that the calls share (chunks.cu).
int check_chunks(const char* call, int x_dtype, long long tokens, int kv_heads, int head_dim, int cache_dtype,
                 const void* keys, const void* values, const float* key_scales, const float* value_scales,
                 int pages, int page_size, const int32_t* page_tables, int table_stride, const int32_t* starts,
                 const int32_t* positions, int batch, int longest);
int check_rows_aligned(const char* call, const void* a, const void* b);

// For few rows: attention_rows.cu over F16 caches (units of 8 rows, 16-key
// tiles) and attention_codes.cu over 8-bit ones (of 4 or 8, 32-key tiles); the
// warps of a CTA, and the CTAs that an SM holds.
constexpr int ATTENTION_ROWS_WARPS = 8;
constexpr int attention_rows_ctas(int head_dim) { return head_dim > 128 ? 1 : 2; }
constexpr int attention_codes_warps(int head_dim) { return head_dim == 128 ? 4 : 8; }
constexpr int attention_codes_ctas(int head_dim) { return head_dim > 128 ? 1 : head_dim == 128 ? 3 : 2; }
int launch_attention_rows(const AttentionChunksArgs& a, int x_dtype, int head_dim, cudaStream_t stream);
int launch_attention_codes(const AttentionChunksArgs& a, int x_dtype, int head_dim, int rows_per_unit,
                           cudaStream_t stream);
// attention_tiles.cu: `row_tiles` tiles of 128 rows
// a unit (1 or 2; 1 for heads of 256), and the keys of one of its tiles.
int attention_tiles_keys(int head_dim, bool bf16, bool codes);
int launch_attention_tiles(const AttentionChunksArgs& a, int x_dtype, int cache_dtype, int head_dim, int row_tiles,
                           cudaStream_t stream);
// attention_expand.cu: an 8-bit cache's keys and values of the chunks as F16 in
// `memory` (16-byte aligned, expanded_bytes), which then take the cache's place
// in `a`.
size_t expanded_bytes(int batch, int kv_heads, int head_dim, int page_size, int max_key_count);
int launch_attention_expand(AttentionChunksArgs& a, int x_dtype, int head_dim, void* memory, cudaStream_t stream);
// Joins the splits (attention_rows.cu).
int launch_attention_join(const AttentionChunksArgs& a, int x_dtype, int head_dim, int rows_per_unit,
                          int keys_per_tile, cudaStream_t stream);

}  // namespace drift

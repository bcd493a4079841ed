// drift_attention_chunks: the choice of kernel and of splits, and the checks.
// (The window, causality, softcap and sinks are Ops.attention's,
// ops/AttentionOps.scala:113-121.)
#include <cuda_runtime.h>

#include <algorithm>

#include "chunks.cuh"
#include "common.cuh"

namespace drift {

namespace {

constexpr size_t EXPANDED_MOST = size_t(1) << 30;  // bytes

struct Plan {
  int row_tiles;        // attention_tiles' row tiles (0: attention_rows or attention_codes)
  int rows_per_unit;    // rows of a key head that a CTA takes
  int keys_per_tile;
  int splits, tiles_per_split;
  bool expands;         // an 8-bit cache's codes to F16 first
};

struct Call {
  int x_dtype, cache_dtype, batch, longest, group, kv_heads, head_dim, max_key_count, causal, window, first, pages,
      page_size;
};

// The most key tiles of `width` that a unit of `rows` rows can see
// (SeenTiles::count's bound).
long long tiles_bound(const Call& c, int rows, int width) {
  const long long all = ((long long)c.max_key_count + width - 1) / width;
  if (c.window <= 0) return all;
  const long long tokens = c.causal ? std::min(c.longest, rows / c.group + 2) : c.longest;
  const long long seen = (c.window + tokens) / width + 2 + ((long long)c.first + width - 1) / width;
  return std::min(all, seen);
}

Plan plan_rows(const Call& c) {
  Plan p;
  p.row_tiles = 0;
  p.expands = false;
  const long long rows = (long long)c.longest * c.group;
  const bool codes = c.cache_dtype == DRIFT_I8;
  p.rows_per_unit = codes && rows <= 4 ? 4 : 8;
  p.keys_per_tile = codes ? 32 : 16;
  const long long units = (rows + p.rows_per_unit - 1) / p.rows_per_unit * c.batch * c.kv_heads;
  const long long tiles = std::max(1LL, tiles_bound(c, p.rows_per_unit, p.keys_per_tile));
  const int warps = codes ? attention_codes_warps(c.head_dim) : ATTENTION_ROWS_WARPS;
  const long long slots = (long long)sm_count() * (codes ? attention_codes_ctas(c.head_dim) : attention_rows_ctas(c.head_dim));
  // CTAs for every SM four times over (F16 caches eight: a step of 16 x 8700 to
  // 16384 keys 148 us, and 179 with four; 8-bit ones of 3 sequences 28, and 33 with
  // eight), of a tile a warp at least; two splits while that leaves SMs idle
  // (eight chunks of 40 F32 rows: 100 us, 111 with one)
  const long long wanted =
      std::max(units < slots ? 2LL : 1LL, (codes ? 4LL : 8LL) * sm_count() / std::max(1LL, units));
  const long long splits = std::min(wanted, (tiles + warps - 1) / warps);
  const long long each = (tiles + splits - 1) / splits;
  long long rounds = (each + warps - 1) / warps;
  // (a tile a warp is not worth a second round of CTAs: 12 rows of one
  // sequence over 4096 keys 17.0 us, 18.9 with it; a windowed step of 13 x 1028
  // keys of heads of 256 15.4, 19.2 with it)
  if (rounds == 1 && units * ((tiles + warps - 1) / warps) > slots) rounds = 2;
  p.tiles_per_split = int(rounds * warps);
  p.splits = int((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  return p;
}

// Whether a chunk's rows of a key head go to the tensor-core tiles, by what
// both take on B200 (8 sequences x 8 key heads of 128, the longest of so many
// rows over 4096 keys, the others down to half; us, few rows' kernel and tiles):
// F16 caches BF16 8 rows 35 and 43, 12 rows 40 and 44 (all of them as long: 56 and
// 45); F32 8 rows 37 and 57, 12 rows 43 and 58 (60 and 59). 8-bit ones BF16 32
// rows 63 and 77, 40 rows 90 and 76 (heads of 256: 24 rows 92 and 91, 32 rows 113
// and 93); F32 40 rows 104 and 129, and of one sequence 22 and 25, but 48 rows
// 33 and 25. F32 heads of 256 (8 x 2 key heads): F16 16 rows 35 and 42, 24 rows
// 46 and 43; 8-bit 64 rows 79 and 86, 128 rows 136 and 88.
bool takes_tiles(const Call& c, long long rows) {
  const bool bf16 = c.x_dtype == DRIFT_BF16;
  const bool wide = c.head_dim > 128;
  if (c.cache_dtype == DRIFT_F16) return rows > (wide && !bf16 ? 16 : 8);
  return rows > (bf16 ? (wide ? 24 : 32) : wide ? 64 : 40);
}

// Two row tiles to a CTA or one, and how many splits: what ends first by a model
// of what was measured on B200. A tile takes so many ns for each key and row
// tile (2048 rows of 8 x 4 heads over 4096 and 8192 keys), a CTA 9 us for its
// start and end; the join's partial rows, written and read, pass at 1.7 TB/s.
// CTAs start with the longest (a causal chunk's last rows). Two row tiles
// share a tile's keys: a row tile by itself takes 1.6 times as long (chunk of
// 2048 BF16 rows, 8192 keys: 241 us, 414 with one) but keeps all SMs at work
// where there are few (1500 F32 tokens of 4 x 4 heads: 67 us, 84 with two).
Plan plan_tiles(const Call& c, bool converts, double slower, double& least) {
  constexpr double CTA_NS = 9000, JOIN_NS = 3000, PARTS_BYTES_A_NS = 1700;
  const bool bf16 = c.x_dtype == DRIFT_BF16;
  const double key_ns = bf16 ? (c.head_dim > 128 ? 20 : c.head_dim > 64 ? 7.7 : 6.5) * slower
                             : (c.head_dim > 128 ? 35 : c.head_dim > 64 ? 14.5 : 10) * slower;
  const long long rows = (long long)c.longest * c.group;
  Plan best;
  least = -1;
  for (int row_tiles = c.head_dim > 128 || rows <= 128 ? 1 : 2; row_tiles > 0; --row_tiles) {
    Plan p;
    p.row_tiles = row_tiles;
    p.expands = false;
    p.rows_per_unit = 128 * row_tiles;
    p.keys_per_tile = attention_tiles_keys(c.head_dim, bf16, converts);
    // (F32 rows of heads of 256 have two CTAs)
    const long long units = (rows + p.rows_per_unit - 1) / p.rows_per_unit * c.batch * c.kv_heads * (!bf16 && c.head_dim > 128 ? 2 : 1);
    const long long tiles = std::max(1LL, tiles_bound(c, p.rows_per_unit, p.keys_per_tile));
    const double tile_ns = p.keys_per_tile * key_ns * (row_tiles == 2 ? 2.0 : c.head_dim > 128 ? 1.0 : 1.6);
    const double cta_ns = row_tiles == 2 ? CTA_NS : 0.7 * CTA_NS;
    // the fewest tiles of a unit, and the mean
    const double fewest = c.causal && c.window == 0 ? double(tiles) * (c.max_key_count - c.longest) / c.max_key_count : double(tiles);
    const double mean = (tiles + fewest) / 2;
    const double parts_bytes = 8.0 * rows * c.batch * c.kv_heads * c.head_dim;  // of a split, there and back
    long long last = 0;
    for (long long splits = 1; splits <= 64 && splits <= tiles; ++splits) {
      const long long each = (tiles + splits - 1) / splits;
      if (each == last) continue;
      last = each;
      const double ctas = units * std::max(1.0, splits * mean / tiles);
      const double longest = each * tile_ns + cta_ns, shortest = std::min(double(each), fewest) * tile_ns + cta_ns;
      const double shared = (units * mean * tile_ns + ctas * cta_ns) / sm_count() + shortest;
      const double rounds = double((units * splits + sm_count() - 1) / sm_count());
      const double cost = std::max(longest, std::min(rounds * longest, shared)) +
                          (splits > 1 ? JOIN_NS + splits * parts_bytes / PARTS_BYTES_A_NS : 0);
      if (least >= 0 && cost >= least) continue;
      least = cost;
      p.tiles_per_split = int(each);
      p.splits = int((tiles + each - 1) / each);
      best = p;
    }
  }
  return best;
}

// The same with the choice of expanding an 8-bit cache's codes: two launches
// more (BF16 rows: three), and 3 bytes a value at about 3 TB/s, in at most 1 GiB
// (us, with each unit's own conversion and expanded: three chunks of 1001 BF16
// tokens x 4 heads over 5003 keys 527 and 293, three of 100 over 2000 49 and 55,
// eight of 40 over 4096 104 and 120; 2048 F32 tokens over 8192 1031 and 640, 64
// over 16384 89 and 109). Converting codes makes a tile 2.2 (BF16) and 2.5 times
// as long, scales by key 1.4 times.
Plan plan_all_tiles(const Call& c) {
  constexpr double BYTES_A_NS = 3000;
  double own;
  const bool bf16 = c.x_dtype == DRIFT_BF16;
  const double launches_ns = bf16 ? 16000 : 14000;
  if (c.cache_dtype != DRIFT_I8) return plan_tiles(c, false, 1.0, own);
  const Plan p = plan_tiles(c, true, bf16 ? 2.2 : 2.5, own);
  if (expanded_bytes(c.batch, c.kv_heads, c.head_dim, c.page_size, c.max_key_count) > EXPANDED_MOST) return p;
  const long long seen = c.window > 0 ? std::min((long long)c.max_key_count, (long long)c.window + c.longest + c.first) : c.max_key_count;
  double expanded;
  Plan q = plan_tiles(c, false, bf16 ? 1.0 : 1.4, expanded);
  q.expands = true;
  expanded += launches_ns + 6.0 * seen * c.batch * c.kv_heads * c.head_dim / BYTES_A_NS;
  // (no tiles convert codes for F32 heads of 256)
  return expanded < own || (!bf16 && c.head_dim > 128) ? q : p;
}

Plan plan_chunks(const Call& c) {
  const long long rows = (long long)c.longest * c.group;
  // (the copies' coordinates are 32-bit, the grid's unit axis 16-bit)
  const bool reachable = (long long)c.pages * c.page_size < (1ll << 31) &&
                         (long long)c.pages * c.kv_heads * c.head_dim < (1ll << 31);
  const bool expandable = expanded_bytes(c.batch, c.kv_heads, c.head_dim, c.page_size, c.max_key_count) <= EXPANDED_MOST;
  const bool has_tiles = c.cache_dtype == DRIFT_F16 || c.x_dtype == DRIFT_BF16 || c.head_dim <= 128 || expandable;
  if (takes_tiles(c, rows) && reachable && has_tiles) {
    const Plan p = plan_all_tiles(c);
    if ((rows + p.rows_per_unit - 1) / p.rows_per_unit * p.splits <= 65535) return p;
  }
  return plan_rows(c);
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

// The workspace: partial results, then (from a 128-byte boundary) expanded codes.
size_t parts_bytes(const Plan& p, long long tokens, int q_heads, int head_dim) {
  return p.splits > 1 ? (size_t(tokens) * q_heads * p.splits * (head_dim + 2) * sizeof(float) + 127) / 128 * 128 : 0;
}
size_t workspace_bytes_of(const Plan& p, const Call& c, long long tokens, int q_heads) {
  return parts_bytes(p, tokens, q_heads, c.head_dim) +
         (p.expands ? expanded_bytes(c.batch, c.kv_heads, c.head_dim, c.page_size, c.max_key_count) : 0);
}

}  // namespace
}  // namespace drift

using namespace drift;

extern "C" {

size_t drift_attention_chunks_workspace_bytes(int x_dtype, int64_t tokens, int q_heads, int kv_heads, int head_dim,
                                              int cache_dtype, int pages, int page_size, int batch, int longest,
                                              int max_key_count, int causal, int window, int first) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0 || pages <= 0 ||
      page_size <= 0 || batch <= 0 || longest <= 0 || max_key_count <= 0)
    return 0;
  const Call c = {x_dtype, cache_dtype, batch, longest, q_heads / kv_heads, kv_heads, head_dim, max_key_count,
                  causal, window, first, pages, page_size};
  return workspace_bytes_of(plan_chunks(c), c, tokens, q_heads);
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
  const Call c = {x_dtype, cache_dtype, batch, longest, group, kv_heads, head_dim, max_key_count, causal,
                  window, first, pages, page_size};
  const Plan p = plan_chunks(c);
  const long long units = ((long long)longest * group + p.rows_per_unit - 1) / p.rows_per_unit;
  // (the kernels count rows of whole units in 32 bits)
  if (units * p.splits > 0x7fffffffll || (long long)longest * q_heads > 0x7fffffffll - 1024)
    return invalid("attention: chunks of %d tokens of %d heads", longest, q_heads);
  const size_t parts = parts_bytes(p, tokens, q_heads, head_dim), needed = workspace_bytes_of(p, c, tokens, q_heads);
  if (needed > workspace_bytes || (needed && !workspace))
    return invalid("attention: a workspace of %zu bytes, %zu needed", workspace_bytes, needed);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return invalid("attention: the workspace does not start on a 16-byte boundary");
  // (two CTAs of F32 heads of 256 read the same rows of q)
  const uintptr_t row_bytes = uintptr_t(tokens) * q_heads * head_dim * (x_dtype == DRIFT_F32 ? 4 : 2);
  const uintptr_t q_at = reinterpret_cast<uintptr_t>(q), out_at = reinterpret_cast<uintptr_t>(out);
  if (q_at < out_at + row_bytes && out_at < q_at + row_bytes) return invalid("attention: q and out overlap");
  AttentionChunksArgs a;
  a.at = {starts, positions, page_tables, tokens, table_stride, pages, page_size, batch, longest, max_key_count};
  a.q = q;
  a.out = out;
  a.keys = keys;
  a.values = values;
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.sinks = sinks;
  a.units = nullptr;
  a.part_o = parts ? static_cast<float*>(workspace) : nullptr;
  a.part_ml = parts ? a.part_o + size_t(tokens) * q_heads * p.splits * head_dim : nullptr;
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
  if (p.expands) DRIFT_TRY(launch_attention_expand(a, x_dtype, head_dim, static_cast<uint8_t*>(workspace) + parts, s));
  if (p.row_tiles) DRIFT_TRY(launch_attention_tiles(a, x_dtype, p.expands ? DRIFT_F16 : cache_dtype, head_dim, p.row_tiles, s));
  else if (cache_dtype == DRIFT_I8) DRIFT_TRY(launch_attention_codes(a, x_dtype, head_dim, p.rows_per_unit, s));
  else DRIFT_TRY(launch_attention_rows(a, x_dtype, head_dim, s));
  if (!parts) return 0;
  return launch_attention_join(a, x_dtype, head_dim, p.rows_per_unit, p.keys_per_tile, s);
}

}  // extern "C"

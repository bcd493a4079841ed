// For attention_chunks over an 8-bit cache where a chunk has several units of
// rows: the sequences' keys and values as F16, once, for attention_tiles' F16
// kernel. The tiles' own converting warps make each tile anew for every unit (one
// takes 2.2 times as long as from an F16 cache).
//
//   BF16 rows: keys16, values16 = code scale / unit, rounded to F16 once
//   F32 rows:  keys16, values16 = code, exactly; and rows of scales for each
//              sequence and head, the values' over their unit (by key)
//
// with powers of two for each sequence, key head and side. BF16 rows' are
// 2^-8 of what the largest scale that a row sees rounds up to, so that a
// quotient is at most 2^15, and 2^-14 and more for scales down to 2^-22 of that,
// where F16 has its 11 bits: what a row has of its keys does not depend on the
// scales beside them. Heads whose scales are farther apart (than 2^20), not
// finite or at the ends of F32's range go by key as F32 rows' do, in a launch of
// the tiles of their own, by a third slower. The tiles multiply scores by the
// keys' unit and results by the values'.
//
// The copies are a paged cache of their own, in the F16 cache's layouts, with
// sequence z's pages from z * page_row on and the table that says so. Only what
// some row may see is written; the tiles mask the rest. Bound by memory: 1 byte
// read and 2 written a value, 4 + 8 bytes a position and head besides.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "chunks.cuh"
#include "common.cuh"
#include "registry.cuh"

namespace drift {

namespace {

constexpr int UNIT_THREADS = 1024;
constexpr int FLIGHT = 4;
constexpr int THREADS = 256;
constexpr int RUN = 16;    // positions of a code chunk, in one page
constexpr int runs_of(int dim) { return dim % 64 ? 8 : 4; }  // of a CTA: as many chunks to every thread

struct ExpandArgs {
  ChunkLayout at;
  const uint8_t* keys;
  const uint8_t* values;
  const float* key_scales;
  const float* value_scales;
  __half* keys16;
  __half* values16;
  float4* units;   // [batch][kv_heads]
  float* key_scales32;    // [batch][kv_heads][page_row page_size]
  float* value_scales32;
  int* table;      // [batch][page_row]
  int* error;
  int kv_heads, page_row, window, first;
  bool always_by_key;
};

// What the rows of a chunk see between them: [low, end) and [0, first).
struct SeenPositions {
  int low, first, end;
  __device__ SeenPositions(const ExpandArgs& a, const Chunk& c) {
    end = c.position + c.tokens;
    low = a.window > 0 ? max(c.position - a.window + 1, 0) : 0;
    first = a.window > 0 ? min(a.first, end) : 0;
  }
  __device__ bool sees(int position) const { return position < end && (position >= low || position < first); }
};

__global__ void __launch_bounds__(UNIT_THREADS) attention_units_kernel(const ExpandArgs a) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  __shared__ uint32_t ends[4][UNIT_THREADS / 32];
  const int head = blockIdx.x, z = blockIdx.y;
  if (head == 0)
    for (int i = threadIdx.x; i < a.page_row; i += UNIT_THREADS) a.table[(long long)z * a.page_row + i] = z * a.page_row + i;
  const Chunk chunk(a.at, z);
  const SeenPositions seen(a, chunk);
  // the largest and (upside down) the smallest of either side's, as bits, which
  // order as numbers do; zeros need none, and of what is no finite positive
  // number it is enough that there is some
  uint32_t most[4] = {0, 0, 0, 0};
  bool odd = false;
  auto look = [&](int from, int to) {
    // four positions of a page to a thread, four times over: two latencies
    // for 16384 positions
#pragma unroll 1
    for (int p0 = from / 4 * 4 + 4 * int(threadIdx.x); p0 < to; p0 += 4 * FLIGHT * UNIT_THREADS) {
      int page[FLIGHT];
#pragma unroll
      for (int n = 0; n < FLIGHT; ++n) {
        const long long p = p0 + 4ll * n * UNIT_THREADS;
        page[n] = p < to ? chunk.table[p / a.at.page_size] : -1;
      }
      float4 x[FLIGHT][2];
#pragma unroll
      for (int n = 0; n < FLIGHT; ++n) {
        const long long p = p0 + 4ll * n * UNIT_THREADS;
        const bool there = page[n] >= 0 && page[n] < a.at.pages;
        const long long at = ((long long)page[n] * a.kv_heads + head) * a.at.page_size + p % a.at.page_size;
        x[n][0] = there ? *reinterpret_cast<const float4*>(a.key_scales + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        x[n][1] = there ? *reinterpret_cast<const float4*>(a.value_scales + at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int n = 0; n < FLIGHT; ++n)
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const float y[4] = {x[n][side].x, x[n][side].y, x[n][side].z, x[n][side].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const long long p = p0 + 4ll * n * UNIT_THREADS + e;
            const uint32_t bits = __float_as_uint(y[e]);
            if (p < from || p >= to || bits == 0) continue;
            odd = odd || bits >= 0x7f800000u;
            if (bits >= 0x7f800000u) continue;
            most[2 * side] = max(most[2 * side], bits);
            most[2 * side + 1] = max(most[2 * side + 1], ~bits);
          }
        }
    }
  };
  if (chunk.tokens > 0) {
    look(0, min(seen.first, seen.low));
    look(seen.low, seen.end);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    most[i] = __reduce_max_sync(0xffffffffu, most[i]);
    if (threadIdx.x % 32 == 0) ends[i][threadIdx.x / 32] = most[i];
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x >= 32) return;
  float top[2];
  bool by_key = a.always_by_key || odd;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, ends[2 * side][threadIdx.x]);
    const uint32_t low = ~__reduce_max_sync(0xffffffffu, ends[2 * side + 1][threadIdx.x]);
    top[side] = __uint_as_float(high);
    // (a side without scales is 0 and 2^32 - 1)
    if (high != 0) by_key = by_key || high - low > 20 << 23 || high > 247 << 23 || high < (side == 0 ? 77 : 27) << 23;
  }
  if (threadIdx.x > 0) return;
  // (all zeros are over one: what they would be over has no inverse)
  auto over = [](float x) { return x > 0.0f ? power_over(x) * (1.0f / 256.0f) : 1.0f; };
  a.units[(long long)z * a.kv_heads + head] =
      by_key ? make_float4(power_over(top[1]), 1.0f, 1.0f, 0.0f) : make_float4(over(top[1]), over(top[0]), 0.0f, 0.0f);
}

// 64 positions of a head (128 where D = 80): a thread takes 16 codes at a time, of a position's
// key or of a dimension's values.
template <int D>
__global__ void __launch_bounds__(THREADS) attention_expand_kernel(const ExpandArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int RUNS = runs_of(D), TASKS = RUNS * 2 * D, PER = TASKS / THREADS;
  static_assert(TASKS % THREADS == 0, "whole rounds");
  const int head = blockIdx.y, z = blockIdx.z;
  const Chunk chunk(a.at, z);
  if (!chunk.ok || chunk.tokens == 0) return;  // (the tiles tell of one that is not)
  const SeenPositions seen(a, chunk);
  const int start = blockIdx.x * RUN * RUNS;
  if (start >= seen.end || (start + RUN * RUNS <= seen.low && start >= seen.first)) return;
  const float4 units = a.units[(long long)z * a.kv_heads + head];
  const bool by_key = units.z != 0.0f;
  const float value_inverse = 1.0f / units.x, key_inverse = 1.0f / units.y;  // exact
  uint4 codes[PER];
  long long from_scales[PER];
  bool there[PER];
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int task = threadIdx.x + THREADS * n, run = task / (2 * D), in = task % (2 * D);
    const int first = start + RUN * run;
    there[n] = false;
    codes[n] = make_uint4(0, 0, 0, 0);
    from_scales[n] = 0;
    if (first >= seen.end) continue;
    const int page = chunk.table[first / a.at.page_size], place = first % a.at.page_size;
    if (page < 0 || page >= a.at.pages) {
      // (what no row sees may be anything)
      bool seen_here = false;
      for (int p = first; p < first + RUN; ++p) seen_here = seen_here || seen.sees(p);
      if (in == 0 && seen_here) chunk_error(a.error);
      continue;
    }
    there[n] = true;
    from_scales[n] = ((long long)page * a.kv_heads + head) * a.at.page_size + place;
    if (in < D)  // key of position in / (D / 16), its chunk in % (D / 16)
      codes[n] = *reinterpret_cast<const uint4*>(
          a.keys + (((long long)page * a.at.page_size + place + in / (D / 16)) * a.kv_heads + head) * D + 16 * (in % (D / 16)));
    else         // values of dimension in - D
      codes[n] = *reinterpret_cast<const uint4*>(
          a.values + (((long long)page * a.kv_heads + head) * D + in - D) * a.at.page_size + place);
  }
#pragma unroll
  for (int n = 0; n < PER; ++n) {
    const int task = threadIdx.x + THREADS * n, run = task / (2 * D), in = task % (2 * D);
    const int first = start + RUN * run;
    if (first >= seen.end) continue;
    const int index = first / a.at.page_size, place = first % a.at.page_size;
    const long long page = (long long)z * a.page_row + index;
    const bool key = in < D;
    float by[RUN];
    if (by_key) {
      if (key && in % (D / 16) == 0) {
        const long long to = ((long long)z * a.kv_heads + head) * a.page_row * a.at.page_size + first + in / (D / 16);
        a.key_scales32[to] = there[n] ? a.key_scales[from_scales[n] + in / (D / 16)] : 0.0f;
        a.value_scales32[to] = there[n] ? a.value_scales[from_scales[n] + in / (D / 16)] * value_inverse : 0.0f;
      }
#pragma unroll
      for (int e = 0; e < RUN; ++e) by[e] = 1.0f;
    } else if (key) {
      const float scale = there[n] ? a.key_scales[from_scales[n] + in / (D / 16)] * key_inverse : 0.0f;
#pragma unroll
      for (int e = 0; e < RUN; ++e) by[e] = scale;
    } else {
#pragma unroll
      for (int e = 0; e < RUN; e += 4) {
        const float4 x = there[n] ? *reinterpret_cast<const float4*>(a.value_scales + from_scales[n] + e)
                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        by[e] = x.x * value_inverse, by[e + 1] = x.y * value_inverse;
        by[e + 2] = x.z * value_inverse, by[e + 3] = x.w * value_inverse;
      }
    }
    const int8_t* c = reinterpret_cast<const int8_t*>(&codes[n]);
    __align__(16) __half2 y[RUN / 2];
#pragma unroll
    for (int e = 0; e < RUN / 2; ++e)
      y[e] = __floats2half2_rn(float(c[2 * e]) * by[2 * e], float(c[2 * e + 1]) * by[2 * e + 1]);
    __half* to = key ? a.keys16 + ((page * a.at.page_size + place + in / (D / 16)) * a.kv_heads + head) * D + 16 * (in % (D / 16))
                     : a.values16 + ((page * a.kv_heads + head) * D + in - D) * a.at.page_size + place;
    reinterpret_cast<uint4*>(to)[0] = reinterpret_cast<const uint4*>(y)[0];
    reinterpret_cast<uint4*>(to)[1] = reinterpret_cast<const uint4*>(y)[1];
  }
}

#define DRIFT_EXPAND_REGISTER(D) DRIFT_REGISTER(attention_expand_d##D, (attention_expand_kernel<D>))
DRIFT_EXPAND_REGISTER(64)
DRIFT_EXPAND_REGISTER(80)
DRIFT_EXPAND_REGISTER(128)
DRIFT_EXPAND_REGISTER(256)
DRIFT_REGISTER(attention_units, attention_units_kernel)

template <int D>
int launch_dim(const ExpandArgs& a, cudaStream_t stream) {
  constexpr int POSITIONS = RUN * runs_of(D);
  const unsigned runs = unsigned(((long long)a.at.max_keys + POSITIONS - 1) / POSITIONS);
  const dim3 grid(runs, a.kv_heads, a.at.batch);
  DRIFT_CUDA(launch_pdl(attention_expand_kernel<D>, grid, THREADS, 0, stream, a));
  DRIFT_LAUNCHED("attention_expand");
  return 0;
}

constexpr size_t round_up(size_t bytes) { return (bytes + 127) / 128 * 128; }

}  // namespace

int expanded_page_row(int max_key_count, int page_size) { return int(((long long)max_key_count + page_size - 1) / page_size); }

// (a tile's scales are read whole past the last page)
static size_t scales_bytes(size_t positions, int kv_heads) { return round_up((positions * kv_heads + 128) * sizeof(float)); }

size_t expanded_bytes(int batch, int kv_heads, int head_dim, int page_size, int max_key_count) {
  const size_t pages = size_t(batch) * expanded_page_row(max_key_count, page_size);
  return round_up(size_t(batch) * kv_heads * sizeof(float4)) + round_up(pages * sizeof(int)) +
         2 * round_up(pages * page_size * kv_heads * head_dim * sizeof(__half)) +
         2 * scales_bytes(pages * page_size, kv_heads);
}

int launch_attention_expand(AttentionChunksArgs& a, int x_dtype, int head_dim, void* memory, cudaStream_t stream) {
  ExpandArgs e;
  e.at = a.at;
  e.keys = static_cast<const uint8_t*>(a.keys);
  e.values = static_cast<const uint8_t*>(a.values);
  e.key_scales = a.key_scales;
  e.value_scales = a.value_scales;
  e.error = a.error;
  e.kv_heads = a.kv_heads;
  e.page_row = expanded_page_row(a.at.max_keys, a.at.page_size);
  e.window = a.window;
  e.first = a.first;
  e.always_by_key = x_dtype == DRIFT_F32;
  const size_t pages = size_t(a.at.batch) * e.page_row;
  uint8_t* at = static_cast<uint8_t*>(memory);
  e.units = reinterpret_cast<float4*>(at);
  at += round_up(size_t(a.at.batch) * a.kv_heads * sizeof(float4));
  e.table = reinterpret_cast<int*>(at);
  at += round_up(pages * sizeof(int));
  const size_t side = round_up(pages * a.at.page_size * a.kv_heads * head_dim * sizeof(__half));
  e.keys16 = reinterpret_cast<__half*>(at);
  e.values16 = reinterpret_cast<__half*>(at + side);
  at += 2 * side;
  const size_t scales = scales_bytes(pages * a.at.page_size, a.kv_heads);
  e.key_scales32 = reinterpret_cast<float*>(at);
  e.value_scales32 = reinterpret_cast<float*>(at + scales);
  DRIFT_CUDA(launch_pdl(attention_units_kernel, dim3(a.kv_heads, a.at.batch), UNIT_THREADS, 0, stream, e));
  DRIFT_LAUNCHED("attention_units");
  switch (head_dim) {
    case 64: DRIFT_TRY(launch_dim<64>(e, stream)); break;
    case 80: DRIFT_TRY(launch_dim<80>(e, stream)); break;
    case 128: DRIFT_TRY(launch_dim<128>(e, stream)); break;
    default: DRIFT_TRY(launch_dim<256>(e, stream)); break;
  }
  // the copies in the cache's place
  a.keys = e.keys16;
  a.values = e.values16;
  a.key_scales = e.key_scales32;
  a.value_scales = e.value_scales32;
  a.units = e.units;
  a.at.tables = e.table;
  a.at.table_stride = e.page_row;
  a.at.pages = int(pages);
  return 0;
}

}  // namespace drift

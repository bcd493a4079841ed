// attention_chunks over an F16 cache for few rows: a decoding step.
//
// A unit is a key head of one sequence with up to 8 of the (token, query
// head) rows that read it; a CTA takes one split of the unit's key tiles,
// each of its 8 warps every eighth tile of 16 keys. The products are turned
// round -- scores^T = K q^T and out^T = V^T p^T by mma.sync m16n8k16, keys and
// then dimensions as the 16 rows and the query rows as the 8 columns --
// because there are few query rows: 8 columns leave nothing idle where 16 rows
// would be half empty. Keys and values go from the cache straight into the
// registers that the matrix instruction reads: a lane's 16 bytes of a key row
// (or of a dimension's consecutive positions) become its A fragments by
// numbering the product's inner index as the bytes lie, which the query
// fragments, laid out once in shared memory, follow.
//
// F32 rows: q and the weights are two F16 terms each (x = hi + lo to 2^-22),
// keys and values exact, so the products are F32-grade. BF16 rows: q is one
// term, exactly (after a power of two per row), and a weight is rounded to
// F16 (off by 2^-11 at most, the result's own rounding is 2^-8).
//
// Softmax in F32, a running maximum and sum per warp; the warps meet
// in shared memory, the splits in a second launch (attention_chunks_join_kernel).
//
// Bound by memory: a step of 16 sequences of 8700 to 16384 keys of 8 heads of
// 128 148 us in F32 and 143 in BF16, 822 MB at 5.6 and 5.8 TB/s; of 13 under a
// window of 1024 of 2 heads of 256, 15 us: one CTA an SM, two rounds of tiles to
// a warp behind one another's page numbers, and the join's launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "chunks.cuh"
#include "common.cuh"
#include "registry.cuh"

namespace drift {

namespace {

constexpr int WARPS = ATTENTION_ROWS_WARPS;
constexpr int THREADS = 32 * WARPS;
// A weight is e^WEIGHT_LOG = 2^14 at the row's largest score, and a row of q
// 2^Q_BITS and more at its largest value: F16's second terms stop at 2^-24, which is
// then 2^-38 of the largest weight (it is 2^-19 of a weight of 2^-6 without:
// the typical one of 4096 random scores).
constexpr float WEIGHT_LOG = 9.704060527839234f;
constexpr int Q_BITS = 12;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 x 8 tile of 16-bit values turned round (lane 4 i + j holds row i's
// values 2 j and 2 j + 1).
__device__ __forceinline__ uint32_t turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float2 pair_value(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// How a lane's loads cover rows of D values, 16 of them to a k-step: chunks of
// 16 bytes a lane while whole ones last, then (D = 80) one k-step of 4 values
// a lane. place_of tells which step and lane t have the four values from d on.
template <int D>
struct RowMap {
  static constexpr int PER = 8;                         // values of a 16-byte chunk
  static constexpr int STEPS_PER = PER / 4;             // k-steps of a chunk
  static constexpr int CHUNKS = D / (4 * PER);          // whole chunks
  static constexpr int STEPS = D / 16;
  static constexpr int TAIL = STEPS - CHUNKS * STEPS_PER;  // 0 or 1
  static constexpr int WORDS = 2 * STEPS;               // 32-bit words a lane holds of a row
  static_assert(TAIL <= 1, "one k-step past the chunks at most");
  __device__ static void place_of(int d, int& step, int& t) {
    const int chunk = d / (4 * PER), in = d % (4 * PER);
    step = chunk < CHUNKS ? STEPS_PER * chunk + in % PER / 4 : STEPS_PER * CHUNKS;
    t = chunk < CHUNKS ? in / PER : in / 4;
  }
};

constexpr int TILE = 16;  // keys of a warp's tile

template <int D_, bool BF16_>
struct RowsTraits {
  static constexpr int D = D_;
  static constexpr bool BF16 = BF16_;
  static constexpr int TERMS = BF16 ? 1 : 2;
  static constexpr int CTAS = attention_rows_ctas(D);  // of an SM: registers
  using Map = RowMap<D>;
  static constexpr int ROWS = 8;
  static constexpr int DM = D / 16;      // 16-dimension tiles of the output
  static constexpr int Q_BYTES = Map::STEPS * TERMS * 32 * 8;
  static constexpr int MERGE_BYTES = WARPS * ROWS * (D + 4) * 4;
  static constexpr int BYTES = Q_BYTES > MERGE_BYTES ? Q_BYTES : MERGE_BYTES;
};

template <class T>
struct RowsWarp {
  static constexpr int D = T::D, DM = T::DM;
  using Map = typename T::Map;

  const AttentionChunksArgs& a;
  const Chunk& chunk;
  const SeenTiles& seen;
  const int head, g, t;
  const uint32_t page_magic;  // 2^32 / page_size, up
  int page, place;            // of the tile that is loaded next
  uint32_t k[2][Map::WORDS];  // [row g, g + 8]
  uint2 v[DM][2];             // [16 dimensions][row g, g + 8], positions 4 t .. 4 t + 3

  __device__ RowsWarp(const AttentionChunksArgs& a, const Chunk& c, const SeenTiles& s, int head, int lane)
      : a(a), chunk(c), seen(s), head(head), g(lane / 4), t(lane % 4),
        page_magic(0xffffffffu / uint32_t(a.at.page_size) + 1) {}

  // The page that holds the tile at key0 and its place in it: -1 past the last
  // key, or for a page that the cache does not have.
  __device__ void find_page(int key0) {
    int index = int(__umulhi(uint32_t(key0), page_magic));  // (one too many at most)
    place = key0 - index * a.at.page_size;
    if (place < 0) --index, place += a.at.page_size;
    page = -1;
    if (key0 >= seen.end) return;
    page = chunk.table[index];
    if (page >= 0 && page < a.at.pages) return;
    chunk_error(a.error);
    page = -1;
  }
  // Row r of the score tile, r = g or g + 8, is this position of the tile: the
  // product of weights and values then meets the positions in the order in
  // which a lane's value words hold them.
  __device__ int position_of(int half) const { return 4 * (g / 2) + g % 2 + 2 * half; }

  __device__ void load_keys() {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const __half* row = static_cast<const __half*>(a.keys) +
                          (((long long)page * a.at.page_size + place + position_of(half)) * a.kv_heads + head) * D;
#pragma unroll
      for (int c = 0; c < Map::CHUNKS; ++c) {
        const uint4 x = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(row) + 4 * c + t) : make_uint4(0, 0, 0, 0);
        k[half][4 * c] = x.x, k[half][4 * c + 1] = x.y, k[half][4 * c + 2] = x.z, k[half][4 * c + 3] = x.w;
      }
      if constexpr (Map::TAIL) {
        constexpr int W = 4 * Map::CHUNKS;
        const uint2 x = page >= 0 ? __ldg(reinterpret_cast<const uint2*>(row + Map::CHUNKS * 4 * Map::PER) + t) : make_uint2(0, 0);
        k[half][W] = x.x, k[half][W + 1] = x.y;
      }
    }
  }
  __device__ void load_values() {
    const __half* column = static_cast<const __half*>(a.values) +
                           ((long long)page * a.kv_heads + head) * D * a.at.page_size + place + 4 * t;
#pragma unroll
    for (int m = 0; m < DM; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        v[m][half] = page >= 0 ? __ldg(reinterpret_cast<const uint2*>(column + (16 * m + g + 8 * half) * (long long)a.at.page_size))
                               : make_uint2(0, 0);
  }

  // The A fragments (rows g, g + 8; the step's first and second eight).
  __device__ void key_fragment(int step, uint32_t (&f)[4]) const {
    f[0] = k[0][2 * step], f[2] = k[0][2 * step + 1];
    f[1] = k[1][2 * step], f[3] = k[1][2 * step + 1];
  }
  __device__ void value_fragment(int m, uint32_t (&f)[4]) const {
    f[0] = v[m][0].x, f[2] = v[m][0].y;
    f[1] = v[m][1].x, f[3] = v[m][1].y;
  }
};

// `word` (positions p and p + 1 of a dimension) with zeros for what no row
// sees and for what is not finite; `found` tells of the latter.
__device__ __forceinline__ uint32_t finite_halves(uint32_t word, int p, int end, int lowest, int first, bool& found) {
  const bool low = p < end && (p >= lowest || p < first);
  const bool high = p + 1 < end && (p + 1 >= lowest || p + 1 < first);
  word &= (low ? 0xffffu : 0u) | (high ? 0xffff0000u : 0u);
  const bool low_bad = (word & 0x7c00u) == 0x7c00u, high_bad = (word & 0x7c000000u) == 0x7c000000u;
  found = found || low_bad || high_bad;
  return word & ((low_bad ? 0u : 0xffffu) | (high_bad ? 0u : 0xffff0000u));
}

template <class T>
__global__ void __launch_bounds__(THREADS, T::CTAS) attention_rows_kernel(const AttentionChunksArgs a) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  constexpr int D = T::D, ROWS = T::ROWS, TERMS = T::TERMS;
  using Map = typename T::Map;
  using X = typename std::conditional<T::BF16, __nv_bfloat16, float>::type;
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ float q_unit[ROWS];  // the power of two each row was divided by
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;
  const int split = blockIdx.x % a.splits, unit = blockIdx.x / a.splits, head = blockIdx.y, z = blockIdx.z;
  const Chunk chunk(a.at, z);
  if (!chunk.ok && blockIdx.x == 0 && head == 0 && tid == 0) chunk_error(a.error);
  // this unit's rows [row0, row1) of the sequence's tokens x group, row r
  // being token r / group, query head r % group of the key head
  const int row0 = unit * ROWS, row1 = min(row0 + ROWS, chunk.tokens * a.group);
  if (row0 >= row1) return;
  const int token0 = row0 / a.group, token1 = (row1 - 1) / a.group + 1;
  const SeenTiles seen(a, chunk, token0, token1, TILE);
  const int tile0 = split * a.tiles_per_split, tile1 = min(tile0 + a.tiles_per_split, seen.count);
  if (tile0 >= tile1) return;

  RowsWarp<T> w(a, chunk, seen, head, lane);
  int tile = tile0 + warp;
  if (tile < tile1) {
    w.find_page(seen.key_of(tile));
    w.load_keys();
    w.load_values();
    if (tile + WARPS < tile1) w.find_page(seen.key_of(tile + WARPS));
  }

  // q: each row divided by a power of two near its largest value, in F16
  // terms, as B fragments [step][column tile][term][lane]: a warp takes a row,
  // a lane four values at a time, which are a fragment each
  uint2* fragments = reinterpret_cast<uint2*>(shared);
  for (int r = warp; r < ROWS; r += WARPS) {
    constexpr int PER = (D + 127) / 128;
    float x[PER][4] = {};
    if (row0 + r < row1) {
      const int row = row0 + r;
      const X* q = static_cast<const X*>(a.q) + ((chunk.row + row / a.group) * a.q_heads + head * a.group + row % a.group) * D;
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int d = 4 * (lane + 32 * n);
        if (d >= D) continue;
        if constexpr (T::BF16) {
          const uint2 y = *reinterpret_cast<const uint2*>(q + d);
          x[n][0] = __uint_as_float(y.x << 16), x[n][1] = __uint_as_float(y.x & 0xffff0000u);
          x[n][2] = __uint_as_float(y.y << 16), x[n][3] = __uint_as_float(y.y & 0xffff0000u);
        } else {
          const float4 y = *reinterpret_cast<const float4*>(q + d);
          x[n][0] = y.x, x[n][1] = y.y, x[n][2] = y.z, x[n][3] = y.w;
        }
      }
    }
    float largest = 0.0f;
#pragma unroll
    for (int n = 0; n < PER; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) largest = fmaxf(largest, fabsf(x[n][e]));
#pragma unroll
    for (int o = 16; o > 0; o /= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    // 2^(floor(log2 largest) - Q_BITS), from the exponent bits, kept where it
    // and its inverse are normal
    const uint32_t exponent = __float_as_uint(largest) & 0x7f800000u;
    const uint32_t shift = uint32_t(Q_BITS) << 23;
    const float unit_of_row = __uint_as_float(max(exponent, shift + 0x00800000u) - shift);
    if (lane == 0) q_unit[r] = unit_of_row;
    const float inverse = 1.0f / unit_of_row;  // exact
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int d = 4 * (lane + 32 * n);
      if (d >= D) continue;
      const float y[4] = {x[n][0] * inverse, x[n][1] * inverse, x[n][2] * inverse, x[n][3] * inverse};
      const uint2 hi = make_uint2(half_pair(y[0], y[1]), half_pair(y[2], y[3]));
      int step, lt;
      Map::place_of(d, step, lt);
      uint2* to = fragments + step * TERMS * 32 + 4 * r + lt;
      to[0] = hi;
      if constexpr (TERMS == 2) {
        const float2 u = pair_value(hi.x), v = pair_value(hi.y);
        to[32] = make_uint2(half_pair(y[0] - u.x, y[1] - u.y), half_pair(y[2] - v.x, y[3] - v.y));
      }
    }
  }
  __syncthreads();

  // this lane's columns: rows 8 n + 2 t and + 1
  float multiplier[2];
  int position[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * t + e;
      multiplier[e] = a.scale * q_unit[r];
      position[e] = chunk.position + min(row0 + r, row1 - 1) / a.group;
    }
  // what every row sees: keys below `all_end` and from `all_low` on (or below
  // `first`)
  const int first = a.window > 0 ? a.first : 0;
  const int all_end = a.causal ? chunk.position + token0 + 1 : seen.end;
  const int all_low = a.window > 0 ? chunk.position + token1 - a.window : 0;
  const int lowest = a.window > 0 ? chunk.position + token0 - a.window + 1 : 0;  // what some row sees

  float out[T::DM][4];
  float largest[2], sum[2];
  bool taken_out = false;
  largest[0] = largest[1] = -INFINITY;
  sum[0] = sum[1] = 0.0f;
#pragma unroll
  for (int m = 0; m < T::DM; ++m) out[m][0] = out[m][1] = out[m][2] = out[m][3] = 0.0f;

  for (; tile < tile1; tile += WARPS) {
    const int key0 = seen.key_of(tile), next = tile + WARPS;
    float s[4];
    s[0] = s[1] = s[2] = s[3] = 0.0f;
#pragma unroll
    for (int step = 0; step < Map::STEPS; ++step) {
      uint32_t f[4];
      w.key_fragment(step, f);
#pragma unroll
        for (int term = TERMS - 1; term >= 0; --term) {
          const uint2 b = fragments[(step * TERMS + term) * 32 + lane];
          mma_f16(s, f, b.x, b.y);
        }
    }
    // (the keys' registers are the next tile's; its page was looked up a tile ago)
    if (next < tile1) w.load_keys();

    // scores, and each column's largest
    const bool whole = key0 + TILE <= all_end && (key0 >= all_low || key0 + TILE <= first);
    float rescale[2];
    bool grown = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = s[2 * half + e] * multiplier[e];
          if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
          if (!whole) {
            const int key = key0 + w.position_of(half);
            const bool sees = key < seen.end && (!a.causal || key <= position[e]) &&
                              (a.window == 0 || key > position[e] - a.window || key < first);
            x = sees ? x : -INFINITY;
          }
          s[2 * half + e] = x;
          top = fmaxf(top, x);
        }
#pragma unroll
        for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float before = largest[e];
        const float now = fmaxf(before, top - WEIGHT_LOG);
        rescale[e] = weight_of(before, now);
        grown = grown || now > before;
        largest[e] = now;
      }
    if (__any_sync(0xffffffffu, grown)) {
      sum[0] *= rescale[0], sum[1] *= rescale[1];
#pragma unroll
      for (int m = 0; m < T::DM; ++m) {
        out[m][0] *= rescale[0], out[m][1] *= rescale[1];
        out[m][2] *= rescale[0], out[m][3] *= rescale[1];
      }
    }
    uint32_t p[TERMS][2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          y[e] = weight_of(s[2 * half + e], largest[e]);
          sum[e] += y[e];
        }
        const uint32_t hi = half_pair(y[0], y[1]);
        p[0][half] = turn(hi);
        if constexpr (TERMS == 2) {
          const float2 u = pair_value(hi);
          p[1][half] = turn(half_pair(y[0] - u.x, y[1] - u.y));
        }
      }
    // where rows differ in what they see, a value that is not finite must not
    // meet the zero weights of those that do not see it: it is taken out here
    // and added to the rows that see it at the end
    if (!whole) {
#pragma unroll
      for (int m = 0; m < T::DM; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          w.v[m][half].x = finite_halves(w.v[m][half].x, key0 + 4 * t, seen.end, lowest, first, taken_out);
          w.v[m][half].y = finite_halves(w.v[m][half].y, key0 + 4 * t + 2, seen.end, lowest, first, taken_out);
        }
    }
    // (a tile's sums start from zero: the tensor core's drop low bits as a
    // chain grows, F32 additions round)
#pragma unroll
    for (int m = 0; m < T::DM; ++m) {
      uint32_t f[4];
      w.value_fragment(m, f);
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int term = TERMS - 1; term >= 0; --term) mma_f16(o, f, p[term][0], p[term][1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[m][e] += o[e];
    }
    if (next < tile1) {
      w.load_values();
      if (next + WARPS < tile1) w.find_page(seen.key_of(next + WARPS));
    }
  }

  // the warps' results: [warp][row][D] and [warp][row] (largest, sum)
  __syncthreads();  // (past the q fragments)
  float* merged = reinterpret_cast<float*>(shared);
  float2* stats = reinterpret_cast<float2*>(merged + WARPS * ROWS * D);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float total = sum[e];
#pragma unroll
      for (int o = 4; o < 32; o *= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
      const int r = 2 * t + e;
      if (g == 0) stats[warp * ROWS + r] = make_float2(largest[e], total);
#pragma unroll
      for (int m = 0; m < T::DM; ++m) {
        merged[(warp * ROWS + r) * D + 16 * m + g] = out[m][e];
        merged[(warp * ROWS + r) * D + 16 * m + g + 8] = out[m][2 + e];
      }
    }
  taken_out = __syncthreads_or(taken_out);
  for (int i = tid; i < (row1 - row0) * (D / 4); i += THREADS) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row0 + r, q_head = head * a.group + row % a.group;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) top = fmaxf(top, stats[j * ROWS + r].x);
    float total = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < WARPS; ++j) {
      const float2 stat = stats[j * ROWS + r];
      const float f = weight_of(stat.x, top);
      total += stat.y * f;  // (a NaN stays one)
      if (f == 0.0f) continue;
      const float4 y = *reinterpret_cast<const float4*>(merged + (j * ROWS + r) * D + d);
      x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
    }
    if (taken_out) {
      const int own = chunk.position + row / a.group;
      for (int j = tile0; j < tile1; ++j) {
        const int key0 = seen.key_of(j);
        if (key0 + TILE <= all_end && (key0 >= all_low || key0 + TILE <= first)) continue;
        const long long page_stride = (long long)a.kv_heads * D * a.at.page_size;
        const float4 y = not_finite(static_cast<const __half*>(a.values) + ((long long)head * D + d) * a.at.page_size,
                                    page_stride, chunk.table, a.at.pages, a.at.page_size, key0,
                                    min(key0 + TILE, a.causal ? own + 1 : seen.end),
                                    a.window > 0 ? own - a.window + 1 : 0, first);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
    }
    const long long at = (chunk.row + row / a.group) * a.q_heads + q_head;
    if (a.part_o) {
      *reinterpret_cast<float4*>(a.part_o + (at * a.splits + split) * D + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (at * a.splits + split) * 2) = make_float2(top, total);
      continue;
    }
    if (a.sinks) {
      const float sink = a.sinks[q_head], all = fmaxf(top, sink);
      const float f = weight_of(top, all);
      x.x *= f, x.y *= f, x.z *= f, x.w *= f;
      total = total * f + weight_of(sink, all);
    }
    X* to = static_cast<X*>(a.out) + at * D + d;
    const bool any = total != 0.0f;
    to[0] = X(any ? x.x / total : 0.0f), to[1] = X(any ? x.y / total : 0.0f);
    to[2] = X(any ? x.z / total : 0.0f), to[3] = X(any ? x.w / total : 0.0f);
  }
}

// The splits' join, a warp per (token, query head) row: out = sum_s o_s
// e^(m_s - M) / (sum_s l_s e^(m_s - M) + e^(sink - M)), M the largest of the
// m_s and the sink. A row's splits are those that held tiles of its unit, as
// the kernel that wrote them counted them.
struct JoinArgs {
  AttentionChunksArgs a;
  int rows_per_unit, keys_per_tile;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(THREADS) attention_chunks_join_kernel(const JoinArgs j) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  using X = typename std::conditional<BF16, __nv_bfloat16, float>::type;
  const AttentionChunksArgs& a = j.a;
  const int lane = threadIdx.x % 32, z = blockIdx.y;
  const Chunk chunk(a.at, z);
  const long long i = (long long)blockIdx.x * WARPS + threadIdx.x / 32;  // token x q_heads + head
  if (i >= (long long)chunk.tokens * a.q_heads) return;
  const int token = int(i / a.q_heads), head = int(i % a.q_heads);
  const int row0 = (token * a.group + head % a.group) / j.rows_per_unit * j.rows_per_unit;
  const int row1 = min(row0 + j.rows_per_unit, chunk.tokens * a.group);
  const SeenTiles seen(a, chunk, row0 / a.group, (row1 - 1) / a.group + 1, j.keys_per_tile);
  const int splits = seen.splits(a.tiles_per_split);
  const long long at = (chunk.row + token) * a.q_heads + head;
  const float2* stats = reinterpret_cast<const float2*>(a.part_ml) + at * a.splits;
  const float* parts = a.part_o + at * a.splits * D;
  float top = a.sinks ? a.sinks[head] : -INFINITY;
  for (int s = lane; s < splits; s += 32) top = fmaxf(top, stats[s].x);
#pragma unroll
  for (int o = 16; o > 0; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float total = 0.0f;
  constexpr int PER = (D + 127) / 128, FLIGHT = 8;  // splits' rows under way
  float x[PER][4] = {};
  for (int s0 = 0; s0 < splits; s0 += 32) {
    float factor = 0.0f;
    if (s0 + lane < splits) {
      const float2 stat = stats[s0 + lane];
      factor = weight_of(stat.x, top);
      total += stat.y * factor;  // (a NaN stays one)
    }
    const int here = min(32, splits - s0);
    for (int s1 = 0; s1 < here; s1 += FLIGHT) {
      float4 y[FLIGHT][PER];
#pragma unroll
      for (int n = 0; n < FLIGHT; ++n)
#pragma unroll
        for (int c = 0; c < PER; ++c) {
          const int d = 4 * (lane + 32 * c);
          y[n][c] = s1 + n < here && d < D ? *reinterpret_cast<const float4*>(parts + (long long)(s0 + s1 + n) * D + d)
                                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
      for (int n = 0; n < FLIGHT; ++n) {
        const float f = __shfl_sync(0xffffffffu, factor, (s1 + n) % 32);
        if (s1 + n >= here || f == 0.0f) continue;
#pragma unroll
        for (int c = 0; c < PER; ++c)
          x[c][0] += y[n][c].x * f, x[c][1] += y[n][c].y * f, x[c][2] += y[n][c].z * f, x[c][3] += y[n][c].w * f;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (a.sinks) total += weight_of(a.sinks[head], top);
  const bool any = total != 0.0f;
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int d = 4 * (lane + 32 * c);
    if (d >= D) continue;
    X* to = static_cast<X*>(a.out) + at * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = X(any ? x[c][e] / total : 0.0f);
  }
}

template <class T>
int launch_rows(const AttentionChunksArgs& a, cudaStream_t stream) {
  static PerDevice configured;
  DRIFT_TRY(ensure_shared_memory(configured, attention_rows_kernel<T>, T::BYTES));
  const int units = (a.at.longest * a.group + T::ROWS - 1) / T::ROWS;
  DRIFT_CUDA(launch_pdl(attention_rows_kernel<T>, dim3(unsigned(units) * a.splits, a.kv_heads, a.at.batch), THREADS,
                        T::BYTES, stream, a));
  DRIFT_LAUNCHED("attention_rows");
  return 0;
}

#define DRIFT_ROWS_REGISTER(D)                                                            \
  DRIFT_REGISTER(attention_rows_bf16_d##D, (attention_rows_kernel<RowsTraits<D, true>>))  \
  DRIFT_REGISTER(attention_rows_f32_d##D, (attention_rows_kernel<RowsTraits<D, false>>))
DRIFT_ROWS_REGISTER(64)
DRIFT_ROWS_REGISTER(80)
DRIFT_ROWS_REGISTER(128)
DRIFT_ROWS_REGISTER(256)
#define DRIFT_JOIN_REGISTER(D)                                                            \
  DRIFT_REGISTER(attention_chunks_join_f32_d##D, (attention_chunks_join_kernel<D, false>)) \
  DRIFT_REGISTER(attention_chunks_join_bf16_d##D, (attention_chunks_join_kernel<D, true>))
DRIFT_JOIN_REGISTER(64)
DRIFT_JOIN_REGISTER(80)
DRIFT_JOIN_REGISTER(128)
DRIFT_JOIN_REGISTER(256)

}  // namespace

template <int D>
static int launch_dim(const AttentionChunksArgs& a, bool bf16, cudaStream_t stream) {
  return bf16 ? launch_rows<RowsTraits<D, true>>(a, stream) : launch_rows<RowsTraits<D, false>>(a, stream);
}

int launch_attention_rows(const AttentionChunksArgs& a, int x_dtype, int head_dim, cudaStream_t stream) {
  const bool bf16 = x_dtype == DRIFT_BF16;
  switch (head_dim) {
    case 64: return launch_dim<64>(a, bf16, stream);
    case 80: return launch_dim<80>(a, bf16, stream);
    case 128: return launch_dim<128>(a, bf16, stream);
    default: return launch_dim<256>(a, bf16, stream);
  }
}

template <int D>
static int launch_join(const JoinArgs& j, bool bf16, cudaStream_t stream) {
  const long long rows = (long long)j.a.at.longest * j.a.q_heads;
  const dim3 grid(unsigned((rows + WARPS - 1) / WARPS), j.a.at.batch);
  if (bf16) DRIFT_CUDA(launch_pdl(attention_chunks_join_kernel<D, true>, grid, THREADS, 0, stream, j));
  else DRIFT_CUDA(launch_pdl(attention_chunks_join_kernel<D, false>, grid, THREADS, 0, stream, j));
  DRIFT_LAUNCHED("attention_chunks_join");
  return 0;
}

int launch_attention_join(const AttentionChunksArgs& a, int x_dtype, int head_dim, int rows_per_unit,
                          int keys_per_tile, cudaStream_t stream) {
  const JoinArgs j = {a, rows_per_unit, keys_per_tile};
  const bool bf16 = x_dtype == DRIFT_BF16;
  switch (head_dim) {
    case 64: return launch_join<64>(j, bf16, stream);
    case 80: return launch_join<80>(j, bf16, stream);
    case 128: return launch_join<128>(j, bf16, stream);
    default: return launch_join<256>(j, bf16, stream);
  }
}

}  // namespace drift

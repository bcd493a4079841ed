// attention_chunks over an 8-bit cache for few rows: a decoding step, drafted
// tokens.
//
// A unit is a key head of one sequence with up to ROWS of the (token, query
// head) rows that read it; a CTA takes one split of the unit's key tiles, each
// of its warps every fourth (or eighth) tile of 32 keys. Both products run on the int8
// tensor cores, turned round -- scores^T = K q^T and out^T = V^T p^T by
// mma.sync m16n8k32, keys and then dimensions as the 16 rows, the few query
// rows as columns -- with the codes as they lie in the cache: a lane's 16
// bytes of a key row, its 8 bytes of a dimension's positions, are A fragments
// without a conversion (converting them to F16 was two thirds of 1470
// instructions a tile). What is converted is the small side: a row of q and
// a tile's weights become whole numbers, split into balanced base-256 digits
// (bytes of (x + 0x808080) ^ 0x808080), a column for each row and digit. The
// sums are exact; they start from the bits of 1.5 x 2^23, so that they are F32
// numbers without a conversion (|sum| < 2^22), and their digits are joined in
// F32. A key's scale multiplies its score, a value's its weight.
//
// What the conversion rounds: q to 2^-30 of its row's largest value and a row's
// 32 products of weight and value scale in a tile to 2^-30 of the largest of them
// (BF16 rows of more than four, in three digits: 2^-22), each row and tile over a
// power of two of its own. So a row does not depend on what it
// does not see, a key of much weight costs no other tile's keys bits, and in
// its own none if its value is small (a row's largest code is 127, so its scale
// is its size). Steps of the warp's largest weight instead lost a tenth of the
// result where one of 16384 keys has ten times the weight of the others and a
// value of zero.
//
// Softmax in F32, a base and a sum a row and warp; the base moves when some
// weight passes 2^3 (and one vote a tile tells). The warps meet in shared
// memory, the splits in a second launch (attention_chunks_join_kernel).
//
// Bound by latency at 12 warps an SM (168 registers: a tile of codes on its way
// in each): about 1200 instructions a tile of 32 keys take 51 % of the issue
// slots and 37 % of DRAM's rate; a warp waits on fixed latencies and on global
// loads, about an issue's time each. A step of 16 sequences of 8700 to 16384
// keys of 8 heads of 128, F32, 115 us, 3.7 TB/s of codes and scales; one of 4096
// keys 11 us, two launches' latencies; 8 sequences' up to 5 drafts over up to
// 4096 keys 53 us, three units of eight rows a sequence and head.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "chunks.cuh"
#include "common.cuh"
#include "registry.cuh"

namespace drift {

namespace {

constexpr int TILE = 32;   // keys of a warp's tile
constexpr int PITCH = 36;  // words of a row's weights in shared memory: rows on different banks
constexpr int ZERO = 0x4b400000;  // the bits of 1.5 x 2^23
constexpr float ZERO_VALUE = 12582912.0f;
constexpr float GROWTH = 8.0f;    // a weight that moves its base
constexpr int UNIT_GROWTH = 40 << 23;  // a tile's unit over the output's, in exponent bits, that moves the latter

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same as a new sum.
__device__ __forceinline__ void mma_s8_new(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(ZERO));
}

// The digits of x, the least in the lowest byte, each -128 to 127.
__device__ __forceinline__ uint32_t digits(int x) { return (uint32_t(x) + 0x00808080u) ^ 0x00808080u; }

// Byte `digit` of each of four words.
__device__ __forceinline__ uint32_t digit_of(const uint4& x, uint32_t digit) {
  const uint32_t pick = digit | (digit + 4) << 4;
  return __byte_perm(__byte_perm(x.x, x.y, pick), __byte_perm(x.z, x.w, pick), 0x5410);
}

// The larger, a NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// Packed: up to four rows, column c of digit tile j being row c % 4's digit 2 j
// + c / 4; otherwise up to eight, with a tile for each digit. (Sixteen or
// twenty-four rows to a warp shared its keys but left registers for eight warps
// an SM: drafts of 12 rows 49 us, in units of eight 40; of 20, 70 and 51.)
template <int D_, bool BF16_, bool PACKED_>
struct CodesTraits {
  static constexpr int D = D_;
  static constexpr bool BF16 = BF16_, PACKED = PACKED_;
  static constexpr int ROWS = PACKED ? 4 : 8;
  // As many warps as registers leave an SM without spills: sixteen of 128, for
  // heads of 128 twelve of 168 (a step of 16 x 8700 to 16384 keys: sixteen, spilling,
  // 191 us, twelve 113, eight 135), for more rows and wider heads eight. In
  // CTAs of four, one's start and end run under the others.
  static constexpr int WARPS = attention_codes_warps(D), THREADS = 32 * WARPS;
  static constexpr int CTAS = attention_codes_ctas(D);
  static constexpr int DIGITS = PACKED || !BF16 ? 4 : 3, Q_DIGITS = DIGITS, P_DIGITS = DIGITS;
  static constexpr int Q_TILES = PACKED ? Q_DIGITS / 2 : Q_DIGITS;
  static constexpr int P_TILES = PACKED ? P_DIGITS / 2 : P_DIGITS;
  static constexpr int Q_BITS = DIGITS == 4 ? 29 : 21;           // of the largest value's leading bit
  static constexpr int P_BITS = P_DIGITS == 4 ? 29 : 21;         // the same for a tile's products
  static constexpr int CHUNKS = D / 64, TAIL = D % 64 / 16;      // 16-byte chunks a lane has of a key row; 4 bytes
  static constexpr int STEPS = 2 * CHUNKS + TAIL, WORDS = 4 * CHUNKS + TAIL;
  static constexpr int DM = D / 16;
  static constexpr int Q_BYTES = STEPS * Q_TILES * 32 * 8;
  static constexpr int P_BYTES = WARPS * ROWS * PITCH * 4;
  static constexpr int MERGE_BYTES = WARPS * ROWS * (D + 4) * 4;
  static constexpr int BYTES = Q_BYTES + P_BYTES > MERGE_BYTES ? Q_BYTES + P_BYTES : MERGE_BYTES;
};

template <class T>
struct CodesWarp {
  static constexpr int D = T::D;
  const AttentionChunksArgs& a;
  const Chunk& chunk;
  const SeenTiles& seen;
  const int head, g, t;
  const uint32_t page_magic;              // 2^32 / page_size, up
  int k_page[2], k_place[2], v_page, v_place;  // of the tile that is loaded next
  uint32_t k[2][2][T::WORDS];             // [16 keys][row g, g + 8]
  uint2 v[T::DM][2];                      // [16 dimensions][row g, g + 8], positions 8 t .. 8 t + 7
  float k_scale[2][2], v_scale[2][2];

  __device__ CodesWarp(const AttentionChunksArgs& a, const Chunk& c, const SeenTiles& s, int head, int lane)
      : a(a), chunk(c), seen(s), head(head), g(lane / 4), t(lane % 4),
        page_magic(0xffffffffu / uint32_t(a.at.page_size) + 1) {}

  // The page that holds `position` and the place in it; -1 past the last key,
  // or for a page that the cache does not have.
  __device__ void find(int position, int& page, int& place) const {
    int index = int(__umulhi(uint32_t(position), page_magic));  // (one too many at most)
    place = position - index * a.at.page_size;
    if (place < 0) --index, place += a.at.page_size;
    page = -1;
    if (position >= seen.end) return;
    page = chunk.table[index];
    if (page >= 0 && page < a.at.pages) return;
    chunk_error(a.error);
    page = -1;
  }
  __device__ void find_pages(int key0) {
    find(key0, k_page[0], k_place[0]);
    find(key0 + 16, k_page[1], k_place[1]);
    v_page = t < 2 ? k_page[0] : k_page[1];
    v_place = (t < 2 ? k_place[0] : k_place[1]) + 8 * (t % 2);
  }

  __device__ void load_keys() {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int place = k_place[m] + g + 8 * half;
        const bool there = k_page[m] >= 0;
        const uint8_t* row = static_cast<const uint8_t*>(a.keys) +
                             (((long long)k_page[m] * a.at.page_size + place) * a.kv_heads + head) * D;
#pragma unroll
        for (int c = 0; c < T::CHUNKS; ++c) {
          const uint4 x = there ? __ldg(reinterpret_cast<const uint4*>(row) + 4 * c + t) : make_uint4(0, 0, 0, 0);
          k[m][half][4 * c] = x.x, k[m][half][4 * c + 1] = x.y, k[m][half][4 * c + 2] = x.z, k[m][half][4 * c + 3] = x.w;
        }
        if constexpr (T::TAIL)
          k[m][half][4 * T::CHUNKS] = there ? __ldg(reinterpret_cast<const uint32_t*>(row + 64 * T::CHUNKS) + t) : 0;
        const long long at = ((long long)k_page[m] * a.kv_heads + head) * a.at.page_size + place;
        k_scale[m][half] = there ? __ldg(a.key_scales + at) : 0.0f;
        v_scale[m][half] = there ? __ldg(a.value_scales + at) : 0.0f;
      }
  }
  __device__ void load_values() {
    const uint8_t* column = static_cast<const uint8_t*>(a.values) +
                            ((long long)v_page * a.kv_heads + head) * D * a.at.page_size + v_place;
#pragma unroll
    for (int m = 0; m < T::DM; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        v[m][half] = v_page >= 0 ? __ldg(reinterpret_cast<const uint2*>(column + (16 * m + g + 8 * half) * (long long)a.at.page_size))
                                 : make_uint2(0, 0);
  }
};

template <class T>
__global__ void __launch_bounds__(T::THREADS, T::CTAS) attention_codes_kernel(const AttentionChunksArgs a) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  constexpr int D = T::D, ROWS = T::ROWS, WARPS = T::WARPS, THREADS = T::THREADS;
  constexpr bool PACKED = T::PACKED;
  using X = typename std::conditional<T::BF16, __nv_bfloat16, float>::type;
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ float q_unit[ROWS];  // what a step of a row of q is worth
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

  CodesWarp<T> w(a, chunk, seen, head, lane);
  int tile = tile0 + warp;
  if (tile < tile1) {
    w.find_pages(seen.key_of(tile));
    w.load_keys();
    w.load_values();
    if (tile + WARPS < tile1) w.find_pages(seen.key_of(tile + WARPS));
  }

  // q in whole numbers of a power of two that gives its largest value
  // Q_BITS + 1 bits, as B fragments of digits [step][digit tile][lane]: a warp
  // takes a row, a lane four values at a time, which are a digit's word each
  uint32_t* fragments = reinterpret_cast<uint32_t*>(shared);
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
    bool finite = true;
#pragma unroll
    for (int n = 0; n < PER; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        largest = fmaxf(largest, fabsf(x[n][e]));
        finite = finite && fabsf(x[n][e]) <= 3.402823466e38f;
      }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    finite = __all_sync(0xffffffffu, finite);
    // (kept where the unit and its inverse are normal; a row that is not
    // finite has a NaN for a unit, and so for every score)
    constexpr uint32_t SHIFT = uint32_t(T::Q_BITS) << 23;
    const uint32_t exponent = max(__float_as_uint(largest) & 0x7f800000u, SHIFT + 0x01000000u) - SHIFT;
    if (lane == 0) q_unit[r] = finite ? __uint_as_float(exponent) : __int_as_float(0x7fc00000);
    const float inverse = __uint_as_float(0x7f000000u - exponent);
#pragma unroll
    for (int n = 0; n < PER; ++n) {
      const int d = 4 * (lane + 32 * n);
      if (d >= D) continue;
      const uint4 y = make_uint4(digits(__float2int_rn(x[n][0] * inverse)), digits(__float2int_rn(x[n][1] * inverse)),
                                 digits(__float2int_rn(x[n][2] * inverse)), digits(__float2int_rn(x[n][3] * inverse)));
      // where a lane of the product has these bytes of a key row: two steps
      // to a chunk of 64, then the tail's first sixteen (of 32: zeros follow)
      const bool tail = d >= 64 * T::CHUNKS;
      const int step = tail ? 2 * T::CHUNKS : d / 64 * 2 + d / 8 % 2, lt = tail ? d / 4 % 4 : d / 16 % 4;
      const int word = tail ? 0 : d / 4 % 2;
#pragma unroll
      for (int digit = 0; digit < T::Q_DIGITS; ++digit) {
        const int tile = PACKED ? digit / 2 : digit, column = PACKED ? digit % 2 * 4 + r : r;
        uint32_t* to = fragments + ((step * T::Q_TILES + tile) * 32 + 4 * column + lt) * 2;
        to[word] = digit_of(y, digit);
        if (tail) to[1] = 0;
      }
    }
  }
  __syncthreads();

  // this lane's columns: rows 2 t and 2 t + 1 (packed: modulo 4)
  float multiplier[2];
  int position[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = PACKED ? (2 * t + e) % 4 : 2 * t + e;
      multiplier[e] = a.scale * q_unit[r];
      position[e] = chunk.position + min(row0 + r, row1 - 1) / a.group;
    }
  // what every row sees: keys below `all_end` and from `all_low` on (or below
  // `first`)
  const int first = a.window > 0 ? a.first : 0;
  const int all_end = a.causal ? chunk.position + token0 + 1 : seen.end;
  const int all_low = a.window > 0 ? chunk.position + token1 - a.window : 0;
  const float low_digit = PACKED && t >= 2 ? 256.0f : 1.0f;  // the worth of a packed lane's lower digit

  float out[T::DM][4];
  float base[2], sum[2];
  int o_unit[2];  // what a row's output is over, a power of two as exponent bits
  o_unit[0] = o_unit[1] = 1 << 23;
  base[0] = base[1] = -INFINITY;
  sum[0] = sum[1] = 0.0f;
#pragma unroll
  for (int m = 0; m < T::DM; ++m) out[m][0] = out[m][1] = out[m][2] = out[m][3] = 0.0f;
  float* weights = reinterpret_cast<float*>(shared + T::Q_BYTES) + warp * ROWS * PITCH;

  for (; tile < tile1; tile += WARPS) {
    const int key0 = seen.key_of(tile), next = tile + WARPS;
    const bool whole = key0 + TILE <= all_end && (key0 >= all_low || key0 + TILE <= first);
    // scores [row tile][16 keys][(key g, columns 2 t, 2 t + 1), (key g + 8, the same)]
    float s[2][4];
    int acc[2][T::Q_TILES][4];
#pragma unroll
    for (int step = 0; step < T::STEPS; ++step) {
      uint2 b[T::Q_TILES];
#pragma unroll
      for (int j = 0; j < T::Q_TILES; ++j)
        b[j] = reinterpret_cast<const uint2*>(fragments)[(step * T::Q_TILES + j) * 32 + lane];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const bool both = step < 2 * T::CHUNKS;
        const int word = 2 * step;
        const uint32_t f[4] = {w.k[m][0][word], w.k[m][1][word], both ? w.k[m][0][both ? word + 1 : 0] : 0,
                               both ? w.k[m][1][both ? word + 1 : 0] : 0};
#pragma unroll
        for (int j = 0; j < T::Q_TILES; ++j) {
          if (step == 0) mma_s8_new(acc[m][j], f, b[j].x, b[j].y);
          else mma_s8(acc[m][j], f, b[j].x, b[j].y);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = 0.0f;
#pragma unroll
        for (int j = T::Q_TILES - 1; j >= 0; --j) {
          const float y = __int_as_float(acc[m][j][e]) - ZERO_VALUE;
          x = j == T::Q_TILES - 1 ? y : fmaf(x, PACKED ? 65536.0f : 256.0f, y);
        }
        if (PACKED) {
          x *= low_digit;
          x += __shfl_xor_sync(0xffffffffu, x, 2);
        }
        s[m][e] = x;
      }
    float k_scale[2][2], v_scale[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half) k_scale[m][half] = w.k_scale[m][half], v_scale[m][half] = w.v_scale[m][half];
    if (next < tile1) w.load_keys();  // on their way under the rest of this tile
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key = key0 + 16 * m + g + 8 * half;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = s[m][2 * half + e] * multiplier[e] * k_scale[m][half];
            if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
            if (!whole) {
              const bool sees = key < seen.end && (!a.causal || key <= position[e]) &&
                                (a.window == 0 || key > position[e] - a.window || key < first);
              x = sees ? x : -INFINITY;
            }
            s[m][2 * half + e] = x;
          }
      }
    // weights with the bases as they are; where one passes GROWTH (or is a
    // NaN, or a row has no base yet) they move
    float p[2][4];
    bool move = false;
    auto weigh = [&]() {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[m][e] = weight_of(s[m][e], base[e % 2]);
            move = move || !(p[m][e] <= GROWTH);
          }
    };
    weigh();
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(s[0][e], s[0][e + 2]), fmaxf(s[1][e], s[1][e + 2]));
#pragma unroll
          for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float now = fmaxf(base[e], top), f = weight_of(base[e], now);
          base[e] = now;
          sum[e] *= f;
#pragma unroll
          for (int m = 0; m < T::DM; ++m) out[m][e] *= f, out[m][e + 2] *= f;
        }
      weigh();
    }
    // products of weights and values' scales, [row][key] in shared memory: a
    // product's columns are rows
    __syncwarp();  // (the tile before is read)
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = p[m][2 * half + e];
          sum[e] += x;
          float y = x * v_scale[m][half];
          if (!whole && x == 0.0f) y = 0.0f;  // (a hidden value's scale may be a NaN)
          if (!PACKED || t < 2) weights[(2 * t + e) * PITCH + 16 * m + g + 8 * half] = y;
        }
    __syncwarp();
    // a row's largest, the power of two at or below it, and the products as
    // whole numbers of steps: this lane has eight keys' of row g (packed: g % 4)
    const float4* from = reinterpret_cast<const float4*>(weights + (PACKED ? g % 4 : g) * PITCH + 8 * t);
    const float4 y0 = from[0], y1 = from[1];
    float y[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
    float top = max_nan(max_nan(max_nan(y[0], y[1]), max_nan(y[2], y[3])), max_nan(max_nan(y[4], y[5]), max_nan(y[6], y[7])));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int tile_unit = max(__float_as_int(top) & 0x7f800000, 1 << 23);
    if (tile_unit < 64 << 23) {  // (its inverse times the steps would be past F32's range)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= 18446744073709551616.0f;
    }
    const float steps = __uint_as_float((uint32_t(254 + T::P_BITS) << 23) - uint32_t(tile_unit + (tile_unit < 64 << 23 ? 64 << 23 : 0)));
    uint4 x0, x1;
    x0.x = digits(__float2int_rn(y[0] * steps)), x0.y = digits(__float2int_rn(y[1] * steps));
    x0.z = digits(__float2int_rn(y[2] * steps)), x0.w = digits(__float2int_rn(y[3] * steps));
    x1.x = digits(__float2int_rn(y[4] * steps)), x1.y = digits(__float2int_rn(y[5] * steps));
    x1.z = digits(__float2int_rn(y[6] * steps)), x1.w = digits(__float2int_rn(y[7] * steps));
    uint32_t b[T::P_TILES][2];
#pragma unroll
    for (int j = 0; j < T::P_TILES; ++j) {
      const uint32_t digit = PACKED ? 2 * j + g / 4 : j;
      b[j][0] = digit_of(x0, digit);
      b[j][1] = digit_of(x1, digit);
    }
    // what a step is worth to this lane's columns, over their outputs' units;
    // a product that is not finite makes its row NaNs
    float worth[2];
    {
      int over[2];
      bool grown = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = PACKED ? (2 * t + e) % 4 : 2 * t + e;
        over[e] = __shfl_sync(0xffffffffu, tile_unit, 4 * r);
        if (over[e] == 0x7f800000) sum[e] = __int_as_float(0x7fc00000);
        over[e] -= o_unit[e];
        grown = grown || over[e] > UNIT_GROWTH;
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (over[e] <= UNIT_GROWTH) continue;
          const float f = __int_as_float(max((127 << 23) - over[e], 0));
          o_unit[e] += over[e];
          over[e] = 0;
#pragma unroll
          for (int m = 0; m < T::DM; ++m) out[m][e] *= f, out[m][e + 2] *= f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) worth[e] = __int_as_float(max(over[e] + ((127 - T::P_BITS) << 23), 0));
    }
#pragma unroll
    for (int m = 0; m < T::DM; ++m) {
      const uint32_t f[4] = {w.v[m][0].x, w.v[m][1].x, w.v[m][0].y, w.v[m][1].y};
      int acc[T::P_TILES][4];
#pragma unroll
      for (int j = 0; j < T::P_TILES; ++j) {
        mma_s8_new(acc[j], f, b[j][0], b[j][1]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = 0.0f;
#pragma unroll
        for (int j = T::P_TILES - 1; j >= 0; --j) {
          const float y = __int_as_float(acc[j][e]) - ZERO_VALUE;
          x = j == T::P_TILES - 1 ? y : fmaf(x, PACKED ? 65536.0f : 256.0f, y);
        }
        out[m][e] = fmaf(x, worth[e % 2], out[m][e]);
      }
    }
    if (next < tile1) {
      w.load_values();
      if (next + WARPS < tile1) w.find_pages(seen.key_of(next + WARPS));
    }
  }

  // the warps' results: [warp][row][D] and [warp][row] (base, sum)
  __syncthreads();  // (past the fragments and the weights)
  float* merged = reinterpret_cast<float*>(shared);
  float2* stats = reinterpret_cast<float2*>(merged + WARPS * ROWS * D);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float total = sum[e];
#pragma unroll
      for (int o = 4; o < 32; o *= 2) total += __shfl_xor_sync(0xffffffffu, total, o);
      const int r = 2 * t + e;
      const bool writes = !PACKED || t < 2;
      if (g == 0 && writes) stats[warp * ROWS + r] = make_float2(base[e], total);
#pragma unroll
      for (int m = 0; m < T::DM; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = out[m][2 * half + e] * low_digit * __int_as_float(o_unit[e]);
          if (PACKED) x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (writes) merged[(warp * ROWS + r) * D + 16 * m + g + 8 * half] = x;
        }
    }
  __syncthreads();
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

template <class T>
int launch_codes(const AttentionChunksArgs& a, cudaStream_t stream) {
  static PerDevice configured;
  DRIFT_TRY(ensure_shared_memory(configured, attention_codes_kernel<T>, T::BYTES));
  const int units = (a.at.longest * a.group + T::ROWS - 1) / T::ROWS;
  DRIFT_CUDA(launch_pdl(attention_codes_kernel<T>, dim3(unsigned(units) * a.splits, a.kv_heads, a.at.batch), T::THREADS,
                        T::BYTES, stream, a));
  DRIFT_LAUNCHED("attention_codes");
  return 0;
}

template <int D, bool BF16>
int launch_rows_of(const AttentionChunksArgs& a, int rows_per_unit, cudaStream_t stream) {
  if (rows_per_unit == 4) return launch_codes<CodesTraits<D, BF16, true>>(a, stream);
  return launch_codes<CodesTraits<D, BF16, false>>(a, stream);
}

template <int D>
int launch_dim(const AttentionChunksArgs& a, bool bf16, int rows_per_unit, cudaStream_t stream) {
  return bf16 ? launch_rows_of<D, true>(a, rows_per_unit, stream) : launch_rows_of<D, false>(a, rows_per_unit, stream);
}

#define DRIFT_CODES_REGISTER(D)                                                                          \
  DRIFT_REGISTER(attention_codes_f32_d##D##_r4, (attention_codes_kernel<CodesTraits<D, false, true>>))  \
  DRIFT_REGISTER(attention_codes_f32_d##D##_r8, (attention_codes_kernel<CodesTraits<D, false, false>>)) \
  DRIFT_REGISTER(attention_codes_bf16_d##D##_r4, (attention_codes_kernel<CodesTraits<D, true, true>>))  \
  DRIFT_REGISTER(attention_codes_bf16_d##D##_r8, (attention_codes_kernel<CodesTraits<D, true, false>>))
DRIFT_CODES_REGISTER(64)
DRIFT_CODES_REGISTER(80)
DRIFT_CODES_REGISTER(128)
DRIFT_CODES_REGISTER(256)

}  // namespace

int launch_attention_codes(const AttentionChunksArgs& a, int x_dtype, int head_dim, int rows_per_unit,
                           cudaStream_t stream) {
  const bool bf16 = x_dtype == DRIFT_BF16;
  switch (head_dim) {
    case 64: return launch_dim<64>(a, bf16, rows_per_unit, stream);
    case 80: return launch_dim<80>(a, bf16, rows_per_unit, stream);
    case 128: return launch_dim<128>(a, bf16, rows_per_unit, stream);
    default: return launch_dim<256>(a, bf16, rows_per_unit, stream);
  }
}

}  // namespace drift

// The paged cache written and read for a batch of sequences' new tokens at
// once: F16 caches, in Ops.cacheWrite's layout (ops/KvCache.scala:12-23), and
// 8-bit ones of the same layout -- codes [pages][page offset][kv_heads][D] and
// [pages][kv_heads][D][page offset], with an F32 scale per (position, head) of
// either side, [pages][kv_heads][page offset].
//
// A row x of D values is kept as scale s = fl(max |x| / 127) and codes
// c = rint(x / s), halves to the even code: a value is off by at most s / 2 (codes
// end at 127, which only subnormal scales, rounded by more than 2^-8, can pass).
// The quotient is decided exactly (quantize()), so a code never depends on how
// a division rounds. A row that holds a NaN or an infinity has no step: its
// scale is NaN and it reads back as NaNs.
//
// A CTA takes 16 consecutive positions (an aligned sixteenth-row of a page) of
// one head, or of a few: their rows in, the keys out as rows, the values out
// transposed, through shared memory, 16 positions of a dimension in one 16-byte
// store (32 for F16). Bound by memory, (4 or 2) + 1 bytes a value: 16 x 4096
// positions of 8 heads of 128 back to BF16 58 us, 5.4 TB/s; 4 x 4099 from BF16
// 59 us, 2.8 TB/s (a CTA's chain of loads, largest value, codes and turned
// stores; F32 rows, twice the bytes in, 61 us). Few rows take 3 us, a launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "chunks.cuh"
#include "common.cuh"
#include "registry.cuh"

namespace drift {

namespace {

constexpr int RUN = 16;       // positions of a CTA
constexpr int THREADS = 256;  // 8 warps, two rows of keys and two of values of a head each
// Heads of a CTA that reads: enough loads under way to hide the three dependent
// ones before them (16 x 4096 positions of 8 heads 58 us, 77 with one). One
// that writes takes one: its rows wait in registers for their largest value,
// and with four there were two CTAs an SM (4 x 4099 positions 110 us, 85 with one).
constexpr int read_heads(int dim) { return dim > 128 ? 2 : 4; }

// x's code for step s > 0: rint(x / s) as if in exact arithmetic. c is within
// one of it; x - c s is exact in one fused operation (both are multiples of
// x's or s's last place, and the difference is below s), so comparing twice
// it with s decides.
__device__ __forceinline__ int quantize(float x, float s) {
  float c = rintf(x / s);
  const float r = fmaf(-c, s, x), twice = 2.0f * r;
  const bool odd = int(c) & 1;
  if (twice > s || (twice == s && odd)) c += 1.0f;
  else if (twice < -s || (twice == -s && odd)) c -= 1.0f;
  return int(fminf(fmaxf(c, -127.0f), 127.0f));
}
__device__ __noinline__ uint32_t quantize_exactly(float x0, float x1, float x2, float x3, float s) {
  return (uint32_t(quantize(x0, s)) & 255) | (uint32_t(quantize(x1, s)) & 255) << 8 |
         (uint32_t(quantize(x2, s)) & 255) << 16 | uint32_t(quantize(x3, s)) << 24;
}
// Four codes by s's reciprocal where that cannot be wrong: x times it is within
// 127 * 2^-23 < 2^-16 of x / s, so only a product that close to a half between
// two codes needs the above, as do steps so small that they lost bits. Added to
// 1.5 x 2^23 a product rounds to a whole number in the sum's low bits. (With
// a conversion and a branch a value 4 x 4099 positions of 8 heads of 64 took 62
// us, 56 so, of 2 heads of 256 30 and 27.)
__device__ __forceinline__ uint32_t quantize_four(const float (&x)[4], float s, float reciprocal) {
  constexpr float ZERO = 12582912.0f;
  uint32_t codes[4];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float sum = fmaf(x[e], reciprocal, ZERO);
    codes[e] = __float_as_uint(sum);
    off = fmaxf(off, fabsf(fmaf(x[e], reciprocal, ZERO - sum)));
  }
  if (!(s > 0.0f)) return 0;  // a row of zeros, or one without a step
  if (off >= 0.4999f || s < 7.9e-31f) return quantize_exactly(x[0], x[1], x[2], x[3], s);
  return __byte_perm(__byte_perm(codes[0], codes[1], 0x0040), __byte_perm(codes[2], codes[3], 0x0040), 0x5410);
}

template <typename X>
__device__ __forceinline__ void load_four(const X* row, float (&x)[4]);
template <>
__device__ __forceinline__ void load_four(const float* row, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(row);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <>
__device__ __forceinline__ void load_four(const __nv_bfloat16* row, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(row);
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void store_four(float* row, const float (&x)[4]) {
  *reinterpret_cast<float4*>(row) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_four(__nv_bfloat16* row, const float (&x)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  uint2 v;
  v.x = *reinterpret_cast<const uint32_t*>(&a), v.y = *reinterpret_cast<const uint32_t*>(&b);
  *reinterpret_cast<uint2*>(row) = v;
}

// The run of positions that CTA (block, head, sequence) handles.
struct Run {
  int lo, hi;            // its offsets in the 16 that are new tokens: [lo, hi)
  long long row;         // the row of offset 0's token (may be before the chunk)
  long long page;
  int offset;            // of the run in its page
  bool missing;          // the page is none of the cache's
  __device__ Run(const ChunkLayout& a, const Chunk& c, int block, int* error) {
    lo = hi = 0;
    missing = false;
    if ((long long)block * RUN >= (long long)c.tokens + RUN) return;  // (start below stays an int)
    const int start = (c.position / RUN + block) * RUN;
    lo = max(c.position - start, 0);
    hi = min(c.position + c.tokens - start, RUN);
    row = c.row + (start - c.position);
    page = 0;
    offset = start % a.page_size;
    if (hi <= lo) return;
    page = c.table[start / a.page_size];
    missing = page < 0 || page >= a.pages;
    if (missing && threadIdx.x == 0) chunk_error(error);
  }
};

struct WriteArgs {
  ChunkLayout at;
  const void* k;
  const void* v;
  void* keys;
  void* values;
  float* key_scales;
  float* value_scales;
  int kv_heads;
  int* error;
};

// Codes are int8_t or __half (no scale).
template <int D, typename X, typename Code>
__global__ void __launch_bounds__(THREADS, D <= 128 ? 6 : 4) cache_write_chunks_kernel(const WriteArgs a) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  constexpr bool CODES = sizeof(Code) == 1;
  constexpr int PER = (D + 127) / 128;  // groups of four values a lane has of a row
  __shared__ __align__(16) Code turned[RUN][D + 16];  // the values' rows
  const int block = blockIdx.x, head = blockIdx.y, z = blockIdx.z;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Chunk chunk(a.at, z);
  if (!chunk.ok && block == 0 && head == 0 && threadIdx.x == 0) chunk_error(a.error);
  const Run run(a.at, chunk, block, a.error);
  if (run.hi <= run.lo || run.missing) return;
  // rows 0-15 are the run's keys, 16-31 its values; warp w takes 4 of them
  float x[4][PER][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = warp + 8 * (i % 2);
    const X* from = static_cast<const X*>(i < 2 ? a.k : a.v) + ((run.row + p) * a.kv_heads + head) * D;
    const bool in = p >= run.lo && p < run.hi;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int d = 4 * (lane + 32 * j);
      if (in && d < D) load_four(from + d, x[i][j]);
      else x[i][j][0] = x[i][j][1] = x[i][j][2] = x[i][j][3] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = warp + 8 * (i % 2);
    const bool in = p >= run.lo && p < run.hi;
    float scale = 0.0f, reciprocal = 0.0f;
    if constexpr (CODES) {
      float largest = 0.0f;
      float zero = 0.0f;  // NaN once a value is infinite or NaN
#pragma unroll
      for (int j = 0; j < PER; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          largest = fmaxf(largest, fabsf(x[i][j][e]));
          zero = fmaf(x[i][j][e], 0.0f, zero);
        }
#pragma unroll
      for (int o = 16; o > 0; o /= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      const bool finite = __all_sync(0xffffffffu, zero == 0.0f);
      scale = finite ? largest / 127.0f : __int_as_float(0x7fc00000);
      if (in && lane == 0)
        (i < 2 ? a.key_scales : a.value_scales)[(run.page * a.kv_heads + head) * a.at.page_size + run.offset + p] =
            scale;
      reciprocal = 1.0f / scale;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int d = 4 * (lane + 32 * j);
      if (d >= D) continue;
      __align__(16) Code codes[4];
      if constexpr (CODES) *reinterpret_cast<uint32_t*>(codes) = quantize_four(x[i][j], scale, reciprocal);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e) codes[e] = __float2half_rn(x[i][j][e]);
      Code* to = i < 2 ? static_cast<Code*>(a.keys) +
                             ((run.page * a.at.page_size + run.offset + p) * a.kv_heads + head) * D + d
                       : &turned[p][d];
      if (i >= 2 || in) {
        if constexpr (CODES) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(codes);
        else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(codes);
      }
    }
  }
  __syncthreads();
  Code* values = static_cast<Code*>(a.values) + (run.page * a.kv_heads + head) * (long long)D * a.at.page_size + run.offset;
  const bool whole = run.lo == 0 && run.hi == RUN;
  for (int d = threadIdx.x; d < D; d += THREADS) {
    __align__(16) Code column[RUN];
#pragma unroll
    for (int p = 0; p < RUN; ++p) column[p] = turned[p][d];
    Code* to = values + (long long)d * a.at.page_size;
    if (whole) {
#pragma unroll
      for (int j = 0; j < int(sizeof(column)) / 16; ++j)
        reinterpret_cast<uint4*>(to)[j] = reinterpret_cast<const uint4*>(column)[j];
    } else {
#pragma unroll
      for (int p = 0; p < RUN; ++p)
        if (p >= run.lo && p < run.hi) to[p] = column[p];
    }
  }
}

struct ReadArgs {
  ChunkLayout at;
  const void* keys;
  const void* values;
  const float* key_scales;
  const float* value_scales;
  void* k;
  void* v;
  int kv_heads;
  int* error;
};

// The reverse: a value is code x scale, rounded once to F32 (and once to BF16).
template <int D, typename X, typename Code>
__global__ void __launch_bounds__(THREADS) cache_read_chunks_kernel(const ReadArgs a) {
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  constexpr bool CODES = sizeof(Code) == 1;
  constexpr int PER = (D + 127) / 128, HEADS = read_heads(D);
  __shared__ __align__(16) Code turned[HEADS][RUN][D + 16];
  const int block = blockIdx.x, head0 = blockIdx.y * HEADS, z = blockIdx.z;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Chunk chunk(a.at, z);
  if (!chunk.ok && block == 0 && head0 == 0 && threadIdx.x == 0) chunk_error(a.error);
  const Run run(a.at, chunk, block, a.error);
  if (run.hi <= run.lo) return;
  const int heads = min(HEADS, a.kv_heads - head0);
  const Code* keys = static_cast<const Code*>(a.keys) +
                     ((run.page * a.at.page_size + run.offset) * a.kv_heads + head0) * (long long)D;
  const Code* values = static_cast<const Code*>(a.values) +
                       (run.page * a.kv_heads + head0) * (long long)D * a.at.page_size + run.offset;
  // (the sixteen positions are one page's: those that are not the chunk's are
  // read with it and not written out)
  using Four = typename std::conditional<CODES, uint32_t, uint2>::type;
  constexpr int WORDS = int(sizeof(Code)) * RUN / 16, COLUMNS = (HEADS * D + THREADS - 1) / THREADS;
  uint4 columns[COLUMNS][WORDS];
#pragma unroll
  for (int n = 0; n < COLUMNS; ++n) {
    const int d = threadIdx.x + THREADS * n;
#pragma unroll
    for (int j = 0; j < WORDS; ++j)
      columns[n][j] = d < heads * D && !run.missing
                          ? reinterpret_cast<const uint4*>(values + (long long)d * a.at.page_size)[j]
                          : make_uint4(0, 0, 0, 0);
  }
  Four held[HEADS][2][PER];
  float scale[HEADS][4];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const bool there = h < heads && !run.missing;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int d = 4 * (lane + 32 * j);
        held[h][i][j] = Four{};
        if (d < D && there)
          held[h][i][j] = *reinterpret_cast<const Four*>(keys + ((long long)(warp + 8 * i) * a.kv_heads + h) * D + d);
      }
    const long long scales = (run.page * a.kv_heads + head0 + h) * a.at.page_size + run.offset;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      scale[h][i] = CODES && there ? (i < 2 ? a.key_scales : a.value_scales)[scales + warp + 8 * (i % 2)] : 1.0f;
  }
#pragma unroll
  for (int n = 0; n < COLUMNS; ++n) {
    const int d = threadIdx.x + THREADS * n;
    if (d >= HEADS * D) break;
    const Code* column = reinterpret_cast<const Code*>(columns[n]);
#pragma unroll
    for (int p = 0; p < RUN; ++p) turned[d / D][p][d % D] = column[p];
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h >= heads) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = warp + 8 * (i % 2);
      if (p < run.lo || p >= run.hi) continue;
      X* to = static_cast<X*>(i < 2 ? a.k : a.v) + ((run.row + p) * a.kv_heads + head0 + h) * D;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int d = 4 * (lane + 32 * j);
        if (d >= D) continue;
        const Four four = i < 2 ? held[h][i % 2][j] : *reinterpret_cast<const Four*>(&turned[h][p][d]);
        const Code* codes = reinterpret_cast<const Code*>(&four);
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = CODES ? float(codes[e]) * scale[h][i] : float(codes[e]);
        store_four(to + d, x);
      }
    }
  }
}

#define DRIFT_CHUNKS_REGISTER(D)                                                                   \
  DRIFT_REGISTER(cache_write_chunks_i8_f32_d##D, (cache_write_chunks_kernel<D, float, int8_t>))           \
  DRIFT_REGISTER(cache_write_chunks_i8_bf16_d##D, (cache_write_chunks_kernel<D, __nv_bfloat16, int8_t>))  \
  DRIFT_REGISTER(cache_write_chunks_f16_f32_d##D, (cache_write_chunks_kernel<D, float, __half>))          \
  DRIFT_REGISTER(cache_write_chunks_f16_bf16_d##D, (cache_write_chunks_kernel<D, __nv_bfloat16, __half>)) \
  DRIFT_REGISTER(cache_read_chunks_i8_f32_d##D, (cache_read_chunks_kernel<D, float, int8_t>))             \
  DRIFT_REGISTER(cache_read_chunks_i8_bf16_d##D, (cache_read_chunks_kernel<D, __nv_bfloat16, int8_t>))    \
  DRIFT_REGISTER(cache_read_chunks_f16_f32_d##D, (cache_read_chunks_kernel<D, float, __half>))            \
  DRIFT_REGISTER(cache_read_chunks_f16_bf16_d##D, (cache_read_chunks_kernel<D, __nv_bfloat16, __half>))
DRIFT_CHUNKS_REGISTER(64)
DRIFT_CHUNKS_REGISTER(80)
DRIFT_CHUNKS_REGISTER(128)
DRIFT_CHUNKS_REGISTER(256)

// Blocks of 16 positions that a chunk of `longest` tokens can touch.
unsigned run_blocks(int longest) { return unsigned((longest + RUN - 2) / RUN + 1); }

template <int D>
int launch_write(const WriteArgs& a, int x_dtype, int cache_dtype, cudaStream_t stream) {
  const bool bf16 = x_dtype == DRIFT_BF16, codes = cache_dtype == DRIFT_I8;
  auto kernel = codes ? (bf16 ? cache_write_chunks_kernel<D, __nv_bfloat16, int8_t> : cache_write_chunks_kernel<D, float, int8_t>)
                      : (bf16 ? cache_write_chunks_kernel<D, __nv_bfloat16, __half> : cache_write_chunks_kernel<D, float, __half>);
  DRIFT_CUDA(launch_pdl(kernel, dim3(run_blocks(a.at.longest), a.kv_heads, a.at.batch), THREADS, 0, stream, a));
  DRIFT_LAUNCHED("cache_write_chunks");
  return 0;
}

template <int D>
int launch_read(const ReadArgs& a, int x_dtype, int cache_dtype, cudaStream_t stream) {
  const bool bf16 = x_dtype == DRIFT_BF16, codes = cache_dtype == DRIFT_I8;
  auto kernel = codes ? (bf16 ? cache_read_chunks_kernel<D, __nv_bfloat16, int8_t> : cache_read_chunks_kernel<D, float, int8_t>)
                      : (bf16 ? cache_read_chunks_kernel<D, __nv_bfloat16, __half> : cache_read_chunks_kernel<D, float, __half>);
  DRIFT_CUDA(launch_pdl(kernel, dim3(run_blocks(a.at.longest), (a.kv_heads + read_heads(D) - 1) / read_heads(D), a.at.batch), THREADS, 0, stream, a));
  DRIFT_LAUNCHED("cache_read_chunks");
  return 0;
}

}  // namespace

// The checks that the three calls share; `tokens` rows of x, `longest` of
// them in one chunk at most.
int check_chunks(const char* call, int x_dtype, long long tokens, int kv_heads, int head_dim, int cache_dtype,
                 const void* keys, const void* values, const float* key_scales, const float* value_scales,
                 int pages, int page_size, const int32_t* page_tables, int table_stride, const int32_t* starts,
                 const int32_t* positions, int batch, int longest) {
  if (x_dtype != DRIFT_F32 && x_dtype != DRIFT_BF16)
    return invalid("%s takes F32 (or BF16), not %s", call, dtype_name(x_dtype));
  if (cache_dtype != DRIFT_F16 && cache_dtype != DRIFT_I8)
    return invalid("%s: a cache of %s (F16 or I8)", call, dtype_name(cache_dtype));
  if (page_size <= 0 || page_size % 16 != 0) return invalid("pages of %d tokens: not a multiple of 16", page_size);
  if (head_dim != 64 && head_dim != 80 && head_dim != 128 && head_dim != 256)
    return invalid("%s: heads of %d (kernels take 64, 80, 128, 256)", call, head_dim);
  if (pages <= 0 || kv_heads <= 0 || kv_heads > 65535) return invalid("%s: a cache of %d pages, %d heads", call, pages, kv_heads);
  if (tokens < 0 || tokens > 0x7fffffffll || batch < 0 || batch > 65535 || longest < 0)
    return invalid("%s: %lld tokens of %d sequences, %d of one at most", call, tokens, batch, longest);
  // (positions are 32-bit numbers, and so is a page table's span)
  if (!page_tables || table_stride <= 0 || (long long)table_stride * page_size < longest ||
      (long long)table_stride * page_size > 0x7fffffffll - 1024)
    return invalid("a page table of %d pages for %d positions", table_stride, longest);
  if (tokens == 0 || batch == 0 || longest == 0) return 0;
  if (!starts || !positions || !keys || !values) return invalid("%s: a null tensor", call);
  if (cache_dtype == DRIFT_I8 && (!key_scales || !value_scales)) return invalid("%s: an 8-bit cache without scales", call);
  if ((reinterpret_cast<uintptr_t>(keys) | reinterpret_cast<uintptr_t>(values)) & 15)
    return invalid("%s: the cache does not start on a 16-byte boundary", call);
  if ((reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales)) & 15)
    return invalid("%s: the cache's scales do not start on a 16-byte boundary", call);
  return 0;
}

int check_rows_aligned(const char* call, const void* a, const void* b) {
  if (!a || !b) return invalid("%s: a null tensor", call);
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15)
    return invalid("%s: a tensor does not start on a 16-byte boundary", call);
  return 0;
}

}  // namespace drift

using namespace drift;

extern "C" {

int drift_cache_write_chunks(int x_dtype, const void* k, const void* v, int64_t tokens, int kv_heads,
                             int head_dim, int cache_dtype, void* keys, void* values, float* key_scales,
                             float* value_scales, int pages, int page_size, const int32_t* page_tables,
                             int table_stride, const int32_t* starts, const int32_t* positions, int batch,
                             int longest, drift_stream_t stream) {
  DRIFT_TRY(check_chunks("cacheWrite", x_dtype, tokens, kv_heads, head_dim, cache_dtype, keys, values, key_scales,
                         value_scales, pages, page_size, page_tables, table_stride, starts, positions, batch, longest));
  if (tokens == 0 || batch == 0 || longest == 0) return 0;
  DRIFT_TRY(check_rows_aligned("cacheWrite", k, v));
  const WriteArgs a = {{starts, positions, page_tables, tokens, table_stride, pages, page_size, batch, longest,
                        table_stride * page_size},
                       k, v, keys, values, key_scales, value_scales, kv_heads, device_error_word()};
  const cudaStream_t s = cudaStream_t(stream);
  switch (head_dim) {
    case 64: return launch_write<64>(a, x_dtype, cache_dtype, s);
    case 80: return launch_write<80>(a, x_dtype, cache_dtype, s);
    case 128: return launch_write<128>(a, x_dtype, cache_dtype, s);
    default: return launch_write<256>(a, x_dtype, cache_dtype, s);
  }
}

int drift_cache_read_chunks(int x_dtype, void* k, void* v, int64_t tokens, int kv_heads, int head_dim,
                            int cache_dtype, const void* keys, const void* values, const float* key_scales,
                            const float* value_scales, int pages, int page_size, const int32_t* page_tables,
                            int table_stride, const int32_t* starts, const int32_t* positions, int batch,
                            int longest, drift_stream_t stream) {
  DRIFT_TRY(check_chunks("cacheRead", x_dtype, tokens, kv_heads, head_dim, cache_dtype, keys, values, key_scales,
                         value_scales, pages, page_size, page_tables, table_stride, starts, positions, batch, longest));
  if (tokens == 0 || batch == 0 || longest == 0) return 0;
  DRIFT_TRY(check_rows_aligned("cacheRead", k, v));
  const ReadArgs a = {{starts, positions, page_tables, tokens, table_stride, pages, page_size, batch, longest,
                        table_stride * page_size},
                      keys, values, key_scales, value_scales, k, v, kv_heads, device_error_word()};
  const cudaStream_t s = cudaStream_t(stream);
  switch (head_dim) {
    case 64: return launch_read<64>(a, x_dtype, cache_dtype, s);
    case 80: return launch_read<80>(a, x_dtype, cache_dtype, s);
    case 128: return launch_read<128>(a, x_dtype, cache_dtype, s);
    default: return launch_read<256>(a, x_dtype, cache_dtype, s);
  }
}

}  // extern "C"

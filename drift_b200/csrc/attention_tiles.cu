// attention_chunks for chunks of many rows, on the tensor cores (tcgen05). A
// unit is a key head of one sequence with 128 MT of the (token, query head)
// rows that read it; a CTA takes one split of the unit's key tiles. Per tile
// of KEYS keys and tile i of 128 rows:
//
//   S_i = Q_i K^T      (TMEM; Q and K in shared memory)
//   P_i = e^(scale S_i - base)  beside S_i, as F16 (softmax warps: a thread
//                       has a row, its base and its sum, in F32)
//   O_i (+)= P_i V     (TMEM; V^T in shared memory, as the cache has it)
//
// The F16 cache's layouts are the tensor core's own K-major operands -- keys
// [..][D], values [D][..positions] -- so pages come straight into shared memory
// by TMA tensor copies, a page's run of 16, 32 or 64 positions at a time (the
// largest that divides the page): runs of keys are rows of the 128-byte
// swizzled tile, and a run of values is a tile of its own, in the swizzle as
// wide as the run. An 8-bit cache's codes come the same way into a buffer of
// their own, from which converting warps write them as F16 into the operands,
// exactly; a key's scale multiplies its scores, and a value's its weights, in
// F32 (BY_KEY). Where a chunk has several units of rows its codes come expanded to
// an F16 cache of the call's own (attention_expand.cu), with their scales by
// position (SCALED), or for BF16 rows with their scales in them where those are of
// like size. Values' scales are over a power of two, of all that some row sees
// (SCALED) or of those so far.
//
// Where scales are by key, a row's base is set by its largest product of weight
// and value scale, since that is what is rounded to F16: so its bits are its own,
// whatever scales the rows beside it see. (With codes converted over the largest
// scale, as was, a key's scale and its product were rounded one after the other,
// twice the error, and a hidden scale of 2^25 times the rest left a row no bits.)
//
// The order: Q K^T of the next tile is issued as soon as the softmax threads
// have taken S into registers, P V when P is there. So the tensor core works
// under the softmax and the softmax under the products, and what bounds a tile
// is the longer of the two: for D = 128 the tensor core's 16 + 10 products of
// 64 and 52 clocks for 80 keys and 256 rows. TMEM's 512 columns set the tile's
// keys: MT S, MT P, MT outputs. Measured: a chunk of 2048 BF16 tokens of 32 heads
// of 128 over 8192 keys 241 us, 1000 TFLOP/s, the special function unit (an
// exponential a score) and the tensor core each busy for 59 % of a full SM's time
// (51 % on average: 256 CTAs on 148 SMs); 1500 F32 tokens of 16 heads 71 us; 6000
// BF16 tokens of 8 heads of 64 under a window of 1024 52 us: 192 CTAs on 148 SMs, each 11 tiles, 4 of them at an edge, and its
// start and end (the exponentials are under half of it on an SM with two CTAs).
//
// BF16 rows (TERMS = 1): q is exact in F16 after a power of two per row; P's
// rounding to F16 (2^-11) is 1/8 of the result's own (2^-8). O stays in TMEM.
// A weight is at most 2^15 or the row's base moves: the sum of a tile's
// weights tells, so that a tile's largest score is looked for only then (and
// in the first tile, to set the base), and the weights made again and O
// rescaled. Looking for it in every tile took 27 % of a tile's softmax.
// F32 rows (TERMS = 2): q and P are two F16 terms each (hi + lo, to 2^-22), the
// products of both summed. The tensor core's F32 sums drop low bits as a chain
// grows, so a tile's P V starts a new O, and the softmax threads add it to
// their row's running output in registers.
//
// F32 rows of heads of 256 have a CTA for each half of the values' dimensions.
//
// MT = 2 (D <= 128) shares a tile's keys and values between two row tiles. MT =
// 1 (heads of 256, whose outputs fill TMEM, and units of 128 rows) has two S.
//
// Warps: first the softmax, four for 128 rows; then one for the copies, two for
// the tensor core (Q K^T, P V), and for an F16 cache one for the edges: in a
// tile that some row sees only in part it takes values that are not finite out
// of V, since such a value times a zero weight would reach rows that do not see it
// (they are added at the end, to the rows that do). A softmax warp passes over
// a tile that none of its rows sees. An 8-bit cache has
// converting warps. Every wait is bounded; one that gives up sets device error
// 2, and the CTA drains its copies and products, frees its TMEM and returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "chunks.cuh"
#include "common.cuh"
#include "registry.cuh"
#include "tc_common.cuh"
#include "tma_host.cuh"

namespace drift {

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr int ROW_TILE = 128;
constexpr uint32_t TMEM_COLUMNS = 512;
// A weight is 2^WEIGHT_BITS at the row's largest score when its base is set,
// and the base moves when a tile's weights sum to more than MOST_WEIGHT. F32
// rows: 2^WEIGHT_BITS_2, and it moves when one would pass 8 times that; a
// second term stops at F16's 2^-24, so a weight is off by 2^-37 of the largest
// (with 2^8 and a growth of 2^6 by 2^-33: 4e-5 of the result where an early
// key has ten times the weight of 65536 others, and no value).
constexpr float WEIGHT_BITS = 8.0f, MOST_WEIGHT = 32768.0f;
constexpr float WEIGHT_BITS_2 = 12.0f, MOST_BITS_2 = 15.0f;
// By key it is products that this holds for, and a bound of them (the largest
// score and the tile's largest scale) that moves a base: a little lower, so that
// the two's difference seldom does.
constexpr float WEIGHT_BITS_BY_KEY = 6.0f, WEIGHT_BITS_2_BY_KEY = 11.0f;
// A row of q is 2^Q_BITS and more at its largest value, so that its second
// terms end far below F16's last bit, 2^-24.
constexpr int Q_BITS = 8;

template <int D_, int KEYS_, int MT_, bool CODES_, int TERMS_, bool SCALED_>
struct TileTraits {
  static constexpr int D = D_, KEYS = KEYS_, MT = MT_, TERMS = TERMS_;
  // F32 rows of heads of 256: a CTA takes 128 of the values' dimensions (a row's
  // running output is in registers), and both make the weights
  static constexpr int DV = TERMS == 2 && D > 128 ? 128 : D, PARTS = D / DV;
  static constexpr bool CODES = CODES_, SCALED = SCALED_;  // SCALED: expanded codes
  static constexpr bool BY_KEY = CODES || SCALED;
  static constexpr int UNIT = ROW_TILE * MT;
  static constexpr int SOFTMAX_WARPS = 4 * MT;
  // Q K^T and P V have a warp each: a wait costs one about 100 clocks even when
  // there is nothing to wait for, and six of them and the products' issue were
  // longer than the products (for the codes of F32 rows they are not).
  static constexpr bool TWO_ISSUE = !(CODES && TERMS == 2);
  static constexpr int COPY_WARP = SOFTMAX_WARPS, QK_WARP = COPY_WARP + 1, PV_WARP = QK_WARP + TWO_ISSUE;
  static constexpr int EDGE_WARP = PV_WARP + 1, EDGE_THREADS = 32;
  // Converting codes for BF16 rows takes eight warps, two to a scheduler (with
  // one, latencies made a tile 6400 clocks long); for F32 rows, at half the
  // rate, two. The softmax warps take the registers that the others leave.
  static constexpr bool WIDE = CODES && TERMS == 1;
  static constexpr int CONVERT_WARP = WIDE ? EDGE_WARP + 1 : EDGE_WARP;
  static constexpr int CONVERT_THREADS = WIDE ? 256 : 64;
  static constexpr int THREADS = 32 * (SOFTMAX_WARPS + 4 + (WIDE ? 8 : 0));
  static constexpr bool MOVES_REGISTERS = MT == 2 || WIDE;  // (255 a thread are there otherwise)
  static constexpr int LAUNCH_REGISTERS = 65536 / THREADS / 8 * 8;
  static constexpr int OTHER_REGISTERS = TERMS == 2 ? 56 : !WIDE ? 88 : MT == 2 ? 48 : 88;
  static constexpr int SHARE =
      (THREADS * LAUNCH_REGISTERS - (THREADS - 32 * SOFTMAX_WARPS) * OTHER_REGISTERS) / (32 * SOFTMAX_WARPS) / 8 * 8;
  static constexpr int SOFTMAX_REGISTERS = SHARE > 232 ? 232 : SHARE;
  static constexpr int ROUND_THREADS = 32 * SOFTMAX_WARPS + EDGE_THREADS;
  static constexpr int PANELS = (D + 63) / 64;             // 64-column panels of a row
  static constexpr int Q_PANEL = ROW_TILE * 128;           // bytes
  static constexpr int Q_BYTES = PANELS * Q_PANEL;         // one term of one row tile
  static constexpr int K_PANEL = KEYS * 128;
  static constexpr int K_BYTES = PANELS * K_PANEL;
  static constexpr int V_BYTES = KEYS * DV * 2;
  static constexpr int V_STAGE = (V_BYTES + 1023) / 1024 * 1024;
  static constexpr int CODE_BYTES = KEYS * D;              // of one side of a tile
  static constexpr int CODE_STAGE = (CODE_BYTES + 127) / 128 * 128;
  static constexpr int K_AT = MT * TERMS * Q_BYTES;
  // what the copies fill: the operands, or codes, twice where that fits; and
  // the operands three times where that does (a copy's 1400 clocks from when
  // its stage is free are a tile's time)
  static constexpr int SCALE_ROWS = TERMS == 1 ? 2 : 3;    // the keys', the values' and (there is room) their logarithms
  static constexpr int bytes_of(int stages, int code_stages) {
    return K_AT + stages * (K_BYTES + V_STAGE) + (CODES ? code_stages * 2 * CODE_STAGE : 0) +
           (CODES ? stages * SCALE_ROWS * KEYS * 4 + code_stages * 2 * KEYS * 4 : 0) +
           (SCALED ? SOFTMAX_WARPS * KEYS * 4 : 0) + 384;
  }
  static constexpr int LIMIT = 232448;
  static constexpr int CODE_STAGES = bytes_of(2, 2) <= LIMIT ? 2 : 1;
  static constexpr int STAGES = bytes_of(3, CODE_STAGES) <= LIMIT ? 3 : 2;
  static constexpr int COPY_STAGES = CODES ? CODE_STAGES : STAGES;
  static constexpr int V_AT = K_AT + STAGES * K_BYTES;
  static constexpr int CODES_AT = V_AT + STAGES * V_STAGE;  // [COPY_STAGES][2]
  static constexpr int SCALES_AT = CODES_AT + (CODES ? COPY_STAGES * 2 * CODE_STAGE : 0);  // [STAGES][SCALE_ROWS][KEYS]
  static constexpr int COPIED_SCALES_AT = SCALES_AT + (CODES ? STAGES * SCALE_ROWS * KEYS * 4 : 0);  // [COPY_STAGES][2][KEYS]
  static constexpr int WARP_SCALES_AT = COPIED_SCALES_AT + (CODES ? COPY_STAGES * 2 * KEYS * 4 : 0);  // [SOFTMAX_WARPS][KEYS]
  static constexpr int BARRIERS_AT = WARP_SCALES_AT + (SCALED ? SOFTMAX_WARPS * KEYS * 4 : 0);
  static constexpr int BYTES = BARRIERS_AT + 384;  // 38 barriers and a few words
  // TMEM: S of row tile i, or (MT = 1) of every other tile; P and O of row tile i
  static constexpr int S_COLUMNS = (KEYS + 31) / 32 * 32;
  static constexpr int P_COLUMN = S_COLUMNS + KEYS, P_COLUMNS = TERMS * KEYS / 2;
  static constexpr int O_COLUMN = int(TMEM_COLUMNS) - MT * ((DV + 31) / 32 * 32), O_COLUMNS = (DV + 31) / 32 * 32;
  static_assert(P_COLUMN + MT * P_COLUMNS <= O_COLUMN, "TMEM");
  static_assert(KEYS % 16 == 0 && KEYS <= 128 && P_COLUMN % 8 == 0, "whole steps");
  static_assert(TERMS == 1 || (DV <= 128 && KEYS == 64), "the running output of a row in registers");
  static_assert(BYTES <= LIMIT, "shared memory");
};

template <int REGISTERS>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGISTERS));
}
template <int REGISTERS>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGISTERS));
}

// K-major operand rows of 32, 64 or 128 bytes in the swizzle of that width,
// 8-row groups apart by eight rows.
__device__ __forceinline__ uint64_t operand_desc(uint32_t address, uint32_t row_bytes) {
  uint64_t d = uint64_t((address >> 4) & 0x3fff);
  d |= uint64_t(1) << 16;
  d |= uint64_t((8 * row_bytes) >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(row_bytes == 128 ? 2 : row_bytes == 64 ? 4 : 6) << 61;
  return d;
}

__device__ __forceinline__ void mma_ss_warp(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

// 32 columns of this thread's lane; the values are there after tmem_load_wait.
__device__ __forceinline__ void tmem_load_32_async(uint32_t address, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void tmem_load_16_async(uint32_t address, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(address)
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store_8(uint32_t address, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(address),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_load_8_async(uint32_t address, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(address)
               : "memory");
}
__device__ __forceinline__ void tmem_store_4(uint32_t address, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
// N columns of this thread's lane, in as few instructions as there are.
template <int N>
__device__ __forceinline__ void tmem_load_async(uint32_t address, float* v) {
  if constexpr (N >= 32) {
    tmem_load_32_async(address, v);
    if constexpr (N > 32) tmem_load_async<N - 32>(address + 32, v + 32);
  } else if constexpr (N >= 16) {
    tmem_load_16_async(address, v);
    if constexpr (N > 16) tmem_load_async<N - 16>(address + 16, v + 16);
  } else {
    static_assert(N == 8, "columns by eights");
    tmem_load_8_async(address, v);
  }
}
__device__ __forceinline__ void tmem_load_16(uint32_t address, float* v) {
  tmem_load_16_async(address, v);
  tmem_load_wait();
}
__device__ __forceinline__ void tmem_store_16(uint32_t address, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(address),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_store(uint32_t address, const uint32_t* r) {
  if constexpr (N >= 16) {
    tmem_store_16(address, r);
    if constexpr (N > 16) tmem_store<N - 16>(address + 16, r + 16);
  } else if constexpr (N >= 8) {
    tmem_store_8(address, r);
    if constexpr (N > 8) tmem_store<N - 8>(address + 8, r + 8);
  } else {
    static_assert(N == 4, "columns by fours");
    tmem_store_4(address, r);
  }
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The largest of three, a NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Pairs: one instruction for two F32 operations.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// What F16 leaves of a pair.
__device__ __forceinline__ uint32_t left_pair(float a, float b, uint32_t pair) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&pair));
  return half_pair(a - h.x, b - h.y);
}

// Four codes as two pairs of F16: a byte u = code + 128 under the exponent of
// 1024 is 1024 + u, less 1152.
__device__ __forceinline__ uint2 code_pairs(uint32_t codes) {
  const uint32_t u = codes ^ 0x80808080u;
  const __half2 less = __half2half2(__ushort_as_half(0x6480));  // 1152
  uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), less);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), less);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// softcap tanh(y): near zero y times a polynomial in its square (least squares
// on Chebyshev points of |y| <= NEAR, reweighted towards the least largest
// relative error, 1e-9), farther off 1 - 2 / (1 + e^(2 y)). The cut is where
// tanh is 1/2: from there on the difference is no smaller than what is taken from
// 1, and loses one bit at most.
constexpr float NEAR = 0.55f;
__device__ __forceinline__ float capped_near(float y) {
  const float u = y * y;
  float p = fmaf(u, -0.006235556676983833f, 0.021039674058556557f);
  p = fmaf(u, p, -0.053842708468437195f);
  p = fmaf(u, p, 0.13332460820674896f);
  p = fmaf(u, p, -0.3333331048488617f);
  return fmaf(y * u, p, y);
}
__device__ __forceinline__ float capped_far(float y) {
  return 1.0f - __fdividef(2.0f, 1.0f + exp2_approx(2.0f * LOG2E * y));
}

struct TileArgs {
  AttentionChunksArgs a;
  int run;  // positions a copy takes of a page: 16, 32 or 64
};

template <class T>
__global__ void __launch_bounds__(T::THREADS, 1)
attention_tiles_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                       const TileArgs args) {
  constexpr int D = T::D, DV = T::DV, KEYS = T::KEYS, MT = T::MT, TERMS = T::TERMS, STAGES = T::STAGES;
  constexpr bool CODES = T::CODES, SCALED = T::SCALED, BY_KEY = T::BY_KEY;
  using X = typename std::conditional<TERMS == 1, __nv_bfloat16, float>::type;
  pdl_trigger();  // the next kernel may launch and wait for this one
  pdl_wait();     // what the kernels before this one wrote is visible
  const AttentionChunksArgs& a = args.a;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int head = blockIdx.x / T::PARTS, part = blockIdx.x % T::PARTS, z = blockIdx.y;
  // the last rows first: under a causal mask they see the most keys
  const int at = gridDim.z - 1 - blockIdx.z, split = at % a.splits, unit = at / a.splits;
  const Chunk chunk(a.at, z);
  if (!chunk.ok && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) chunk_error(a.error);
  const int row0 = unit * T::UNIT, row1 = min(row0 + T::UNIT, chunk.tokens * a.group);
  if (row0 >= row1) return;
  const int token0 = row0 / a.group, token1 = (row1 - 1) / a.group + 1;
  const SeenTiles seen(a, chunk, token0, token1, KEYS);
  const int tile0 = split * a.tiles_per_split, tile1 = min(tile0 + a.tiles_per_split, seen.count);
  if (tile0 >= tile1) return;
  const int tiles = tile1 - tile0;
  // (BF16 rows' expanded codes: those of a head whose scales are by key are the
  // SCALED launch's, the others' the F16 cache's)
  float4 units = make_float4(1.0f, 1.0f, 0.0f, 0.0f);
  if (!CODES && a.units) {
    units = a.units[(long long)z * a.kv_heads + head];
    if (SCALED != (units.z != 0.0f)) return;
  }
  // what some row sees: keys below seen.end that are `lowest` or later or
  // below `first`; what every row sees: below all_end, from all_low on (or
  // below `first`)
  const int first = a.window > 0 ? a.first : 0;
  const int lowest = a.window > 0 ? chunk.position + token0 - a.window + 1 : 0;
  const int all_end = a.causal ? chunk.position + token0 + 1 : seen.end;
  const int all_low = a.window > 0 ? chunk.position + token1 - a.window : 0;
  auto whole = [&](int key0) { return key0 + KEYS <= all_end && (key0 >= all_low || key0 + KEYS <= first); };

  extern __shared__ __align__(1024) uint8_t shared[];
  const uint32_t base = tc::smem_u32(shared);
  if (base & 1023) {  // (the operands' swizzles want it; a kernel without static shared memory has it)
    if (tid == 0 && a.error) atomicCAS(a.error, 0, 2);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(shared + T::BARRIERS_AT);
  uint64_t* q_full = bars;             // [2]
  uint64_t* k_full = bars + 2;         // [STAGES] each
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* scales_full = v_empty + STAGES;
  uint64_t* s_full = scales_full + STAGES;  // [2]: of row tile i, or of buffer i
  uint64_t* s_empty = s_full + 2;           // [2]
  uint64_t* p_full = s_empty + 2;           // [2]: of row tile i
  uint64_t* pv_done = p_full + 2;           // [2]: P is read, O written
  uint64_t* edge_found = pv_done + 2;       // [2] each, of every other edge tile (two may be under way):
  uint64_t* edge_clean = edge_found + 2;    // its values are there; they are clean
  uint64_t* codes_full = edge_clean + 2;    // [COPY_STAGES][2]: of the keys, of the values
  uint64_t* codes_empty = codes_full + 4;   // [COPY_STAGES][2]
  uint64_t* drained = codes_empty + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* taken_out = abort + 1;
  volatile int* copied = abort + 2;         // [2]: tiles whose keys, values were asked for
  volatile float* v_unit = reinterpret_cast<volatile float*>(abort + 4);  // [STAGES]: what values' scales are over,
  volatile float* v_most = v_unit + STAGES;                               // and the largest of a tile's
  float* scales = reinterpret_cast<float*>(shared + T::SCALES_AT);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&q_full[i], ROW_TILE);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&s_empty[i], ROW_TILE);
      tc::mbar_init(&p_full[i], ROW_TILE);
      tc::mbar_init(&pv_done[i], 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      tc::mbar_init(&k_full[s], CODES ? T::CONVERT_THREADS : 1);
      tc::mbar_init(&k_empty[s], 1);
      tc::mbar_init(&v_full[s], CODES ? T::CONVERT_THREADS : 1);
      tc::mbar_init(&v_empty[s], 1);
      tc::mbar_init(&scales_full[s], T::CONVERT_THREADS);
    }
    for (int s = 0; s < 4; ++s) {
      tc::mbar_init(&codes_full[s], 1);
      tc::mbar_init(&codes_empty[s], T::CONVERT_THREADS);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&edge_found[i], 1);
      tc::mbar_init(&edge_clean[i], T::EDGE_THREADS);
    }
    tc::mbar_init(drained, 1 + T::TWO_ISSUE);
    *abort = 0;
    *taken_out = 0;
    copied[0] = copied[1] = 0;
    tc::fence_barrier_init();
  }
  __syncwarp();
  if (warp == 0) tc::tmem_alloc(tmem_slot, TMEM_COLUMNS);
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return tc::mbar_wait_warp(bar, parity, abort, a.error); };

  if constexpr (T::MOVES_REGISTERS) {
    if (warp < T::SOFTMAX_WARPS) more_registers<T::SOFTMAX_REGISTERS>();
    else fewer_registers<T::OTHER_REGISTERS>();
  }

  if (warp < T::SOFTMAX_WARPS) {
    // ---- softmax: this thread's row of row tile i --------------------------------------
    const int i = warp / 4, r = tid % ROW_TILE, row = row0 + ROW_TILE * i + r;
    const bool real = row < row1;
    const int token = (real ? row : row1 - 1) / a.group, q_head = head * a.group + row % a.group;
    const uint32_t lanes = uint32_t(32 * (warp % 4)) << 16;
    const long long row_at = (chunk.row + token) * a.q_heads + q_head;
    // q, divided by a power of two (and by the scale's sign), into the
    // swizzled panels of its terms: a warp takes its 32 rows, a few at a time,
    // a lane eight values of one
    float multiplier;
    const uint32_t group_magic = a.group > 1 ? 0xffffffffu / uint32_t(a.group) + 1 : 0;  // (2^32 / group, up)
    {
      constexpr int CHUNKS = D / 8, LANES = CHUNKS <= 8 ? 8 : CHUNKS <= 16 ? 16 : 32;  // of a row
      constexpr int AT_ONCE = 32 / LANES, PASSES = LANES, FLIGHT = TERMS == 2 ? 4 : 8;
      const int c = lane % LANES, part = lane / LANES;
      const int tile_row0 = row0 + ROW_TILE * i + 32 * (warp % 4);
      const int tile_token0 = tile_row0 / a.group, tile_head0 = tile_row0 % a.group;
      // (rows past the unit's are zeros, and so are the last panel's columns past D)
      auto load = [&](int pass, uint4 (&x)[TERMS]) {
        const int from = tile_row0 + pass * AT_ONCE + part;
#pragma unroll
        for (int n = 0; n < TERMS; ++n) x[n] = make_uint4(0, 0, 0, 0);
        if (c >= CHUNKS || from >= row1) return;
        // (row x's token past the first: x below 48 over at most 16, exactly)
        const int x_row = tile_head0 + pass * AT_ONCE + part, tokens = a.group > 1 ? int(__umulhi(x_row, group_magic)) : x_row;
        const X* q = static_cast<const X*>(a.q) +
                     ((chunk.row + tile_token0 + tokens) * a.q_heads + head * a.group + x_row - tokens * a.group) * D + 8 * c;
#pragma unroll
        for (int n = 0; n < TERMS; ++n) x[n] = reinterpret_cast<const uint4*>(q)[n];
      };
      multiplier = 0.0f;
#pragma unroll 1
      for (int pass0 = 0; pass0 < PASSES; pass0 += FLIGHT) {
        uint4 held[FLIGHT][TERMS];
#pragma unroll
        for (int n = 0; n < FLIGHT; ++n) load(pass0 + n, held[n]);
#pragma unroll
        for (int n = 0; n < FLIGHT; ++n) {
          float x[8];
          const uint32_t* w = reinterpret_cast<const uint32_t*>(held[n]);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = __uint_as_float(TERMS == 2 ? w[e % (4 * TERMS)] : e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
          float largest = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(x[e]));
#pragma unroll
          for (int o = 1; o < LANES; o *= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
          // 2^(floor(log2 largest) - Q_BITS), kept where it and its inverse
          // are normal (NaNs and infinities stay what they are)
          constexpr uint32_t SHIFT = uint32_t(Q_BITS) << 23;
          const uint32_t exponent = max(__float_as_uint(largest) & 0x7f800000u, SHIFT + 0x01000000u) - SHIFT;
          const float unit_inverse = __uint_as_float(0x7f000000u - exponent);
          const float by = a.scale < 0.0f ? -unit_inverse : a.scale > 0.0f ? unit_inverse : 0.0f;
          const int pass = pass0 + n;
          const uint32_t own = __shfl_sync(0xffffffffu, exponent, lane % AT_ONCE * LANES);
          if (lane / AT_ONCE == pass) multiplier = fabsf(a.scale) * __uint_as_float(own);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= by;
          const uint4 hi = make_uint4(half_pair(x[0], x[1]), half_pair(x[2], x[3]), half_pair(x[4], x[5]), half_pair(x[6], x[7]));
          const int to_row = 32 * (warp % 4) + pass * AT_ONCE + part;
          if (c < T::PANELS * 8) {
            uint8_t* to = shared + i * TERMS * T::Q_BYTES + to_row * 128 + c / 8 * T::Q_PANEL + 16 * ((c % 8) ^ (to_row % 8));
            *reinterpret_cast<uint4*>(to) = hi;
            if constexpr (TERMS == 2)
              *reinterpret_cast<uint4*>(to + T::Q_BYTES) =
                  make_uint4(left_pair(x[0], x[1], hi.x), left_pair(x[2], x[3], hi.y), left_pair(x[4], x[5], hi.z),
                             left_pair(x[6], x[7], hi.w));
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(&q_full[i]);
    }
    const float value_unit = units.x;
    multiplier *= units.y;
    // (a softcap leaves natural units behind; and never zero, which a hidden
    // score of -infinity may not meet: with a scale of zero it is q that is)
    const float m2 = a.softcap > 0.0f ? LOG2E : fmaxf(multiplier * LOG2E, 1.17549435e-38f);
    const int position = chunk.position + token;
    const int hi = a.causal ? position + 1 : seen.end;
    // (not below 0: a window of no limit less a key's position is past 32 bits)
    const int lo = a.window > 0 ? max(position - a.window + 1, 0) : 0;
    // what all of this warp's rows see (from `all_low` to `all_end`, and below
    // `first`), and what some row sees
    const int warp_row0 = row0 + ROW_TILE * i + 32 * (warp % 4), warp_row1 = min(warp_row0 + 32, row1);
    const int token_first = chunk.position + warp_row0 / a.group, token_last = chunk.position + max(warp_row1 - 1, 0) / a.group;
    const int all_end = a.causal ? token_first + 1 : seen.end, some_end = a.causal ? token_last + 1 : seen.end;
    const int all_low = a.window > 0 ? token_last - a.window + 1 : 0, some_low = a.window > 0 ? token_first - a.window + 1 : 0;
    const uint32_t o_at = tmem + lanes + T::O_COLUMN + i * T::O_COLUMNS, p_at = tmem + lanes + T::P_COLUMN + i * T::P_COLUMNS;

    float base2 = -INFINITY, sum = 0.0f;  // weights are 2^(score in base 2 - base2)
    float unit = 0.0f;                    // and, for codes, values' scales are over this
    float total[TERMS == 2 ? DV : 1] = {};  // the running output (F32 rows)
    // the last tile's output, which the tensor core has left in O
    auto take_output = [&]() {
      if constexpr (TERMS == 2) {
#pragma unroll
        for (int c = 0; c < DV; c += 16) {
          float o[16];
          tmem_load_16(o_at + c, o);
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float2 x = add2(make_float2(total[c + e], total[c + e + 1]), make_float2(o[e], o[e + 1]));
            total[c + e] = x.x, total[c + e + 1] = x.y;
          }
        }
      }
    };
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      const int b = MT == 2 ? i : j & 1, stage = j % STAGES;
      // (expanded codes' scales, and the largest of the values', off the way)
      constexpr int HELD = (KEYS + 31) / 32;  // a lane has of a tile (reads up to 31 past it)
      float held_k[HELD], held_v[HELD], most_scale = 1.0f;
      if constexpr (SCALED) {
        const long long at = ((long long)z * a.kv_heads + head) * a.at.table_stride * a.at.page_size + seen.key_of(tile0 + j) + lane;
#pragma unroll
        for (int n = 0; n < HELD; ++n) held_k[n] = a.key_scales[at + 32 * n], held_v[n] = a.value_scales[at + 32 * n];
        uint32_t most = 0;  // (what is past the last key may be anything)
#pragma unroll
        for (int n = 0; n < HELD; ++n)
          if (__float_as_uint(held_v[n]) <= 0x3f800000u) most = max(most, __float_as_uint(held_v[n]));
        most_scale = __uint_as_float(__reduce_max_sync(0xffffffffu, most));
      }
      if (!(ok = wait(&s_full[b], MT == 2 ? j & 1 : (j >> 1) & 1))) break;
      // P and O are free (and O complete) when the last tile's P V is done
      auto settled = [&]() {
        if (j == 0) return true;
        if (!wait(&pv_done[i], (j - 1) & 1)) return false;
        tc::fence_after_sync();
        return true;
      };
      const int key0 = seen.key_of(tile0 + j);
      if (warp_row0 >= row1 || key0 >= some_end || (key0 + KEYS <= some_low && key0 >= first)) {
        // no row of the warp sees the tile: weights of zero
        tc::mbar_arrive(&s_empty[b]);
        if (!(ok = settled())) break;
        if (TERMS == 2 && j > 0) take_output();
        const uint32_t zeros[8] = {};
#pragma unroll
        for (int c = 0; c < T::P_COLUMNS; c += 8) tmem_store_8(p_at + c, zeros);
        tc::tmem_store_wait();
        tc::fence_before_sync();
        tc::mbar_arrive(&p_full[i]);
        continue;
      }
      if (CODES && !(ok = wait(&scales_full[stage], (j / STAGES) & 1))) break;
      tc::fence_after_sync();
      float s[KEYS];
      tmem_load_async<KEYS>(tmem + lanes + b * T::S_COLUMNS, s);
      tmem_load_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(&s_empty[b]);

      // (expanded codes' scales: one kind after the other in a row of the warp's own)
      float* warp_scales = reinterpret_cast<float*>(shared + T::WARP_SCALES_AT) + warp * KEYS;
      const float* k_scales = SCALED ? warp_scales : scales + stage * T::SCALE_ROWS * KEYS;
      const float* v_scales = SCALED ? warp_scales : k_scales + KEYS;
      const float* logarithms = SCALED ? warp_scales : v_scales + KEYS;
      auto share = [&](const float (&x)[HELD]) {
        __syncwarp();  // (what it held before is read)
#pragma unroll
        for (int n = 0; n < HELD; ++n)
          if (KEYS % 32 == 0 || lane + 32 * n < KEYS) warp_scales[lane + 32 * n] = x[n];
        __syncwarp();
      };
      if constexpr (SCALED) share(held_k);
      const float now_unit = CODES ? float(v_unit[stage]) : 0.0f;
      if constexpr (BY_KEY) {
#pragma unroll
        for (int c = 0; c < KEYS; c += 4) {
          const float4 x = *reinterpret_cast<const float4*>(k_scales + c);
          const float2 u = mul2(make_float2(s[c], s[c + 1]), make_float2(x.x, x.y));
          const float2 v = mul2(make_float2(s[c + 2], s[c + 3]), make_float2(x.z, x.w));
          s[c] = u.x, s[c + 1] = u.y, s[c + 2] = v.x, s[c + 3] = v.y;
        }
      }
      if (a.softcap > 0.0f) {
        // (where no score of the warp's rows is far from zero, the usual case,
        // the far form's two special functions a score are left out: of 1500 F32
        // rows of 16 heads, 98 us with them)
        const float inverse = multiplier / a.softcap;
        float far = 0.0f;
#pragma unroll
        for (int c = 0; c < KEYS; c += 2) far = max3(far, fabsf(s[c]), fabsf(s[c + 1]));
        if (__any_sync(0xffffffffu, !(far * fabsf(inverse) <= NEAR))) {
#pragma unroll
          for (int c = 0; c < KEYS; ++c) {
            const float y = s[c] * inverse;
            s[c] = a.softcap * (fabsf(y) <= NEAR ? capped_near(y) : capped_far(y));
          }
        } else {
#pragma unroll
          for (int c = 0; c < KEYS; ++c) s[c] = a.softcap * capped_near(s[c] * inverse);
        }
      }
      const bool edge = !(key0 + KEYS <= all_end && (key0 >= all_low || key0 + KEYS <= first));
      if (edge) {
        // a bit for each key that the row sees
        auto below = [](int n) { return n <= 0 ? 0u : 0xffffffffu >> max(32 - n, 0); };
#pragma unroll
        for (int c = 0; c < KEYS; c += 32) {
          const int at = key0 + c;
          const uint32_t sees = below(hi - at) & (~below(lo - at) | below(first - at));
#pragma unroll
          for (int e = 0; e < 32 && c + e < KEYS; ++e)
            if (!(sees >> e & 1)) s[c + e] = -INFINITY;
        }
      }
      // the row's base from this tile's largest score (BY_KEY: its largest
      // product's logarithm), and what is summed in it
      bool not_a_number = false;
      auto rebase = [&](float top) {
        not_a_number = top != top;
        float g = 1.0f;
        if constexpr (CODES) {
          if (now_unit > unit) {
            // values' scales are over 2^over times as much: as products stay
            // what they are, the base falls and the weights' sum grows, as far
            // as it has room (the outputs take the rest)
            if (unit > 0.0f) {
              const int over = (__float_as_int(now_unit) - __float_as_int(unit)) >> 23;
              const int falls = min(over, max(227 - (__float_as_int(sum) >> 23), 0));
              base2 -= float(falls);
              sum = ldexpf(sum, falls);
              g = exp2f(float(falls - over));
            }
            unit = now_unit;
          }
        }
        // (a row without a base takes one; a base that is too high stays)
        constexpr float BITS = TERMS == 2 ? (BY_KEY ? WEIGHT_BITS_2_BY_KEY : WEIGHT_BITS_2) : BY_KEY ? WEIGHT_BITS_BY_KEY : WEIGHT_BITS;
        const float now = fmaxf(base2, top - BITS);
        const float f = base2 == -INFINITY ? 0.0f : exp2f(base2 - now);
        g *= f;
        base2 = now;
        sum *= f;
        if constexpr (TERMS == 2) {
#pragma unroll
          for (int c = 0; c < DV; ++c) total[c] *= g;
        } else if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < DV; c += 16) {
            float o[16];
            tmem_load_16(o_at + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= g;
            tmem_store_16(o_at + c, reinterpret_cast<const uint32_t*>(o));
          }
        }
      };
      auto largest_score = [&]() {
        float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < KEYS - 4; c += 8)
#pragma unroll
          for (int n = 0; n < 4; ++n) tops[n] = max3(tops[n], s[c + 2 * n], s[c + 2 * n + 1]);
#pragma unroll
        for (int n = 0; n < 4; ++n) tops[n] = max3(tops[n], tops[n], s[KEYS - 4 + n]);
        return max3(tops[0], tops[1], max3(tops[2], tops[2], tops[3])) * m2;
      };
      // by key: of a product. (NaNs do not count: a hidden key's scale may be one,
      // and a score that is makes its row NaNs by its weight.)
      auto largest_product = [&]() {
        if constexpr (SCALED) {
          float x[HELD];
#pragma unroll
          for (int n = 0; n < HELD; ++n) x[n] = logarithm(held_v[n]);
          share(x);
        }
        float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < KEYS; c += 4) {
          float4 l;
          if constexpr (SCALED || T::SCALE_ROWS == 3) l = *reinterpret_cast<const float4*>(logarithms + c);
          else l = make_float4(logarithm(v_scales[c]), logarithm(v_scales[c + 1]), logarithm(v_scales[c + 2]), logarithm(v_scales[c + 3]));
          const float2 x = fma2(make_float2(s[c], s[c + 1]), make_float2(m2, m2), make_float2(l.x, l.y));
          const float2 y = fma2(make_float2(s[c + 2], s[c + 3]), make_float2(m2, m2), make_float2(l.z, l.w));
          tops[0] = fmaxf(tops[0], fmaxf(x.x, x.y)), tops[1] = fmaxf(tops[1], fmaxf(y.x, y.y));
        }
        return fmaxf(tops[0], tops[1]);
      };
      if constexpr (CODES) most_scale = v_most[stage];
      uint32_t p[KEYS / 2], p_low[TERMS == 2 ? KEYS / 2 : 1];
      // the weights and their sum (a tile's own: short chains)
      auto weigh = [&]() {
        // (a NaN makes the whole row NaNs)
        const float less = not_a_number ? __int_as_float(0x7fc00000) : base2 == -INFINITY ? 0.0f : -base2;
        float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int e = 0; e < KEYS / 2; e += 2) {
          float4 by;
          if constexpr (BY_KEY) by = *reinterpret_cast<const float4*>(v_scales + 2 * e);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float s0 = s[2 * (e + n)], s1 = s[2 * (e + n) + 1];
            float2 w = fma2(make_float2(s0, s1), make_float2(m2, m2), make_float2(less, less));
            w = make_float2(exp2_approx(w.x), exp2_approx(w.y));
            part = add2(part, w);
            if constexpr (BY_KEY) {
              w = mul2(w, n == 0 ? make_float2(by.x, by.y) : make_float2(by.z, by.w));
              if (edge) {  // (a hidden value's scale may be a NaN)
                w.x = s0 == -INFINITY ? 0.0f : w.x;
                w.y = s1 == -INFINITY ? 0.0f : w.y;
              }
            }
            p[e + n] = half_pair(w.x, w.y);
            if constexpr (TERMS == 2) p_low[e + n] = left_pair(w.x, w.y, p[e + n]);
          }
        }
        return part.x + part.y;
      };
      if constexpr (TERMS == 2) {
        if (!(ok = settled())) break;
        if (j > 0) take_output();
        // (no product is past its weight times the tile's largest scale)
        float top = largest_score();
        if constexpr (BY_KEY) top += logarithm(most_scale);
        const bool grown = !(top <= base2 + MOST_BITS_2) || (CODES && now_unit > unit);
        if (__any_sync(0xffffffffu, grown)) {
          if constexpr (BY_KEY) top = largest_product();
          rebase(top);
        }
        if constexpr (SCALED) share(held_v);
        sum += weigh();
      } else {
        // the bases stay unless a weight might not fit; in the first tile, and
        // where a row without one sees keys, they are set
        bool slow = j == 0;
        if constexpr (SCALED) share(held_v);
        float part = 0.0f;
        if (!slow) {
          part = weigh();
          const bool sees = key0 < hi && (key0 + KEYS > lo || key0 < first);
          const bool over = !(part * most_scale <= MOST_WEIGHT) || (base2 == -INFINITY && sees) ||
                            (CODES && now_unit > unit);
          slow = __any_sync(0xffffffffu, over);
        }
        if (!(ok = settled())) break;
        if (slow) {
          rebase(BY_KEY ? largest_product() : largest_score());
          if constexpr (SCALED) share(held_v);
          part = weigh();
        }
        sum += part;
      }
      tmem_store<KEYS / 2>(p_at, p);
      if constexpr (TERMS == 2) tmem_store<KEYS / 2>(p_at + KEYS / 2, p_low);
      tc::tmem_store_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(&p_full[i]);
    }
    if (ok) ok = wait(&pv_done[i], (tiles - 1) & 1);
    float all_sum = sum;
    if constexpr (!CODES) asm volatile("bar.sync 1, %0;" ::"n"(T::ROUND_THREADS) : "memory");  // (taken_out is final)
    if (ok) {
      tc::fence_after_sync();
      take_output();
      // (two factors: what values are over may be at either end of F32's range)
      const float over = CODES ? unit : value_unit;  // (an F16 cache's is 1)
      float scale = 1.0f;
      if (!a.part_o) {
        if (a.sinks) {
          // the sink's weight in the row's units, or the row's in the sink's
          const float sink = a.sinks[q_head] * LOG2E, all = fmaxf(base2, sink);
          const float f = base2 == -INFINITY ? 0.0f : exp2f(base2 - all);
          all_sum = all_sum * f + exp2f(sink - all);
          scale = f;
        }
        scale = all_sum != 0.0f ? scale / all_sum : 0.0f;
      } else {
        // (BY_KEY over 2^15: products up to that, times what values are over, may pass F32's range)
        constexpr float PART_BITS = BY_KEY ? 15.0f : 0.0f;
        scale = BY_KEY ? 1.0f / 32768.0f : 1.0f;
        if (real && part == 0)
          *reinterpret_cast<float2*>(a.part_ml + (row_at * a.splits + split) * 2) =
              make_float2((base2 + PART_BITS) * LN2, all_sum * scale);
      }
      // PIECE dimensions of every row at a time, through this warp's part of the
      // row tile's q (which no product reads any more): a row to a thread goes
      // in, a row to neighbouring threads comes out
      constexpr int PIECE = DV % 32 == 0 && ROW_TILE * 144 <= TERMS * T::Q_BYTES ? 32 : 16;
      const bool wide = TERMS == 2 || a.part_o;
      const int size = wide ? 4 : 2, pitch = PIECE * size + 16;
      const long long row_bytes = (a.part_o ? (long long)a.splits : 1ll) * D * size;
      uint8_t* out = a.part_o ? reinterpret_cast<uint8_t*>(a.part_o + (long long)split * D) : static_cast<uint8_t*>(a.out);
      out += part * DV * size;
      uint8_t* stage = shared + i * TERMS * T::Q_BYTES + 32 * (warp % 4) * pitch;
      static_assert(ROW_TILE * (PIECE * 4 + 16) <= TERMS * T::Q_BYTES, "a piece of every row");
      const int lanes_to_row = PIECE * size / 16, at_once = 32 / lanes_to_row;  // 2 to 8, 16 to 4
      const int tile_row0 = row0 + ROW_TILE * i + 32 * (warp % 4);
      const int tile_token0 = tile_row0 / a.group, tile_head0 = tile_row0 % a.group;
#pragma unroll
      for (int c = 0; c < DV; c += PIECE) {
        float o[PIECE];
        if constexpr (TERMS == 2) {
#pragma unroll
          for (int e = 0; e < PIECE; ++e) o[e] = total[c + e];
        } else {
          tmem_load_async<PIECE>(o_at + c, o);
          tmem_load_wait();
        }
#pragma unroll
        for (int e = 0; e < PIECE; ++e) o[e] = o[e] * scale * over;
        if (!BY_KEY && *taken_out && real) {
#pragma unroll 1
          for (int j = 0; j < tiles; ++j) {
            const int key0 = seen.key_of(tile0 + j);
            if (whole(key0)) continue;
            const int end = min(key0 + KEYS, hi);
#pragma unroll
            for (int e = 0; e < PIECE; e += 4) {
              const float4 y = not_finite(static_cast<const __half*>(a.values) + ((long long)head * D + part * DV + c + e) * a.at.page_size,
                                          (long long)a.kv_heads * D * a.at.page_size, chunk.table, a.at.pages,
                                          a.at.page_size, key0, end, lo, first);
              o[e] += y.x, o[e + 1] += y.y, o[e + 2] += y.z, o[e + 3] += y.w;
            }
          }
        }
        __syncwarp();  // (the piece before is out of the way)
        uint8_t* own = stage + lane * pitch;
        if (wide) {
#pragma unroll
          for (int e = 0; e < PIECE; e += 4)
            *reinterpret_cast<float4*>(own + 4 * e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < PIECE; e += 8) {
            __align__(16) __nv_bfloat162 y[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) y[n] = __floats2bfloat162_rn(o[e + 2 * n], o[e + 2 * n + 1]);
            *reinterpret_cast<uint4*>(own + 2 * e) = *reinterpret_cast<const uint4*>(y);
          }
        }
        __syncwarp();
        for (int x = lane / lanes_to_row; x < 32; x += at_once) {
          if (tile_row0 + x >= row1) break;
          const int x_row = tile_head0 + x, tokens = a.group > 1 ? int(__umulhi(x_row, group_magic)) : x_row;
          const long long to = (chunk.row + tile_token0 + tokens) * a.q_heads + head * a.group + x_row - tokens * a.group;
          *reinterpret_cast<uint4*>(out + to * row_bytes + c * size + 16 * (lane % lanes_to_row)) =
              *reinterpret_cast<const uint4*>(stage + x * pitch + 16 * (lane % lanes_to_row));
        }
        __syncwarp();
      }
    }
  } else if (warp == T::COPY_WARP) {
    // ---- copies: a lane per run of a tile's keys, then of its values --------------------
    const int run = args.run, runs = KEYS / run;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      const int stage = j % T::COPY_STAGES;
      const uint32_t used = ((j / T::COPY_STAGES) & 1) ^ 1;
      const int key = seen.key_of(tile0 + j) + lane * run;
      // past the last key, or a page that the cache does not have: out of the
      // maps' range, which reads as zeros
      int page = a.at.pages;
      if (lane < runs && key < seen.end) {
        page = chunk.table[key / a.at.page_size];
        if (page < 0 || page >= a.at.pages) {
          chunk_error(a.error);
          page = a.at.pages;
        }
      }
      const int place = key % a.at.page_size;
      const int k_row = page * a.at.page_size + (page < a.at.pages ? place : 0);
      const int v_row = (page * a.kv_heads + (page < a.at.pages ? head : 0)) * D + part * DV;
      const uint32_t codes = base + T::CODES_AT + stage * 2 * T::CODE_STAGE + lane * run * D;
      // codes come with the scales of their pages' runs (zeros for the others')
      const long long scales_row = ((long long)page * a.kv_heads + head) * a.at.page_size + place;
      float* copied_scales = reinterpret_cast<float*>(shared + T::COPIED_SCALES_AT) + stage * 2 * KEYS + lane * run;
      const bool there = page < a.at.pages;
      const int bytes = T::CODE_BYTES + 4 * run * __popc(__ballot_sync(0xffffffffu, there));
      auto copy_scales = [&](const float* from, float* to, uint64_t* bar) {
        if (there) tc::bulk_load(to, from + scales_row, 4 * run, bar);
      };
      auto clear_scales = [&](float* to) {
        if (CODES && lane < runs && !there)
          for (int n = 0; n < run; n += 4) *reinterpret_cast<float4*>(to + n) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      };
      if (j >= T::COPY_STAGES && !(ok = wait(CODES ? &codes_empty[2 * stage] : &k_empty[stage], used))) break;
      uint64_t* full = CODES ? &codes_full[2 * stage] : &k_full[stage];
      clear_scales(copied_scales);
      __syncwarp();
      if (lane == 0) {
        tc::mbar_expect_tx(full, CODES ? bytes : T::K_BYTES);
        copied[0] = j + 1;
      }
      __syncwarp();
      if (lane < runs) {
        if constexpr (CODES) {
          tma_load_3d(codes, &key_map, full, 0, head, k_row);
          copy_scales(a.key_scales, copied_scales, full);
        } else {
#pragma unroll
          for (int p = 0; p < T::PANELS; ++p)
            tma_load_3d(base + T::K_AT + stage * T::K_BYTES + p * T::K_PANEL + lane * run * 128, &key_map, full, 64 * p,
                        head, k_row);
        }
      }
      if (j >= T::COPY_STAGES && !(ok = wait(CODES ? &codes_empty[2 * stage + 1] : &v_empty[stage], used))) break;
      full = CODES ? &codes_full[2 * stage + 1] : &v_full[stage];
      clear_scales(copied_scales + KEYS);
      __syncwarp();
      if (lane == 0) {
        tc::mbar_expect_tx(full, CODES ? bytes : T::V_BYTES);
        copied[1] = j + 1;
      }
      __syncwarp();
      if (lane < runs)
        tma_load_2d(CODES ? codes + T::CODE_STAGE : base + T::V_AT + stage * T::V_STAGE + lane * run * DV * 2, &value_map,
                    full, place, v_row);
      if (CODES && lane < runs) copy_scales(a.value_scales, copied_scales + KEYS, full);
      __syncwarp();
    }
  } else if (warp == T::QK_WARP || warp == T::PV_WARP) {
    // ---- tensor core --------------------------------------------------------------------
    constexpr uint32_t qk = tc::instr_desc_f16(ROW_TILE, KEYS), pv = tc::instr_desc_f16(ROW_TILE, DV);
    const int run = CODES ? 16 : args.run;  // keys of a piece of V
    const uint32_t run_shift = run == 64 ? 2 : run == 32 ? 1 : 0, run_bytes = uint32_t(run) * DV * 2;  // 2^shift steps
    int edges_told = 0, edges = 0;
    // (second terms first, while the sums are small)
    auto scores = [&](int j, int i, int b) {
      const uint64_t k = operand_desc(base + T::K_AT + (j % STAGES) * T::K_BYTES, 128);
#pragma unroll
      for (int term = TERMS - 1; term >= 0; --term) {
        const uint64_t q = operand_desc(base + (i * TERMS + term) * T::Q_BYTES, 128);
#pragma unroll
        for (int step = 0; step < D / 16; ++step)
          mma_ss_warp(tmem + b * T::S_COLUMNS, q + ((step / 4 * T::Q_PANEL + step % 4 * 32) >> 4),
                      k + ((step / 4 * T::K_PANEL + step % 4 * 32) >> 4), qk, term < TERMS - 1 || step > 0);
      }
      tc::mma_commit_warp(&s_full[b]);
    };
    // (false if the weights did not come)
    auto outputs = [&](int j, int i) {
      const uint64_t v = operand_desc(base + T::V_AT + (j % STAGES) * T::V_STAGE, 2 * run);
      if (!wait(&p_full[i], j & 1)) return false;
      tc::fence_after_sync();
#pragma unroll
      for (int term = TERMS - 1; term >= 0; --term)
#pragma unroll
        for (int step = 0; step < KEYS / 16; ++step) {
          const uint32_t at = (step >> run_shift) * run_bytes + (step & ((1u << run_shift) - 1)) * 32;
          tc::mma_f16_ts_warp(tmem + T::O_COLUMN + i * T::O_COLUMNS,
                              tmem + T::P_COLUMN + i * T::P_COLUMNS + term * KEYS / 2 + 8 * step, v + (at >> 4), pv,
                              (TERMS == 1 && j > 0) || term < TERMS - 1 || step > 0);
        }
      if (i == MT - 1) tc::mma_commit_warp(&v_empty[j % STAGES]);
      tc::mma_commit_warp(&pv_done[i]);
      return true;
    };
    auto keys_ready = [&](int j) { return wait(&k_full[j % STAGES], (j / STAGES) & 1); };
    // (the edge warp is told of an edge tile while the tile before is at work)
    auto tell_edge = [&](int j) {
      if (CODES || j >= tiles || whole(seen.key_of(tile0 + j))) return true;
      if (!wait(&v_full[j % STAGES], (j / STAGES) & 1)) return false;
      if (lane == 0) tc::mbar_arrive(&edge_found[edges_told & 1]);
      ++edges_told;
      return true;
    };
    auto values_ready = [&](int j) {
      if (!CODES && !whole(seen.key_of(tile0 + j))) {
        const int edge = edges++;
        return wait(&edge_clean[edge & 1], (edge >> 1) & 1);
      }
      return wait(&v_full[j % STAGES], (j / STAGES) & 1);
    };
    // scores of tile j (two row tiles: when theirs of the last are read; with
    // two S, when those of the one before are)
    auto next_scores = [&](int j) {
      if (!keys_ready(j)) return false;
      for (int i = 0; i < MT; ++i) {
        const int b = MT == 2 ? i : j & 1;
        if (MT == 2 && j > 0 && !wait(&s_empty[b], (j - 1) & 1)) return false;
        if (MT == 1 && j > 1 && !wait(&s_empty[b], ((j - 2) >> 1) & 1)) return false;
        tc::fence_after_sync();
        scores(j, i, b);
      }
      tc::mma_commit_warp(&k_empty[j % STAGES]);
      return true;
    };
    bool ok = true;
    const bool does_scores = warp == T::QK_WARP, does_outputs = warp == T::PV_WARP;
    if (does_scores) {
      for (int i = 0; i < MT && ok; ++i) ok = wait(&q_full[i], 0);
      if (ok) ok = next_scores(0);
    }
    if (does_outputs && ok) ok = tell_edge(0);
    for (int j = 0; j < tiles && ok; ++j) {
      if (does_scores && j + 1 < tiles && !(ok = next_scores(j + 1))) break;
      if (!does_outputs) continue;
      if (!(ok = tell_edge(j + 1))) break;
      if (!(ok = values_ready(j))) break;
      for (int i = 0; i < MT && ok; ++i) ok = outputs(j, i);
    }
  } else if (CODES && warp >= T::CONVERT_WARP) {
    // ---- conversion: codes to F16 operands, and the tile's scales ------------------------
    constexpr int N = T::CONVERT_THREADS, CHUNKS = D / 16;  // 16-byte chunks of a key's codes
    const int t = tid - 32 * T::CONVERT_WARP;
    const int run = args.run;
    auto seen_key = [&](int key) { return key < seen.end && (key >= lowest || key < first); };
    // a tile's scales, of every 32nd key from this lane's, zeros where no row
    // sees the key (each warp finds the largest for itself)
    constexpr int PER = (KEYS + 31) / 32;
    auto load_scales = [&](int key0, bool check, const float* from, float (&x)[PER]) {
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        const int k = lane + 32 * n;
        x[n] = k < KEYS && (!check || seen_key(key0 + k)) ? from[k] : 0.0f;
      }
    };
    auto largest_scale = [](const float (&x)[PER]) {  // of those that are finite
      float most = 0.0f;
#pragma unroll
      for (int n = 0; n < PER; ++n) most = x[n] <= 3.402823466e38f ? fmaxf(most, x[n]) : most;
#pragma unroll
      for (int o = 16; o > 0; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      return most;
    };
    float v_power = 0.0f;
    bool ok = true;
    for (int j = 0; j < tiles; ++j) {
      const int stage = j % STAGES, key0 = seen.key_of(tile0 + j);
      const uint32_t used = ((j / STAGES) & 1) ^ 1;
      const int copy_stage = j % T::COPY_STAGES;
      const uint32_t copy_phase = (j / T::COPY_STAGES) & 1;
      const uint8_t* k_codes = shared + T::CODES_AT + copy_stage * 2 * T::CODE_STAGE;
      const uint8_t* v_codes = k_codes + T::CODE_STAGE;
      // keys: a thread takes a row, or every second or fourth chunk of one
      constexpr int TO_ROW = CHUNKS % 4 == 0 && N >= 4 * KEYS ? 4 : CHUNKS % 2 == 0 && N >= 2 * KEYS ? 2 : 1;  // threads
      const int row = t % KEYS, share = t / KEYS;
      const bool has_row = share < TO_ROW;
      const float* k_from = reinterpret_cast<const float*>(shared + T::COPIED_SCALES_AT) + copy_stage * 2 * KEYS;
      const float* v_from = k_from + KEYS;
      const bool check = !whole(key0);
      if (j >= STAGES && !(ok = wait(&k_empty[stage], used))) break;
      if (!(ok = wait(&codes_full[2 * copy_stage], copy_phase))) break;
      const float own_k = (!check || seen_key(key0 + row)) ? k_from[row] : 0.0f;
      if (has_row) {
        uint8_t* k = shared + T::K_AT + stage * T::K_BYTES + row * 128;
        constexpr int TAKES = CHUNKS / TO_ROW;  // chunks a thread takes
        // (each eight lanes' chunks on different banks; loads ahead of the
        // stores, which the compiler cannot tell apart)
        auto chunk_of = [&](int n) {
          return CHUNKS == 4 ? (TO_ROW * n + share + row / 2) % 4 : CHUNKS % 8 == 0 ? (TO_ROW * n + share + row) % CHUNKS : n;
        };
        constexpr int FLIGHT = TAKES % 4 == 0 ? 4 : TAKES;
#pragma unroll
        for (int n0 = 0; n0 < TAKES; n0 += FLIGHT) {
          uint4 x[FLIGHT];
#pragma unroll
          for (int n = 0; n < FLIGHT; ++n) x[n] = *reinterpret_cast<const uint4*>(k_codes + row * D + 16 * chunk_of(n0 + n));
#pragma unroll
          for (int n = 0; n < FLIGHT; ++n) {
            const int c = chunk_of(n0 + n);
            const uint2 y0 = code_pairs(x[n].x), y1 = code_pairs(x[n].y), y2 = code_pairs(x[n].z), y3 = code_pairs(x[n].w);
            uint8_t* to = k + c / 4 * T::K_PANEL;
            *reinterpret_cast<uint4*>(to + 16 * ((2 * (c % 4)) ^ (row % 8))) =
                make_uint4(y0.x, y0.y, y1.x, y1.y);
            *reinterpret_cast<uint4*>(to + 16 * ((2 * (c % 4) + 1) ^ (row % 8))) =
                make_uint4(y2.x, y2.y, y3.x, y3.y);
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(&k_full[stage]);
      tc::mbar_arrive(&codes_empty[2 * copy_stage]);
      // scales: the stage's were last read by the softmax before the P V that
      // freed its values
      if (j >= STAGES && !(ok = wait(&v_empty[stage], used))) break;
      if (!(ok = wait(&codes_full[2 * copy_stage + 1], copy_phase))) break;
      float v_scale[PER];
      load_scales(key0, check, v_from, v_scale);
      const float most = largest_scale(v_scale);
      if (most > v_power) v_power = power_over(most);
      const float v_inverse = 1.0f / (v_power > 0.0f ? v_power : 1.0f);
      float* to_scales = scales + stage * T::SCALE_ROWS * KEYS + row;
      const float own_v = !check || seen_key(key0 + row) ? v_from[row] * v_inverse : 0.0f;
      to_scales[0] = own_k;
      to_scales[KEYS] = own_v;
      if constexpr (T::SCALE_ROWS == 3) to_scales[2 * KEYS] = logarithm(own_v);
      if (t == 0) v_unit[stage] = v_power, v_most[stage] = most * v_inverse;
      tc::mbar_arrive(&scales_full[stage]);
      // values: a thread takes sixteen positions of every (DIMS)th dimension
      constexpr int GROUPS = KEYS / 16, DIMS = N / GROUPS;
      const int per = run / 16;
      const int group = t % per + per * (t / (DIMS * per)), first_d = t / per % DIMS;
      const bool has_group = group < GROUPS;
      if (has_group) {
        uint8_t* v = shared + T::V_AT + stage * T::V_STAGE + group * (D * 32);
        const uint8_t* from = v_codes + group / per * (run * D) + group % per * 16;
        constexpr int TAKES = (D + DIMS - 1) / DIMS, FLIGHT = TAKES % 4 == 0 ? 4 : TAKES;
#pragma unroll
        for (int n0 = 0; n0 < TAKES; n0 += FLIGHT) {
          uint4 x[FLIGHT];
#pragma unroll
          for (int n = 0; n < FLIGHT; ++n) {
            const int d = first_d + DIMS * (n0 + n);
            x[n] = d < D ? *reinterpret_cast<const uint4*>(from + d * run) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int n = 0; n < FLIGHT; ++n) {
            const int d = first_d + DIMS * (n0 + n);
            if (d >= D) break;
            const uint2 y0 = code_pairs(x[n].x), y1 = code_pairs(x[n].y), y2 = code_pairs(x[n].z), y3 = code_pairs(x[n].w);
            uint8_t* to = v + d * 32;  // (rows of 32 bytes, their halves exchanged in every other four)
            const int c = d / 4 % 2;
            *reinterpret_cast<uint4*>(to + 16 * c) = make_uint4(y0.x, y0.y, y1.x, y1.y);
            *reinterpret_cast<uint4*>(to + 16 * (1 - c)) = make_uint4(y2.x, y2.y, y3.x, y3.y);
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(&v_full[stage]);
      tc::mbar_arrive(&codes_empty[2 * copy_stage + 1]);
    }
  } else if (!CODES && warp == T::EDGE_WARP) {
    // ---- edges: values that are not finite, out of the tiles seen in part -----------------
    bool ok = true;
    int edges = 0;
    const int run = args.run, row_bytes = 2 * run, chunks = run / 8;  // 16-byte chunks of a run's row
    for (int j = 0; j < tiles && ok; ++j) {
      const int key0 = seen.key_of(tile0 + j);
      if (whole(key0)) continue;
      const int edge = edges++;
      if (!(ok = wait(&edge_found[edge & 1], (edge >> 1) & 1))) break;
      if (!(ok = wait(&v_full[j % STAGES], (j / STAGES) & 1))) break;
      uint8_t* v = shared + T::V_AT + (j % STAGES) * T::V_STAGE;
      bool found = false;
      // (several loads under way: the look is a chain of latencies otherwise,
      // 2000 clocks long, and a window has an edge tile in every second)
      constexpr int CHECKS = T::V_BYTES / 512, FLIGHT = CHECKS % 8 == 0 ? 8 : 5;
      static_assert(T::V_BYTES % 512 == 0 && CHECKS % FLIGHT == 0, "whole rounds of a warp");
      // (an exponent of all ones carries into the sign's place)
      auto full = [](uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; };
#pragma unroll 1
      for (int n0 = lane; n0 < T::V_BYTES / 16; n0 += 32 * FLIGHT) {
        uint4 held[FLIGHT];
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) held[f] = *reinterpret_cast<const uint4*>(v + 16 * (n0 + 32 * f));
        uint32_t bad = 0;
#pragma unroll
        for (int f = 0; f < FLIGHT; ++f) bad |= full(held[f].x) | full(held[f].y) | full(held[f].z) | full(held[f].w);
        if (!bad) continue;
#pragma unroll 1
        for (int n = n0; n < n0 + 32 * FLIGHT; n += 32) {
          uint4 x = *reinterpret_cast<uint4*>(v + 16 * n);
          uint32_t* w = reinterpret_cast<uint32_t*>(&x);
          uint32_t any = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t is = full(w[e]);
            any |= is;
            w[e] &= (is & 0x8000u ? 0u : 0xffffu) | (is & 0x80000000u ? 0u : 0xffff0000u);
          }
          if (!any) continue;
          *reinterpret_cast<uint4*>(v + 16 * n) = x;
          // which keys: the run, and the chunk in its row before the swizzle
          // (which exchanges 16-byte chunks by the address bits 7 and up)
          const int in_run = 16 * n % (run * DV * 2), d = in_run / row_bytes;
          const int swizzle = row_bytes == 128 ? d % 8 : row_bytes == 64 ? d / 2 % 4 : d / 4 % 2;
          const int key = key0 + 16 * n / (run * DV * 2) * run + 8 * ((n % chunks) ^ swizzle);
          for (int e = 0; e < 8; ++e)
            found = found || (key + e < seen.end && (key + e >= lowest || key + e < first));
        }
      }
      if (found) *taken_out = 1;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc::mbar_arrive(&edge_clean[edge & 1]);
    }
    asm volatile("bar.arrive 1, %0;" ::"n"(T::ROUND_THREADS) : "memory");
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*abort) {
    // a wait gave up: what is on its way lands before shared memory and TMEM go
    int none = 0;
    if (tid == 32 * T::COPY_WARP)
      for (int side = 0; side < 2; ++side) {
        const int n = copied[side];
        uint64_t* full = CODES ? codes_full + side : side == 0 ? k_full : v_full;
        for (int j = max(0, n - T::COPY_STAGES); j < n; ++j)
          tc::mbar_wait(&full[j % T::COPY_STAGES * (CODES ? 2 : 1)], (j / T::COPY_STAGES) & 1, &none, nullptr);
      }
    if (warp == T::QK_WARP || warp == T::PV_WARP) {
      tc::mma_commit_warp(drained);
      tc::mbar_wait_warp(drained, 0, &none, nullptr);
    }
    __syncthreads();
  }
  if (warp == 0) tc::tmem_dealloc(tmem, TMEM_COLUMNS);
}

// Keys of a tile: what TMEM holds beside the outputs (P_COLUMN's assertion);
// F32 rows and heads of 256 have no room in registers or shared memory for more.
// Codes of heads of 64 go by 64 for BF16 rows, whose softmax takes scales as well
// (a chunk of 2 x 100 tokens x 4 heads over 2048 keys 18 us, 22 by 128, spilling).
constexpr int tile_of(int head_dim, int terms, bool codes) {
  return terms == 2 || head_dim > 128 ? 64 : head_dim > 80 ? 80 : head_dim > 64 ? 96 : codes ? 64 : 128;
}

template <int D, int MT, bool CODES, int TERMS, bool SCALED>
int launch_tiles(const AttentionChunksArgs& a, cudaStream_t stream) {
  using T = TileTraits<D, tile_of(D, TERMS, CODES), MT, CODES, TERMS, SCALED>;
  TileArgs args;
  args.a = a;
  const int ps = a.at.page_size;
  // the largest piece that pages and tiles are made of
  args.run = ps % 64 == 0 && T::KEYS % 64 == 0 ? 64 : ps % 32 == 0 && T::KEYS % 32 == 0 ? 32 : 16;
  const uint64_t positions = uint64_t(a.at.pages) * ps;
  constexpr uint64_t SIZE = CODES ? 1 : 2;
  CUtensorMap key_map, value_map;
  {
    const uint64_t dims[3] = {uint64_t(D), uint64_t(a.kv_heads), positions};
    const uint64_t strides[2] = {uint64_t(D) * SIZE, uint64_t(a.kv_heads) * D * SIZE};
    const uint32_t box[3] = {CODES ? uint32_t(D) : 64u, 1, uint32_t(args.run)};
    DRIFT_TRY(encode_cache_tiles(&key_map, a.keys, CODES, 3, dims, strides, box, CODES ? 0 : 128));
  }
  {
    const uint64_t dims[2] = {uint64_t(ps), uint64_t(a.at.pages) * a.kv_heads * D};
    const uint64_t strides[1] = {uint64_t(ps) * SIZE};
    const uint32_t box[2] = {uint32_t(args.run), uint32_t(T::DV)};
    DRIFT_TRY(encode_cache_tiles(&value_map, a.values, CODES, 2, dims, strides, box, CODES ? 0 : 2 * args.run));
  }
  static PerDevice configured;
  if (T::MOVES_REGISTERS && !configured.done()) {
    // the warps' shares come out of what a block is launched with; more than
    // that would be waited for without end
    cudaFuncAttributes attributes;
    DRIFT_CUDA(cudaFuncGetAttributes(&attributes, attention_tiles_kernel<T>));
    if (attributes.numRegs < T::LAUNCH_REGISTERS)
      return invalid("attention: a kernel of %d registers, built for %d", attributes.numRegs, T::LAUNCH_REGISTERS);
  }
  DRIFT_TRY(ensure_shared_memory(configured, attention_tiles_kernel<T>, T::BYTES));
  const unsigned units = unsigned((a.at.longest * a.group + T::UNIT - 1) / T::UNIT);
  DRIFT_CUDA(launch_pdl(attention_tiles_kernel<T>, dim3(a.kv_heads * T::PARTS, a.at.batch, units * a.splits), T::THREADS, T::BYTES,
                        stream, key_map, value_map, args));
  DRIFT_LAUNCHED("attention_tiles");
  return 0;
}

template <int D, int MT>
int launch_types(const AttentionChunksArgs& a, bool codes, bool bf16, cudaStream_t stream) {
  if (bf16 && codes) return launch_tiles<D, MT, true, 1, false>(a, stream);
  if (bf16) {
    // (expanded codes with their scales in them, and by key: what is the other's
    // returns at once)
    DRIFT_TRY((launch_tiles<D, MT, false, 1, false>(a, stream)));
    return a.units ? launch_tiles<D, MT, false, 1, true>(a, stream) : 0;
  }
  if (!codes) return a.units ? launch_tiles<D, MT, false, 2, true>(a, stream) : launch_tiles<D, MT, false, 2, false>(a, stream);
  if constexpr (D <= 128) return launch_tiles<D, MT, true, 2, false>(a, stream);
  else return invalid("attention: no tiles that convert codes for F32 heads of %d", D);
}

#define DRIFT_TILES_REGISTER_AS(D, MT, codes, terms, scaled, name) \
  DRIFT_REGISTER(name, (attention_tiles_kernel<TileTraits<D, tile_of(D, terms, codes), MT, codes, terms, scaled>>))
#define DRIFT_TILES_REGISTER_BF16(D, MT)                                            \
  DRIFT_TILES_REGISTER_AS(D, MT, false, 1, false, attention_tiles_f16_bf16_d##D##_m##MT)    \
  DRIFT_TILES_REGISTER_AS(D, MT, true, 1, false, attention_tiles_i8_bf16_d##D##_m##MT)      \
  DRIFT_TILES_REGISTER_AS(D, MT, false, 1, true, attention_tiles_expanded_bf16_d##D##_m##MT)
#define DRIFT_TILES_REGISTER(D, MT)                                                 \
  DRIFT_TILES_REGISTER_BF16(D, MT)                                                  \
  DRIFT_TILES_REGISTER_AS(D, MT, false, 2, false, attention_tiles_f16_f32_d##D##_m##MT)     \
  DRIFT_TILES_REGISTER_AS(D, MT, true, 2, false, attention_tiles_i8_f32_d##D##_m##MT)  \
  DRIFT_TILES_REGISTER_AS(D, MT, false, 2, true, attention_tiles_expanded_f32_d##D##_m##MT)
DRIFT_TILES_REGISTER(64, 1)
DRIFT_TILES_REGISTER(64, 2)
DRIFT_TILES_REGISTER(80, 1)
DRIFT_TILES_REGISTER(80, 2)
DRIFT_TILES_REGISTER(128, 1)
DRIFT_TILES_REGISTER(128, 2)
DRIFT_TILES_REGISTER_BF16(256, 1)
DRIFT_TILES_REGISTER_AS(256, 1, false, 2, false, attention_tiles_f16_f32_d256_m1)
DRIFT_TILES_REGISTER_AS(256, 1, false, 2, true, attention_tiles_expanded_f32_d256_m1)

}  // namespace

int attention_tiles_keys(int head_dim, bool bf16, bool codes) { return tile_of(head_dim, bf16 ? 1 : 2, codes); }

int launch_attention_tiles(const AttentionChunksArgs& a, int x_dtype, int cache_dtype, int head_dim, int row_tiles,
                           cudaStream_t stream) {
  const bool bf16 = x_dtype == DRIFT_BF16, codes = cache_dtype == DRIFT_I8;
  switch (head_dim) {
    case 64: return row_tiles == 2 ? launch_types<64, 2>(a, codes, bf16, stream) : launch_types<64, 1>(a, codes, bf16, stream);
    case 80: return row_tiles == 2 ? launch_types<80, 2>(a, codes, bf16, stream) : launch_types<80, 1>(a, codes, bf16, stream);
    case 128: return row_tiles == 2 ? launch_types<128, 2>(a, codes, bf16, stream) : launch_types<128, 1>(a, codes, bf16, stream);
    default: return launch_types<256, 1>(a, codes, bf16, stream);
  }
}

}  // namespace drift

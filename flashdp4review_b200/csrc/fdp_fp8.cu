// Products in 8-bit floating point (e4m3) with one scale for each block of 128 numbers of the contraction.
//
//   Y[m, n] = sum_kb s_a[m, kb] * s_w[n / 128, kb] * sum_{k in kb} q_a[m, k] q_w[n, k]  (+ bias[n])
//
// Activations and gradients have a scale for each row and 128 columns, so that no number of one sample depends on another
// sample's (per-sample clipping needs that); weights one for each 128 x 128 block, which serves both the forward product
// and the input gradient.  Scales are powers of two, the smallest that brings a block's largest finite magnitude to at
// most 448: dividing by one and multiplying by two of them is exact, so the only roundings are those to e4m3, those of
// the accumulation and the last one.  A number that is not finite becomes a NaN (e4m3 has no infinity).
//
// The matrix instruction applies the scales itself (kind::mxf8f6f4, block_scale): it takes one exponent a row for 32 numbers
// out of TMEM, and here the four instructions of a K block take the same one.  A word of TMEM holds the exponents of four
// K blocks, so they are copied there once for every 512 numbers.  Exponents lie in memory as that copy wants them, in
// units of 128 rows x 4 K blocks, 512 bytes: row r's word at (r % 32) * 16 + r / 32 * 4.
#include <cuda_fp8.h>

#include "fdp_async.cuh"
#include "fdp_kernels.h"
#include "fdp_tcgen05.cuh"
#include "fdp_vec8.cuh"

namespace fdp {
namespace {

// ---- quantisation -----------------------------------------------------------------------------------
// exponent k of the smallest power of two with amax <= 448 * 2^k (448 = 1.75 * 2^8); 0 for a block of zeros; not below -126,
// so that 2^k and 2^-k are both normal numbers
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  if (amax_bits == 0) return 0;
  const int k = static_cast<int>(amax_bits >> 23) - 127 - ((amax_bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7);
  return k < -126 ? -126 : k;
}
__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }
__device__ __forceinline__ uint32_t exponent_byte(int k) { return static_cast<uint32_t>(k + 127); }
// Eight adjacent numbers, as they are loaded, and their largest magnitude as the bits of an fp32 number (0x7F800000 or more
// where one is not finite).  16-bit magnitudes are compared two at a time as the whole numbers that order like them.
template <typename T> struct Eight { Vec8<T> raw; };
template <typename T>
__device__ __forceinline__ uint32_t largest_bits(const Eight<T>& a) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.raw.v);
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
    return m;
  } else {
    const uint32_t m = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
    return max(m & 0xFFFFu, m >> 16);
  }
}
template <typename T> __device__ __forceinline__ uint32_t as_fp32_bits(uint32_t m) { return m; }
template <> __device__ __forceinline__ uint32_t as_fp32_bits<__nv_bfloat16>(uint32_t m) { return m << 16; }
template <> __device__ __forceinline__ uint32_t as_fp32_bits<__half>(uint32_t m) { return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m)))); }
// the same without what is not finite
template <typename T>
__device__ __forceinline__ uint32_t largest_finite_bits(const Eight<T>& a) {
  float f[8];
  unpack8(a.raw, f);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(f[e]) & 0x7FFFFFFFu;
    m = max(m, b < 0x7F800000u ? b : 0u);
  }
  return m;
}
// times 2^-k as e4m3 (round to nearest even; nothing saturates: the block's largest is at most 448).  STRANGE: a block with
// numbers that are not finite, which become NaNs.
template <typename T, bool STRANGE>
__device__ __forceinline__ uint2 to_e4m3x8(const Eight<T>& a, float inv) {
  float f[8];
  unpack8(a.raw, f);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float2 p = make_float2(f[4 * h + 2 * j], f[4 * h + 2 * j + 1]);
      if (STRANGE) {
        if ((__float_as_uint(p.x) & 0x7F800000u) == 0x7F800000u) p.x = __uint_as_float(0x7FC00000u);
        if ((__float_as_uint(p.y) & 0x7F800000u) == 0x7F800000u) p.y = __uint_as_float(0x7FC00000u);
      }
      w[h] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(p.x * inv, p.y * inv), __NV_SATFINITE, __NV_E4M3)) << (16 * j);
    }
  }
  return make_uint2(w[0], w[1]);
}

// eight numbers of a row from column `col` on; what lies past the row's end is 0
template <typename T, bool VEC>
__device__ __forceinline__ Eight<T> load_row8(const T* row, int col, int cols) {
  Eight<T> r{};
  if (VEC) {
    if (col < cols) r.raw = load8(row + col);
  } else {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = col + e < cols ? row[col + e] : from_f32<T>(0.f);
    r.raw = *reinterpret_cast<const Vec8<T>*>(t);
  }
  return r;
}

// Rows: a half warp takes 128 columns of a row at a time, a block 16 rows x four blocks of columns: a row's four exponents are a
// word of the unit described above.  HBM-bound: 3 bytes an element of 16 bits (2 read, 1 written), 5 of 32.
constexpr int QKB = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, uint32_t* __restrict__ packed,
                                                       float* __restrict__ scales, int rows, int cols, int pitch, int kblocks, int row_tiles) {
  const int hw = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int group = blockIdx.x / row_tiles, r0 = (blockIdx.x - group * row_tiles) * 16, kb0 = group * QKB;
  const int row = r0 + hw;
  pdl_trigger();
  if (row >= rows) return;            // (a half warp as a whole; the shuffles are its own)
  const uint32_t half = 0xFFFFu << (threadIdx.x & 16);
  const T* xr = x + static_cast<size_t>(row) * cols;
  uint8_t* qr = q + static_cast<size_t>(row) * pitch;
  Eight<T> f[QKB];
#pragma unroll
  for (int i = 0; i < QKB; ++i) f[i] = load_row8<T, VEC>(xr, (kb0 + i) * 128 + l * 8, cols);      // (nothing past the last column)
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < QKB; ++i) {
    const int col = (kb0 + i) * 128 + l * 8;
    uint32_t m = largest_bits(f[i]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half, m, o));
    m = as_fp32_bits<T>(m);
    uint2 w;
    int k;
    if (m < 0x7F800000u) {
      k = scale_exponent(m);
      w = to_e4m3x8<T, false>(f[i], power_of_two(-k));
    } else {
      m = largest_finite_bits(f[i]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(half, m, o));
      k = scale_exponent(m);
      w = to_e4m3x8<T, true>(f[i], power_of_two(-k));
    }
    if (col < pitch) *reinterpret_cast<uint2*>(qr + col) = w;
    word |= exponent_byte(k) << (8 * i);
    if (scales != nullptr && l == 0 && kb0 + i < kblocks) scales[static_cast<size_t>(kb0 + i) * rows + row] = power_of_two(k);
  }
  if (packed != nullptr && l == 0) {
    const int groups = (kblocks + 3) / 4, in = row & 127;
    packed[(static_cast<size_t>(row >> 7) * groups + group) * 128 + (in & 31) * 4 + (in >> 5)] = word;
  }
}

// 4 x 4 bytes transposed: out[j] holds byte j of in[0..3]
__device__ __forceinline__ void transpose4(const uint32_t in[4], uint32_t out[4]) {
  const uint32_t a = __byte_perm(in[0], in[1], 0x5140), b = __byte_perm(in[2], in[3], 0x5140);   // bytes 0 and 1 of the pairs
  const uint32_t c = __byte_perm(in[0], in[1], 0x7362), d = __byte_perm(in[2], in[3], 0x7362);   // bytes 2 and 3
  out[0] = __byte_perm(a, b, 0x5410);
  out[1] = __byte_perm(a, b, 0x7632);
  out[2] = __byte_perm(c, d, 0x5410);
  out[3] = __byte_perm(c, d, 0x7632);
}
// Weights: one block a 128 x 128 block, written as it lies and transposed (both products contract over adjacent bytes).  A
// half warp holds eight rows of it, a thread 8 x 8 numbers, whose bytes it transposes in registers.
constexpr int WT_PITCH = 128 + 16;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fp8_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ q, uint8_t* __restrict__ qt,
                                                         float* __restrict__ scales, uint8_t* __restrict__ packed, uint8_t* __restrict__ packed_t,
                                                         int rows, int cols, int pitch, int pitch_t, int row_blocks, int col_blocks) {
  __shared__ __align__(16) uint8_t tile[128 * WT_PITCH];
  __shared__ uint32_t red[8];
  const int hw = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int rb = blockIdx.x / col_blocks, cb = blockIdx.x - rb * col_blocks;
  const int r0 = rb * 128 + hw * 8, c = cb * 128 + l * 8;
  pdl_trigger();
  Eight<T> f[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = Eight<T>{};
    if (r0 + i < rows) f[i] = load_row8<T, VEC>(w + static_cast<size_t>(r0 + i) * cols, c, cols);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, largest_bits(f[i]));
  auto block_largest = [&](uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) v = max(v, red[i]);
    return v;
  };
  m = as_fp32_bits<T>(block_largest(m));
  const bool strange = m >= 0x7F800000u;
  if (strange) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, largest_finite_bits(f[i]));
    __syncthreads();
    m = block_largest(m);
  }
  const int k = scale_exponent(m);
  const float inv = power_of_two(-k);
  if (threadIdx.x == 0) scales[blockIdx.x] = power_of_two(k);
  if (threadIdx.x < 128) {            // the same exponent for 128 rows, of the matrix and of its transpose
    const int at = (threadIdx.x & 31) * 16 + (threadIdx.x >> 5) * 4;
    packed[(static_cast<size_t>(rb) * ((col_blocks + 3) / 4) + cb / 4) * 512 + at + cb % 4] = static_cast<uint8_t>(exponent_byte(k));
    packed_t[(static_cast<size_t>(cb) * ((row_blocks + 3) / 4) + rb / 4) * 512 + at + rb % 4] = static_cast<uint8_t>(exponent_byte(k));
  }
  uint2 b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    b[i] = strange ? to_e4m3x8<T, true>(f[i], inv) : to_e4m3x8<T, false>(f[i], inv);
    if (r0 + i < rows && c < pitch) *reinterpret_cast<uint2*>(q + static_cast<size_t>(r0 + i) * pitch + c) = b[i];
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {          // columns 4 half .. 4 half + 3 of the thread's eight
    uint32_t lo[4], hi[4], in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = half ? b[i].y : b[i].x;
    transpose4(in, lo);
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = half ? b[4 + i].y : b[4 + i].x;
    transpose4(in, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint2*>(tile + (l * 8 + half * 4 + j) * WT_PITCH + hw * 8) = make_uint2(lo[j], hi[j]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int piece = threadIdx.x + i * 256, tc = piece >> 3, tr = (piece & 7) * 16;
    if (cb * 128 + tc < cols && rb * 128 + tr < pitch_t)
      *reinterpret_cast<uint4*>(qt + static_cast<size_t>(cb * 128 + tc) * pitch_t + rb * 128 + tr) = *reinterpret_cast<const uint4*>(tile + tc * WT_PITCH + tr);
  }
}

// ---- the product --------------------------------------------------------------------------------------
// A persistent, warp-specialised kernel: warp 0 copies (TMA, 128-byte swizzle), warp 1 issues the matrix instructions and owns
// TMEM, warps 2 to 9 store, two on each TMEM lane quarter.  CTAS = 2: a cluster of two CTAs works on 256 rows, each
// loads its 128 rows of A and half of the tile's columns of B, the even one issues for both (every CTA needs the exponents
// of all the tile's columns).  Both operands are K-major; a stage of the ring is one K block, 128 bytes a row.
//
// (Before: kind::f8f6f4 and the scales in the epilogue, where a K block's accumulator was added to fp32 registers times both
// scales.  A hand-off is a commit, a wait, the accumulator's loads and an arrival across the pair, with two accumulators in
// turn about 900 cycles for every 512 cycles of matrix instructions: 8192 rows 4096 -> 11008 386 us.)
// (Tried: tiles of 256 x 192 with two accumulators, so that a pair's store runs beside the next tile's products.  What long thin
// products wait for is their operands from L2, of which smaller tiles read more: with the quantisation of 16384 rows
// 1024 -> 4096 78 us against 70, 8192 rows 4096 -> 11008 300 against 284, 8192 rows 2048 -> 2048 55 against 60.)
//
// The tensor cores add into their fp32 accumulators by truncation, up to a unit in the last place a step, 2^-23, and all of one
// sign; a K block has four steps.  So an accumulator is handed over after a number of K blocks and added to registers, rounded to
// nearest: F8_CHAIN of them for fp32 outputs, and F8_CHAIN_16 for 16-bit ones, whose 512 steps lose at most 2^-14, an eighth to a quarter
// of fp16's half step (2^-11 to 2^-12).  Contractions of up to 16384 columns have one chain.  (With a single chain of any length 262144
// columns lost 2^-10.)
constexpr int F8_BM = 128, F8_THREADS = 320, F8_RING = 160 * 1024, F8_CHAIN = 8, F8_CHAIN_16 = 128;
template <int CTAS, int BN> struct F8Tile {
  static constexpr int A_BYTES = F8_BM * 128, B_BYTES = BN / CTAS * 128, STG = A_BYTES + B_BYTES;
  static constexpr int STAGES = F8_RING / STG < 8 ? F8_RING / STG : 8;
  static constexpr int ACCS = (TMEM_COLS - 32) / BN < 2 ? 1 : 2;
  static constexpr int WC = BN / 2;          // columns of an epilogue warp
  static constexpr int SF_BYTES = 512 + BN * 4;     // exponents of a stage: 128 rows of A, BN of B, four K blocks
  static constexpr int SMEM = F8_RING + 1024 + 8 * BOX_BYTES + STAGES * SF_BYTES + 256;
};
static_assert(F8Tile<2, 256>::SMEM <= 227 * 1024 && F8Tile<1, 128>::SMEM <= 227 * 1024, "shared memory of one CTA");
constexpr int F8_SF_COL = TMEM_COLS - 32;    // TMEM columns of the exponents: 4 of A's, then BN / 32 of B's

struct Fp8Args {
  int M, N, kblocks;
  int tiles_m, tiles_n, m_group, split, chain;
  void* out; int out_dt; int direct_out;
  const void* bias; int bias_dt;
  float* parts;                             // split > 1: [unit][CTA][epilogue warp][WC / 32][1024]
  int* sticky;
};

template <int CTAS>
__device__ __forceinline__ void f8_mma(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t sf_a,
                                       uint32_t sf_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 a, {%1, %2};\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::%7.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %5, [%8], [%9], p;\n\t}"
      ::"r"(tmem_d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "n"(CTAS), "r"(sf_a), "r"(sf_b) : "memory");
}
// 32 x 16 bytes of shared memory (a unit of exponents: eight rows 128 bytes apart, no swizzle) to four columns of TMEM, in
// every lane quarter; in both CTAs of a pair.  Runs in order with the matrix instructions issued before and after it.
template <int CTAS>
__device__ __forceinline__ void f8_copy_exponents(uint32_t tmem, uint32_t saddr) {
  const uint32_t lo = (saddr >> 4) & 0x3FFF, hi = (128u >> 4) | (1u << 14);
  asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::%3.32x128b.warpx4 [%0], d;\n\t}"
               ::"r"(tmem), "r"(lo), "r"(hi), "n"(CTAS) : "memory");
}
// e4m3 x e4m3 -> fp32, both operands K-major, exponent scales (UE8M0); `sf` is the byte of the scales' words
__host__ __device__ constexpr uint32_t f8_idesc(int ctas, int n, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>((F8_BM * ctas) >> 4) << 24) |
         (static_cast<uint32_t>(sf) << 29);
}

// v[0..31] += bias[n..n+31], the same numbers in every lane: 16-byte loads where they may be
__device__ __forceinline__ void f8_add_bias(const void* bias, int dt, int n, int N, float v[32]) {
  if (n + 32 <= N && (reinterpret_cast<uintptr_t>(bias) & 15) == 0) {
    if (dt == FDP_F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(bias) + n) + j);
        v[4 * j] += b.x; v[4 * j + 1] += b.y; v[4 * j + 2] += b.z; v[4 * j + 3] += b.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(bias) + n) + j);
        float b[8];
        if (dt == FDP_BF16) unpack16<__nv_bfloat16>(raw, b); else unpack16<__half>(raw, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * j + e] += b[e];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n + j < N) v[j] += load_as(bias, dt, n + j);
  }
}

// rows of a warp's box one by one: an output that the copy engine cannot write
template <typename T>
__device__ __forceinline__ void f8_store_rows(T* out, size_t ld, uint32_t box, int rows, int lane, bool in) {
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = r0 + k;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[k]) : "r"(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (in && r0 + k < rows) out[static_cast<size_t>(r0 + k) * ld] = from_f32<T>(v[k]);
  }
}

template <int CTAS, int BN>
__global__ void __launch_bounds__(F8_THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmSA,
                const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ Fp8Args args) {
  using L = F8Tile<CTAS, BN>;
  constexpr int NST = L::STAGES, NACC = L::ACCS, WC = L::WC, STG = L::STG;
  const uint32_t cta_rank = CTAS == 2 ? cluster_ctarank() : 0u;
  const bool is_leader = cta_rank == 0;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw), base = (raw_addr + 1023u) & ~1023u;
  const uint32_t boxes = base + F8_RING, exps = boxes + 8 * BOX_BYTES, bar_base = exps + NST * L::SF_BYTES;
  uint8_t* bar_gen = smem_raw + (bar_base - raw_addr);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (8 + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (16 + a); };
  auto tfree_bar = [&](int a) { return bar_base + 8u * (18 + a); };
  const uint32_t drain_bar = bar_base + 8u * 20;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bar_gen + 8 * 21);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_gen + 8 * 21 + 4);
  const WaitCtx wctx{abort_flag, nullptr, args.sticky, WAIT_LIMIT_CYCLES};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int units = args.tiles_m * args.tiles_n * args.split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int a = 0; a < NACC; ++a) { mbar_init(tfull_bar(a), 1); mbar_init(tfree_bar(a), 8 * CTAS); }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (CTAS == 2) {
    __syncthreads();
    cluster_sync_all();      // the peer's barriers must be initialised before anything is signalled across the pair
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::%2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(const_cast<uint32_t*>(tmem_slot))), "r"(TMEM_COLS), "n"(CTAS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::%0.sync.aligned;" ::"n"(CTAS) : "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  pdl_wait();
  const int wid = blockIdx.x / CTAS, wstep = gridDim.x / CTAS;
  const uint32_t tmem_base = *tmem_slot;

  // unit -> tile, K blocks.  Tiles are walked in groups of m_group tile rows, so that the CTAs that run together share operands.
  auto decode = [&](int u, int& m0, int& n0, int& k0, int& k1) {
    const int tile = u / args.split, part = u - tile * args.split;
    k0 = static_cast<int>(static_cast<long long>(args.kblocks) * part / args.split);
    k1 = static_cast<int>(static_cast<long long>(args.kblocks) * (part + 1) / args.split);
    const int per_group = args.m_group * args.tiles_n;
    const int g = tile / per_group, r = tile - g * per_group;
    const int gm = min(args.m_group, args.tiles_m - g * args.m_group);
    m0 = (g * args.m_group + r % gm) * (F8_BM * CTAS) + static_cast<int>(cta_rank) * F8_BM;
    n0 = r / gm * BN;
  };

  if (warp == 0) {
    // ================= copies =================
    int stage = 0; uint32_t phase = 0;
    bool ok = true;
    const int kgroups = (args.kblocks + 3) / 4;
    for (int u = wid; u < units && ok; u += wstep) {
      int m0, n0, k0, k1;
      decode(u, m0, n0, k0, k1);
      for (int kb = k0; kb < k1; ++kb) {
        if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, wctx, 21)) { ok = false; break; }
        if (elect_one()) {
          const bool exponents = kb == k0 || kb % 4 == 0;
          const uint32_t sa = base + stage * STG, sb = sa + L::A_BYTES, se = exps + stage * L::SF_BYTES;
          const uint32_t lbar = CTAS == 1 ? full_bar(stage) : mapa_u32(full_bar(stage), 0);
          if (is_leader) mbar_expect_tx(full_bar(stage), CTAS * (STG + (exponents ? L::SF_BYTES : 0)));
          const int nb = n0 + static_cast<int>(cta_rank) * (BN / CTAS);
          auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1) {
            if (CTAS == 1) tma_load_2d(dst, map, c0, c1, lbar); else tma_load_2d_pair(dst, map, c0, c1, lbar);
          };
          if (exponents) {
            load(se, &tmSA, 0, m0 / 128 * kgroups + kb / 4);
#pragma unroll
            for (int j = 0; j < BN / 128; ++j) load(se + 512 + j * 512, &tmSB, 0, (n0 / 128 + j) * kgroups + kb / 4);
          }
          load(sa, &tmA, kb * 128, m0);
          load(sb, &tmB, kb * 128, nb);
        }
        __syncwarp();
        if (++stage == NST) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok && lane == 0 && is_leader) {
      // wait (bounded) for the copies already in flight before the CTA may leave
      for (int s = 0; s < NST; ++s) {
        const long long t0 = clock64();
        const uint32_t ph = (s < stage) ? phase : (phase ^ 1u);
        while (!mbar_try(full_bar(s), ph) && clock64() - t0 < WAIT_LIMIT_CYCLES / 8) {}
      }
    }
  } else if (warp == 1) {
    // ================= matrix instructions: the whole warp walks, one elected lane issues =================
    if (is_leader) {
      int stage = 0; uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      const Desc a0 = make_desc(base, 0, 1024), b0 = make_desc(base + L::A_BYTES, 0, 1024);
      const uint32_t sf_a = tmem_base + F8_SF_COL, sf_b = sf_a + 4;
      auto commit = [&](uint32_t bar) { if (CTAS == 1) tc_commit(bar); else tc_commit_pair(bar); };
      for (int u = wid; u < units && ok; u += wstep) {
        int m0, n0, k0, k1;
        decode(u, m0, n0, k0, k1);
        for (int kb = k0; kb < k1 && ok; ++it) {
          const int acc = it % NACC, end = min(k1, kb + args.chain), first = kb;
          if (!mbar_wait_warp(tfree_bar(acc), ((it / NACC) & 1u) ^ 1u, wctx, 22)) { ok = false; break; }
          for (; kb < end; ++kb) {
            if (!mbar_wait_warp(full_bar(stage), phase, wctx, 23)) { ok = false; break; }
            tc_fence_after();
            const uint32_t so = static_cast<uint32_t>(stage * STG) >> 4;
            if (elect_one()) {
              if (kb == k0 || kb % 4 == 0) {
                const uint32_t se = exps + stage * L::SF_BYTES;
                f8_copy_exponents<CTAS>(sf_a, se);
#pragma unroll
                for (int j = 0; j < BN / 128; ++j) f8_copy_exponents<CTAS>(sf_b + 4 * j, se + 512 + j * 512);
              }
              const uint32_t idesc = f8_idesc(CTAS, BN, 0) | (static_cast<uint32_t>(kb & 3) << 4) | (static_cast<uint32_t>(kb & 3) << 29);
#pragma unroll
              for (int k = 0; k < 4; ++k)        // 32 numbers, 32 bytes, each
                f8_mma<CTAS>(tmem_base + acc * BN, a0.lo + so + 2 * k, a0.hi, b0.lo + so + 2 * k, b0.hi, idesc, sf_a, sf_b, kb > first || k > 0 ? 1u : 0u);
              commit(empty_bar(stage));
              if (kb + 1 == end) commit(tfull_bar(acc));
            }
            __syncwarp();
            if (++stage == NST) { stage = 0; phase ^= 1u; }
          }
        }
      }
      if (!ok && elect_one()) {
        // let the instructions already issued finish before TMEM is released
        commit(drain_bar);
        const long long t0 = clock64();
        while (!mbar_try(drain_bar, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES / 8) {}
      }
    }
  } else {
    // ================= epilogue =================
    const int quarter = warp & 3, ew = warp - 2, chalf = ew >> 2;
    const uint32_t box = boxes + ew * BOX_BYTES;
    int it = 0;
    bool ok = true;
    for (int u = wid; u < units && ok; u += wstep) {
      int m0, n0, k0, k1;
      decode(u, m0, n0, k0, k1);
      const int nw = n0 + chalf * WC;
      float acc_r[WC];
      for (int kb = k0; kb < k1; kb += args.chain, ++it) {
        const int acc = it % NACC;
        if (!mbar_wait_warp(tfull_bar(acc), (it / NACC) & 1u, wctx, 24)) { ok = false; break; }
        tc_fence_after();
        const uint32_t tb = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * BN + chalf * WC;
        if (kb == k0) {
#pragma unroll
          for (int c4 = 0; c4 < WC / 32; ++c4) tc_ld32(tb + c4 * 32, reinterpret_cast<uint32_t*>(acc_r) + c4 * 32);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int c4 = 0; c4 < WC / 32; ++c4) {
            uint32_t r[32];
            tc_ld32(tb + c4 * 32, r);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) acc_r[c4 * 32 + j] += __uint_as_float(r[j]);
          }
        }
        tc_fence_before();               // the accumulator has been read: back to the matrix warp
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 1 || is_leader) mbar_arrive(tfree_bar(acc));
          else mbar_arrive_cluster(mapa_u32(tfree_bar(acc), 0));
        }
      }
      if (!ok) break;
      const int row0 = m0 + quarter * 32;
      if (row0 >= args.M) continue;
      if (args.split > 1) {
        float* dst = args.parts + ((static_cast<size_t>(u) * CTAS + cta_rank) * 8 + ew) * (WC * 32);
#pragma unroll
        for (int c4 = 0; c4 < WC / 32; ++c4)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            reinterpret_cast<float4*>(dst + c4 * 1024)[j * 32 + lane] =
                make_float4(acc_r[c4 * 32 + 4 * j], acc_r[c4 * 32 + 4 * j + 1], acc_r[c4 * 32 + 4 * j + 2], acc_r[c4 * 32 + 4 * j + 3]);
        continue;
      }
#pragma unroll
      for (int c4 = 0; c4 < WC / 32; ++c4) {
        const int n = nw + c4 * 32;
        if (n >= args.N) break;
        float* v = acc_r + c4 * 32;
        if (args.bias != nullptr) f8_add_bias(args.bias, args.bias_dt, n, args.N, v);
        if (args.direct_out || args.out_dt == FDP_F32) {
          box_wait(lane);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            box_put(box, lane, j, __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
          if (!args.direct_out) {
            box_send(box, &tmOut, n, row0, lane);
          } else {
            __syncwarp();
            const int rows = min(BOX_ROWS, args.M - row0);
            const size_t at = static_cast<size_t>(row0) * args.N + n + lane;
            const bool in = n + lane < args.N;
            if (args.out_dt == FDP_F32) f8_store_rows(static_cast<float*>(args.out) + at, args.N, box, rows, lane, in);
            else if (args.out_dt == FDP_BF16) f8_store_rows(static_cast<__nv_bfloat16*>(args.out) + at, args.N, box, rows, lane, in);
            else f8_store_rows(static_cast<__half*>(args.out) + at, args.N, box, rows, lane, in);
            __syncwarp();
          }
        } else {
          // 16-bit: two chunks of 32 columns fill a box (a lone one is sent half full; the map's box is 64 wide, so it waits
          // for its second half only where the matrix has one)
          if ((c4 & 1) == 0) box_wait(lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 w = args.out_dt == FDP_BF16 ? pack16<__nv_bfloat16>(v + 8 * j) : pack16<__half>(v + 8 * j);
            box_put(box, lane, 4 * (c4 & 1) + j, w.x, w.y, w.z, w.w);
          }
          if ((c4 & 1) == 1 || n + 32 >= args.N) box_send(box, &tmOut, n - 32 * (c4 & 1), row0, lane);
        }
      }
    }
  }
  // ================= teardown =================
  if (warp >= 2) box_drain(lane);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CTAS == 2) cluster_sync_all();   // neither CTA leaves (or frees TMEM) while its peer may still signal it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::%2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS), "n"(CTAS) : "memory");
  }
}

// the parts of a K split, added in order, with the bias
template <int CTAS, int BN>
__global__ void __launch_bounds__(256) fp8_join_kernel(const __grid_constant__ Fp8Args args) {
  constexpr int WC = F8Tile<CTAS, BN>::WC, UNIT = CTAS * F8_BM * BN;
  pdl_wait();
  // a thread takes four columns of a row: rows of a box lie 16 bytes apart
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const int tile = static_cast<int>(i / (UNIT / 4)), e = static_cast<int>(i % (UNIT / 4)) * 4;
  if (tile >= args.tiles_m * args.tiles_n) return;
  const int wbox = e / 1024, in_box = e % 1024;
  const int c4 = wbox % (WC / 32), cw = wbox / (WC / 32), ew = cw % 8, rank = cw / 8;
  // epilogue warp ew is warp ew + 2 of its CTA: lane quarter (ew + 2) % 4, column half ew / 4
  const int per_group = args.m_group * args.tiles_n;
  const int g = tile / per_group, r = tile - g * per_group;
  const int gm = min(args.m_group, args.tiles_m - g * args.m_group);
  const int row = (g * args.m_group + r % gm) * (F8_BM * CTAS) + rank * F8_BM + ((ew + 2) & 3) * 32 + (in_box % 128) / 4;
  const int n = r / gm * BN + (ew >> 2) * WC + c4 * 32 + in_box / 128 * 4;
  if (row >= args.M || n >= args.N) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < args.split; ++p) {
    const float4 t = *reinterpret_cast<const float4*>(args.parts + (static_cast<size_t>(tile) * args.split + p) * UNIT + e);
    v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
  }
  for (int k = 0; k < 4 && n + k < args.N; ++k)
    store_as(args.out, args.out_dt, static_cast<size_t>(row) * args.N + n + k, v[k] + (args.bias != nullptr ? load_as(args.bias, args.bias_dt, n + k) : 0.f));
}

bool make_bytes_map(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {128, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// units of exponents, 128 words each, of ceil(rows / 128) x ceil(kblocks / 4)
bool make_exponents_map(CUtensorMap* m, const void* base, int rows, int kblocks) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>(ceil_div(rows, 128)) * ceil_div(kblocks, 4)};
  const cuuint64_t strides[1] = {512};
  const cuuint32_t box[2] = {128, 1};
  const cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CTAS, int BN>
int gemm_launch(const Fp8Args& args_in, const void* a, int pitch_a, const void* sa, const void* w, int pitch_w, const void* sw, int K, const Fp8Plan& pl,
                cudaStream_t s) {
  static std::mutex mu;
  static bool done[64];
  if (!smem_opt_in(done, mu, fp8_gemm_kernel<CTAS, BN>, F8Tile<CTAS, BN>::SMEM)) return FDP_ERR_LAUNCH;
  Fp8Args args = args_in;
  args.tiles_m = ceil_div(args.M, F8_BM * CTAS);
  args.tiles_n = ceil_div(args.N, BN);
  args.split = pl.split;
  args.m_group = args.tiles_m < 8 ? args.tiles_m : 8;
  args.sticky = sticky_status_slot();
  args.chain = args.out_dt == FDP_F32 ? F8_CHAIN : F8_CHAIN_16;
  CUtensorMap ma, mb, msa, msb, mo;
  if (!make_bytes_map(&ma, a, args.M, K, pitch_a, F8_BM) || !make_bytes_map(&mb, w, args.N, K, pitch_w, BN / CTAS) ||
      !make_exponents_map(&msa, sa, args.M, args.kblocks) || !make_exponents_map(&msb, sw, args.N, args.kblocks))
    return FDP_ERR_LAUNCH;
  args.direct_out = static_cast<size_t>(args.N) * dtype_size(args.out_dt) % 16 != 0 || !aligned16(args.out);
  if (args.direct_out || args.split > 1) mo = ma;
  else if (!make_out_map(&mo, args.out, args.M, args.N, args.out_dt)) return FDP_ERR_LAUNCH;
  const int units = args.tiles_m * args.tiles_n * args.split, workers = launch_sms() / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CTAS * (units < workers ? units : workers));
  cfg.blockDim = dim3(F8_THREADS);
  cfg.dynamicSmemBytes = F8Tile<CTAS, BN>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (CTAS == 2) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = 2; attr[na].val.clusterDim.y = 1; attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (pdl_enabled()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr; cfg.numAttrs = na;
  if (cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<CTAS, BN>, ma, mb, msa, msb, mo, args) != cudaSuccess) { cudaGetLastError(); return FDP_ERR_LAUNCH; }
  note_launch();
  if (args.split > 1) {
    const size_t threads = static_cast<size_t>(args.tiles_m) * args.tiles_n * (CTAS * F8_BM * BN / 4);
    launch_dependent(fp8_join_kernel<CTAS, BN>, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s, args);
    note_launch();
  }
  return FDP_OK;
}

template <typename T>
void rows_typed(const void* x, uint8_t* q, uint32_t* packed, float* scales, int rows, int cols, int pitch, cudaStream_t s) {
  const int kblocks = ceil_div(cols, 128), row_tiles = ceil_div(rows, 16);
  const unsigned grid = static_cast<unsigned>(row_tiles) * ceil_div(kblocks, QKB);
  const T* xt = static_cast<const T*>(x);
  if (cols % 8 == 0 && aligned16(x)) fp8_rows_kernel<T, true><<<grid, 256, 0, s>>>(xt, q, packed, scales, rows, cols, pitch, kblocks, row_tiles);
  else fp8_rows_kernel<T, false><<<grid, 256, 0, s>>>(xt, q, packed, scales, rows, cols, pitch, kblocks, row_tiles);
  note_launch();
}
template <typename T>
void weight_typed(const void* w, uint8_t* q, uint8_t* qt, float* scales, uint8_t* packed, uint8_t* packed_t, int rows, int cols, int pitch, int pitch_t,
                  cudaStream_t s) {
  const int cb = ceil_div(cols, 128), rb = ceil_div(rows, 128);
  const unsigned grid = static_cast<unsigned>(rb) * cb;
  const T* wt = static_cast<const T*>(w);
  if (cols % 8 == 0 && aligned16(w)) fp8_weight_kernel<T, true><<<grid, 256, 0, s>>>(wt, q, qt, scales, packed, packed_t, rows, cols, pitch, pitch_t, rb, cb);
  else fp8_weight_kernel<T, false><<<grid, 256, 0, s>>>(wt, q, qt, scales, packed, packed_t, rows, cols, pitch, pitch_t, rb, cb);
  note_launch();
}

}  // namespace

void fp8_rows(const void* x, void* q, void* packed, float* scales, int rows, int cols, int pitch, int dt, cudaStream_t s) {
  uint8_t* b = static_cast<uint8_t*>(q);
  uint32_t* p = static_cast<uint32_t*>(packed);
  if (dt == FDP_F32) rows_typed<float>(x, b, p, scales, rows, cols, pitch, s);
  else if (dt == FDP_BF16) rows_typed<__nv_bfloat16>(x, b, p, scales, rows, cols, pitch, s);
  else rows_typed<__half>(x, b, p, scales, rows, cols, pitch, s);
}
void fp8_weight(const void* w, void* q, void* qt, float* scales, void* packed, void* packed_t, int rows, int cols, int pitch, int pitch_t, int dt,
                cudaStream_t s) {
  uint8_t *b = static_cast<uint8_t*>(q), *bt = static_cast<uint8_t*>(qt), *p = static_cast<uint8_t*>(packed), *pt = static_cast<uint8_t*>(packed_t);
  if (dt == FDP_F32) weight_typed<float>(w, b, bt, scales, p, pt, rows, cols, pitch, pitch_t, s);
  else if (dt == FDP_BF16) weight_typed<__nv_bfloat16>(w, b, bt, scales, p, pt, rows, cols, pitch, pitch_t, s);
  else weight_typed<__half>(w, b, bt, scales, p, pt, rows, cols, pitch, pitch_t, s);
}

// Pair tiles of 256 x 256, single CTAs' of 128 x 128, or those cut along K, whichever is expected to take least: a K block of
// either tile takes about 0.27 us (the pair's is the tensor cores' time, the small tile's the time of its 32 KB from L2).  A
// pair's tile takes 1.6 us beside them, a small one, whose store runs beside the next tile's products, 0.4; the pair starts and
// ends half a microsecond slower (512 x 768 -> 768 bf16 with the quantisation 7.1 us in small tiles, 8.6 in pairs; 2048 x
// 2048 -> 2048, where the small tiles take two rounds, 15.8 and 14.2).  The parts of a cut go to L2 and back and take a
// launch to be added up.
Fp8Plan fp8_plan(int M, int N, int K) {
  constexpr double BLOCK = 0.27, PAIR_TILE = 1.6, PAIR = 1.3, TILE = 0.4, ONE = 0.8, JOIN = 3.0, PARTS_BYTES_A_US = 5e6;
  const int kb = ceil_div(K, 128);
  const long long pairs = static_cast<long long>(ceil_div(M, 256)) * ceil_div(N, 256), tiles = static_cast<long long>(ceil_div(M, 128)) * ceil_div(N, 128);
  Fp8Plan pl{2, 256, 1, 0};
  double best = static_cast<double>((pairs + 73) / 74) * (kb * BLOCK + PAIR_TILE) + PAIR;
  for (int split = 1; split <= 16 && split <= kb; split *= 2) {
    const double rows = M < 128 ? (M + 31) / 32 * 32 : 128;
    const double parts = split > 1 ? static_cast<double>(tiles) * split * rows * 128 * 4 : 0.0;
    const double cost = static_cast<double>((tiles * split + 147) / 148) * (ceil_div(kb, split) * BLOCK + TILE) + ONE + (split > 1 ? JOIN + 2 * parts / PARTS_BYTES_A_US : 0.0);
    if (cost < best) { best = cost; pl = Fp8Plan{1, 128, split, 0}; }
  }
  if (pl.split > 1) pl.parts_bytes = static_cast<size_t>(tiles) * pl.split * F8_BM * pl.bn * sizeof(float);
  return pl;
}

int fp8_gemm(const void* a, int pitch_a, const void* sa, const void* w, int pitch_w, const void* sw, const void* bias, int bias_dt, void* out, int M,
             int N, int K, int out_dt, float* parts, const Fp8Plan& pl, cudaStream_t s) {
  Fp8Args args{};
  args.M = M; args.N = N; args.kblocks = ceil_div(K, 128);
  args.out = out; args.out_dt = out_dt; args.bias = bias; args.bias_dt = bias_dt; args.parts = parts;
  if (pl.ctas == 2) return gemm_launch<2, 256>(args, a, pitch_a, sa, w, pitch_w, sw, K, pl, s);
  return gemm_launch<1, 128>(args, a, pitch_a, sa, w, pitch_w, sw, K, pl, s);
}

}  // namespace fdp

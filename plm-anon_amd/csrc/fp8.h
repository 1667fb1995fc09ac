// Rows of e4m3 codes with a power of two per block of 128 along K, as the 8-bit kernels see them: activations [M, K]
// and weights [N, K] alike.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 rows by 16 columns over 128 of K and takes a power of two for each
// row and each column (32 of K at a time; all four are the block's here), so a block's scales cost no instruction of
// their own and the sum over blocks is one chain of such products in fp32. Where in K a lane's 32 bytes lie is free as long
// as both operands agree: in pieces of 8, so that four lanes' pieces of 16-bit values are 64 bytes of a row. With r = row % 16,
// f = row / 16, b = k / 128, h = k / 64 % 2, p = k / 32 % 2, g = k / 8 % 4, j = k % 8:
//   code   byte ((b * fragments + f) * 2 + h) * 1024 + g * 256 + r * 16 + p * 8 + j
//   scale  byte ((b / 4) * fragments + f) * 64 + r * 4 + b % 4, holding the exponent + 127
// Lane l = 16 g + r reads 16 bytes at 16 l of either half: 1 KiB side by side per load, from memory and from LDS.
// Codes past K are zero, and so are scales (2^-127); rows past the last hold anything, since a row's codes reach only its own outputs.
// A gate/up weight's fragments alternate: fragment 2 j has gate rows [16 j, 16 j + 16), fragment 2 j + 1 the up rows.
#pragma once

#include "kv_cache.h"

namespace plm {

// Two values in 16 bits each, as to_bits16 rounds them, by one instruction.
template <int DT>
__device__ __forceinline__ uint32_t two_bits16(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  if constexpr (DT == DT_BF16) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, pair));
  } else {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, pair));
  }
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;           // of K
constexpr int64_t kFp8Bytes = 2048;      // of a fragment: 16 rows x 128 codes
constexpr int64_t kFp8ScaleBytes = 64;   // of a fragment's four blocks

__host__ __device__ constexpr int64_t fp8_frags(int64_t rows) { return (rows + 15) / 16; }
__host__ __device__ constexpr int64_t fp8_blocks(int64_t k) { return (k + kFp8Block - 1) / kFp8Block; }
__host__ __device__ constexpr int64_t fp8_codes_bytes(int64_t rows, int64_t k) { return fp8_frags(rows) * fp8_blocks(k) * kFp8Bytes; }
__host__ __device__ constexpr int64_t fp8_scales_bytes(int64_t rows, int64_t k) {
  return fp8_frags(rows) * ((fp8_blocks(k) + 3) / 4) * kFp8ScaleBytes;
}

__device__ __forceinline__ int64_t fp8_code_at(int64_t frags, int64_t row, int64_t k) {
  return ((k >> 7) * frags + (row >> 4)) * kFp8Bytes + ((k >> 6) & 1) * 1024 + ((k >> 3) & 3) * 256 + (row & 15) * 16 +
         ((k >> 5) & 1) * 8 + (k & 7);
}
// Where in K the four pieces of eight of a lane lie, in its codes' order.
__device__ __forceinline__ int fp8_piece_at(int64_t kb, int lane, int i) { return static_cast<int>(kb) * kFp8Block + i * 32 + (lane >> 4) * 8; }
__device__ __forceinline__ int64_t fp8_scale_at(int64_t frags, int64_t row, int64_t block) {
  return ((block >> 2) * frags + (row >> 4)) * kFp8ScaleBytes + (row & 15) * 4 + (block & 3);
}

// A block's scale, and after the last block's zeros up to the next multiple of four.
__device__ __forceinline__ void fp8_put_scale(uint8_t* scales, int64_t frags, int64_t row, int64_t block, int64_t blocks, uint8_t e) {
  uint8_t* at = scales + fp8_scale_at(frags, row, block);
  *at = e;
  if (block == blocks - 1)
    for (int i = 1; i < 4 - static_cast<int>(block & 3); ++i) at[i] = 0;
}

// Where a weight's row lies: of gate/up the halves' fragments alternate (n: rows of both, a multiple of 32).
__device__ __forceinline__ int64_t fp8_place(int64_t row, int64_t n, bool gate_up) {
  if (!gate_up) return row;
  const int64_t half = n >> 1, up = row >= half ? 1 : 0, i = row - up * half;
  return ((i >> 4) * 2 + up) * 16 + (i & 15);
}

__device__ __forceinline__ uint8_t fp8_exponent(float scale) { return static_cast<uint8_t>(__builtin_bit_cast(uint32_t, scale) >> 23); }
__device__ __forceinline__ float fp8_power(uint32_t exponent) { return __builtin_bit_cast(float, exponent << 23); }
// 1 / scale, for scales up to 2^126.
__device__ __forceinline__ float fp8_inverse(float scale) {
  return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, scale));
}

// |x| for the largest magnitude of a block: what is not finite has no part in it.
__device__ __forceinline__ float fp8_magnitude(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;
}

// The largest magnitude of 32 values of 16 bits, as bits: of finite ones it is their largest, else at least fp8_infinite.
template <int DT>
__device__ __forceinline__ constexpr uint32_t fp8_infinite() {
  return DT == DT_BF16 ? 0x7f80u : 0x7c00u;
}
template <int DT, typename... W>
__device__ __forceinline__ uint32_t fp8_most16(W... words) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 most = {0, 0};
  auto add = [&](u32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
  };
  (add(words), ...);
  return max(static_cast<uint32_t>(most[0]), static_cast<uint32_t>(most[1]));
}

// Codes of four finite 16-bit values, two in a word, over a scale that bounds them.
template <int DT>
__device__ __forceinline__ uint32_t fp8_four(uint32_t lo, uint32_t hi, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 w = {0, 0};
  if constexpr (DT == DT_BF16) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, hi), scale, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, lo), scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(w, __builtin_bit_cast(f16x2, hi), scale, true);
  }
  return __builtin_bit_cast(uint32_t, w);
}

__device__ __forceinline__ uint32_t fp8_four(float a, float b, float c, float d, float scale) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, w);
}

// Codes of 32 values of any kind and their scale; `share` gives the largest magnitude of the lanes that have a block.
template <int DT, typename F>
__device__ __forceinline__ float fp8_round_any(const u32x4 (&raw)[4], F share, i32x8& codes) {
  float v[32], amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = from_bits16<DT>(static_cast<uint16_t>(raw[i >> 3][(i & 7) >> 1] >> (16 * (i & 1))));
    amax = fmaxf(amax, fp8_magnitude(v[i]));
  }
  const float scale = fp8_scale_of(share(amax)), inverse = fp8_inverse(scale);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    codes[i] = static_cast<int>(fp8_word(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse));
  return scale;
}

// c += rows of `a` times rows of `b` over one block, times the scales in the low bytes of sa and sb. The instruction adds
// products in eights (k, k + 1, .., k + 7 of a lane), aligned to the largest sum of two factors' exponents among them (a subnormal
// code's is -6) and cut at 2^-13 of two to that, and the eights' sums in fp32 (measured; so does the older
// v_mfma_f32_16x16x32_fp8_fp8). The cut is toward zero, of either sign alike, so it has no mean where products have both signs. Measured from K = 512 to 65536, of a result's size (rms): 1.5e-5 over
// normal rows and weights, 4e-5 where a hundredth of the rows' channels is 16 times as large; over values of one sign a mean of
// -2.4e-6. bf16's rounding is 1.7e-3, fp16's 2.1e-4 (with the cut of such channels 2.12e-4 for 2.08e-4). Results in fp32 are
// made by fp8_mma_exact.
__device__ __forceinline__ f32x4 fp8_mma(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// The same with every product added in fp32: codes times half their scales are bf16 values, exactly, four products of 32 deep.
// Half, since the largest of a row may have rounded up to 2^128, which bf16 does not hold; sums are a quarter of what they
// stand for (kFp8Exact), without a loss at the other end: products are whole numbers of 2^-148.
constexpr float kFp8Exact = 4.0f;
struct Fp8Exact {
  u32x4 part[4];
};
__device__ __forceinline__ Fp8Exact fp8_exact(i32x8 v, int scale) {
  const float s = 0.5f * fp8_power(static_cast<uint32_t>(scale));
  Fp8Exact e;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    e.part[i] = fp8_eight<DT_BF16>(static_cast<uint32_t>(v[2 * i]), static_cast<uint32_t>(v[2 * i + 1]), s);
  return e;
}
__device__ __forceinline__ f32x4 fp8_mma_exact(const Fp8Exact& a, const Fp8Exact& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = mfma_16x16x32<DT_BF16>(a.part[i], b.part[i], c);
  return c;
}

__device__ __forceinline__ i32x8 fp8_operand(u32x4 lo, u32x4 hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

}  // namespace plm

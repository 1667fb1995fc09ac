// The products over e4m3 rows (plm_fp8_linear): what their kernels share.
#pragma once

#include "fp8.h"
#include "fp8_plan.h"
#include "plm_amd.h"

namespace plm {

struct Fp8Gemm {
  const uint8_t* x;         // codes of [m, k], or rows of 16 bits (x_type: plm_fp8_in)
  const uint8_t* x_scales;
  const uint8_t* w;         // codes of [n, k]
  const uint8_t* w_scales;
  void* y;
  f32x4* partials;          // of products whose K is cut into ranges
  int64_t ldy, x_row;       // x_row: stride of 16-bit rows
  int m, n, k, blocks;      // n: rows of the weight; blocks of K
  int range;                // blocks of a range
  int x_frags, w_frags, x_type, out;  // out: plm_fp8_out
};

// 16 and 8 bytes at any even address, which one store writes: rows of an odd length begin anywhere.
typedef u32x4 fp8_any16 __attribute__((aligned(2)));
typedef u32x2 fp8_any8 __attribute__((aligned(2)));

// g / (1 + e^-g) * u in fp32. With h = e^(-|g| / 2), which has no overflow and underflows where h^2 does twice over, that is
// g / (1 + h^2) u, times h^2 where g is negative: one h with g's part and one with u, as g h^2 underflows long before its
// product with a large u does. The exponent in base 2 is a product's two parts, the second of which is put
// on behind; exponential and reciprocal are the instructions of 1 ulp: 2^-20 of the result at most, for g down to -174, where h
// is normal (largest measured 3.7 times 2^-24; with expf and a division 1.7). 16 instructions for
// about 45 with expf and a division (gate/up of 11264 x 2048 over 4096 rows 85 us for 95).
__device__ __forceinline__ float fp8_silu_mul(float g, float u) {
  constexpr float kHalf = 0x1.715476p-1f, kRest = 0x1.4ae0cp-27f, kLn2 = 0x1.62e43p-1f;   // kHalf + kRest = log2(e) / 2
  const float a = fminf(fabsf(g), 512.0f), t = -a * kHalf;
  const float rest = fmaf(-a, kRest, fmaf(-a, kHalf, -t));
  float h = __builtin_amdgcn_exp2f(t);
  h = fmaf(h, rest * kLn2, h);
  const float p = g * __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f)), f = g < 0.0f ? h : 1.0f;
  return (p * f) * (f * u);
}

// Columns [n, n + 4) of row m, of `columns` in all.
__device__ __forceinline__ void fp8_store4(const Fp8Gemm& a, int m, int n, int columns, f32x4 v) {
  const int64_t at = m * a.ldy + n;
  const int left = columns - n;
  if (a.out == PLM_FP8_F32) {
    float* y = static_cast<float*>(a.y) + at;
    if (left >= 4) {
      *reinterpret_cast<fp8_any16*>(y) = __builtin_bit_cast(u32x4, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) y[j] = v[j];
    }
    return;
  }
  const uint32_t lo = a.out == PLM_FP8_BF16 ? two_bits16<DT_BF16>(v[0], v[1]) : two_bits16<DT_F16>(v[0], v[1]);
  const uint32_t hi = a.out == PLM_FP8_BF16 ? two_bits16<DT_BF16>(v[2], v[3]) : two_bits16<DT_F16>(v[2], v[3]);
  uint16_t* y = static_cast<uint16_t*>(a.y) + at;
  if (left >= 4) {
    *reinterpret_cast<fp8_any8*>(y) = u32x2{lo, hi};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) y[j] = static_cast<uint16_t>((j < 2 ? lo : hi) >> (16 * (j & 1)));
  }
}

// Rows of 16 bits (plm_dtype) into codes and scales.
hipError_t fp8_round(int dtype, const void* x, int64_t x_row, int64_t rows, int64_t k, uint8_t* codes, uint8_t* scales, hipStream_t s);
hipError_t fp8_narrow(Fp8Gemm a, const Fp8Narrow& p, bool act, hipStream_t s);
hipError_t fp8_tile(const Fp8Gemm& a, Fp8TileKind kind, bool act, hipStream_t s);

}  // namespace plm

// Products over e4m3 rows for few rows of X: bound by the weight's bytes.
//
// A workgroup has NF fragments of the weight (16 NF of its rows) and MT of X; its KW wavefronts take every KW-th block of
// K, each operand straight from memory into registers, and their sums are added in LDS in the wavefronts' order.
#include <hip/hip_runtime.h>

#include "fp8_gemm.h"

namespace plm {
namespace {

template <int MT, int NF, int KW, bool ACT, bool EXACT>
__global__ __launch_bounds__(64 * KW) void narrow_kernel(Fp8Gemm a) {
  extern __shared__ __attribute__((aligned(16))) f32x4 red[];   // [KW][NF * MT][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int f0 = blockIdx.x * NF, t0 = blockIdx.y * MT;
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = wave; kb < a.blocks; kb += KW) {
    i32x8 w[NF], x[MT];
    int ws[NF], xs[MT];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int frag = min(f0 + f, a.w_frags - 1);
      const uint8_t* p = a.w + (static_cast<int64_t>(kb) * a.w_frags + frag) * kFp8Bytes + lane * 16;
      w[f] = fp8_operand(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 1024));
      ws[f] = a.w_scales[(static_cast<int64_t>(kb >> 2) * a.w_frags + frag) * kFp8ScaleBytes + (lane & 15) * 4 + (kb & 3)];
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int frag = min(t0 + t, a.x_frags - 1);
      const uint8_t* p = a.x + (static_cast<int64_t>(kb) * a.x_frags + frag) * kFp8Bytes + lane * 16;
      x[t] = fp8_operand(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 1024));
      xs[t] = a.x_scales[(static_cast<int64_t>(kb >> 2) * a.x_frags + frag) * kFp8ScaleBytes + (lane & 15) * 4 + (kb & 3)];
    }
    if constexpr (EXACT) {
      Fp8Exact xe[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xe[t] = fp8_exact(x[t], xs[t]);
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const Fp8Exact we = fp8_exact(w[f], ws[f]);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = fp8_mma_exact(we, xe[t], acc[f][t]);
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = fp8_mma(w[f], x[t], acc[f][t], ws[f], xs[t]);
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[(wave * NF * MT + f * MT + t) * 64 + lane] = acc[f][t];
  __syncthreads();
  constexpr int kOut = ACT ? NF / 2 : NF;
  for (int o = wave; o < kOut * MT; o += KW) {
    const int f = o / MT, t = o - f * MT;
    const int m = (t0 + t) * 16 + (lane & 15);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f}, u = v;
    const int at = (ACT ? 2 * f : f) * MT + t;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      v += red[(k * NF * MT + at) * 64 + lane];
      if constexpr (ACT) u += red[(k * NF * MT + at + MT) * 64 + lane];
    }
    if constexpr (ACT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fp8_silu_mul(v[j], u[j]);
    }
    const int columns = ACT ? a.n / 2 : a.n, n = ((ACT ? f0 / 2 : f0) + f) * 16 + (lane >> 4) * 4;
    if (m < a.m && n < columns) fp8_store4(a, m, n, columns, v);
  }
}

template <int MT, int NF, int KW, bool ACT, bool EXACT>
hipError_t launch(const Fp8Gemm& a, hipStream_t s) {
  constexpr int lds = KW * NF * MT * 1024;
  static_assert(lds <= 64 * 1024, "above 64 KiB a kernel has to ask for its LDS");
  const dim3 grid(static_cast<unsigned>((a.w_frags + NF - 1) / NF), static_cast<unsigned>((a.x_frags + MT - 1) / MT));
  hipLaunchKernelGGL((narrow_kernel<MT, NF, KW, ACT, EXACT>), grid, dim3(64 * KW), lds, s, a);
  return hipGetLastError();
}

template <bool ACT, bool EXACT>
hipError_t pick(const Fp8Gemm& a, hipStream_t s) {
  if (a.x_frags == 1) return launch<1, 2, 8, ACT, EXACT>(a, s);
  if (a.x_frags == 2) return launch<2, 2, 8, ACT, EXACT>(a, s);
  return launch<4, 2, 8, ACT, EXACT>(a, s);
}

}  // namespace

hipError_t fp8_narrow(const Fp8Gemm& a, bool act, hipStream_t s) {
  if (a.out == PLM_FP8_F32) return act ? pick<true, true>(a, s) : pick<false, true>(a, s);
  return act ? pick<true, false>(a, s) : pick<false, false>(a, s);
}

}  // namespace plm

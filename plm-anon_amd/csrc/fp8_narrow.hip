// Products over e4m3 rows for few rows of X: bound by the weight's bytes.
//
// A workgroup has NF fragments of the weight (16 NF of its rows) and MT of X; its KW wavefronts take every KW-th block of
// K, each operand straight from memory into registers, a block ahead, and their sums are added in LDS in the wavefronts'
// order. A CU pulls about 24 GB/s from memory and 94 from its L2, so all of them have to read: where a weight has few rows, K
// is cut into ranges of workgroups, whose partial sums a second launch adds (narrow_plan).
//
// Measured, weights from memory: 50257 x 2048 over 16 rows 21.7 us (4.7 TB/s), over 56 32.5 (of a CU's reads two thirds are X, so
// tiles take it, 27.2), 6144 x 2048 over 56 rows 6.1, 2048 x 2048 over one row 3.4. Four fragments of the weight to a
// workgroup, so that X is read half as often: gate/up 10.2 for 10.7, but the LM head at 56 rows 35 for 33.4, 6144 x 2048 8.7 for
// 6.7. Nontemporal loads of the weight: 2 to 12 % less from memory (down of 2560 x 10240 at 42 rows 11.6 for 12.6), 3 to 30 %
// more for weights that the 256 MB cache still holds (10.2 for 9.1); not done.
//
// Up to 16 rows of 16 bits are rounded to 8 here, by every workgroup for itself (XT: plm_fp8_in): as the rounding of their own
// launch does, without the launch.
#include <hip/hip_runtime.h>

#include "fp8_gemm.h"

namespace plm {
namespace {

template <int MT, int NF>
struct Operands {
  i32x8 w[NF], x[MT];
  int ws[NF], xs[MT];
  u32x4 raw[4];   // of 16-bit rows: this lane's 32 values
};

template <int MT, int NF, int XT>
__device__ __forceinline__ void load(const Fp8Gemm& a, int kb, int f0, int t0, int lane, Operands<MT, NF>& o) {
  const uint8_t* w = a.w + static_cast<int64_t>(kb) * a.w_frags * kFp8Bytes;
  const uint8_t* ws = a.w_scales + static_cast<int64_t>(kb >> 2) * a.w_frags * kFp8ScaleBytes + (kb & 3);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const uint32_t frag = min(f0 + f, a.w_frags - 1);
    const uint8_t* p = w + (frag * static_cast<uint32_t>(kFp8Bytes) + lane * 16);
    o.w[f] = fp8_operand(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 1024));
    o.ws[f] = ws[frag * static_cast<uint32_t>(kFp8ScaleBytes) + (lane & 15) * 4];
  }
  if constexpr (XT == PLM_FP8_CODES) {
    const uint8_t* x = a.x + static_cast<int64_t>(kb) * a.x_frags * kFp8Bytes;
    const uint8_t* xs = a.x_scales + static_cast<int64_t>(kb >> 2) * a.x_frags * kFp8ScaleBytes + (kb & 3);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      // Rows past the last read the first: a single token's is a sixteenth of its fragment.
      const int row_of = (t0 + t) * 16 + (lane & 15), there = row_of < a.m ? row_of : t0 * 16;
      const uint8_t* p = x + (static_cast<uint32_t>(there >> 4) * static_cast<uint32_t>(kFp8Bytes) + (lane >> 4) * 256 + (there & 15) * 16);
      o.x[t] = fp8_operand(*reinterpret_cast<const u32x4*>(p), *reinterpret_cast<const u32x4*>(p + 1024));
      o.xs[t] = xs[static_cast<uint32_t>(there >> 4) * static_cast<uint32_t>(kFp8ScaleBytes) + (there & 15) * 4];
    }
  } else {
    const int r = (lane & 15) < a.m ? lane & 15 : 0;
    const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x) + r * a.x_row;
#pragma unroll
    for (int i = 0; i < 4; ++i)   // past k anything: round_rows puts zeros there
      o.raw[i] = *reinterpret_cast<const u32x4*>(x + min(fp8_piece_at(kb, lane, i), a.k - 8));
  }
}

// The lane's 32 values of a row's block in 8 bits, with the scale of the row's other three lanes too.
template <int MT, int NF, int XT>
__device__ __forceinline__ void round_rows(Operands<MT, NF>& o, int kb, int k, int lane) {
  constexpr int DT = XT == PLM_FP8_ROWS_BF16 ? DT_BF16 : DT_F16;
  if ((kb + 1) * kFp8Block > k) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (fp8_piece_at(kb, lane, i) >= k) o.raw[i] = u32x4{0u, 0u, 0u, 0u};
  }
  const uint32_t most = fp8_most16<DT>(o.raw[0], o.raw[1], o.raw[2], o.raw[3]);
  const uint32_t of_row = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
  const uint32_t amax = max(of_row, static_cast<uint32_t>(__shfl_xor(static_cast<int>(of_row), 32)));
  if (__builtin_expect(__ballot(amax >= fp8_infinite<DT>()) != 0, 0)) {
    const float scale = fp8_round_any<DT>(o.raw, [](float v) { return fmaxf(fmaxf(v, __shfl_xor(v, 16)), __shfl_xor(fmaxf(v, __shfl_xor(v, 16)), 32)); },
                                          o.x[0]);
    o.xs[0] = fp8_exponent(scale);
    return;
  }
  const float scale = fp8_scale_of(from_bits16<DT>(static_cast<uint16_t>(amax)));
#pragma unroll
  for (int i = 0; i < 8; ++i) o.x[0][i] = static_cast<int>(fp8_four<DT>(o.raw[i >> 1][2 * (i & 1)], o.raw[i >> 1][2 * (i & 1) + 1], scale));
  o.xs[0] = fp8_exponent(scale);
}

template <int MT, int NF, int XT, bool EXACT>
__device__ __forceinline__ void multiply(Operands<MT, NF>& o, int kb, int k, int lane, f32x4 (&acc)[NF][MT]) {
  if constexpr (XT != PLM_FP8_CODES) round_rows<MT, NF, XT>(o, kb, k, lane);
  if constexpr (EXACT) {
    Fp8Exact x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = fp8_exact(o.x[t], o.xs[t]);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const Fp8Exact w = fp8_exact(o.w[f], o.ws[f]);
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[f][t] = fp8_mma_exact(w, x[t], acc[f][t]);
    }
  } else {
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[f][t] = fp8_mma(o.w[f], o.x[t], acc[f][t], o.ws[f], o.xs[t]);
  }
}

// A finished fragment's four columns of a lane; `n`: the first of them.
template <bool ACT>
__device__ __forceinline__ void finish(const Fp8Gemm& a, int m, int n, f32x4 v, f32x4 u) {
  if constexpr (ACT) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = fp8_silu_mul(v[j], u[j]);
  }
  const int columns = ACT ? a.n / 2 : a.n;
  if (m < a.m && n < columns) fp8_store4(a, m, n, columns, v);
}

template <int MT, int NF, int KW, int XT, bool ACT, bool EXACT>
__global__ __launch_bounds__(64 * KW) void narrow_kernel(Fp8Gemm a) {
  __shared__ __attribute__((aligned(16))) f32x4 red[KW * NF * MT * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = blockIdx.x * NF, t0 = blockIdx.y * MT;
  const int first = blockIdx.z * a.range, end = min(a.blocks, first + a.range);
  f32x4 acc[NF][MT];
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  int kb = first + wave;
  if (kb < end) {
    Operands<MT, NF> o[2];
    load<MT, NF, XT>(a, kb, f0, t0, lane, o[0]);
#pragma unroll 1
    for (; kb + 2 * KW < end; kb += 2 * KW) {
      load<MT, NF, XT>(a, kb + KW, f0, t0, lane, o[1]);
      multiply<MT, NF, XT, EXACT>(o[0], kb, a.k, lane, acc);
      load<MT, NF, XT>(a, kb + 2 * KW, f0, t0, lane, o[0]);
      multiply<MT, NF, XT, EXACT>(o[1], kb + KW, a.k, lane, acc);
    }
    if (kb + KW < end) {
      load<MT, NF, XT>(a, kb + KW, f0, t0, lane, o[1]);
      multiply<MT, NF, XT, EXACT>(o[0], kb, a.k, lane, acc);
      multiply<MT, NF, XT, EXACT>(o[1], kb + KW, a.k, lane, acc);
    } else {
      multiply<MT, NF, XT, EXACT>(o[0], kb, a.k, lane, acc);
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[((wave * NF + f) * MT + t) * 64 + lane] = EXACT ? acc[f][t] * kFp8Exact : acc[f][t];
  __syncthreads();
  auto sum = [&](int at) {
    f32x4 v = red[at * 64 + lane];
#pragma unroll
    for (int k = 1; k < KW; ++k) v += red[(k * NF * MT + at) * 64 + lane];
    return v;
  };
  if (gridDim.z > 1) {
    // Partial sums [range][fragment of X][fragment of the weight][lane].
    for (int at = wave; at < NF * MT; at += KW) {
      const int f = at / MT, t = at - f * MT;
      if (f0 + f < a.w_frags && t0 + t < a.x_frags)
        a.partials[((static_cast<int64_t>(blockIdx.z) * a.x_frags + t0 + t) * a.w_frags + f0 + f) * 64 + lane] = sum(at);
    }
    return;
  }
  constexpr int kOut = ACT ? NF / 2 : NF;
  for (int at = wave; at < kOut * MT; at += KW) {
    const int f = at / MT, t = at - f * MT, m = (t0 + t) * 16 + (lane & 15);
    if constexpr (ACT) {
      finish<true>(a, m, (f0 / 2 + f) * 16 + (lane >> 4) * 4, sum(2 * f * MT + t), sum((2 * f + 1) * MT + t));
    } else {
      const f32x4 v = sum(at);
      finish<false>(a, m, (f0 + f) * 16 + (lane >> 4) * 4, v, v);
    }
  }
}

// The ranges' partial sums, in their order: a wavefront has a fragment of the output.
template <bool ACT>
__global__ __launch_bounds__(256) void join_kernel(Fp8Gemm a, int ranges, int frags) {
  const int at = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (at >= frags) return;
  const int columns = ACT ? a.w_frags / 2 : a.w_frags, t = at / columns, f = at - t * columns;
  auto sum = [&](int frag) {
    const f32x4* p = a.partials + (static_cast<int64_t>(t) * a.w_frags + frag) * 64 + lane;
    f32x4 v = p[0];
    for (int r = 1; r < ranges; ++r) v += p[static_cast<int64_t>(r) * a.x_frags * a.w_frags * 64];
    return v;
  };
  const f32x4 v = sum(ACT ? 2 * f : f), u = ACT ? sum(2 * f + 1) : v;
  finish<ACT>(a, t * 16 + (lane & 15), f * 16 + (lane >> 4) * 4, v, u);
}

template <int MT, int NF, int KW, int XT, bool ACT, bool EXACT>
void launch(const Fp8Gemm& a, const Fp8Narrow& p, hipStream_t s) {
  const int columns = (a.w_frags + NF - 1) / NF;
  const dim3 grid(static_cast<unsigned>(columns), static_cast<unsigned>((a.x_frags + MT - 1) / MT), static_cast<unsigned>(p.ranges));
  hipLaunchKernelGGL((narrow_kernel<MT, NF, KW, XT, ACT, EXACT>), grid, dim3(64 * KW), 0, s, a);
}

template <int MT, int XT, bool ACT, bool EXACT>
void pick_width(const Fp8Gemm& a, const Fp8Narrow& p, hipStream_t s) {
  if constexpr (XT != PLM_FP8_CODES) {
    if (p.waves == 4) return launch<MT, 2, 4, XT, ACT, EXACT>(a, p, s);
  }
  if constexpr (!ACT) {
    if (p.width == 1) return launch<MT, 1, 8, XT, ACT, EXACT>(a, p, s);
  }
  launch<MT, 2, 8, XT, ACT, EXACT>(a, p, s);
}

template <bool ACT, bool EXACT>
void pick_rows(const Fp8Gemm& a, const Fp8Narrow& p, hipStream_t s) {
  if (a.x_type == PLM_FP8_ROWS_BF16) return pick_width<1, PLM_FP8_ROWS_BF16, ACT, EXACT>(a, p, s);
  if (a.x_type == PLM_FP8_ROWS_F16) return pick_width<1, PLM_FP8_ROWS_F16, ACT, EXACT>(a, p, s);
  switch (p.rows) {
    case 1: return pick_width<1, PLM_FP8_CODES, ACT, EXACT>(a, p, s);
    case 2: return pick_width<2, PLM_FP8_CODES, ACT, EXACT>(a, p, s);
    case 3: return pick_width<3, PLM_FP8_CODES, ACT, EXACT>(a, p, s);
    default: return pick_width<4, PLM_FP8_CODES, ACT, EXACT>(a, p, s);
  }
}

}  // namespace

hipError_t fp8_narrow(Fp8Gemm a, const Fp8Narrow& p, bool act, hipStream_t s) {
  a.range = (a.blocks + p.ranges - 1) / p.ranges;
  const bool exact = a.out == PLM_FP8_F32;
  if (act) exact ? pick_rows<true, true>(a, p, s) : pick_rows<true, false>(a, p, s);
  else exact ? pick_rows<false, true>(a, p, s) : pick_rows<false, false>(a, p, s);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.ranges == 1) return err;
  const int frags = (act ? a.w_frags / 2 : a.w_frags) * a.x_frags;
  const dim3 grid(static_cast<unsigned>((frags + 3) / 4));
  if (act) hipLaunchKernelGGL((join_kernel<true>), grid, dim3(256), 0, s, a, p.ranges, frags);
  else hipLaunchKernelGGL((join_kernel<false>), grid, dim3(256), 0, s, a, p.ranges, frags);
  return hipGetLastError();
}

}  // namespace plm

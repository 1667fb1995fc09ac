// Rows into 8 bits (plm_fp8_rows), with the root-mean-square norm and the residual's addition before it or the norm in
// 16 bits; weights into 8 bits or into the kernels' order (plm_fp8_weight, plm_fp8_pack) and back to values
// (plm_fp8_values). Declared in include/plm_amd.h; order of the bytes: fp8.h.
//
// Norm: t = x + residual, rounded to the model's type (so that the norm of the returned sum is the same); y = t w / sqrt(
// mean(t^2) + eps). The sum of squares is fp64: squares of 16-bit values are exact in fp32, four of them are added in
// fp32 at most. y in fp32 is off by three roundings; a code has 2^20 fp32 values to a step, so of a million values one to
// four would come out on the other side of a border between codes: what is that close is computed in fp64 and
// rounded once, the scale's border likewise.
#include <hip/hip_runtime.h>

#include "fp8.h"
#include "plm_amd.h"

namespace plm {
namespace {

struct RowsArgs {
  const uint16_t* x;
  const uint16_t* residual;
  const uint16_t* weight;  // null: no multiplication
  uint16_t* sum;           // contiguous [rows, k]
  uint16_t* y;             // contiguous [rows, k], or null: codes
  uint8_t* codes;
  uint8_t* scales;
  int64_t x_row, residual_row, frags;
  double eps;
  int rows, k;
};

template <int DT>
__device__ __forceinline__ void unpack8(u32x4 v, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = from_bits16<DT>(static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1))));
}

template <int DT>
__device__ __forceinline__ u32x4 pack8of(const float* x) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = to_bits16<DT>(x[2 * i]) | (static_cast<uint32_t>(to_bits16<DT>(x[2 * i + 1])) << 16);
  return o;
}

// A double as the fp32 value on either side whose last bit is set, if it is not one itself: rounded again to fewer bits that
// is as if rounded once.
__device__ __forceinline__ float odd_float(double v) {
  const float near = static_cast<float>(v);
  const double off = v - static_cast<double>(near);
  uint32_t bits = __builtin_bit_cast(uint32_t, near);
  if (fabs(off) > 0.0 && fabs(off) < __builtin_inf() && (bits & 1u) == 0u)
    bits += (off < 0.0) == ((bits >> 31) != 0u) ? 1u : ~0u;
  return __builtin_bit_cast(float, bits);
}

// Sixteen values of a row from `at`, a multiple of 16 (k is one of 8), zeros past k.
template <int DT>
__device__ __forceinline__ void load16(const uint16_t* row, int at, int k, u32x4 (&v)[2]) {
  v[0] = at < k ? *reinterpret_cast<const u32x4*>(row + at) : u32x4{0u, 0u, 0u, 0u};
  v[1] = at + 8 < k ? *reinterpret_cast<const u32x4*>(row + at + 8) : u32x4{0u, 0u, 0u, 0u};
}

// x + residual, rounded.
template <int DT>
__device__ __forceinline__ void add16(u32x4 (&v)[2], const u32x4 (&r)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[8], y[8];
    unpack8<DT>(v[h], x);
    unpack8<DT>(r[h], y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] += y[i];
    v[h] = pack8of<DT>(x);
  }
}

__device__ __forceinline__ void store16(uint16_t* row, int at, int k, const u32x4 (&v)[2]) {
  if (at < k) *reinterpret_cast<u32x4*>(row + at) = v[0];
  if (at + 8 < k) *reinterpret_cast<u32x4*>(row + at + 8) = v[1];
}

// A row's norm: 1 / sqrt(mean + eps) in both widths.
struct Norm {
  double exact;
  float near;
  bool wide;   // outside of what fp32 steps stay accurate in: every value in fp64
};

// y of sixteen values. `close` gets the bit of each that is within its error (three roundings, 2^-22 is more than twice
// that) of a place where codes may part: at most four bits of mantissa, so 19 zeros at the end.
template <int DT, bool NORM, bool WEIGHT>
__device__ __forceinline__ void normed16(const RowsArgs& a, const Norm& norm, const u32x4 (&v)[2], int at, float (&y)[16],
                                         uint32_t& close) {
  unpack8<DT>(v[0], y);
  unpack8<DT>(v[1], y + 8);
  close = 0;
  if constexpr (NORM) {
    float w[16];
    if constexpr (WEIGHT) {
      u32x4 of[2];
      load16<DT>(a.weight, at, a.k, of);
      unpack8<DT>(of[0], w);
      unpack8<DT>(of[1], w + 8);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      y[i] *= norm.near;
      if constexpr (WEIGHT) y[i] *= w[i];
      const float border = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, y[i]) + 0x40000u) & 0xfff80000u);
      close |= fabsf(y[i] - border) < 0x1p-22f * fabsf(y[i]) || (norm.wide && at + i < a.k) ? 1u << i : 0u;
    }
  }
}

// The values of `close`, in fp64 and rounded to odd.
template <int DT, bool WEIGHT>
__device__ __forceinline__ void normed_exact(const RowsArgs& a, const Norm& norm, const u32x4 (&v)[2], int at, uint32_t close,
                                             float (&y)[16]) {
  for (; close != 0; close &= close - 1) {
    const int j = __builtin_ctz(close);
    uint32_t word = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n)
      if (n == j >> 1) word = v[n >> 2][n & 3];
    double exact = static_cast<double>(from_bits16<DT>(static_cast<uint16_t>(word >> (16 * (j & 1))))) * norm.exact;
    if constexpr (WEIGHT) exact *= static_cast<double>(from_bits16<DT>(a.weight[at + j]));
    const float odd = odd_float(exact);
#pragma unroll
    for (int n = 0; n < 16; ++n)
      if (n == j) y[n] = odd;
  }
}

// Sixteen values of a row, of `row`'s 16-bit v, into the output.
template <int DT, bool NORM, bool WEIGHT, bool E8>
__device__ __forceinline__ void emit16(const RowsArgs& a, const Norm& norm, int64_t row, int at, const u32x4 (&v)[2]) {
  float y[16];
  uint32_t close;
  normed16<DT, NORM, WEIGHT>(a, norm, v, at, y, close);
  if constexpr (NORM) {
    if (E8 || norm.wide) normed_exact<DT, WEIGHT>(a, norm, v, at, close, y);
  }
  if constexpr (!E8) {
    const u32x4 o[2] = {pack8of<DT>(y), pack8of<DT>(y + 8)};
    store16(a.y + row * a.k, at, a.k, o);
  } else {
    // 448 is among the borders above: a value that could lie on either side of it has been computed exactly.
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fp8_magnitude(y[j]));
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    const float scale = fp8_scale_of(amax), inverse = fp8_inverse(scale);
    const int block = at >> 7;
    if (block < static_cast<int>(fp8_blocks(a.k))) {
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = fp8_word(y[4 * j] * inverse, y[4 * j + 1] * inverse, y[4 * j + 2] * inverse, y[4 * j + 3] * inverse);
      *reinterpret_cast<u32x4*>(a.codes + fp8_code_at(a.frags, row, at)) = o;
      if ((threadIdx.x & 7) == 0) fp8_put_scale(a.scales, a.frags, row, block, fp8_blocks(a.k), fp8_exponent(scale));
    }
  }
}

// Chunks of 16 values of a row; whole blocks where codes are written, whose zeros past k are part of them.
template <bool E8>
__device__ __forceinline__ int row_chunks(int k) {
  return E8 ? static_cast<int>(fp8_blocks(k)) * 8 : (k + 15) / 16;
}

// A wavefront takes a row, a lane the sixteen values at 16 (lane + 64 i); eight lanes have a block. HELD chunks stay in
// registers between the sum of squares and the output; the rest of a longer row is read again.
template <int DT, bool RES, bool WEIGHT, bool E8, int HELD>
__global__ __launch_bounds__(1024) void norm_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 6) + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int turns = (row_chunks<E8>(a.k) + 63) / 64;
  const uint16_t* x = a.x + row * a.x_row;
  const uint16_t* residual = RES ? a.residual + row * a.residual_row : nullptr;
  uint16_t* sum = RES ? a.sum + row * a.k : nullptr;
  double squares = 0.0;
  auto add = [&](const u32x4 (&v)[2]) {
    float f[16];
    unpack8<DT>(v[0], f);
    unpack8<DT>(v[1], f + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) squares = fma(static_cast<double>(f[j]), static_cast<double>(f[j]), squares);
  };
  u32x4 held[HELD][2], more[RES ? HELD : 1][2];
#pragma unroll
  for (int i = 0; i < HELD; ++i) {   // every load before the first store, which it may not pass
    load16<DT>(x, 16 * (lane + 64 * i), a.k, held[i]);
    if constexpr (RES) load16<DT>(residual, 16 * (lane + 64 * i), a.k, more[i]);
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    if constexpr (RES) {
      add16<DT>(held[i], more[i]);
      store16(sum, 16 * (lane + 64 * i), a.k, held[i]);
    }
    add(held[i]);
  }
  for (int i = HELD; i < turns; ++i) {
    u32x4 v[2];
    load16<DT>(x, 16 * (lane + 64 * i), a.k, v);
    if constexpr (RES) {
      u32x4 r[2];
      load16<DT>(residual, 16 * (lane + 64 * i), a.k, r);
      add16<DT>(v, r);
      store16(sum, 16 * (lane + 64 * i), a.k, v);
    }
    add(v);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) squares += __shfl_xor(squares, d);
  Norm norm;
  norm.exact = 1.0 / sqrt(squares / a.k + a.eps);
  norm.near = static_cast<float>(norm.exact);
  norm.wide = !(norm.near > 0x1p-100f && norm.near < 0x1p100f);
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (i < turns) emit16<DT, true, WEIGHT, E8>(a, norm, row, 16 * (lane + 64 * i), held[i]);
  for (int i = HELD; i < turns; ++i) {
    u32x4 v[2];
    load16<DT>(RES ? sum : x, 16 * (lane + 64 * i), a.k, v);   // of the sum this lane's own stores
    emit16<DT, true, WEIGHT, E8>(a, norm, row, 16 * (lane + 64 * i), v);
  }
}

// Rows as they are: every 64 chunks of a row a wavefront's of its own.
template <int DT>
__global__ __launch_bounds__(1024) void round_kernel(RowsArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 6) + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const int at = 16 * (static_cast<int>(blockIdx.y) * 64 + static_cast<int>(threadIdx.x & 63));
  u32x4 v[2];
  load16<DT>(a.x + row * a.x_row, at, a.k, v);
  emit16<DT, false, false, true>(a, Norm{0.0, 1.0f, false}, row, at, v);
}

struct WeightArgs {
  const uint16_t* w;       // values to round, row stride ld; or
  const uint8_t* plain;    // codes [n, k], row stride ld, with
  const float* blocks;     // a power of two per 128 x 128, [2 blocks of a half of n with gate_up, blocks of k]
  uint8_t* codes;
  uint8_t* scales;
  int64_t ld, n, k, half, half_blocks, k_blocks;  // half: rows of a half (n without gate_up)
  int gate_up;
};

// A workgroup has a block of 128 x 128: thread t column group t % 16 of 8 values, rows t / 16 + 16 i.
template <int DT, bool PLAIN>
__global__ __launch_bounds__(256) void weight_kernel(WeightArgs a) {
  __shared__ float most[4];
  const int64_t kb = blockIdx.x % a.k_blocks, nb = blockIdx.x / a.k_blocks;
  const int64_t half = nb / a.half_blocks, first = (nb - half * a.half_blocks) * 128;
  const int64_t frags = fp8_frags(a.n), at = kb * kFp8Block + (threadIdx.x & 15) * 8;
  float x[8][8];
  float amax = 0.0f;
  if constexpr (!PLAIN) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t row = first + (threadIdx.x >> 4) + 16 * i;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (row < a.half && at < a.k) v = *reinterpret_cast<const u32x4*>(a.w + (half * a.half + row) * a.ld + at);
      unpack8<DT>(v, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fp8_magnitude(x[i][j]));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  }
  const float scale = PLAIN ? a.blocks[nb * a.k_blocks + kb] : fp8_scale_of(amax), inverse = fp8_inverse(scale);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = first + (threadIdx.x >> 4) + 16 * i;
    if (row >= a.half) continue;
    u32x2 o = {0u, 0u};
    if constexpr (PLAIN) {
      if (at < a.k) o = *reinterpret_cast<const u32x2*>(a.plain + (half * a.half + row) * a.ld + at);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = fp8_word(x[i][4 * j] * inverse, x[i][4 * j + 1] * inverse, x[i][4 * j + 2] * inverse, x[i][4 * j + 3] * inverse);
    }
    const int64_t place = fp8_place(half * a.half + row, a.n, a.gate_up != 0);
    *reinterpret_cast<u32x2*>(a.codes + fp8_code_at(frags, place, at)) = o;
    if ((threadIdx.x & 15) == 0) fp8_put_scale(a.scales, frags, place, kb, a.k_blocks, fp8_exponent(scale));
  }
}

struct ValuesArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* y;   // contiguous [rows, k]
  int64_t rows, k, frags, pieces;
  int gate_up;
};

// A thread has eight values of a row; OUT: plm_fp8_out.
template <int OUT>
__global__ __launch_bounds__(256) void values_kernel(ValuesArgs a) {
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (piece >= a.pieces) return;
  const int64_t per = a.k >> 3, row = piece / per, at = (piece - row * per) << 3;
  const int64_t place = fp8_place(row, a.rows, a.gate_up != 0);
  const u32x2 word = *reinterpret_cast<const u32x2*>(a.codes + fp8_code_at(a.frags, place, at));
  const float scale = fp8_power(a.scales[fp8_scale_at(a.frags, place, at >> 7)]);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = fp8_value(word[j >> 2], j & 3) * scale;
  if constexpr (OUT == PLM_FP8_F32) {
    f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + row * a.k + at);
    y[0] = f32x4{x[0], x[1], x[2], x[3]};
    y[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + row * a.k + at) = pack8of<OUT == PLM_FP8_BF16 ? DT_BF16 : DT_F16>(x);
  }
}

// Rows of a workgroup: a fragment's sixteen write whole lines between them, few rows go to as many CUs.
int rows_per_group(int64_t rows) { return rows >= 4096 ? 16 : rows >= 1024 ? 4 : 1; }

template <int DT, bool RES, bool WEIGHT, bool E8>
void launch_norm(const RowsArgs& a, hipStream_t s) {
  const int per = rows_per_group(a.rows);
  const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per)), block(64 * per);
  if (a.k <= 1024) hipLaunchKernelGGL((norm_kernel<DT, RES, WEIGHT, E8, 1>), grid, block, 0, s, a);
  else if (a.k <= 2048) hipLaunchKernelGGL((norm_kernel<DT, RES, WEIGHT, E8, 2>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((norm_kernel<DT, RES, WEIGHT, E8, 4>), grid, block, 0, s, a);
}

template <int DT>
hipError_t launch_rows(const RowsArgs& a, bool norm, hipStream_t s) {
  const bool res = a.residual != nullptr, weight = a.weight != nullptr, e8 = a.y == nullptr;
  if (!norm) {
    const int per = rows_per_group(a.rows);
    const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per), static_cast<unsigned>((fp8_blocks(a.k) + 7) / 8));
    hipLaunchKernelGGL((round_kernel<DT>), grid, dim3(64 * per), 0, s, a);
  } else if (e8) {
    if (res) weight ? launch_norm<DT, true, true, true>(a, s) : launch_norm<DT, true, false, true>(a, s);
    else weight ? launch_norm<DT, false, true, true>(a, s) : launch_norm<DT, false, false, true>(a, s);
  } else {
    if (res) weight ? launch_norm<DT, true, true, false>(a, s) : launch_norm<DT, true, false, false>(a, s);
    else weight ? launch_norm<DT, false, true, false>(a, s) : launch_norm<DT, false, false, false>(a, s);
  }
  return hipGetLastError();
}

bool sizes_fit(int64_t rows, int64_t k) {
  return rows >= 1 && rows < (int64_t{1} << 24) && k >= 8 && k <= (1 << 24) && k % 8 == 0;
}

template <typename... P>
bool aligned_all(const P*... p) {
  return (... && aligned16_ptr(p));
}

}  // namespace
}  // namespace plm

extern "C" {

size_t plm_fp8_codes_bytes(int64_t rows, int64_t k) {
  return plm::sizes_fit(rows, k) ? static_cast<size_t>(plm::fp8_codes_bytes(rows, k)) : 0;
}

size_t plm_fp8_scales_bytes(int64_t rows, int64_t k) {
  return plm::sizes_fit(rows, k) ? static_cast<size_t>(plm::fp8_scales_bytes(rows, k)) : 0;
}

int plm_fp8_rows(const plm_fp8_rows_call* call, void* stream) {
  using namespace plm;
  if (call == nullptr) return PLM_ERR_ARGUMENT;
  const plm_fp8_rows_call& h = *call;
  if ((h.dtype != PLM_BF16 && h.dtype != PLM_F16) || !sizes_fit(h.rows, h.k) || h.x == nullptr) return PLM_ERR_ARGUMENT;
  const bool norm = h.norm != 0, e8 = h.y == nullptr;
  if (h.x_row < 0 || h.residual_row < 0 || (e8 && (h.codes == nullptr || h.scales == nullptr))) return PLM_ERR_ARGUMENT;
  if (!norm && (!e8 || h.residual != nullptr || h.weight != nullptr)) return PLM_ERR_ARGUMENT;
  if ((h.residual != nullptr) != (h.sum != nullptr)) return PLM_ERR_ARGUMENT;
  if (norm && !(h.eps >= 0x1p-100 && h.eps <= 0x1p100)) return PLM_ERR_ARGUMENT;
  if (h.x_row % 8 != 0 || h.residual_row % 8 != 0 || !aligned_all(h.x, h.residual, h.sum, h.weight, h.y, h.codes, h.scales))
    return PLM_ERR_ALIGNMENT;
  RowsArgs a{};
  a.x = static_cast<const uint16_t*>(h.x);
  a.residual = static_cast<const uint16_t*>(h.residual);
  a.weight = static_cast<const uint16_t*>(h.weight);
  a.sum = static_cast<uint16_t*>(h.sum);
  a.y = static_cast<uint16_t*>(h.y);
  a.codes = static_cast<uint8_t*>(h.codes);
  a.scales = static_cast<uint8_t*>(h.scales);
  a.x_row = h.x_row;
  a.residual_row = h.residual_row;
  a.frags = fp8_frags(h.rows);
  a.eps = h.eps;
  a.rows = static_cast<int>(h.rows);
  a.k = static_cast<int>(h.k);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = h.dtype == PLM_BF16 ? launch_rows<DT_BF16>(a, norm, s) : launch_rows<DT_F16>(a, norm, s);
  return err == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

int plm_fp8_weight(const plm_fp8_weight_call* call, void* stream) {
  using namespace plm;
  if (call == nullptr) return PLM_ERR_ARGUMENT;
  const plm_fp8_weight_call& h = *call;
  const bool plain = h.blocks != nullptr;
  if ((!plain && h.dtype != PLM_BF16 && h.dtype != PLM_F16) || !sizes_fit(h.n, h.k) || h.w == nullptr || h.codes == nullptr ||
      h.scales == nullptr || h.ld < h.k || (h.gate_up != 0 && h.n % 32 != 0))
    return PLM_ERR_ARGUMENT;
  if (h.ld % 8 != 0 || !aligned_all(h.codes, h.scales)) return PLM_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(h.w) % (plain ? 8 : 16) != 0) return PLM_ERR_ALIGNMENT;
  WeightArgs a{};
  a.w = static_cast<const uint16_t*>(h.w);
  a.plain = static_cast<const uint8_t*>(h.w);
  a.blocks = h.blocks;
  a.codes = static_cast<uint8_t*>(h.codes);
  a.scales = static_cast<uint8_t*>(h.scales);
  a.ld = h.ld;
  a.n = h.n;
  a.k = h.k;
  a.gate_up = h.gate_up != 0 ? 1 : 0;
  a.half = a.gate_up ? h.n / 2 : h.n;
  a.half_blocks = fp8_blocks(a.half);
  a.k_blocks = fp8_blocks(h.k);
  const int64_t grid = a.k_blocks * a.half_blocks * (a.gate_up ? 2 : 1);
  if (grid >= (int64_t{1} << 31)) return PLM_ERR_ARGUMENT;
  const dim3 blocks(static_cast<unsigned>(grid));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (plain) hipLaunchKernelGGL((weight_kernel<DT_BF16, true>), blocks, dim3(256), 0, s, a);
  else if (h.dtype == PLM_BF16) hipLaunchKernelGGL((weight_kernel<DT_BF16, false>), blocks, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((weight_kernel<DT_F16, false>), blocks, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

int plm_fp8_values(const void* codes, const void* scales, int64_t rows, int64_t k, int32_t gate_up, int32_t out_type, void* y,
                   void* stream) {
  using namespace plm;
  if (!sizes_fit(rows, k) || codes == nullptr || scales == nullptr || y == nullptr || (gate_up != 0 && rows % 32 != 0) ||
      out_type < PLM_FP8_BF16 || out_type > PLM_FP8_F32)
    return PLM_ERR_ARGUMENT;
  if (!aligned_all(codes, scales, y)) return PLM_ERR_ALIGNMENT;
  const int64_t pieces = rows * (k / 8), grid = (pieces + 255) / 256;
  if (grid >= (int64_t{1} << 31)) return PLM_ERR_ARGUMENT;
  const ValuesArgs a{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), y, rows, k, fp8_frags(rows), pieces,
                     gate_up != 0 ? 1 : 0};
  const dim3 blocks(static_cast<unsigned>(grid));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (out_type == PLM_FP8_BF16) hipLaunchKernelGGL((values_kernel<PLM_FP8_BF16>), blocks, dim3(256), 0, s, a);
  else if (out_type == PLM_FP8_F16) hipLaunchKernelGGL((values_kernel<PLM_FP8_F16>), blocks, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((values_kernel<PLM_FP8_F32>), blocks, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

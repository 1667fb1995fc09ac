// Rows into 8 bits (plm_fp8_rows), with the root-mean-square norm and the residual's addition before it or the norm in
// 16 bits; weights into 8 bits or into the kernels' order (plm_fp8_weight) and back to values (plm_fp8_values). Declared in
// include/plm_amd.h; order of the bytes: fp8.h.
//
// Norm: t = x + residual, rounded to the model's type (so that the norm of the returned sum is the same); y = t w / sqrt(
// mean(t^2) + eps). The sum of squares and the root are fp64. y in fp32 is off by three roundings, 3 of its last places at
// most; a code has 2^20 fp32 values to a step, so of a million values one to four would come out on the other side of a
// border between codes: what is that close is computed in fp64 and rounded once, the scale's border likewise. So is all of
// a row whose root fp32 does not hold well, and in bf16 a lane's values of which one's quotient by the root is subnormal in
// fp32, where a weight of 2^7 or more would bring it back without the bits that it lost.
//
// Measured (replayed over inputs from memory; a large copy 5.1 TB/s). Norm with residual into 8 bits: 8192 x 2048 34.4 us,
// 117 MB, 3.4 TB/s (a row's values are held in registers between the sum and the codes; its 512 workgroups are all there at
// once and read, compute and write nearly in step), 16384 x 2048 61.5, 56 x 2048 4.0. Norm in 16 bits: 8192 x 2048 with
// residual 34.3, 134 MB, 3.9 TB/s; 1 x 1024 2.3, of which 2.2 are a launch. Rounding alone: 8192 x 2048 12.7, 50 MB, 4.0 TB/s.
// Values of 8192 x 2048 in bf16: 15, 3.4 TB/s (10.5 where part of it is cached). A weight of 11264 x 2048: 15.6.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fp8_gemm.h"

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
  for (int i = 0; i < 4; ++i) o[i] = two_bits16<DT>(x[2 * i], x[2 * i + 1]);
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

// Eight values of a row from `at`, a multiple of 8 as k is one; zeros past k.
__device__ __forceinline__ u32x4 load8(const uint16_t* row, int at, int k) {
  return at < k ? *reinterpret_cast<const u32x4*>(row + at) : u32x4{0u, 0u, 0u, 0u};
}

// x + residual, rounded.
template <int DT>
__device__ __forceinline__ u32x4 add8(u32x4 v, u32x4 r) {
  float x[8], y[8];
  unpack8<DT>(v, x);
  unpack8<DT>(r, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] += y[i];
  return pack8of<DT>(x);
}

template <int DT>
__device__ __forceinline__ double squares8(u32x4 v) {
  float x[8];
  unpack8<DT>(v, x);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum = fma(static_cast<double>(x[j]), static_cast<double>(x[j]), sum);
  return sum;
}

// A row's norm: 1 / sqrt(mean + eps) in both widths.
struct Norm {
  double exact;
  float near;
  bool wide;   // outside of where fp32 keeps its steps
};

__device__ __forceinline__ Norm norm_of(double squares, int k, double eps) {
  Norm n;
  n.exact = 1.0 / sqrt(squares / k + eps);
  n.near = static_cast<float>(n.exact);
  n.wide = !(n.near > 0x1p-100f && n.near < 0x1p100f);
  return n;
}

// What of a lane's values fp32 does not settle.
struct Unsettled {
  bool close;   // one is so close to a place where codes may part that fp32 does not tell the side
  bool wide;    // they may have left fp32's range on the way: all of them
};

// y of N / 8 pieces of eight values. Places where codes may part have at most four bits of mantissa, 19 zeros at the end.
// A subnormal quotient is off by 2^-150. Times a weight below 2^7 that is 2^-8 of half of bf16's least step, and the value far
// under the least code.
template <int DT, bool WEIGHT, int N>
__device__ __forceinline__ Unsettled normed(const Norm& norm, const u32x4 (&v)[N / 8], const u32x4 (&w)[N / 8], float (&y)[N]) {
  uint32_t least = ~0u;
  bool wide = norm.wide;
  if constexpr (WEIGHT && DT == DT_BF16) {
    uint32_t any = 0u;
#pragma unroll
    for (int p = 0; p < N / 8; ++p) any |= w[p][0] | w[p][1] | w[p][2] | w[p][3];
    if ((any & 0x40004000u) != 0u) {   // a weight of 2 or more
      uint32_t most = 0u;
#pragma unroll
      for (int p = 0; p < N / 8; ++p) most = max(most, fp8_most16<DT>(w[p]));
      if (most >= 0x4300u) {           // of 2^7
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float t = from_bits16<DT>(static_cast<uint16_t>(v[i >> 3][(i & 7) >> 1] >> (16 * (i & 1))));
          wide = wide || (t != 0.0f && fabsf(t * norm.near) < 0x1p-126f);
        }
      }
    }
  }
#pragma unroll
  for (int p = 0; p < N / 8; ++p) {
    float of[8];
    unpack8<DT>(v[p], y + 8 * p);
    if constexpr (WEIGHT) unpack8<DT>(w[p], of);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[8 * p + i] *= norm.near;
      if constexpr (WEIGHT) y[8 * p + i] *= of[i];
      least = min(least, (__builtin_bit_cast(uint32_t, y[8 * p + i]) + 4u) & 0x7ffffu);
    }
  }
  return {least <= 8u, wide};
}

// What is that close, in fp64 and rounded to odd: one value at a time, as it is rarely more than one of a wavefront's, and read
// again, so that nothing is kept for it. `t` and `weight`: the row and the norm's weights, value i at place(i) of k.
template <int DT, bool WEIGHT, int N, typename P>
__device__ __forceinline__ void normed_exact(const Norm& norm, bool wide, const uint16_t* t, const uint16_t* weight, int k, P place, float (&y)[N]) {
  uint32_t close = wide ? ~0u >> (32 - N) : 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) close |= ((__builtin_bit_cast(uint32_t, y[i]) + 4u) & 0x7ffffu) <= 8u ? 1u << i : 0u;
#pragma unroll 1
  for (; close != 0; close &= close - 1) {
    const int i = __builtin_ctz(close), at = place(i);
    if (at >= k) continue;
    double exact = static_cast<double>(from_bits16<DT>(t[at])) * norm.exact;
    if constexpr (WEIGHT) exact *= static_cast<double>(from_bits16<DT>(weight[at]));
    const float odd = odd_float(exact);
#pragma unroll
    for (int n = 0; n < N; ++n) y[n] = n == i ? odd : y[n];
  }
}

// Codes of N values, and their scale; `share` gives the largest of the lanes that have a block between them. 448 is among the
// borders above: a value that could lie on either side of it has been computed exactly.
template <int N, typename F>
__device__ __forceinline__ float codes_of(const float (&y)[N], F share, uint32_t (&codes)[N / 4]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) most = max(most, __builtin_bit_cast(uint32_t, y[i]) & 0x7fffffffu);
  most = share(most);
  if (__builtin_expect(__ballot(most >= 0x7f800000u) != 0, 0)) {   // not all finite
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) amax = fmaxf(amax, fp8_magnitude(y[i]));
    const float scale = fp8_scale_of(__builtin_bit_cast(float, share(__builtin_bit_cast(uint32_t, amax)))), inverse = fp8_inverse(scale);
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      codes[i] = fp8_word(y[4 * i] * inverse, y[4 * i + 1] * inverse, y[4 * i + 2] * inverse, y[4 * i + 3] * inverse);
    return scale;
  }
  const float scale = fp8_scale_of(__builtin_bit_cast(float, most));
#pragma unroll
  for (int i = 0; i < N / 4; ++i) codes[i] = fp8_four(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3], scale);
  return scale;
}

// Chunks of 16 values of a row, 8 and 8 of every 64; whole blocks where codes are written, whose zeros past k are part of them.
template <bool E8>
__host__ __device__ __forceinline__ int row_chunks(int k) {
  return E8 ? static_cast<int>(fp8_blocks(k)) * 8 : (k + 63) / 64 * 4;
}

// A workgroup has a row, a thread chunks thread + threads i of it, the pieces of eight at 64 (chunk / 4) + 8 (chunk % 4) and 32
// further; eight threads have a block. The first chunk stays in
// registers between the sum of squares and the output; the rest of a row longer than the workgroup is read again. GROUPED: of 128
// workgroups the sixteen of an XCD (number % 8) have the sixteen rows of a fragment; the grid is a multiple of 128.
template <int DT, bool RES, bool WEIGHT, bool E8, bool GROUPED>
__global__ __launch_bounds__(1024) void row_norm_kernel(RowsArgs a) {
  __shared__ double parts[16];
  const int64_t row = GROUPED ? (blockIdx.x & ~127u) | ((blockIdx.x & 7u) << 4) | ((blockIdx.x >> 3) & 15u) : blockIdx.x;
  if (GROUPED && row >= a.rows) return;
  const int threads = blockDim.x, turns = (row_chunks<E8>(a.k) + threads - 1) / threads;
  const uint16_t* x = a.x + row * a.x_row;
  const uint16_t* residual = RES ? a.residual + row * a.residual_row : nullptr;
  uint16_t* sum = RES ? a.sum + row * a.k : nullptr;
  auto read = [&](int at, u32x4 (&v)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v[h] = load8(x, at + 32 * h, a.k);
      if constexpr (RES) {
        v[h] = add8<DT>(v[h], load8(residual, at + 32 * h, a.k));
        if (at + 32 * h < a.k) *reinterpret_cast<u32x4*>(sum + at + 32 * h) = v[h];
      }
    }
    return squares8<DT>(v[0]) + squares8<DT>(v[1]);
  };
  auto weights = [&](int at, u32x4 (&w)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = WEIGHT ? load8(a.weight, at + 32 * h, a.k) : u32x4{0u, 0u, 0u, 0u};
  };
  auto emit = [&](const Norm& norm, int at, const u32x4 (&v)[2], const u32x4 (&w)[2]) {
    float y[16];
    const Unsettled some = normed<DT, WEIGHT, 16>(norm, v, w, y);
    if ((E8 && some.close) || some.wide)
      normed_exact<DT, WEIGHT, 16>(norm, some.wide, RES ? sum : x, a.weight, a.k, [&](int i) { return at + (i >> 3) * 32 + (i & 7); }, y);
    if constexpr (E8) {
      uint32_t c[4];
      const float scale = codes_of<16>(y, [](uint32_t most) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), d)));
        return most;
      }, c);
      const int block = at >> 7;
      if (block < static_cast<int>(fp8_blocks(a.k))) {
        *reinterpret_cast<u32x4*>(a.codes + fp8_code_at(a.frags, row, at)) = u32x4{c[0], c[1], c[2], c[3]};
        if ((threadIdx.x & 7) == 0) fp8_put_scale(a.scales, a.frags, row, block, fp8_blocks(a.k), fp8_exponent(scale));
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (at + 32 * h < a.k) *reinterpret_cast<u32x4*>(a.y + row * a.k + at + 32 * h) = pack8of<DT>(y + 8 * h);
    }
  };

  auto chunk_at = [&](int i) {
    const int chunk = static_cast<int>(threadIdx.x) + threads * i;
    return (chunk >> 2) * 64 + (chunk & 3) * 8;
  };
  const int first = chunk_at(0);
  u32x4 held[2], w[2];
  weights(first, w);
  double squares = read(first, held);
  for (int i = 1; i < turns; ++i) {
    u32x4 v[2];
    squares += read(chunk_at(i), v);
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) squares += __shfl_xor(squares, d);
  if (threads > 64) {
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = squares;
    __syncthreads();
    squares = parts[0];
    for (int i = 1; i < threads >> 6; ++i) squares += parts[i];
  }
  const Norm norm = norm_of(squares, a.k, a.eps);
  emit(norm, first, held, w);
  for (int i = 1; i < turns; ++i) {
    u32x4 v[2], of[2];
    const int at = chunk_at(i);
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = load8(RES ? sum : x, at + 32 * h, a.k);   // of the sum this thread's own
    weights(at, of);
    emit(norm, at, v, of);
  }
}

// The lanes of a row in a wavefront that has a fragment: 16 apart.
__device__ __forceinline__ uint32_t share_row(uint32_t most) {
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
  return max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
}

// A lane's 32 codes of a fragment, 1 KiB side by side per store, and the scales of its rows.
__device__ __forceinline__ void store_fragment(const RowsArgs& a, int64_t frag, int kb, int lane, const uint32_t (&c)[8], float scale) {
  u32x4* to = reinterpret_cast<u32x4*>(a.codes + (kb * a.frags + frag) * kFp8Bytes) + lane;
  to[0] = u32x4{c[0], c[1], c[2], c[3]};
  to[64] = u32x4{c[4], c[5], c[6], c[7]};
  if (lane < 16) fp8_put_scale(a.scales, a.frags, frag * 16 + lane, kb, fp8_blocks(a.k), fp8_exponent(scale));
}

// Sixteen rows of the norm in 8 bits: a wavefront has a fragment, row lane % 16 of it a lane, and has HELD blocks of K,
// which stay in registers. Whole lines are written, where a row to a workgroup
// writes 16 bytes of each.
template <int DT, bool RES, bool WEIGHT, int HELD>
__global__ __launch_bounds__(1024) void fragment_norm_kernel(RowsArgs a) {
  __shared__ double parts[16][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, blocks = static_cast<int>(fp8_blocks(a.k));
  const int64_t frag = blockIdx.x, row = min(frag * 16 + (lane & 15), static_cast<int64_t>(a.rows) - 1);
  const bool there = frag * 16 + (lane & 15) < a.rows;   // rows past the last compute the last one's, and store nothing
  const uint16_t* x = a.x + row * a.x_row;
  const uint16_t* residual = RES ? a.residual + row * a.residual_row : nullptr;
  uint16_t* sum = RES ? a.sum + row * a.k : nullptr;
  u32x4 held[HELD][4];
  double squares = 0.0;
  {
    u32x4 more[HELD][4];
#pragma unroll
    for (int i = 0; i < HELD; ++i)   // every load before the first store, which it may not pass
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        held[i][j] = load8(x, fp8_piece_at(wave + waves * i, lane, j), a.k);
        if constexpr (RES) more[i][j] = load8(residual, fp8_piece_at(wave + waves * i, lane, j), a.k);
      }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (RES) {
          held[i][j] = add8<DT>(held[i][j], more[i][j]);
          const int at = fp8_piece_at(wave + waves * i, lane, j);
          if (at < a.k && there) *reinterpret_cast<u32x4*>(sum + at) = held[i][j];
        }
        squares += squares8<DT>(held[i][j]);
      }
  }
  squares += __shfl_xor(squares, 16);
  squares += __shfl_xor(squares, 32);
  if (lane < 16) parts[wave][lane] = squares;
  __syncthreads();
  squares = parts[0][lane & 15];
  for (int i = 1; i < waves; ++i) squares += parts[i][lane & 15];
  const Norm norm = norm_of(squares, a.k, a.eps);
  auto emit = [&](int kb, const u32x4 (&v)[4]) {
    u32x4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = WEIGHT ? load8(a.weight, fp8_piece_at(kb, lane, j), a.k) : u32x4{0u, 0u, 0u, 0u};
    float y[32];
    const Unsettled some = normed<DT, WEIGHT, 32>(norm, v, w, y);
    if (some.close || some.wide)
      normed_exact<DT, WEIGHT, 32>(norm, some.wide, RES ? sum : x, a.weight, a.k, [&](int i) { return fp8_piece_at(kb, lane, i >> 3) + (i & 7); }, y);
    uint32_t c[8];
    const float scale = codes_of<32>(y, share_row, c);
    store_fragment(a, frag, kb, lane, c, scale);
  };
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (wave + waves * i < blocks) emit(wave + waves * i, held[i]);
}

// Rows as they are: a wavefront has a fragment, its neighbours the blocks of K beside it, so that rows are read on: 8192 x 2048
// 12.7 us for 14.9 where they had the rows below, 8192 x 8192 40.0 for 49.8 (5.0 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void round_kernel(RowsArgs a, int64_t count) {
  const int64_t number = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 6) + (threadIdx.x >> 6);
  if (number >= count) return;
  const int lane = threadIdx.x & 63;
  const int64_t blocks = fp8_blocks(a.k), frag = number / blocks, kb = number - frag * blocks, row = min(frag * 16 + (lane & 15), static_cast<int64_t>(a.rows) - 1);
  u32x4 v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = load8(a.x + row * a.x_row, fp8_piece_at(static_cast<int>(kb), lane, j), a.k);
  uint32_t c[8];
  const uint32_t most = share_row(fp8_most16<DT>(v[0], v[1], v[2], v[3]));
  float scale;
  if (__builtin_expect(__ballot(most >= fp8_infinite<DT>()) != 0, 0)) {
    i32x8 codes;
    scale = fp8_round_any<DT>(v, [](float amax) { return __builtin_bit_cast(float, share_row(__builtin_bit_cast(uint32_t, amax))); }, codes);
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = static_cast<uint32_t>(codes[i]);
  } else {
    scale = fp8_scale_of(from_bits16<DT>(static_cast<uint16_t>(most)));
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = fp8_four<DT>(v[i >> 1][2 * (i & 1)], v[i >> 1][2 * (i & 1) + 1], scale);
  }
  store_fragment(a, frag, static_cast<int>(kb), lane, c, scale);
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
  int64_t rows, k, frags, count;
  int gate_up;
};

// A wavefront has a fragment, its neighbours the blocks of K beside it (8192 x 8192 50 us for 62 where they had the rows below),
// a lane 32 values of a row; OUT: plm_fp8_out.
template <int OUT>
__global__ __launch_bounds__(256) void values_kernel(ValuesArgs a) {
  const int64_t number = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (number >= a.count) return;
  const int lane = threadIdx.x & 63;
  const int64_t blocks = fp8_blocks(a.k), frag = number / blocks, kb = number - frag * blocks;
  const int64_t row = (a.gate_up != 0 ? (frag >> 1) * 16 + (frag & 1) * (a.rows >> 1) : frag * 16) + (lane & 15);
  if (row >= a.rows) return;
  const u32x4* from = reinterpret_cast<const u32x4*>(a.codes + (kb * a.frags + frag) * kFp8Bytes) + lane;
  const u32x4 codes[2] = {from[0], from[64]};
  const float scale = fp8_power(a.scales[fp8_scale_at(a.frags, frag * 16 + (lane & 15), kb)]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int at = fp8_piece_at(static_cast<int>(kb), lane, j);
    if (at >= a.k) continue;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fp8_value(codes[j >> 1][2 * (j & 1) + (i >> 2)], i & 3) * scale;
    if constexpr (OUT == PLM_FP8_F32) {
      f32x4* y = reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + row * a.k + at);
      y[0] = f32x4{x[0], x[1], x[2], x[3]};
      y[1] = f32x4{x[4], x[5], x[6], x[7]};
    } else {
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.y) + row * a.k + at) = pack8of<OUT == PLM_FP8_BF16 ? DT_BF16 : DT_F16>(x);
    }
  }
}

// Rows from which a workgroup has sixteen, and the blocks of K that its registers hold: 4096 x 2048 20.2 us for
// 21.6 with one, 4096 x 4096 34.6 for 39.1, 8192 x 2048 34.4 for 36.9, but 2048 x 2048 16.5 for 12.2 and 512 x 2048 13.5 for 5.7.
constexpr int kFragmentRows = 4096, kFragmentBlocks = 32;

template <int DT, bool RES, bool WEIGHT, bool E8>
void launch_norm(const RowsArgs& a, hipStream_t s) {
  // Wavefronts of a row: a chunk to a thread, in a launch of less than 2^32 threads (three for the most rows).
  const int64_t fit = 0xffffffffll / (64 * ((static_cast<int64_t>(a.rows) + 127) / 128 * 128));
  const int waves = static_cast<int>(std::min({(row_chunks<E8>(a.k) + int64_t{63}) / 64, int64_t{16}, fit}));
  const unsigned rows = static_cast<unsigned>(a.rows);
  if constexpr (E8) {
    const int blocks = static_cast<int>(fp8_blocks(a.k));
    if (a.rows >= kFragmentRows && blocks <= kFragmentBlocks) {
      // Two blocks to a wavefront, so that two workgroups fit a CU at 2048 columns (33.5 us for 35.7 with one of 16).
      const dim3 grid(static_cast<unsigned>(a.frags)), block(64 * (blocks <= 8 ? blocks : blocks <= 16 ? 8 : 16));
      if (blocks <= 8) hipLaunchKernelGGL((fragment_norm_kernel<DT, RES, WEIGHT, 1>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((fragment_norm_kernel<DT, RES, WEIGHT, 2>), grid, block, 0, s, a);
      return;
    }
    // A fragment's rows on one XCD, in whose L2 their pieces of its lines meet: 2048 x 4096 21.8 us for 24.4, 8192 x 8192 115 for
    // 144, 128 x 2048 4.1 for 4.1.
    if (a.rows >= 128) {
      hipLaunchKernelGGL((row_norm_kernel<DT, RES, WEIGHT, true, true>), dim3((rows + 127) / 128 * 128), dim3(64 * waves), 0, s, a);
      return;
    }
  }
  hipLaunchKernelGGL((row_norm_kernel<DT, RES, WEIGHT, E8, false>), dim3(rows), dim3(64 * waves), 0, s, a);
}

template <int DT>
hipError_t launch_rows(const RowsArgs& a, bool norm, hipStream_t s) {
  const bool res = a.residual != nullptr, weight = a.weight != nullptr, e8 = a.y == nullptr;
  if (!norm) {
    const int64_t count = a.frags * fp8_blocks(a.k);
    const int waves = count < 4096 ? 2 : 4;   // 42 x 10240 2.5 us for 2.9 of four, 4096 x 2048 8.0 for 7.7
    hipLaunchKernelGGL((round_kernel<DT>), dim3(static_cast<unsigned>((count + waves - 1) / waves)), dim3(64 * waves), 0, s, a, count);
  } else if (e8) {
    if (res) weight ? launch_norm<DT, true, true, true>(a, s) : launch_norm<DT, true, false, true>(a, s);
    else weight ? launch_norm<DT, false, true, true>(a, s) : launch_norm<DT, false, false, true>(a, s);
  } else {
    if (res) weight ? launch_norm<DT, true, true, false>(a, s) : launch_norm<DT, true, false, false>(a, s);
    else weight ? launch_norm<DT, false, true, false>(a, s) : launch_norm<DT, false, false, false>(a, s);
  }
  return hipGetLastError();
}

// What fits a launch of a wavefront to a fragment, whose threads are less than 2^32, among others.
bool sizes_fit(int64_t rows, int64_t k) {
  return rows >= 1 && rows < (int64_t{1} << 24) && k >= 8 && k <= (1 << 24) && k % 8 == 0 &&
         fp8_frags(rows) * fp8_blocks(k) <= (int64_t{1} << 25);
}

template <typename... P>
bool aligned_all(const P*... p) {
  return (... && aligned16_ptr(p));
}

}  // namespace

hipError_t fp8_round(int dtype, const void* x, int64_t x_row, int64_t rows, int64_t k, uint8_t* codes, uint8_t* scales, hipStream_t s) {
  RowsArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.codes = codes;
  a.scales = scales;
  a.x_row = x_row;
  a.frags = fp8_frags(rows);
  a.rows = static_cast<int>(rows);
  a.k = static_cast<int>(k);
  return dtype == PLM_BF16 ? launch_rows<DT_BF16>(a, false, s) : launch_rows<DT_F16>(a, false, s);
}

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
  const int64_t count = fp8_frags(rows) * fp8_blocks(k), grid = (count + 3) / 4;
  const ValuesArgs a{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), y, rows, k, fp8_frags(rows), count,
                     gate_up != 0 ? 1 : 0};
  const dim3 blocks(static_cast<unsigned>(grid));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (out_type == PLM_FP8_BF16) hipLaunchKernelGGL((values_kernel<PLM_FP8_BF16>), blocks, dim3(256), 0, s, a);
  else if (out_type == PLM_FP8_F16) hipLaunchKernelGGL((values_kernel<PLM_FP8_F16>), blocks, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((values_kernel<PLM_FP8_F32>), blocks, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

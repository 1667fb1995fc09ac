// Products over e4m3 rows for many rows of X: bound by the matrix cores.
//
// A workgroup has a tile of 16 WN FN rows of the weight x 16 WM FM rows of X, a wavefront FN x FM fragments of it. X comes
// into LDS (four sets, two blocks of K ahead), the weight's operands straight from memory into registers, a block ahead: read
// from LDS too, both operands of 256 x 256 took LDS as many cycles as the products take the matrix cores. The fragments'
// order is what a wavefront's 16-byte reads want: no bank met twice, no address to compute.
//
// One barrier a block, in its middle, where the next block's set must have arrived; the operand that the next block
// begins with is read before this one's end, so the matrix cores do not run dry at either. Workgroups stay, and the loads run
// ahead into the next tile while the last one is stored.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fp8_gemm.h"

namespace plm {
namespace {

typedef __attribute__((address_space(3))) void* LdsPtr;

__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, u32x4* to, uint32_t lane_offset, uint32_t offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)to, 16, static_cast<int>(lane_offset), static_cast<int>(offset), 0, 0);
}

// A barrier, before which all of a wavefront's loads but its last N have arrived. (A fence would wait for every load into LDS.)
// No wait for reads of LDS is needed: what a set held has been multiplied before the barrier after which it is overwritten.
template <int N>
__device__ __forceinline__ void tile_sync() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A lane's offset, seen anew: what is added to it then goes into an instruction's own offset, not into registers of its own
// that the compiler would compute ahead of the loop (it spilled a dozen).
__device__ __forceinline__ int anew(int offset) {
  asm volatile("" : "+v"(offset));
  return offset;
}

template <int J>
__device__ __forceinline__ f32x4 mma_at(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, J, sa, J, sb);
}

// Two fragments' four columns of a row in each lane to eight of one: lanes 16 g + r have columns [8 (g / 2), 8 (g / 2) + 8) of
// fragment g % 2, row r, so that rows are stored 64 bytes at a time.
__device__ __forceinline__ u32x4 eight_columns(u32x2 a, u32x2 b) {
  const auto lo = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

template <int DT>
__device__ __forceinline__ u32x2 four16(f32x4 v) {
  return u32x2{to_bits16<DT>(v[0]) | (static_cast<uint32_t>(to_bits16<DT>(v[1])) << 16),
               to_bits16<DT>(v[2]) | (static_cast<uint32_t>(to_bits16<DT>(v[3])) << 16)};
}

struct Tiles {
  int n, m, per_xcd;
};

// Each XCD has a contiguous run of tiles, in groups of kGroup tiles of X, whose weights it reads once for all of the group.
constexpr int kGroup = 4;

__device__ __forceinline__ void place_of(const Tiles& g, int tile, int& tn, int& tm) {
  const int group = tile / (kGroup * g.n), rest = tile - group * (kGroup * g.n);
  const int deep = min(kGroup, g.m - group * kGroup);
  tn = rest / deep;
  tm = group * kGroup + rest - tn * deep;
}

template <int WN, int WM, int FN, int FM, int AHEAD, int DT, bool ACT>
__global__ __launch_bounds__(64 * WN * WM) void tile_kernel(Fp8Gemm a, Tiles tiles) {
  constexpr int kWaves = WN * WM, TN = WN * FN, TM = WM * FM, kX = 2 * TM / kWaves;
  static_assert(AHEAD == 1 || AHEAD == 3, "operands of two or four blocks");
  static_assert(2 * TM % kWaves == 0 && FM % 2 == 0, "every wavefront stages as many pieces of 1 KiB");
  __shared__ __attribute__((aligned(16))) u32x4 set0[TM * 128], set1[TM * 128], set2[TM * 128], set3[TM * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int base = (blockIdx.x & 7) * tiles.per_xcd, count = min(tiles.per_xcd, tiles.n * tiles.m - base);
  const int stride = gridDim.x >> 3;
  int local = blockIdx.x >> 3;
  if (local >= count) return;
  const int wn = wave / WM, wm = wave - wn * WM, at_lane = lane * 16;
  const uint32_t w_block = static_cast<uint32_t>(a.w_frags) * kFp8Bytes, x_block = static_cast<uint32_t>(a.x_frags) * kFp8Bytes;
  const uint32_t w_scale_block = static_cast<uint32_t>(a.w_frags) * kFp8ScaleBytes;
  const uint32_t x_scale_block = static_cast<uint32_t>(a.x_frags) * kFp8ScaleBytes;

  // Four blocks of K from kb on: an operand's bytes there, and where in it a block's fragment lies. Fragments past the operand's
  // last are the next block's first, or zeros without traffic past its end; they reach no output that is stored. So are
  // the weight's blocks past K; X has its last one again there, since a set's older codes may be another row's NaN.
  struct Group {
    __amdgpu_buffer_rsrc_t w, x;
    int kb;
  };
  auto group_at = [&](int kb, bool in) {
    const uint32_t left = in ? static_cast<uint32_t>(min(a.blocks - kb, 4)) : 0u;
    return Group{make_rsrc(a.w + static_cast<int64_t>(kb) * w_block, left * w_block),
                 make_rsrc(a.x + static_cast<int64_t>(kb) * x_block, left * x_block), kb};
  };
  // Pieces [i0, i1) of a block of X into a set, and of the weight's operands into registers: 1 KiB a load.
  auto stage = [&](const Group& g, int t0, int j, u32x4* set, int i0, int i1) {
    const uint32_t at = static_cast<uint32_t>(min(j, a.blocks - 1 - g.kb)) * x_block + static_cast<uint32_t>(t0) * kFp8Bytes;
#pragma unroll
    for (int i = 0; i < kX; ++i)
      if (i >= i0 && i < i1) load_lds16(g.x, set + (i * kWaves + wave) * 64, at_lane + wave * 1024, at + i * (kWaves * 1024));
  };
  auto weights = [&](const Group& g, int f0, int j, i32x8 (&w)[FN], int i0, int i1) {
    const uint32_t at = static_cast<uint32_t>(j) * w_block + static_cast<uint32_t>(f0) * kFp8Bytes;
    const int here = anew(at_lane);
#pragma unroll
    for (int f = 0; f < FN; ++f) {
      if (f < i0 || f >= i1) continue;
      // Two fragments are within the 4 KiB of an instruction's own offset.
      const int from = static_cast<int>(at + (f & ~1) * kFp8Bytes), in_lane = here + (f & 1) * static_cast<int>(kFp8Bytes);
      w[f] = fp8_operand(__builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(g.w, in_lane, from, 0)),
                         __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(g.w, in_lane + 1024, from, 0)));
    }
  };
  // Four blocks' scales of fragments [f, f1) of an operand, a byte each. Past K they are zeros, which stand for 2^-127.
  auto scales = [&](const uint8_t* from, uint32_t block, int kb, bool in, int first, int i0, int i1, int* s) {
    const int here = anew((lane & 15) * 4);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(from + static_cast<int64_t>(kb >> 2) * block, in ? block : 0u);
#pragma unroll
    for (int i = i0; i < i1; ++i) s[i] = __builtin_amdgcn_raw_buffer_load_b32(r, here + i * 64, first * static_cast<int>(kFp8ScaleBytes), 0);
  };

  f32x4 acc[FN][FM];
  int ws[FN], xs[FM], next_ws[FN];
  i32x8 w[AHEAD + 1][FN], xo[2];
  const int x_at = wm * FM * 128 + lane;
  int f0, t0;
  place_of(tiles, base + local, f0, t0);
  f0 = f0 * TN + wn * FN;
  t0 *= TM;
  scales(a.w_scales, w_scale_block, 0, true, f0, 0, FN, next_ws);
  scales(a.x_scales, x_scale_block, 0, true, t0 + wm * FM, 0, FM, xs);
  Group now = group_at(0, true);
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) weights(now, f0, j, w[j], 0, FN);
  stage(now, t0, 0, set0, 0, kX);
  stage(now, t0, 1, set1, 0, kX);
  stage(now, t0, 2, set2, 0, kX);
  tile_sync<2 * kX>();   // the first set's have arrived
  xo[0] = fp8_operand(set0[x_at], set0[x_at + 64]);
  const int columns = ACT ? a.n / 2 : a.n;

  // The wait before the barrier: of the loads since the next set's, the set after it (kX) and the weight's next operands (2 FN)
  // may be outstanding. A barrier alone does not wait for loads into LDS.
#define PLM_HALF(J, SET, NEXT, FROM, LOAD)                                                                                \
  _Pragma("unroll") for (int t = FROM; t < FROM + FM / 2; ++t) {                                                          \
    const u32x4* p = t + 1 < FM ? SET + x_at + (t + 1) * 128 : NEXT + x_at;                                               \
    xo[(t + 1) & 1] = fp8_operand(p[0], p[64]);                                                                           \
    _Pragma("unroll") for (int f = 0; f < FN; ++f)                                                                        \
        acc[f][t] = mma_at<J>(w[J % (AHEAD + 1)][f], xo[t & 1], acc[f][t], ws[f], xs[t]);                                 \
    LOAD;                                                                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                                    \
  }
#define PLM_STEP(J, SET, NEXT, LAST, MORE, COUNT)                                                                         \
  PLM_HALF(J, SET, NEXT, 0,                                                                                               \
           MORE; weights(J + AHEAD < 4 ? now : next, J + AHEAD < 4 ? f0 : fn, (J + AHEAD) & 3, w[(J + AHEAD) % (AHEAD + 1)], \
                         t * 2 * FN / FM, (t + 1) * 2 * FN / FM))                                                         \
  tile_sync<kX + 2 * FN * (AHEAD == 1 ? 1 : 2) + COUNT>();                                                                \
  PLM_HALF(J, SET, NEXT, FM / 2,                                                                                          \
           MORE; stage(J == 0 ? now : next, J == 0 ? t0 : tn, (J + 3) & 3, LAST, (t - FM / 2) * 2 * kX / FM,              \
                       (t + 1 - FM / 2) * 2 * kX / FM))

  for (;;) {
    const bool more = local + stride < count;
    int f1 = 0, t1 = 0;
    if (more) {
      place_of(tiles, base + local + stride, f1, t1);
      f1 = f1 * TN + wn * FN;
      t1 *= TM;
    }
#pragma unroll
    for (int f = 0; f < FN; ++f)
#pragma unroll
      for (int t = 0; t < FM; ++t) acc[f][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int kb = 0; kb < a.blocks; kb += 4) {
      const bool last = kb + 4 >= a.blocks, in = !last || more;
      const int fn = last ? f1 : f0, tn = last ? t1 : t0;
      const Group next = group_at(last ? 0 : kb + 4, in);
#pragma unroll
      for (int f = 0; f < FN; ++f) ws[f] = next_ws[f];
      PLM_STEP(0, set0, set1, set3, , 0)
      PLM_STEP(1, set1, set2, set0, , 0)
      PLM_STEP(2, set2, set3, set1, , 0)
      scales(a.w_scales, w_scale_block, next.kb, in, fn, 0, FN, next_ws);
      PLM_STEP(3, set3, set0, set2, scales(a.x_scales, x_scale_block, next.kb, in, tn + wm * FM, t, t + 1, xs), FN + FM / 2)
      now = next;
    }

    constexpr int kOut = ACT ? FN / 2 : FN;
    const int n0 = f0 / (ACT ? 2 : 1) * 16, column = anew(lane);
#pragma unroll
    for (int t = 0; t < FM; ++t) {
      const int m = (t0 + wm * FM + t) * 16 + (column & 15);
      f32x4 v[kOut];
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        v[f] = acc[ACT ? 2 * f : f][t];
        if constexpr (ACT) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[f][j] = fp8_silu_mul(v[f][j], acc[2 * f + 1][t][j]);
        }
      }
      if (kOut % 2 == 0 && n0 + kOut * 16 <= columns) {
#pragma unroll
        for (int f = 0; f + 1 < kOut; f += 2) {
          const u32x4 o = eight_columns(four16<DT>(v[f]), four16<DT>(v[f + 1]));
          const int n = n0 + (f + ((column >> 4) & 1)) * 16 + (column >> 5) * 8;
          if (m < a.m) *reinterpret_cast<fp8_any16*>(static_cast<uint16_t*>(a.y) + m * a.ldy + n) = o;
        }
      } else if (m < a.m) {
#pragma unroll
        for (int f = 0; f < kOut; ++f) {
          const int n = n0 + f * 16 + (column >> 4) * 4;
          uint16_t* y = static_cast<uint16_t*>(a.y) + m * a.ldy + n;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < columns) y[j] = to_bits16<DT>(v[f][j]);
        }
      }
    }
    if (!more) break;
    local += stride;
    f0 = f1;
    t0 = t1;
  }
#undef PLM_STEP
#undef PLM_HALF
  __builtin_amdgcn_s_waitcnt(0x0f70);   // no load may arrive in this workgroup's LDS after its end
}

template <int WN, int WM, int FN, int FM, int AHEAD, int DT, bool ACT>
hipError_t launch(const Fp8Gemm& a, hipStream_t s) {
  const int tiles_n = (a.w_frags + WN * FN - 1) / (WN * FN), tiles_m = (a.x_frags + WM * FM - 1) / (WM * FM);
  const int64_t tiles = static_cast<int64_t>(tiles_n) * tiles_m, per_xcd = (tiles + 7) / 8;
  if (tiles >= (int64_t{1} << 28)) return hipErrorInvalidValue;
  // As many workgroups as the CUs of an XCD hold at once, by their LDS.
  constexpr int64_t resident = kFp8Cus / 8 * (4 * WM * FM * 2048 > 80 * 1024 ? 1 : 2);
  hipLaunchKernelGGL((tile_kernel<WN, WM, FN, FM, AHEAD, DT, ACT>), dim3(static_cast<unsigned>(8 * std::min(per_xcd, resident))),
                     dim3(64 * WN * WM), 0, s, a, Tiles{tiles_n, tiles_m, static_cast<int>(per_xcd)});
  return hipGetLastError();
}

template <int DT, bool ACT>
hipError_t pick(const Fp8Gemm& a, Fp8TileKind kind, hipStream_t s) {
  switch (kind) {   // fragments of a tile: kFp8Tiles
    case kTile64x64: return launch<2, 1, 2, 4, 3, DT, ACT>(a, s);
    case kTile128x64: return launch<4, 1, 2, 4, 3, DT, ACT>(a, s);
    case kTile128x128: return launch<4, 1, 2, 8, 3, DT, ACT>(a, s);
    default: return launch<4, 2, 4, 8, 1, DT, ACT>(a, s);
  }
}

}  // namespace

hipError_t fp8_tile(const Fp8Gemm& a, Fp8TileKind kind, bool act, hipStream_t s) {
  if (a.out == PLM_FP8_BF16) return act ? pick<DT_BF16, true>(a, kind, s) : pick<DT_BF16, false>(a, kind, s);
  return act ? pick<DT_F16, true>(a, kind, s) : pick<DT_F16, false>(a, kind, s);
}

}  // namespace plm

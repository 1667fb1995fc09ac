// Products over e4m3 rows for many rows of X: bound by the matrix cores.
//
// A workgroup has a tile of rows of the weight x rows of X, a wavefront FD x FS fragments of it. One operand comes into LDS (four
// sets, two blocks of K ahead), the other's fragments straight from memory into registers, a block ahead or three: read
// from LDS too, both operands of 256 x 256 took LDS as many cycles as the products take the matrix cores (8192 x 8192 x 2048
// 137 us). The fragments' order is what a wavefront's 16-byte reads want: no bank met twice, no address to compute.
//
// One barrier a block, in its middle, where the next block's set must have arrived; the operand that the next block
// begins with is read before this one's end, so the matrix cores do not run dry at either. Workgroups stay, and the loads run
// ahead into the next tile while the last one is stored.
//
// Tiles of 128 x 256 are for products of about as many of them as CUs: 4096 x 2048 x 5632 45 us for 51 with 128 x 128 and 56 with
// 256 x 256, 1024 x 8192 x 8192 64, 70 and 82.
//
// Measured, rows in 8 bits, weights from memory: 8192 x 8192 x 2048 112 us (2450 TFLOP/s; 26 us of it is what the stores take a
// copy), 8192^3 370 (2970), 2048 x 8192 x 8192 94. Of the last 70 remain with no loads at all: the products and the
// barriers, at the clock that they leave.
//
// Results in fp32 are sums of bf16 products, exact ones: a fragment's codes times their scales, 16 conversions for each of an
// operand's, 128 x 64 and 128 x 128 only. 2048 x 8192 x 2048 69 us (1000 TFLOP/s, of the 1650 that bf16's products reach; each
// wavefront converts all of X), 65 with tiles of 256 x 128, 127 the way of few rows.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "fp8_gemm.h"
#include "fp8_waits.h"

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
  return u32x2{two_bits16<DT>(v[0], v[1]), two_bits16<DT>(v[2], v[3])};
}

constexpr int kExact = -1;

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

// D is the operand whose fragments a wavefront reads into registers, FD of them, S the one that goes through LDS, FS; WL: S is the
// weight, else X. Weights are read from memory and X mostly from L2, so that the largest tiles, whose registers hold one block
// ahead only, have the weight in LDS: 8192 x 8192 x 2048 112.3 us for 117.4.
// DT: the result's, 16 bits, or kExact: fp32, of products added in fp32.
template <int WD, int WS, int FD, int FS, int AHEAD, bool WL, int DT, bool ACT>
__global__ __launch_bounds__(64 * WD * WS) void tile_kernel(Fp8Gemm a, Tiles tiles) {
  constexpr int kWaves = WD * WS, TD = WD * FD, TS = WS * FS, kStaged = 2 * TS / kWaves;
  constexpr int TN = WL ? TS : TD, TM = WL ? TD : TS, FN = WL ? FS : FD, FM = WL ? FD : FS;
  constexpr bool kWide = DT == kExact;
  static_assert(!kWide || !WL, "the exact products have X in LDS");
  static_assert(AHEAD == 1 || AHEAD == 3, "operands of two or four blocks");
  static_assert(2 * TS % kWaves == 0 && FS % 2 == 0, "every wavefront stages as many pieces of 1 KiB");
  constexpr Fp8TileLoads kLoads{FD, FS, kStaged, AHEAD};
  __shared__ __attribute__((aligned(16))) u32x4 set0[TS * 128], set1[TS * 128], set2[TS * 128], set3[TS * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int base = (blockIdx.x & 7) * tiles.per_xcd, count = min(tiles.per_xcd, tiles.n * tiles.m - base);
  const int stride = gridDim.x >> 3;
  int local = blockIdx.x >> 3;
  if (local >= count) return;
  const int wd = wave / WS, ws = wave - wd * WS, at_lane = lane * 16;
  const uint8_t *d_codes = WL ? a.x : a.w, *s_codes = WL ? a.w : a.x;
  const uint8_t *d_scales = WL ? a.x_scales : a.w_scales, *s_scales = WL ? a.w_scales : a.x_scales;
  const uint32_t d_frags = WL ? a.x_frags : a.w_frags, s_frags = WL ? a.w_frags : a.x_frags;
  const uint32_t d_block = d_frags * static_cast<uint32_t>(kFp8Bytes), s_block = s_frags * static_cast<uint32_t>(kFp8Bytes);
  const uint32_t d_scale_block = d_frags * static_cast<uint32_t>(kFp8ScaleBytes);
  const uint32_t s_scale_block = s_frags * static_cast<uint32_t>(kFp8ScaleBytes);

  // Four blocks of K from kb on: an operand's bytes there, and where in it a block's fragment lies. Fragments past the operand's
  // last are the next block's first, or zeros without traffic past its end; they reach no output that is stored. So are
  // D's blocks past K; S has its last one again there, since a set's older codes may be another row's NaN.
  struct Group {
    __amdgpu_buffer_rsrc_t d, s;
    int kb;
  };
  auto group_at = [&](int kb, bool in) {
    const uint32_t left = in ? static_cast<uint32_t>(min(a.blocks - kb, 4)) : 0u;
    return Group{make_rsrc(d_codes + static_cast<int64_t>(kb) * d_block, left * d_block),
                 make_rsrc(s_codes + static_cast<int64_t>(kb) * s_block, left * s_block), kb};
  };
  // Pieces [i0, i1) of a block of S into a set, and of D's operands into registers: 1 KiB a load.
  auto stage = [&](const Group& g, int s0, int j, u32x4* set, int i0, int i1) {
    const uint32_t at = static_cast<uint32_t>(min(j, a.blocks - 1 - g.kb)) * s_block + static_cast<uint32_t>(s0) * kFp8Bytes;
#pragma unroll
    for (int i = 0; i < kStaged; ++i)
      if (i >= i0 && i < i1) load_lds16(g.s, set + (i * kWaves + wave) * 64, at_lane + wave * 1024, at + i * (kWaves * 1024));
  };
  auto direct = [&](const Group& g, int d0, int j, i32x8 (&o)[FD], int i0, int i1) {
    const uint32_t at = static_cast<uint32_t>(j) * d_block + static_cast<uint32_t>(d0) * kFp8Bytes;
    const int here = anew(at_lane);
#pragma unroll
    for (int i = 0; i < FD; ++i) {
      if (i < i0 || i >= i1) continue;
      // Two fragments are within the 4 KiB of an instruction's own offset.
      const int from = static_cast<int>(at + (i & ~1) * kFp8Bytes), in_lane = here + (i & 1) * static_cast<int>(kFp8Bytes);
      o[i] = fp8_operand(__builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(g.d, in_lane, from, 0)),
                         __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(g.d, in_lane + 1024, from, 0)));
    }
  };
  // Four blocks' scales of fragments [f, f1) of an operand, a byte each. Past K they are zeros, which stand for 2^-127.
  auto scales = [&](const uint8_t* from, uint32_t block, int kb, bool in, int first, int i0, int i1, int* s) {
    const int here = anew((lane & 15) * 4);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(from + static_cast<int64_t>(kb >> 2) * block, in ? block : 0u);
#pragma unroll
    for (int i = i0; i < i1; ++i) s[i] = __builtin_amdgcn_raw_buffer_load_b32(r, here + i * 64, first * static_cast<int>(kFp8ScaleBytes), 0);
  };

  f32x4 acc[FD][FS];
  int ds[FD], ss[FS], next_ds[FD];
  i32x8 d[AHEAD + 1][FD], so[2];
  [[maybe_unused]] Fp8Exact exact[FD];
  const int s_at = ws * FS * 128 + lane;
  // The tile's first fragments: of this wavefront's D, and of S.
  auto first_of = [&](int tile, int& d0, int& s0) {
    int tn, tm;
    place_of(tiles, tile, tn, tm);
    d0 = (WL ? tm : tn) * TD + wd * FD;
    s0 = (WL ? tn : tm) * TS;
  };
  int d0, s0;
  first_of(base + local, d0, s0);
  scales(d_scales, d_scale_block, 0, true, d0, 0, FD, next_ds);
  scales(s_scales, s_scale_block, 0, true, s0 + ws * FS, 0, FS, ss);
  Group now = group_at(0, true);
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) direct(now, d0, j, d[j], 0, FD);
  stage(now, s0, 0, set0, 0, kStaged);
  stage(now, s0, 1, set1, 0, kStaged);
  stage(now, s0, 2, set2, 0, kStaged);
  tile_sync<fp8_first_wait(kLoads)>();   // the first set's have arrived, and the second's where step 0 does not wait for them
  so[0] = fp8_operand(set0[s_at], set0[s_at + 64]);
  const int columns = ACT ? a.n / 2 : a.n;

  // The wait before the barrier (fp8_waits.h): the loads issued since the next set's may be in flight. A barrier alone does not wait
  // for loads into LDS.
#define PLM_HALF(J, SET, NEXT, FROM, LOAD)                                                                                \
  _Pragma("unroll") for (int t = FROM; t < FROM + FS / 2; ++t) {                                                          \
    const u32x4* p = t + 1 < FS ? SET + s_at + (t + 1) * 128 : NEXT + s_at;                                               \
    so[(t + 1) & 1] = fp8_operand(p[0], p[64]);                                                                           \
    [[maybe_unused]] Fp8Exact other;                                                                                      \
    if constexpr (kWide) other = fp8_exact(so[t & 1], ss[t] >> (8 * J) & 255);                                            \
    _Pragma("unroll") for (int i = 0; i < FD; ++i)                                                                        \
        acc[i][t] = kWide ? fp8_mma_exact(exact[i], other, acc[i][t])                                                     \
                    : WL  ? mma_at<J>(so[t & 1], d[J % (AHEAD + 1)][i], acc[i][t], ss[t], ds[i])                          \
                          : mma_at<J>(d[J % (AHEAD + 1)][i], so[t & 1], acc[i][t], ds[i], ss[t]);                         \
    LOAD;                                                                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                                    \
  }
#define PLM_STEP(J, SET, NEXT, LAST, MORE)                                                                                \
  if constexpr (kWide) {                                                                                                  \
    _Pragma("unroll") for (int i = 0; i < FD; ++i) exact[i] = fp8_exact(d[J % (AHEAD + 1)][i], ds[i] >> (8 * J) & 255);   \
  }                                                                                                                       \
  PLM_HALF(J, SET, NEXT, 0,                                                                                               \
           MORE; direct(J + AHEAD < 4 ? now : next, J + AHEAD < 4 ? d0 : dn, (J + AHEAD) & 3, d[(J + AHEAD) % (AHEAD + 1)], \
                        t * 2 * FD / FS, (t + 1) * 2 * FD / FS))                                                          \
  tile_sync<fp8_step_wait(kLoads, J)>();                                                                                  \
  PLM_HALF(J, SET, NEXT, FS / 2,                                                                                          \
           MORE; stage(J == 0 ? now : next, J == 0 ? s0 : sn, (J + 3) & 3, LAST, (t - FS / 2) * 2 * kStaged / FS,         \
                       (t + 1 - FS / 2) * 2 * kStaged / FS))

  for (;;) {
    const bool more = local + stride < count;
    int d1 = 0, s1 = 0;
    if (more) first_of(base + local + stride, d1, s1);
#pragma unroll
    for (int i = 0; i < FD; ++i)
#pragma unroll
      for (int t = 0; t < FS; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int kb = 0; kb < a.blocks; kb += 4) {
      const bool last = kb + 4 >= a.blocks, in = !last || more;
      const int dn = last ? d1 : d0, sn = last ? s1 : s0;
      const Group next = group_at(last ? 0 : kb + 4, in);
#pragma unroll
      for (int i = 0; i < FD; ++i) ds[i] = next_ds[i];
      PLM_STEP(0, set0, set1, set3, )
      PLM_STEP(1, set1, set2, set0, )
      PLM_STEP(2, set2, set3, set1, )
      scales(d_scales, d_scale_block, next.kb, in, dn, 0, FD, next_ds);
      PLM_STEP(3, set3, set0, set2, scales(s_scales, s_scale_block, next.kb, in, sn + ws * FS, t, t + 1, ss))
      now = next;
    }

    constexpr int kOut = ACT ? FN / 2 : FN;
    const int n0 = (WL ? s0 + ws * FS : d0) / (ACT ? 2 : 1) * 16, m0 = (WL ? d0 : s0 + ws * FS) * 16, column = anew(lane);
#pragma unroll
    for (int t = 0; t < FM; ++t) {
      const int m = m0 + t * 16 + (column & 15);
      f32x4 v[kOut];
      auto sum = [&](int g) {
        const f32x4 s = WL ? acc[t][g] : acc[g][t];
        return kWide ? s * kFp8Exact : s;
      };
#pragma unroll
      for (int f = 0; f < kOut; ++f) {
        v[f] = sum(ACT ? 2 * f : f);
        if constexpr (ACT) {
          const f32x4 u = sum(2 * f + 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[f][j] = fp8_silu_mul(v[f][j], u[j]);
        }
      }
      if constexpr (kWide) {
#pragma unroll
        for (int f = 0; f < kOut; ++f) {
          const int n = n0 + f * 16 + (column >> 4) * 4;
          if (m < a.m && n < columns) fp8_store4(a, m, n, columns, v[f]);
        }
      } else if (kOut % 2 == 0 && n0 + kOut * 16 <= columns) {
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
    d0 = d1;
    s0 = s1;
  }
#undef PLM_STEP
#undef PLM_HALF
  __builtin_amdgcn_s_waitcnt(0x0f70);   // no load may arrive in this workgroup's LDS after its end
}

template <int WD, int WS, int FD, int FS, int AHEAD, bool WL, int DT, bool ACT>
hipError_t launch(const Fp8Gemm& a, hipStream_t s) {
  constexpr int TN = WL ? WS * FS : WD * FD, TM = WL ? WD * FD : WS * FS;
  const int tiles_n = (a.w_frags + TN - 1) / TN, tiles_m = (a.x_frags + TM - 1) / TM;
  const int64_t tiles = static_cast<int64_t>(tiles_n) * tiles_m, per_xcd = (tiles + 7) / 8;
  if (tiles >= (int64_t{1} << 28)) return hipErrorInvalidValue;
  // As many workgroups as the CUs of an XCD hold at once, by their LDS.
  constexpr int64_t resident = kFp8Cus / 8 * (4 * WS * FS * 2048 > 80 * 1024 ? 1 : 2);
  hipLaunchKernelGGL((tile_kernel<WD, WS, FD, FS, AHEAD, WL, DT, ACT>), dim3(static_cast<unsigned>(8 * std::min(per_xcd, resident))),
                     dim3(64 * WD * WS), 0, s, a, Tiles{tiles_n, tiles_m, static_cast<int>(per_xcd)});
  return hipGetLastError();
}

template <int DT, bool ACT>
hipError_t pick(const Fp8Gemm& a, Fp8TileKind kind, hipStream_t s) {
  switch (kind) {
    case kTile64x64: return launch<2, 1, 2, 4, 3, false, DT, ACT>(a, s);
    case kTile128x64: return launch<4, 1, 2, 4, 3, false, DT, ACT>(a, s);
    case kTile128x128: return launch<4, 1, 2, 8, 3, false, DT, ACT>(a, s);
    case kTile128x256: return launch<4, 2, 2, 8, 3, false, DT, ACT>(a, s);
    default: return launch<4, 2, 4, 8, 1, true, DT, ACT>(a, s);
  }
}

template <bool ACT>
hipError_t pick_exact(const Fp8Gemm& a, Fp8TileKind kind, hipStream_t s) {
  return kind == kTile128x64 ? launch<4, 1, 2, 4, 3, false, kExact, ACT>(a, s) : launch<4, 1, 2, 8, 1, false, kExact, ACT>(a, s);
}

}  // namespace

hipError_t fp8_tile(const Fp8Gemm& a, Fp8TileKind kind, bool act, hipStream_t s) {
  if (a.out == PLM_FP8_F32) return act ? pick_exact<true>(a, kind, s) : pick_exact<false>(a, kind, s);
  if (a.out == PLM_FP8_BF16) return act ? pick<DT_BF16, true>(a, kind, s) : pick<DT_BF16, false>(a, kind, s);
  return act ? pick<DT_F16, true>(a, kind, s) : pick<DT_F16, false>(a, kind, s);
}

}  // namespace plm

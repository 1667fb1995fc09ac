// The second launch of an attention whose sequences are cut: joins the ranges' partial results,
//   out = sum_j 2^(m_j - m) o_j / sum_j 2^(m_j - m) l_j, m the largest m_j.
// A launch of its own: joined by the last workgroup of each group to finish, a group's partial results came through one
// CU, past its caches, at about 50 GB/s (a round's 56 rows over 4007 tokens: 16 groups of 16 ranges, 11 us of 25).
// Here a workgroup takes eight columns of a group, thread by thread four dimensions of one.
#include "attend.h"

namespace plm {

template <int DT, int COLS>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
  constexpr int kSlices = COLS / kJoinColumns;
  __shared__ float weight[kAttendMost][kJoinColumns], sums[kAttendMost][kJoinColumns], total[kJoinColumns];
  const int slice = blockIdx.x % kSlices;
  const AttendItem it = attend_item<COLS, true>(a, blockIdx.x / kSlices, threadIdx.x & 63);
  if (it.ranges < 2) return;
  const KvSeq seq = kv_seq(a.rows, it.b, a.cache.page_shift);
  const int first = it.tile * COLS + slice * kJoinColumns;  // column of the sequence
  const int live = min(kJoinColumns, seq.rows * a.group - first);
  if (live <= 0) return;
  const int pad = 64 * a.cache.chunks, dim = a.cache.dim;
  const int64_t apart = attend_slot_floats(COLS, pad) * a.cache.heads;  // from a range to the next
  const float* slot = a.partials + it.slot * attend_slot_floats(COLS, pad);
  for (int i = threadIdx.x; i < it.ranges * kJoinColumns; i += 256) {
    const int range = i / kJoinColumns, c = i % kJoinColumns;
    const float* from = slot + range * apart + COLS * pad + slice * kJoinColumns + c;
    weight[range][c] = c < live ? from[0] : 0.0f;
    sums[range][c] = c < live ? from[COLS] : 0.0f;
  }
  __syncthreads();
  if (threadIdx.x < kJoinColumns) {
    const int c = threadIdx.x;
    constexpr float none = -__builtin_inff();
    float top = none, sum = 0.0f;
    for (int range = 0; range < it.ranges; ++range) top = fmaxf(top, weight[range][c]);
    for (int range = 0; range < it.ranges; ++range) {
      const float m = weight[range][c], x = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      weight[range][c] = x;
      sum += x * sums[range][c];
    }
    total[c] = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing is zero
  }
  __syncthreads();
  const int quads = dim >> 2;
  for (int i = threadIdx.x; i < live * quads; i += 256) {
    const int c = i / quads, e = (i - c * quads) << 2;
    const float* from = slot + (slice * kJoinColumns + c) * pad + e;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int base = 0; base < it.ranges; base += 8) {
      f32x4 part[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) part[k] = *reinterpret_cast<const f32x4*>(from + min(base + k, it.ranges - 1) * apart);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (base + k < it.ranges) sum += part[k] * weight[base + k][c];
    }
    sum *= total[c];
    const int column = first + c, row = column / a.group;
    uint16_t* at = a.out + (static_cast<int64_t>(seq.start + row) * a.heads + it.head * a.group + column - row * a.group) * dim;
    *reinterpret_cast<u32x2*>(at + e) = u32x2{pack2<DT>(sum[0], sum[1]), pack2<DT>(sum[2], sum[3])};
  }
}

namespace {

template <int COLS>
hipError_t join_go(int32_t dtype, const AttendArgs& a, unsigned groups, hipStream_t s) {
  const unsigned grid = groups * (COLS / kJoinColumns);
  if (dtype == PLM_BF16) attend_join_kernel<DT_BF16, COLS><<<grid, 256, 0, s>>>(a);
  else attend_join_kernel<DT_F16, COLS><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t attend_join(int32_t dtype, const AttendArgs& a, int columns, unsigned groups, hipStream_t s) {
  switch (columns) {
    case 16: return join_go<16>(dtype, a, groups, s);
    case 32: return join_go<32>(dtype, a, groups, s);
    case 64: return join_go<64>(dtype, a, groups, s);
    case 128: return join_go<128>(dtype, a, groups, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace plm

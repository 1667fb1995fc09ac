// The second launch of an attention whose sequences are cut: joins the ranges' partial results,
//   out = sum_j 2^(m_j - m) o_j / sum_j 2^(m_j - m) l_j, m the largest m_j.
// A launch of its own: joined by the last workgroup of each group to finish, a group's partial results came through one
// CU, past its caches, at about 50 GB/s (a round's 56 rows over 4007 tokens: 11 us of 25).
// Here a workgroup takes `take` columns of a group at a time, thread by thread four dimensions of one. Bound by latency
// (the lengths, the maxima and sums, the results: one after the other): 5.3 us behind that round's 3.7 MB of partial
// results, 5.6 behind the 1 MB of two sequences of 131004 tokens.
#include "attend.h"

namespace plm {

template <int DT, int COLS>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, int take, int slices, int items) {
  __shared__ float weight[kJoinColumns][kAttendMost], total[kJoinColumns];
  __shared__ f32x4 parts[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pad = 64 * a.cache.chunks, dim = a.cache.dim, quads = dim >> 2;
  const int64_t apart = attend_slot_floats(COLS, pad) * a.cache.heads;  // from a range to the next
  // A thread's share: every `lanes`-th range of four dimensions of a column.
  const int work = take * quads, lanes = 256 / work, share = threadIdx.x / work;
  const int c = (threadIdx.x - share * work) / quads, e = (threadIdx.x - share * work - c * quads) << 2;
  for (int index = blockIdx.x; index < items; index += gridDim.x) {
    const AttendItem it = attend_item<COLS, true>(a, index / slices, lane);
    if (it.ranges < 2) return;
    const int slice = index % slices;
    const int first = it.tile * COLS + slice * take;  // column of the sequence
    const int live = min(take, it.seq.rows * a.group - first);
    if (live <= 0) continue;
    const float* slot = a.partials + it.slot * attend_slot_floats(COLS, pad);
    // The first eight of the thread's loads go with the maxima's and sums'.
    const bool mine = share < lanes && c < live;
    const float* from = slot + (slice * take + c) * pad + e;
    f32x4 part[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (mine) part[k] = *reinterpret_cast<const f32x4*>(from + min(share + k * lanes, it.ranges - 1) * apart);
    // A wavefront per column, a lane per range.
    static_assert(kAttendMost == 64, "a lane per range");
    for (int x = wave; x < live; x += 4) {
      const float* at = slot + min(lane, it.ranges - 1) * apart + COLS * pad + slice * take + x;
      const float m = lane < it.ranges ? at[0] : -__builtin_inff(), l = at[COLS];
      float top = m;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      const float y = lane >= it.ranges ? 0.0f : m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      weight[x][lane] = y;
      const float sum = wave_total(lane < it.ranges ? y * l : 0.0f);
      if (lane == 0) total[x] = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing is zero
    }
    __syncthreads();
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) {
      for (int base = share; base < it.ranges; base += 8 * lanes) {
        if (base != share) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            part[k] = *reinterpret_cast<const f32x4*>(from + min(base + k * lanes, it.ranges - 1) * apart);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (base + k * lanes < it.ranges) sum += part[k] * weight[c][base + k * lanes];
      }
    }
    parts[threadIdx.x] = sum;
    __syncthreads();
    if (share == 0 && c < live) {
      for (int k = 1; k < lanes; ++k) sum += parts[threadIdx.x + k * work];
      sum *= total[c];
      const int column = first + c, row = column / a.group;
      uint16_t* at = a.out + (static_cast<int64_t>(it.seq.start + row) * a.heads + it.head * a.group + column - row * a.group) * dim;
      *reinterpret_cast<u32x2*>(at + e) = u32x2{pack2<DT>(sum[0], sum[1]), pack2<DT>(sum[2], sum[3])};
    }
    __syncthreads();
  }
}

namespace {

template <int COLS>
hipError_t join_go(int32_t dtype, const AttendArgs& a, int64_t groups, int columns, hipStream_t s) {
  // Few columns per workgroup while the device has room for more of them, each of which costs a look at the lengths:
  // cut decodes one at a time. What the grid does not cover is taken in turns.
  const int quads = a.cache.dim / 4;
  int take = 1;
  while (take < kJoinColumns && 2 * take * quads <= 256 && groups * ((columns + take - 1) / take) > 512) take *= 2;
  const int slices = (columns + take - 1) / take;
  const int items = static_cast<int>(groups) * slices;
  const unsigned grid = static_cast<unsigned>(items < 2048 ? items : 2048);
  if (dtype == PLM_BF16) attend_join_kernel<DT_BF16, COLS><<<grid, 256, 0, s>>>(a, take, slices, items);
  else attend_join_kernel<DT_F16, COLS><<<grid, 256, 0, s>>>(a, take, slices, items);
  return hipGetLastError();
}

}  // namespace

hipError_t attend_join(int32_t dtype, const AttendArgs& a, int columns, int64_t groups, hipStream_t s) {
  const int64_t most = static_cast<int64_t>(a.rows.max_rows) * a.group;
  const int live = static_cast<int>(most < columns ? most : columns);
  switch (columns) {
    case 16: return join_go<16>(dtype, a, groups, live, s);
    case 32: return join_go<32>(dtype, a, groups, live, s);
    case 64: return join_go<64>(dtype, a, groups, live, s);
    case 128: return join_go<128>(dtype, a, groups, live, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace plm

// Attention of a call's rows over the paged cache (plm_attend, include/plm_amd.h).
//
// Per query: softmax over the visible tokens of scale * q . k, times the values, in one pass over the
// tokens with the running maximum m and sum l of the exponentials (base 2: the scale carries log2 e).
//
// Orientation: a wavefront computes S^T = K Q^T (16 tokens x 16 columns per MFMA chain, a column being
// one query: row * group + head of the group) and O^T = V^T P^T. The accumulator registers of S^T (lane
// l: tokens 4 (l / 16) + r of column l % 16) are, rounded, the B operand of the second product with no
// move between lanes, since the values are laid out for that order of tokens (kv_cache.h); the output
// comes out with 16 consecutive dimensions per lane. Keys and values go from memory straight into
// operand registers: 16 bytes per lane, 1 KiB per load, no LDS.
//
// A workgroup's W wavefronts take every W-th step of 32 tokens of one range of one (sequence, tile of
// columns, key head), and are joined through LDS at the end. Ranges of the same (sequence, tile, head)
// are joined by the last of their workgroups to finish, through partial results in device memory.
#pragma once

#include "kv_cache.h"

namespace plm {

struct AttendArgs {
  KvCache cache;
  KvRows rows;
  const uint16_t* q;
  uint16_t* out;  // contiguous [total, heads, dim]
  int64_t q_row, q_head;
  const int64_t* positions;  // [total]; null: context + row
  const uint32_t* mask;      // [mask_rows, mask_words]; null: causal
  int* counters;             // one per (sequence, tile, head) of several ranges, zero between calls
  float* partials;           // slots of attend_slot_floats(columns, padded dim)
  float scale;               // times log2 e
  int heads, group, window, sinks, mask_rows, mask_words;
  int target;   // workgroups that the work is split over, at most; 0: never split
  int least;    // steps of a range, at least
  int most;     // ranges per group, at most
};

constexpr int kStep = 32;  // tokens of a step

__host__ __device__ constexpr int64_t attend_slot_floats(int columns, int padded) {
  return static_cast<int64_t>(columns) * (padded + 2);
}

// A sequence's share of the work, the same in every workgroup.
struct AttendShare {
  int tiles, steps;
};

template <int COLS>
__device__ __forceinline__ AttendShare attend_share(const AttendArgs& a, int b) {
  AttendShare s{0, 0};
  if (b >= a.rows.seqs) return s;
  const KvSeq seq = kv_seq(a.rows, b, a.cache.page_shift);
  if (seq.rows == 0) return s;
  s.tiles = (seq.rows * a.group + COLS - 1) / COLS;
  // With a window, the first row's place says where it begins: where a later row's place is before it,
  // the ranges get longer, and that is all.
  const int64_t place = a.positions != nullptr ? a.positions[seq.start] : seq.context;
  const int hi = (seq.context + seq.rows + kStep - 1) / kStep;
  int lo = 0;
  if (a.window > 0) lo = static_cast<int>(min(max(place + 1 - a.window, int64_t{0}), static_cast<int64_t>(hi) * kStep)) / kStep;
  s.steps = hi - lo + min((a.sinks + kStep - 1) / kStep, lo);
  return s;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(v, d);
    if (lane >= d) v += below;
  }
  return v;
}

struct AttendItem {
  int b, tile, head, range, ranges;  // ranges == 0: nothing to do
  int group;                         // number of the (sequence, tile, head) among those of several ranges
  int slot;                          // first of the group's partial slots, in steps of `heads`
};

// Which range of which group workgroup `index` takes. The work of the whole call (steps x tiles x heads,
// from the lengths on the device) is cut so that about `target` workgroups share it evenly, whatever the
// sequences' lengths and the table's width: a launch sized on the host alone would have to cut the widest
// sequence the table could hold. Every wavefront scans the sequences by itself, 64 at a time.
template <int COLS>
__device__ __forceinline__ AttendItem attend_item(const AttendArgs& a, int index, int lane) {
  const int heads = a.cache.heads;
  AttendItem it{};
  int chunk = 1 << 30;
  AttendShare own = attend_share<COLS>(a, lane);
  if (a.target > 0) {
    int64_t load = 0;
    for (int base = 0; base < a.rows.seqs; base += 64) {
      const AttendShare s = base == 0 ? own : attend_share<COLS>(a, base + lane);
      load += static_cast<int64_t>(s.tiles) * s.steps;
    }
    load = wave_sum64(load) * heads;
    chunk = static_cast<int>(min(max((load + a.target - 1) / a.target, static_cast<int64_t>(a.least)), int64_t{1} << 30));
  }
  int items = 0, groups = 0, slots = 0;
  for (int base = 0; base < a.rows.seqs; base += 64) {
    const AttendShare s = base == 0 ? own : attend_share<COLS>(a, base + lane);
    const int ranges = min(max((s.steps + chunk - 1) / chunk, 1), a.most);
    const int mine = s.tiles * ranges * heads;
    const int to = wave_scan(mine, lane);
    // Only groups of several ranges have a counter and slots.
    const int split = ranges > 1 ? s.tiles * heads : 0;
    const int group_to = a.target > 0 ? wave_scan(split, lane) : 0;
    const int slot_to = a.target > 0 ? wave_scan(split * ranges, lane) : 0;
    const uint64_t past = __ballot(items + to > index);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int first = items + __shfl(to - mine, at);
      it.b = base + at;
      it.ranges = __shfl(ranges, at);
      const int tiles = __shfl(s.tiles, at);
      const int rest = index - first;
      if (rest < 0 || tiles < 1) return AttendItem{};
      it.head = rest % heads;
      const int x = rest / heads;
      it.range = x % it.ranges;
      it.tile = tiles - 1 - x / it.ranges;  // a causal tile's work grows with its number: the longest first
      it.group = groups + __shfl(group_to, at) - tiles * heads + it.tile * heads + it.head;
      it.slot = slots + __shfl(slot_to, at) - tiles * it.ranges * heads + it.tile * it.ranges * heads + it.head;
      it.b = __builtin_amdgcn_readfirstlane(it.b);
      it.ranges = __builtin_amdgcn_readfirstlane(it.ranges);
      it.head = __builtin_amdgcn_readfirstlane(it.head);
      it.range = __builtin_amdgcn_readfirstlane(it.range);
      it.tile = __builtin_amdgcn_readfirstlane(it.tile);
      it.group = __builtin_amdgcn_readfirstlane(it.group);
      it.slot = __builtin_amdgcn_readfirstlane(it.slot);
      return it;
    }
    items += __shfl(to, 63);
    groups += __shfl(group_to, 63);
    slots += __shfl(slot_to, 63);
  }
  return it;
}

// The lane's value and its partner's, 32 (WIDE) or 16 lanes away, in either order.
template <bool WIDE>
__device__ __forceinline__ void lane_pair(float v, float& a, float& b) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  uint32_t lo, hi;  // copies: a bit cast of a vector's element reads its first one
  if constexpr (WIDE) {
    const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    lo = p[0], hi = p[1];
  } else {
    const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    lo = p[0], hi = p[1];
  }
  a = __builtin_bit_cast(float, lo);
  b = __builtin_bit_cast(float, hi);
}

// Maximum and sum over the four lanes that hold a column's tokens (lanes l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float column_max(float v) {
  float a, b;
  lane_pair<true>(v, a, b);
  lane_pair<false>(fmaxf(a, b), a, b);
  return fmaxf(a, b);
}

__device__ __forceinline__ float column_sum(float v) {
  float a, b;
  lane_pair<true>(v, a, b);
  lane_pair<false>(a + b, a, b);
  return a + b;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return to_bits16<DT>(a) | (static_cast<uint32_t>(to_bits16<DT>(b)) << 16);
}

// Whether a 16-bit pair holds an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool pair_not_finite(uint32_t w) {
  constexpr uint32_t e = DT == DT_BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

constexpr float kMinusInf = -__builtin_inff();
// The running maximum follows a larger one only where that is more than this (base 2) above it, so most
// steps leave the accumulators alone; exponentials then reach 2^kSlack, exact in fp32 sums. fp16
// probabilities carry 2^kShift besides (out of both sums at the end), so that small ones stay normal:
// 2^(kSlack + kShift) is inside fp16.
constexpr float kSlack = 6.0f;
template <int DT>
constexpr float kShift = DT == DT_F16 ? 8.0f : 0.0f;

// A wavefront's state and its walk over tokens.
template <int DT, bool E8, int C, int NC>
struct AttendWave {
  static constexpr int kLoads = E8 ? 1 : 2;  // of 16 bytes per lane, unit and chunk
  static constexpr int kUnitBytes = 1024 * kLoads;

  struct Step {
    u32x4 k[2][C][kLoads], v[2][C][kLoads];
    float ks[2], vs[2];
    bool held[2];  // the unit's page is a page of the cache
  };

  f32x4 o[NC][C][4];
  u32x4 q[NC][C][2];
  float m[NC], l[NC];
  float ref;  // largest scale of the values so far: the accumulators are in its units
  int page_id, page_first;  // lane i: page number page_first + i of the sequence
  float page_ks, page_vs;

  __device__ __forceinline__ void pages(const AttendArgs& a, int b, int head, int number, int last, int lane) {
    page_first = number;
    const int at = number + lane;
    int id = -1;
    if (at < last && at < a.rows.width) id = a.rows.table[b * a.rows.table_stride + at];
    const bool good = id >= 0 && id < a.cache.pages;
    page_id = good ? id : -1;
    if constexpr (E8) {
      page_ks = good ? a.cache.k_scale[static_cast<int64_t>(id) * a.cache.heads + head] : 0.0f;
      page_vs = good ? a.cache.v_scale[static_cast<int64_t>(id) * a.cache.heads + head] : 0.0f;
      float most = page_vs;
#pragma unroll
      for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x));
      most = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, most)));
      if (most > ref) {
        const float less = ref / most;
        ref = most;
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][c][j] *= less;
      }
    }
  }

  __device__ __forceinline__ void fetch(const AttendArgs& a, int b, int head, int t0, int last_page, int lane, Step& s) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = t0 + 16 * u;
      const int number = t >> a.cache.page_shift;
      if (number < page_first || number >= page_first + 64) pages(a, b, head, number, last_page, lane);
      const int id = __builtin_amdgcn_readlane(page_id, number - page_first);
      s.held[u] = id >= 0;
      if constexpr (E8) {
        s.ks[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, page_ks), number - page_first));
        s.vs[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, page_vs), number - page_first));
      }
      const int unit = (t & (a.cache.page - 1)) >> 4;
      const int64_t at = ((static_cast<int64_t>(max(id, 0)) * a.cache.heads + head) * (a.cache.page >> 4) + unit) *
                         (a.cache.chunks * kUnitBytes);
      const char* k = a.cache.k + at;
      const char* v = a.cache.v + at;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < kLoads; ++h) {
          const uint32_t off = c * kUnitBytes + h * 1024 + lane * 16;
          // Dimensions past the head's are not read: 16 (keys) or 4 (values) of them per lane.
          s.k[u][c][h] = 64 * c + 16 * (lane >> 4) < a.cache.dim ? *reinterpret_cast<const u32x4*>(k + off) : u32x4{0u, 0u, 0u, 0u};
          s.v[u][c][h] = 64 * c + 4 * (lane & 15) < a.cache.dim ? *reinterpret_cast<const u32x4*>(v + off) : u32x4{0u, 0u, 0u, 0u};
        }
    }
  }
};

template <int DT, bool E8, int C, int NC, int W>
__global__ __launch_bounds__(64 * W) void attend_kernel(AttendArgs a) {
  constexpr int COLS = 16 * NC, PAD = 64 * C;
  extern __shared__ char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const AttendItem it = attend_item<COLS>(a, blockIdx.x, lane);
  if (it.ranges == 0) return;
  KvSeq seq = kv_seq(a.rows, it.b, a.cache.page_shift);
  seq.start = __builtin_amdgcn_readfirstlane(seq.start);
  seq.rows = __builtin_amdgcn_readfirstlane(seq.rows);
  seq.context = __builtin_amdgcn_readfirstlane(seq.context);
  const int columns = seq.rows * a.group;
  const int dim = a.cache.dim;

  using Wave = AttendWave<DT, E8, C, NC>;
  Wave w;
  w.ref = 0.0f;
  w.page_first = -64;
  int row[NC], place[NC], window_lo[NC], head_of[NC];
  bool real[NC];
  constexpr int kFar = 1 << 30;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int x = it.tile * COLS + 16 * n + col;
    real[n] = x < columns;
    row[n] = min(x, columns - 1) / a.group;
    head_of[n] = it.head * a.group + min(x, columns - 1) % a.group;
    const int64_t at = seq.start + row[n];
    const int64_t p = a.positions != nullptr ? a.positions[at] : seq.context + row[n];
    place[n] = static_cast<int>(min(max(p, static_cast<int64_t>(-kFar)), static_cast<int64_t>(kFar)));
    window_lo[n] = a.window > 0 ? max(place[n] - a.window + 1, 0) : 0;
    const uint16_t* from = a.q + at * a.q_row + head_of[n] * a.q_head;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = 64 * c + 16 * g + 8 * h;
        w.q[n][c][h] = real[n] && e < dim ? *reinterpret_cast<const u32x4*>(from + e) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 2; ++j) w.o[n][c][2 * h + j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    w.m[n] = kMinusInf;
    w.l[n] = 0.0f;
  }

  // The tile's tokens: [0, 32 sink_steps) and [32 first, end).
  const int end = seq.context + seq.rows;
  const int row_lo = it.tile * COLS / a.group, row_hi = min((it.tile + 1) * COLS, columns) - 1;
  const int tile_end = a.mask != nullptr ? end : seq.context + row_hi / a.group + 1;
  const int whole = a.mask != nullptr ? seq.context : seq.context + row_lo + 1;  // seen by every column, window apart
  int lo_least = 0, lo_most = 0;
  if (a.window > 0) {
    lo_least = kFar;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      lo_least = min(lo_least, window_lo[n]);
      lo_most = max(lo_most, window_lo[n]);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
      lo_least = min(lo_least, __shfl_xor(lo_least, x));
      lo_most = max(lo_most, __shfl_xor(lo_most, x));
    }
    // Under a mask the window holds for the context alone: the rows' own tokens are always walked.
    if (a.mask != nullptr) lo_least = min(lo_least, seq.context);
    lo_least = __builtin_amdgcn_readfirstlane(lo_least);
    lo_most = __builtin_amdgcn_readfirstlane(lo_most);
  }
  const int last_step = (tile_end + kStep - 1) / kStep;
  const int first = min(lo_least / kStep, last_step);
  const int sink_steps = min((a.sinks + kStep - 1) / kStep, first);
  const int steps = sink_steps + last_step - first;
  const int from = static_cast<int>(static_cast<int64_t>(steps) * it.range / it.ranges);
  const int to = static_cast<int>(static_cast<int64_t>(steps) * (it.range + 1) / it.ranges);
  const int last_page = (end + a.cache.page - 1) >> a.cache.page_shift;
  auto token_of = [&](int s) { return kStep * (s < sink_steps ? s : first + s - sink_steps); };

  auto compute = [&](const typename Wave::Step& s, int t0) {
    const bool edge = t0 + kStep > whole || (a.window > 0 && t0 < lo_most && t0 + kStep > a.sinks) || !s.held[0] || !s.held[1];
    // S^T of both units, all columns.
    f32x4 score[NC][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int n = 0; n < NC; ++n) score[n][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        u32x4 k0, k1;
        if constexpr (E8) {
          const u32x4 x = s.k[u][c][0];
          k0 = fp8_eight<DT>(x[0], x[1], 1.0f);
          k1 = fp8_eight<DT>(x[2], x[3], 1.0f);
        } else {
          k0 = s.k[u][c][0];
          k1 = s.k[u][c][1];
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          score[n][u] = mfma_16x16x32<DT>(k0, w.q[n][c][0], score[n][u]);
          score[n][u] = mfma_16x16x32<DT>(k1, w.q[n][c][1], score[n][u]);
        }
      }
    }
    u32x4 p[NC];
    uint32_t seen_bits[NC];  // bit 4 u + r: token t0 + 16 u + 4 g + r is seen by the lane's column
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u) score[n][u] *= E8 ? a.scale * s.ks[u] : a.scale;
      if (edge) {
        seen_bits[n] = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int t = t0 + 16 * u + 4 * g + r;
            const bool near = t >= window_lo[n] || t < a.sinks;
            bool seen;
            if (a.mask == nullptr) {
              seen = near && t <= seq.context + row[n];
            } else if (t < seq.context) {
              seen = near;
            } else {
              const int i = t - seq.context;
              seen = i < seq.rows && (i >> 5) < a.mask_words && row[n] < a.mask_rows &&
                     ((a.mask[static_cast<int64_t>(row[n]) * a.mask_words + (i >> 5)] >> (i & 31)) & 1u) != 0;
            }
            seen = seen && t < end && s.held[u];
            seen_bits[n] |= static_cast<uint32_t>(seen) << (4 * u + r);
            score[n][u][r] = seen ? score[n][u][r] : kMinusInf;
          }
      }
      float top = kMinusInf;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, score[n][u][r]);
      top = column_max(top);
      if (__any(top > w.m[n] + kSlack)) {
        const float next = fmaxf(w.m[n], top);
        const float less = w.m[n] == next ? 1.0f : __builtin_amdgcn_exp2f(w.m[n] - next);
        w.m[n] = next;
        w.l[n] *= less;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) w.o[n][c][j] *= less;
      }
      const float base = w.m[n] == kMinusInf ? 0.0f : w.m[n] - kShift<DT>;
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(score[n][i / 4][i % 4] - base);
        w.l[n] += e[i];
      }
      // Probabilities in the model's type, as its matrix product takes them; their sum is of the fp32 ones.
#pragma unroll
      for (int i = 0; i < 4; ++i) p[n][i] = pack2<DT>(e[2 * i], e[2 * i + 1]);
    }
    // O^T += V^T P^T: operand j of a chunk has dimensions 4 (l % 16) + j as rows.
    const float less = w.ref > 0.0f ? 1.0f / w.ref : 0.0f;
    float ratio[2] = {1.0f, 1.0f};
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};  // per pair of tokens: 16-bit masks of those that any column may see
    if constexpr (E8) {
      ratio[0] = s.vs[0] * less;
      ratio[1] = s.vs[1] * less;
    }
    if (edge) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int t = t0 + 16 * u + 4 * g + 2 * r;
          keep[2 * u + r] = (s.held[u] && t < end ? 0xffffu : 0u) | (s.held[u] && t + 1 < end ? 0xffff0000u : 0u);
        }
    }
    auto values_of = [&](int c, int j) {
      u32x4 v;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (E8) {
          v[2 * u] = fp8_pair<DT>(s.v[u][c][0][j], ratio[u], false);
          v[2 * u + 1] = fp8_pair<DT>(s.v[u][c][0][j], ratio[u], true);
        } else {
          v[2 * u] = s.v[u][c][j / 2][2 * (j & 1)];
          v[2 * u + 1] = s.v[u][c][j / 2][2 * (j & 1) + 1];
        }
      }
      return v;
    };
    if (!edge) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 v = values_of(c, j);
#pragma unroll
          for (int n = 0; n < NC; ++n) w.o[n][c][j] = mfma_16x16x32<DT>(v, p[n], w.o[n][c][j]);
        }
      return;
    }
    // A value that is not finite where some columns do not look: 0 * it would reach them. Where an
    // operand has one, its tokens go one at a time, and only the columns that see a token take its result.
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 v = values_of(c, j);
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] &= keep[i];
          odd = odd || pair_not_finite<DT>(v[i]);
        }
        if (!__any(odd)) {
#pragma unroll
          for (int n = 0; n < NC; ++n) w.o[n][c][j] = mfma_16x16x32<DT>(v, p[n], w.o[n][c][j]);
          continue;
        }
#pragma unroll 1
        for (int x = 0; x < kStep; ++x) {
          const int slot = ((x >> 4) << 2) | (x & 3);  // the token's place among a lane's eight
          const int holder = (x & 15) >> 2;            // the lanes that hold it
          const uint32_t half = holder == g ? 0xffffu << (16 * (slot & 1)) : 0u;
          u32x4 only;
#pragma unroll
          for (int i = 0; i < 4; ++i) only[i] = (slot >> 1) == i ? half : 0u;
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            const bool sees = ((__shfl(static_cast<int>(seen_bits[n]), holder * 16 + col) >> slot) & 1) != 0;
            const f32x4 sum = mfma_16x16x32<DT>(v & only, p[n] & only, w.o[n][c][j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) w.o[n][c][j][r] = sees ? sum[r] : w.o[n][c][j][r];
          }
        }
      }
  };

  {
    typename Wave::Step next;
    int s = from + wave;
    if (s < to) w.fetch(a, it.b, it.head, token_of(s), last_page, lane, next);
    while (s < to) {
      const typename Wave::Step now = next;
      const int t0 = token_of(s);
      s += W;
      if (s < to) w.fetch(a, it.b, it.head, token_of(s), last_page, lane, next);
      compute(now, t0);
    }
  }

  // Every wavefront's result in plain units, then joined by halves through LDS.
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    w.l[n] = column_sum(w.l[n]);
    if constexpr (E8) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) w.o[n][c][j] *= w.ref;
    }
  }
  constexpr int kWaveFloats = NC * (C * 16 + 2) * 64;
  float* shared = reinterpret_cast<float*>(lds);
  for (int half = W / 2; half > 0; half >>= 1) {
    if (half != W / 2) __syncthreads();
    if (wave >= half && wave < 2 * half) {
      float* to_ = shared + (wave - half) * kWaveFloats + lane;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) to_[((n * C + c) * 16 + j * 4 + r) * 64] = w.o[n][c][j][r];
        to_[(NC * C * 16 + 2 * n) * 64] = w.m[n];
        to_[(NC * C * 16 + 2 * n + 1) * 64] = w.l[n];
      }
    }
    __syncthreads();
    if (wave < half) {
      const float* other = shared + wave * kWaveFloats + lane;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const float m = other[(NC * C * 16 + 2 * n) * 64], l = other[(NC * C * 16 + 2 * n + 1) * 64];
        const float top = fmaxf(w.m[n], m);
        const float x = w.m[n] == top ? 1.0f : __builtin_amdgcn_exp2f(w.m[n] - top);
        const float y = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        w.m[n] = top;
        w.l[n] = w.l[n] * x + l * y;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              w.o[n][c][j][r] = w.o[n][c][j][r] * x + other[((n * C + c) * 16 + j * 4 + r) * 64] * y;
      }
    }
  }

  if (it.ranges == 1) {
    if (wave != 0) return;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (!real[n]) continue;
      const float inverse = w.l[n] == 0.0f ? 0.0f : 1.0f / w.l[n];  // a row that sees nothing is zero
      uint16_t* at = a.out + (static_cast<int64_t>(seq.start + row[n]) * a.heads + head_of[n]) * dim;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = 64 * c + 16 * g;
        u32x4 word[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // dimensions e + 2 i, e + 2 i + 1
          const int r = i / 2, j = 2 * (i & 1);
          word[i / 4][i % 4] = pack2<DT>(w.o[n][c][j][r] * inverse, w.o[n][c][j + 1][r] * inverse);
        }
        if (e < dim) *reinterpret_cast<u32x4*>(at + e) = word[0];
        if (e + 8 < dim) *reinterpret_cast<u32x4*>(at + e + 8) = word[1];
      }
    }
    return;
  }

  // A range of several: the partial result goes to the group's slot `range`; the group's last workgroup
  // joins them. Slot: [COLS][PAD] sums, then [COLS] maxima and [COLS] sums of exponentials.
  constexpr uint32_t kSlotBytes = static_cast<uint32_t>(attend_slot_floats(COLS, PAD) * 4);
  const int heads = a.cache.heads;
  if (wave == 0) {
    char* mine = reinterpret_cast<char*>(a.partials) + static_cast<int64_t>(it.slot + it.range * heads) * kSlotBytes;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(mine, kSlotBytes);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (!real[n]) continue;
      const int at = 16 * n + col;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const f32x4 x = {w.o[n][c][0][r], w.o[n][c][1][r], w.o[n][c][2][r], w.o[n][c][3][r]};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), rs,
                                                 (at * PAD + 64 * c + 16 * g + 4 * r) * 4, 0, kCoherent);
        }
      if (g == 0) {
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, w.m[n]), rs, (COLS * PAD + at) * 4, 0, kCoherent);
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, w.l[n]), rs, (COLS * PAD + COLS + at) * 4, 0, kCoherent);
      }
    }
  }
  if (!arrive_last(a.counters + it.group, it.ranges)) return;
  // Weights of the ranges per column in LDS, then every thread joins four dimensions of a column.
  const int live = min(COLS, columns - it.tile * COLS);
  float* weight = shared;                     // [ranges][COLS]
  float* total = weight + a.most * COLS;      // [COLS]
  auto slot_of = [&](int range) {
    return reinterpret_cast<const char*>(a.partials) + static_cast<int64_t>(it.slot + range * heads) * kSlotBytes;
  };
  for (int i = threadIdx.x; i < it.ranges * COLS; i += 64 * W) {
    const int range = i / COLS, c = i % COLS;
    weight[i] = c < live ? collect(reinterpret_cast<const float*>(slot_of(range)) + COLS * PAD + c) : kMinusInf;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < live) {
    float top = kMinusInf, sum = 0.0f;
    for (int range = 0; range < it.ranges; ++range) top = fmaxf(top, weight[range * COLS + threadIdx.x]);
    for (int range = 0; range < it.ranges; ++range) {
      const float m = weight[range * COLS + threadIdx.x];
      const float x = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      weight[range * COLS + threadIdx.x] = x;
      sum += x * collect(reinterpret_cast<const float*>(slot_of(range)) + COLS * PAD + COLS + threadIdx.x);
    }
    total[threadIdx.x] = sum == 0.0f ? 0.0f : 1.0f / sum;
  }
  __syncthreads();
  const int quads = dim >> 2;
  for (int i = threadIdx.x; i < live * quads; i += 64 * W) {
    const int c = i / quads, e = (i - c * quads) << 2;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int range = 0; range < it.ranges; ++range) {
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(slot_of(range), kSlotBytes);
      const f32x4 x = __builtin_bit_cast(
          f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, (c * PAD + e) * 4, 0, kCoherent));
      sum += x * weight[range * COLS + c];
    }
    sum *= total[c];
    const int x = it.tile * COLS + c;
    uint16_t* at = a.out + (static_cast<int64_t>(seq.start + x / a.group) * a.heads + it.head * a.group + x % a.group) * dim;
    *reinterpret_cast<u32x2*>(at + e) = u32x2{pack2<DT>(sum[0], sum[1]), pack2<DT>(sum[2], sum[3])};
  }
}

// Columns of a tile and wavefronts of a workgroup for heads of C chunks, by the columns that the longest
// sequence may have per key head.
inline int attend_column_tiles(int chunks, int64_t columns) {
  if (columns <= 16) return 1;
  if (columns <= 32 || chunks > 2) return 2;
  return 4;
}

hipError_t attend_bf16_e4m3(const AttendArgs& a, int tiles, unsigned grid, hipStream_t s);
hipError_t attend_bf16_model(const AttendArgs& a, int tiles, unsigned grid, hipStream_t s);
hipError_t attend_f16_e4m3(const AttendArgs& a, int tiles, unsigned grid, hipStream_t s);
hipError_t attend_f16_model(const AttendArgs& a, int tiles, unsigned grid, hipStream_t s);

constexpr int kAttendMost = 64;  // ranges per group, at most

template <int DT, bool E8, int C, int NC>
hipError_t attend_launch(const AttendArgs& a, unsigned grid, hipStream_t s) {
  constexpr int W = NC == 1 ? 8 : 4;
  constexpr size_t join = static_cast<size_t>(W / 2) * NC * (C * 16 + 2) * 64 * 4;
  constexpr size_t weights = static_cast<size_t>(kAttendMost + 1) * 16 * NC * 4;
  constexpr size_t bytes = join > weights ? join : weights;
  auto* kern = &attend_kernel<DT, E8, C, NC, W>;
  if (bytes > 64 * 1024) {
    static const hipError_t raised = hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (raised != hipSuccess) return raised;
  }
  kern<<<grid, 64 * W, bytes, s>>>(a);
  return hipGetLastError();
}

template <int DT, bool E8>
hipError_t attend_pick(const AttendArgs& a, int tiles, unsigned grid, hipStream_t s) {
  switch (a.cache.chunks * 8 + tiles) {
    case 8 + 1: return attend_launch<DT, E8, 1, 1>(a, grid, s);
    case 8 + 2: return attend_launch<DT, E8, 1, 2>(a, grid, s);
    case 8 + 4: return attend_launch<DT, E8, 1, 4>(a, grid, s);
    case 16 + 1: return attend_launch<DT, E8, 2, 1>(a, grid, s);
    case 16 + 2: return attend_launch<DT, E8, 2, 2>(a, grid, s);
    case 16 + 4: return attend_launch<DT, E8, 2, 4>(a, grid, s);
    case 24 + 1: return attend_launch<DT, E8, 3, 1>(a, grid, s);
    case 24 + 2: return attend_launch<DT, E8, 3, 2>(a, grid, s);
    case 32 + 1: return attend_launch<DT, E8, 4, 1>(a, grid, s);
    case 32 + 2: return attend_launch<DT, E8, 4, 2>(a, grid, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace plm

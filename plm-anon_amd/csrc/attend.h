// Attention of a call's rows over the paged cache (plm_attend, include/plm_amd.h).
//
// Per query: softmax over the visible tokens of scale * q . k, times the values, in one pass over the
// tokens with the running maximum m and sum l of the exponentials (base 2: the scale carries log2 e).
//
// Orientation: a wavefront computes S^T = K Q^T (16 tokens x 16 columns per MFMA chain, a column being
// one query: row * group + head of the group) and O^T = V^T P^T. The accumulator registers of S^T (lane
// l: tokens 4 (l / 16) + r of column l % 16) are, rounded (and, up to 32 columns, once more what that
// loses), the B operand of the second product with no move between lanes, since the values are laid out
// for that order of tokens (kv_cache.h); the output comes out with 16 consecutive dimensions per lane.
// Keys and values go from memory straight into operand registers: 16 bytes per lane, 1 KiB per load, no LDS.
//
// A workgroup's wavefronts (four, or as many as a CU holds) take the steps of 32 tokens of one range of one (sequence,
// tile of columns, key head) in turn, and are joined through LDS at the end. Ranges of the same (sequence, tile, head)
// leave partial results in device memory, which a second launch joins (attend_join.hip).
#pragma once

#include <type_traits>

#include "attend_plan.h"
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
  float* partials;           // slots of attend_slot_floats(columns, padded dim)
  int64_t window;            // 0: none
  float scale;               // times log2 e
  int heads, group, sinks, mask_rows, mask_words;
  int target;   // workgroups that the work is split over, at most; 0: never split
  float per_target;  // a little more than 1 / target
  int least;    // steps of a range, at least
  int whole;    // a group of so many steps is not cut
  int wide;     // workgroups of attend_wide wavefronts, where that is more
  int walkers;  // workgroups of the launch that walk; those after them clear (kv_clear)
};

// The first token of the window of a row at `position`, held to 2^30, which no cache's tokens reach. Positions and windows
// are what the caller says, in 64 bits: neither needs to have to do with the cache's size.
__device__ __forceinline__ int window_first(const AttendArgs& a, int64_t position) {
  return position < a.window ? 0 : static_cast<int>(min(position - a.window + 1, int64_t{1} << 30));
}

// A sequence's share of the work, the same in every workgroup.
struct AttendShare {
  int tiles, steps;
  KvSeq seq;
};

template <int COLS>
__device__ __forceinline__ AttendShare attend_share(const AttendArgs& a, int b) {
  AttendShare s{0, 0, {0, 0, 0}};
  if (b >= a.rows.seqs) return s;
  const KvSeq seq = s.seq = kv_seq(a.rows, b, a.cache.page_shift);
  if (seq.rows == 0) return s;
  s.tiles = (seq.rows * a.group + COLS - 1) / COLS;
  const int hi = (seq.context + seq.rows + kStep - 1) / kStep;
  int lo = 0;
  if (a.window > 0) {
    // The first row's place says where the window begins: where a later row's is before it, the ranges get longer, and
    // that is all.
    lo = min(window_first(a, a.positions != nullptr ? a.positions[seq.start] : seq.context) / kStep, hi);
  }
  s.steps = hi - lo + min((a.sinks + kStep - 1) / kStep, lo);
  return s;
}

// Inclusive sums over the wavefront's lanes, by DPP: shifts inside rows of 16, then the rows' last lanes handed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = scan_step<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);  // row_bcast 15 into rows 1 and 3
  return scan_step<0x143, 0xc>(v);  // row_bcast 31 into rows 2 and 3
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float scan_step(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_total(float v) {
  v = scan_step<0x111, 0xf>(v);
  v = scan_step<0x112, 0xf>(v);
  v = scan_step<0x114, 0xf>(v);
  v = scan_step<0x118, 0xf>(v);
  v = scan_step<0x142, 0xa>(v);
  v = scan_step<0x143, 0xc>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

struct AttendItem {
  int b, tile, head, range, ranges;  // ranges == 0: nothing to do
  int slot;                          // the group's first partial slot; its ranges' are `heads` slots apart
  KvSeq seq;
};

// Which range of which group (sequence, tile, key head) workgroup `index` takes; with JOIN, which group of several
// ranges is number `index`. The work of the whole call (steps x tiles x heads, from the lengths on the device) is cut
// so that about `target` workgroups share it evenly, whatever the sequences' lengths and the table's width: a launch
// cut on the host alone would have to go by the longest sequence that the table could hold. Every wavefront scans the
// sequences by itself, 64 at a time.
template <int COLS, bool JOIN>
__device__ __forceinline__ AttendItem attend_item(const AttendArgs& a, int index, int lane) {
  const int heads = a.cache.heads;
  AttendItem it{};
  int chunk = 1 << 30;
  const AttendShare own = attend_share<COLS>(a, lane);
  if (a.target > 0) {
    // In fp32, rounded up by more than its sums can be off: a chunk is never less than load / target.
    float load = 0.0f;
    for (int base = 0; base < a.rows.seqs; base += 64) {
      const AttendShare s = base == 0 ? own : attend_share<COLS>(a, base + lane);
      load += static_cast<float>(s.tiles) * static_cast<float>(s.steps);
    }
    const float cut = ceilf(wave_total(load) * static_cast<float>(heads) * a.per_target);
    chunk = max(static_cast<int>(fminf(cut, static_cast<float>(1 << 30))), a.least);
  }
  int items = 0, slots = 0;
  for (int base = 0; base < a.rows.seqs; base += 64) {
    const AttendShare s = base == 0 ? own : attend_share<COLS>(a, base + lane);
    const int ranges = s.steps <= a.whole ? 1 : min(max((s.steps + chunk - 1) / chunk, 1), kAttendMost);
    const int split = ranges > 1 ? s.tiles * heads : 0;  // groups of several ranges: they alone have slots
    const int mine = JOIN ? split : s.tiles * heads * ranges;
    const int to = wave_scan(mine);
    const int slot_to = a.target > 0 ? wave_scan(split * ranges) : 0;
    const uint64_t past = __ballot(items + to > index);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      it.b = base + at;
      it.ranges = of(ranges);
      const int tiles = of(s.tiles), rest = index - (items + of(to - mine));
      // Sequences that claim the same rows again and again can add up to more than 32 bits hold: nobody's work.
      if (static_cast<uint32_t>(rest) >= static_cast<uint32_t>(of(mine))) return AttendItem{};
      const int x = rest / heads;
      it.head = rest - x * heads;
      if constexpr (JOIN) {
        it.tile = x;
      } else {
        const int y = x / it.ranges;
        it.range = x - y * it.ranges;
        it.tile = tiles - 1 - y;  // a causal tile's work grows with its number: the longest first
      }
      it.slot = slots + of(slot_to) + (it.tile - tiles) * it.ranges * heads + it.head;
      it.seq = {of(s.seq.start), of(s.seq.rows), of(s.seq.context)};
      return it;
    }
    items += __builtin_amdgcn_readlane(to, 63);
    slots += __builtin_amdgcn_readlane(slot_to, 63);
  }
  return it;
}

__device__ __forceinline__ void attend_clear(const AttendArgs& a) {
  kv_clear(a.rows, a.cache.page_shift, a.out, static_cast<int64_t>(a.heads) * (a.cache.dim >> 3), blockIdx.x - a.walkers,
           gridDim.x - a.walkers);
}

// The larger of two, NaN if either is: unlike fmaxf it needs no quieting of its operands, and three values are one
// instruction. A score that is NaN makes its row NaN, whatever the maximum.
__device__ __forceinline__ float larger_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }

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
  lane_pair<false>(larger_of(a, b), a, b);
  return larger_of(a, b);
}

__device__ __forceinline__ float column_sum(float v) {
  float a, b;
  lane_pair<true>(v, a, b);
  lane_pair<false>(a + b, a, b);
  return a + b;
}

// Two values in the model's type, rounded to nearest even, as one word.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// What two values lose in pack2's word, in the model's type.
template <int DT>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t word) {
  return pack2<DT>(a - from_bits16<DT>(static_cast<uint16_t>(word)), b - from_bits16<DT>(static_cast<uint16_t>(word >> 16)));
}

// Whether a 16-bit pair holds an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool pair_not_finite(uint32_t w) {
  constexpr uint32_t e = DT == DT_BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// Whether any of four e4m3 codes is NaN (all seven bits below the sign).
__device__ __forceinline__ bool fp8_not_finite(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }

// Scales are at least this (a masked score times a scale of zero would be NaN).
constexpr float kLeastScale = 1.0f / 18446744073709551616.0f;
constexpr float kMinusInf = -__builtin_inff();
// The running maximum follows a larger one only where that is more than this (base 2) above it, so most
// steps leave the accumulators alone; exponentials then reach 2^kSlack, exact in fp32 sums. fp16
// probabilities carry 2^kShift besides (out of both sums at the end), so that small ones stay normal:
// 2^(kSlack + kShift) is inside fp16.
constexpr float kSlack = 6.0f;
template <int DT>
constexpr float kShift = DT == DT_F16 ? 8.0f : 0.0f;

// 8-bit values under fp16 rows are taken as codes times (page scale / `ref`), the accumulators being in units of `ref`, a
// power of two. Ratios in [2^-5, 2^6] make every code a normal fp16 number, so no bit is lost; where the scales of a
// step's pages leave that range `ref` moves, and the accumulators with it, in fp32. A page that a row does not see, or
// barely, thus takes nothing from the others. bf16 holds codes times any scale: its accumulators are in plain units.
template <int DT, bool E8>
constexpr bool kUnits = E8 && DT == DT_F16;
// Pages below this are left out: no value of theirs, 448 times it at most, reaches half of fp16's least (2^-25).
constexpr float kSilent = 0x1p-34f;

// Moves `ref` to where the pages' scales `vs` (0: no page) have ratios in range; false where no place is, 2^11 apart.
template <int N>
__device__ __forceinline__ bool unit_for(const float (&vs)[N], float& ref) {
  // Powers of two are compared by their bits, which the scalar unit does.
  constexpr int step = 1 << 23;
  int hi = 0, lo = 0x7f000000;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int bits = __builtin_bit_cast(int, vs[u]), x = bits >= __builtin_bit_cast(int, kSilent) ? bits : 0;
    hi = max(hi, x);
    lo = x > 0 ? min(lo, x) : lo;
  }
  const int at = __builtin_bit_cast(int, ref);
  if (hi == 0 || (hi - at <= 6 * step && at - lo <= 5 * step)) return true;
  if (hi - lo > 11 * step) return false;
  ref = __builtin_bit_cast(float, hi - lo > 5 * step ? lo + 5 * step : hi);
  return true;
}

// What accumulators in units of `from` are multiplied by to be in units of `to`. (Bounded: scales that far apart are no
// page's whose values fp16 holds, and zeros have to stay zeros.)
__device__ __forceinline__ float unit_ratio(float from, float to) { return fminf(from / to, 0x1p120f); }

// Token x of a step's 32: its place among the eight of the lanes that hold it.
struct TokenOf {
  int slot, holder;
  u32x4 only;  // masks that leave this token alone
  __device__ __forceinline__ TokenOf(int x, int g) {
    slot = ((x >> 4) << 2) | (x & 3);
    holder = (x & 15) >> 2;
    const uint32_t half = holder == g ? 0xffffu << (16 * (slot & 1)) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) only[i] = (slot >> 1) == i ? half : 0u;
  }
  // Whether the lane's column sees it, from the bits of the lanes that hold it.
  __device__ __forceinline__ bool seen(uint32_t bits, int step, int col) const {
    return ((__shfl(static_cast<int>(bits), holder * 16 + col) >> (8 * step + slot)) & 1) != 0;
  }
};

template <int DT>
__device__ __forceinline__ void take_token(u32x4 v, u32x4 p, bool sees, f32x4& o) {
  const f32x4 sum = mfma_16x16x32<DT>(v, p, o);
#pragma unroll
  for (int r = 0; r < 4; ++r) o[r] = sees ? sum[r] : o[r];
}

// The queries of a wavefront's NC x 16 columns: lane l has column l % 16 of each sixteen.
template <int NC>
struct AttendColumns {
  int row[NC], head[NC], window_lo[NC];
  bool real[NC];  // others repeat the sequence's last column and are not stored

  __device__ __forceinline__ void set(const AttendArgs& a, const KvSeq& seq, const AttendItem& it, int first, int columns,
                                      int col) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int x = first + 16 * n + col, y = min(x, columns - 1);
      real[n] = x < columns;
      row[n] = y / a.group;
      head[n] = it.head * a.group + y - row[n] * a.group;
      window_lo[n] = 0;
      if (a.window > 0) window_lo[n] = window_first(a, a.positions != nullptr ? a.positions[seq.start + row[n]] : seq.context + row[n]);
    }
  }

  // Bit 4 u + r: column n sees token t0 + 16 u + 4 g + r; units without a page (`held`) are not seen. Called where a
  // step is at an edge of what its columns see.
  template <int UNITS>
  __device__ __forceinline__ uint32_t seen_bits(const AttendArgs& a, const KvSeq& seq, int n, int t0, int g,
                                                uint32_t held) const {
    const int end = a.mask != nullptr ? seq.context + seq.rows : seq.context + row[n] + 1;
    uint64_t own = ~uint64_t{0};  // bit i: token t0 + i by the mask
    if (a.mask != nullptr && t0 + 16 * UNITS > seq.context) {
      // The 16 UNITS bits from own row t0 - context on: three words of the row cover them.
      const int i0 = max(t0 - seq.context, 0);
      const uint32_t* from = a.mask + static_cast<int64_t>(row[n]) * a.mask_words;
      uint32_t word[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int at = (i0 >> 5) + i;
        word[i] = at < a.mask_words && row[n] < a.mask_rows ? from[at] : 0u;
      }
      const uint64_t low = word[0] | static_cast<uint64_t>(word[1]) << 32, high = word[1] | static_cast<uint64_t>(word[2]) << 32;
      own = (low >> (i0 & 31) & 0xffffffffu) | (high >> (i0 & 31)) << 32;
      const int before = seq.context - t0;  // tokens of the context come first
      if (before > 0) own = own << before | ((uint64_t{1} << before) - 1);
    }
    // What is left of the step's tokens by the row's end and the window, as bits like `own`.
    const auto below = [](int n) { return n <= 0 ? uint64_t{0} : n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1; };
    uint64_t near = ~below(window_lo[n] - t0) | below(a.sinks - t0);
    if (a.mask != nullptr) near |= ~below(seq.context - t0);
    own &= near & below(end - t0);
    const uint64_t mine = own >> (4 * g);
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) bits |= ((held >> u) & 1u ? static_cast<uint32_t>(mine >> (16 * u)) & 15u : 0u) << (4 * u);
    return bits;
  }

  template <int DT, int C>
  __device__ __forceinline__ void queries(const AttendArgs& a, const KvSeq& seq, int g, u32x4 (&q)[NC][C][2]) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const uint16_t* from = a.q + (seq.start + row[n]) * a.q_row + head[n] * a.q_head;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = 64 * c + 16 * g + 8 * h;
          q[n][c][h] = real[n] && e < a.cache.dim ? *reinterpret_cast<const u32x4*>(from + e) : u32x4{0u, 0u, 0u, 0u};
        }
    }
  }

  // The finished sums over l, in the model's type.
  template <int DT, int C>
  __device__ __forceinline__ void store(const AttendArgs& a, const KvSeq& seq, int g, const f32x4 (&o)[NC][C][4],
                                        const float (&l)[NC]) const {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      if (!real[n]) continue;
      const float inverse = l[n] == 0.0f ? 0.0f : 1.0f / l[n];  // a row that sees nothing is zero
      uint16_t* at = a.out + (static_cast<int64_t>(seq.start + row[n]) * a.heads + head[n]) * a.cache.dim;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int e = 64 * c + 16 * g;
        u32x4 word[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // dimensions e + 2 i, e + 2 i + 1
          const int r = i / 2, j = 2 * (i & 1);
          word[i / 4][i % 4] = pack2<DT>(o[n][c][j][r] * inverse, o[n][c][j + 1][r] * inverse);
        }
        if (e < a.cache.dim) *reinterpret_cast<u32x4*>(at + e) = word[0];
        if (e + 8 < a.cache.dim) *reinterpret_cast<u32x4*>(at + e + 8) = word[1];
      }
    }
  }
};

// The tokens that a tile of columns looks at: steps of `STEP` tokens, the sinks' first, then from the window's
// (or the sequence's) first on. Step s begins at token_of(s).
template <int STEP>
struct AttendWalk {
  int whole;            // tokens before this are seen by every column, the window apart
  int lo_most, sinks;   // tokens from lo_most on, and before `sinks`, are inside every column's window
  int sink_steps, first, steps;
  int from, to;         // the range's steps

  template <int NC>
  __device__ __forceinline__ void set(const AttendArgs& a, const KvSeq& seq, const AttendItem& it, int cols, int columns,
                                      const AttendColumns<NC>& c, int lo_least) {
    const int row_lo = it.tile * cols / a.group, row_hi = (min((it.tile + 1) * cols, columns) - 1) / a.group;
    const int end = a.mask != nullptr ? seq.context + seq.rows : seq.context + row_hi + 1;
    whole = a.mask != nullptr ? seq.context : seq.context + row_lo + 1;
    sinks = a.sinks;
    // Under a mask the window holds for the context alone: the rows' own tokens are always walked.
    if (a.mask != nullptr) lo_least = min(lo_least, seq.context);
    const int last = (end + STEP - 1) / STEP;
    first = min(lo_least / STEP, last);
    sink_steps = min((min(a.sinks, 1 << 29) + STEP - 1) / STEP, first);
    steps = sink_steps + last - first;
    // At most 2^24 steps (a table holds 2^29 tokens) and kAttendMost ranges: inside 32 bits.
    const uint32_t n = static_cast<uint32_t>(steps), r = static_cast<uint32_t>(it.range), all = static_cast<uint32_t>(it.ranges);
    from = all == 1 ? 0 : static_cast<int>(n * r / all);
    to = all == 1 ? steps : static_cast<int>(n * (r + 1) / all);
  }
  __device__ __forceinline__ int token_of(int s) const { return STEP * (s < sink_steps ? s : first + s - sink_steps); }
  __device__ __forceinline__ bool edge(int t0) const { return t0 + STEP > whole || (t0 < lo_most && t0 + STEP > sinks); }
};

// Least and largest first token of the columns' windows over the sixteen lanes of a group (0 without a window).
template <int NC>
__device__ __forceinline__ void window_bounds(const AttendArgs& a, const AttendColumns<NC>& c, int& least, int& most) {
  least = most = 0;
  if (a.window <= 0) return;
  least = 1 << 30;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    least = min(least, c.window_lo[n]);
    most = max(most, c.window_lo[n]);
  }
#pragma unroll
  for (int x = 8; x > 0; x >>= 1) {
    least = min(least, __shfl_xor(least, x));
    most = max(most, __shfl_xor(most, x));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);
}

// A partial result's slot: [cols][pad] sums, then [cols] maxima and [cols] sums of exponentials.
template <int NC, int C>
__device__ __forceinline__ void attend_publish(const AttendArgs& a, const AttendItem& it, int cols, int first, int g, int col,
                                               const AttendColumns<NC>& c, const f32x4 (&o)[NC][C][4], const float (&m)[NC],
                                               const float (&l)[NC]) {
  constexpr int PAD = 64 * C;
  float* mine = a.partials + static_cast<int64_t>(it.slot + it.range * a.cache.heads) * attend_slot_floats(cols, PAD);
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    if (!c.real[n]) continue;
    const int at = first + 16 * n + col;
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<f32x4*>(mine + at * PAD + 64 * k + 16 * g + 4 * r) =
            f32x4{o[n][k][0][r], o[n][k][1][r], o[n][k][2][r], o[n][k][3][r]};
    if (g == 0) {
      mine[cols * PAD + at] = m[n];
      mine[cols * PAD + cols + at] = l[n];
    }
  }
}

// Chunk c of the unit at byte `at` (the same in every lane). Dimensions past the head's, in the last chunk, are not
// read: a lane whose are (`inside` false) gets zeros. ONCE: no other workgroup reads them, so they are not to stay in the
// caches (bit 1 of the load's last operand: nontemporal).
template <bool E8, int C, bool ONCE>
__device__ __forceinline__ void load_chunk_of(__amdgpu_buffer_rsrc_t rs, int c, int lane, bool inside, u32x4 (&x)[E8 ? 1 : 2]) {
#pragma unroll
  for (int h = 0; h < (E8 ? 1 : 2); ++h) {
    const uint32_t off = static_cast<uint32_t>((c * (E8 ? 1 : 2) + h) * 1024 + lane * 16);
    const uint32_t at = c == C - 1 && !inside ? kOutOfRange : off;
    if constexpr (ONCE) x[h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, static_cast<int>(at), 0, 2));
    else x[h] = buffer_load16(rs, at);
  }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t unit_rsrc(const char* base, int64_t at, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base) + static_cast<uint64_t>(at);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(p >> 32));
  return make_rsrc(reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo), bytes);
}

template <bool E8, int C, bool ONCE>
__device__ __forceinline__ void load_unit(const char* base, int64_t at, int lane, bool inside, u32x4 (&x)[C][E8 ? 1 : 2]) {
  const __amdgpu_buffer_rsrc_t rs = unit_rsrc(base, at, C * (E8 ? 1024 : 2048));
#pragma unroll
  for (int c = 0; c < C; ++c) load_chunk_of<E8, C, ONCE>(rs, c, lane, inside, x[c]);
}

// A wavefront's state and its walk over tokens.
template <int DT, bool E8, int C, int NC, bool ONCE>
struct AttendWave {
  static constexpr int kLoads = E8 ? 1 : 2;  // of 16 bytes per lane, unit and chunk
  static constexpr int kUnitBytes = 1024 * kLoads;

  // Where a step's two units are.
  struct Place {
    int64_t at[2];
    float ks[2], vs[2];
    bool held[2];  // the unit's page is a page of the cache
  };

  u32x4 k[2][C][kLoads], v[2][C][kLoads];
  f32x4 o[NC][C][4];
  u32x4 q[NC][C][2];
  float m[NC], l[NC];
  float ref;  // the accumulators' unit (kUnits)
  int page_id, page_first;  // lane i: page number page_first + i of the sequence
  float page_ks, page_vs;

  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      m[n] = kMinusInf;
      l[n] = 0.0f;
    }
    ref = 0.0f;
    page_first = -64;
  }

  __device__ __forceinline__ void pages(const AttendArgs& a, int b, int head, int number, int last, int lane) {
    page_first = number;
    const int at = number + lane;
    int id = -1;
    if (at < last && at < a.rows.width) id = a.rows.table[b * a.rows.table_stride + at];
    const bool good = id >= 0 && id < a.cache.pages;
    page_id = good ? id : -1;
    if constexpr (E8) {
      page_ks = good ? fmaxf(a.cache.k_scale[static_cast<int64_t>(id) * a.cache.heads + head], kLeastScale) : kLeastScale;
      page_vs = good ? a.cache.v_scale[static_cast<int64_t>(id) * a.cache.heads + head] : 0.0f;
    }
  }

  // The accumulators in units of `to`.
  __device__ __forceinline__ void follow(float to) {
    if (to == ref) return;
    const float by = unit_ratio(ref, to);
    ref = to;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j] *= by;
  }

  __device__ __forceinline__ Place place(const AttendArgs& a, int b, int head, int t0, int last_page, int lane) {
    Place s;
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
      // A page of one head is at most 128 KiB, a page of all heads 128 MiB.
      const uint32_t page_bytes = static_cast<uint32_t>(a.cache.page >> 4) * (C * kUnitBytes);
      s.at[u] = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(max(id, 0))) * (page_bytes * a.cache.heads) +
                                     page_bytes * static_cast<uint32_t>(head) + static_cast<uint32_t>(unit) * (C * kUnitBytes));
    }
    return s;
  }

  __device__ __forceinline__ void keys(const AttendArgs& a, const Place& s, int lane) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_unit<E8, C, ONCE>(a.cache.k, s.at[u], lane, 16 * (lane >> 4) < a.cache.dim - 64 * (C - 1), k[u]);
  }
  __device__ __forceinline__ void values(const AttendArgs& a, const Place& s, int lane) {
#pragma unroll
    for (int u = 0; u < 2; ++u) load_unit<E8, C, ONCE>(a.cache.v, s.at[u], lane, 4 * (lane & 15) < a.cache.dim - 64 * (C - 1), v[u]);
  }
};

// 16 NC columns. Bound, where contexts are long, by the bytes of the keys and values, each read once and used by one
// wavefront: hence no LDS in the loop, and a key head's whole group of queries as columns of one tile. 64 sequences of
// 4500 tokens on average, 16 heads of 128 over 4 in 8 bits: 62 us for 296 MB, 4.8 TB/s with the join (a large copy reaches
// 5.1); two of 131004 tokens 51 us for 268 MB, 5.3 TB/s; 32 windows of 1024 tokens, 16 key heads in 16 bits, 49 us for 270
// MB, 5.5 TB/s. Where they are short, by a workgroup's beginning and end (arguments, lengths, table, scales, first loads, join:
// 6000 to 7000 cycles): 500 tokens 6.7 us. Four wavefronts per workgroup there (with eight the first of these took 70 us); groups of
// middling length that all find a CU are taken whole by as many as it holds (attend_plan).
template <int DT, bool E8, int C, int NC, bool ONCE, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(attend_waves(E8, C, NC)))) void attend_kernel(AttendArgs a) {
  constexpr int COLS = 16 * NC;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  if (static_cast<int>(blockIdx.x) >= a.walkers) return attend_clear(a);
  const AttendItem it = attend_item<COLS, false>(a, blockIdx.x, lane);
  if (it.ranges == 0) return;
  const KvSeq& seq = it.seq;
  const int columns = seq.rows * a.group;

  using Wave = AttendWave<DT, E8, C, NC, ONCE>;
  Wave w;
  AttendColumns<NC> cols;
  cols.set(a, seq, it, it.tile * COLS, columns, col);
  cols.template queries<DT, C>(a, seq, g, w.q);
  AttendWalk<kStep> walk;
  int lo_least;
  window_bounds(a, cols, lo_least, walk.lo_most);
  walk.set(a, seq, it, COLS, columns, cols, lo_least);
  const int end = seq.context + seq.rows;
  const int last_page = (end + a.cache.page - 1) >> a.cache.page_shift;

  // One step. Keys and values have one set of registers each, refilled for the wavefront's next step as soon as the
  // product that reads them is issued, so about a step's bytes are in flight throughout.
  // CAREFUL: a value that is not finite was met in a step that some columns do not see whole, where 0 * it would reach
  // them, or a step's two pages have scales too far apart for one unit (unit_for). The walk is then done again with one
  // token at a time in such steps: apart from the usual one, whose registers it would take.
  typename Wave::Place s;
  bool odd = false;
  auto step = [&](auto careful, int number) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const int t0 = walk.token_of(number);
    const bool more = !CAREFUL && number + W < walk.to;
    const bool edge = walk.edge(t0) || !s.held[0] || !s.held[1];
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
          const u32x4 x = w.k[u][c][0];
          k0 = fp8_eight<DT>(x[0], x[1], 1.0f);
          k1 = fp8_eight<DT>(x[2], x[3], 1.0f);
        } else {
          k0 = w.k[u][c][0];
          k1 = w.k[u][c][1];
        }
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          score[n][u] = mfma_16x16x32<DT>(k0, w.q[n][c][0], score[n][u]);
          score[n][u] = mfma_16x16x32<DT>(k1, w.q[n][c][1], score[n][u]);
        }
      }
    }
    typename Wave::Place next = s;
    if (more) {
      next = w.place(a, it.b, it.head, walk.token_of(number + W), last_page, lane);
      w.keys(a, next, lane);
    }
    uint32_t seen[NC];
    if (edge) {
      const uint32_t held = static_cast<uint32_t>(s.held[0]) | static_cast<uint32_t>(s.held[1]) << 1;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        seen[n] = cols.template seen_bits<2>(a, seq, n, t0, g, held);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) score[n][u][r] = (seen[n] >> (4 * u + r)) & 1u ? score[n][u][r] : kMinusInf;
      }
      // Tokens that are no one's, past the end or of a page that is not there, have values of zero.
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int live = s.held[u] ? min(max(end - (t0 + 16 * u + 4 * g), 0), 4) : 0;  // of the lane's four tokens
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int h = 0; h < Wave::kLoads; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (E8) {
                w.v[u][c][h][i] &= live == 4 ? ~0u : (1u << (8 * live)) - 1u;
                odd = odd || fp8_not_finite(w.v[u][c][h][i]);
              } else {
                const int two = min(max(live - 2 * (i & 1), 0), 2);
                w.v[u][c][h][i] &= two == 2 ? ~0u : (1u << (16 * two)) - 1u;
                odd = odd || pair_not_finite<DT>(w.v[u][c][h][i]);
              }
            }
      }
    }
    u32x4 p[NC], rest[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u) score[n][u] *= E8 ? a.scale * s.ks[u] : a.scale;
      float top = kMinusInf;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = larger_of(top, score[n][u][r]);
      top = column_max(top);
      if (__any(top > w.m[n] + kSlack)) {
        const float next = larger_of(w.m[n], top);
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
      // Probabilities in two parts of the model's type, as its matrix product takes them: 2^-16 off at most (fp16 2^-22), so
      // that the output's rounding is the only one that shows. The matrix cores have the time: single tokens 61.9 us with the
      // rest for 61.5, a round of 56 rows 17.3 for 16.7, and the error against 64 bits 0.0017 of the values for 0.0023.
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[n][i] = pack2<DT>(e[2 * i], e[2 * i + 1]);
        rest[n][i] = rest2<DT>(e[2 * i], e[2 * i + 1], p[n][i]);
      }
    }
    // O^T += V^T P^T: operand j of a chunk has dimensions 4 (l % 16) + j as rows.
    float ratio[2] = {1.0f, 1.0f};
    bool apart = false;
    auto ratios = [&]() {
      const float less = kUnits<DT, E8> ? (w.ref > 0.0f ? 1.0f / w.ref : 0.0f) : 1.0f;
      ratio[0] = s.vs[0] * less;
      ratio[1] = s.vs[1] * less;
    };
    if constexpr (kUnits<DT, E8>) {
      float ref = w.ref;
      apart = !unit_for(s.vs, ref);
      odd = odd || apart;
      w.follow(ref);
    }
    if constexpr (E8) ratios();
    auto values_of = [&](int c, int j) {
      u32x4 v;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (E8) {
          v[2 * u] = fp8_pair<DT>(w.v[u][c][0][j], ratio[u], false);
          v[2 * u + 1] = fp8_pair<DT>(w.v[u][c][0][j], ratio[u], true);
        } else {
          v[2 * u] = w.v[u][c][j / 2][2 * (j & 1)];
          v[2 * u + 1] = w.v[u][c][j / 2][2 * (j & 1) + 1];
        }
      }
      return v;
    };
    if (!CAREFUL || !(edge || apart)) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x4 v = values_of(c, j);
#pragma unroll
          for (int n = 0; n < NC; ++n) w.o[n][c][j] = mfma_16x16x32<DT>(v, rest[n], mfma_16x16x32<DT>(v, p[n], w.o[n][c][j]));
        }
    } else {
      if (!edge) {
#pragma unroll
        for (int n = 0; n < NC; ++n) seen[n] = ~0u;
      }
      // Units apart one after the other, each with its own page's scale for a unit of the accumulators.
      const float first = s.vs[0], second = s.vs[1];
#pragma unroll 1
      for (int u = 0; u < (apart ? 2 : 1); ++u) {
        if (apart) {
          const float to = u == 0 ? first : second;
          if (to >= kSilent) w.follow(to);
          ratios();
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u32x4 v = values_of(c, j);
#pragma unroll 1
            for (int x = 16 * u; x < (apart ? 16 * u + 16 : kStep); ++x) {
              const TokenOf t(x, g);
#pragma unroll
              for (int n = 0; n < NC; ++n) {
                const bool sees = t.seen(seen[n], 0, col);
                take_token<DT>(v & t.only, p[n] & t.only, sees, w.o[n][c][j]);
                take_token<DT>(v & t.only, rest[n] & t.only, sees, w.o[n][c][j]);
              }
            }
          }
      }
    }
    s = next;
    if (more) w.values(a, s, lane);
  };

  w.begin();
  if (walk.from + wave < walk.to) {
    s = w.place(a, it.b, it.head, walk.token_of(walk.from + wave), last_page, lane);
    w.keys(a, s, lane);
    w.values(a, s, lane);
    for (int number = walk.from + wave; number < walk.to; number += W) step(std::false_type{}, number);
    if (__any(odd)) {
      w.begin();
#pragma unroll 1
      for (int number = walk.from + wave; number < walk.to; number += W) {
        s = w.place(a, it.b, it.head, walk.token_of(number), last_page, lane);
        w.keys(a, s, lane);
        w.values(a, s, lane);
        step(std::true_type{}, number);
      }
    }
  }

  // The wavefronts' results, in plain units, meet in LDS; each then joins some of the 4 C parts of the dimensions: part p is
  // register p % 4 (4 consecutive dimensions of 16) of chunk p / 4.
  constexpr int kWaveFloats = NC * (C * 16 + 2) * 64;
  float* shared = reinterpret_cast<float*>(lds);
  {
    float* mine = shared + wave * kWaveFloats + lane * 4;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float scale = kUnits<DT, E8> ? w.ref : 1.0f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(mine + ((n * C + c) * 4 + r) * 256) =
              f32x4{w.o[n][c][0][r], w.o[n][c][1][r], w.o[n][c][2][r], w.o[n][c][3][r]} * scale;
      float* ends = shared + wave * kWaveFloats + NC * C * 1024 + n * 128 + lane;
      ends[0] = w.m[n];
      ends[64] = column_sum(w.l[n]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    float top = kMinusInf, m[W], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      m[i] = shared[i * kWaveFloats + NC * C * 1024 + n * 128 + lane];
      top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      m[i] = m[i] == top ? 1.0f : __builtin_amdgcn_exp2f(m[i] - top);
      sum += m[i] * shared[i * kWaveFloats + NC * C * 1024 + n * 128 + 64 + lane];
    }
    if (!cols.real[n]) continue;
    const bool last = it.ranges == 1;
    const float inverse = !last ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing is zero
    constexpr int PAD = 64 * C;
    float* slot = a.partials + static_cast<int64_t>(it.slot + it.range * a.cache.heads) * attend_slot_floats(COLS, PAD);
    const int x = 16 * n + col;
    uint16_t* out = a.out + (static_cast<int64_t>(seq.start + cols.row[n]) * a.heads + cols.head[n]) * a.cache.dim;
#pragma unroll
    for (int first = 0; first < 4 * C; first += W) {
      const int part = first + wave, e = 64 * (part / 4) + 16 * g + 4 * (part % 4);
      if (4 * C % W != 0 && part >= 4 * C) break;
      f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < W; ++i)
        o += *reinterpret_cast<const f32x4*>(shared + i * kWaveFloats + (n * C * 4 + part) * 256 + lane * 4) * m[i];
      o *= inverse;
      if (!last) *reinterpret_cast<f32x4*>(slot + x * PAD + e) = o;
      else if (e < a.cache.dim) *reinterpret_cast<u32x2*>(out + e) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
    }
    if (!last && g == 0 && wave == 0) {
      slot[COLS * PAD + x] = top;
      slot[COLS * PAD + COLS + x] = sum;
    }
  }
}

hipError_t attend_bf16_e4m3(const AttendArgs& a, int columns, unsigned grid, hipStream_t s);
hipError_t attend_bf16_model(const AttendArgs& a, int columns, unsigned grid, hipStream_t s);
hipError_t attend_f16_e4m3(const AttendArgs& a, int columns, unsigned grid, hipStream_t s);
hipError_t attend_f16_model(const AttendArgs& a, int columns, unsigned grid, hipStream_t s);

// Joins the groups of several ranges, `groups` at most.
hipError_t attend_join(int32_t dtype, const AttendArgs& a, int columns, int64_t groups, hipStream_t s);

}  // namespace plm

// How an attention call is launched (plm_attend): which kernel, over how many workgroups, cut or not. Sizes in, a plan out:
// plain C++, without the device.
#pragma once

#include <algorithm>
#include <cstdint>

namespace plm {

constexpr int kStep = 32;        // tokens of a step
constexpr int kWaves = 4;        // wavefronts of a workgroup, but for wide ones (attend_wide)
constexpr int kAttendMost = 64;  // ranges per group, at most
constexpr int kJoinColumns = 8;  // columns that a workgroup of the joining launch takes at a time, at most

constexpr int64_t attend_slot_floats(int columns, int padded) {
  return static_cast<int64_t>(columns) * (padded + 2);
}

// Wavefronts per SIMD to leave registers for: as many as hold the accumulators, the queries and a step's keys and
// values without spilling (512 registers over them).
constexpr int attend_waves(bool e8, int chunks, int nc) {
  if (chunks == 1) return nc == 1 ? 4 : 3;
  if (chunks == 2) return e8 && nc == 1 ? 3 : 2;
  return e8 || chunks == 3 ? 2 : 1;
}

// Wavefronts of a workgroup that fills a CU.
constexpr int attend_wide(bool e8, int chunks) { return 4 * attend_waves(e8, chunks, 1); }

constexpr int64_t kNarrowWork = 24000;  // groups of 16 columns times steps
constexpr int64_t kWideGroups = 256, kWideSteps = 100, kWideAlone = 56, kWideBytes = 448 * 1024;

struct AttendPlan {
  int columns;        // of a workgroup's tile
  int target, least, whole, wide;  // AttendArgs
  int64_t grid, groups, bytes;
};

// The launch of a call, from what the host knows: sizes, never the lengths. The work is cut on the device (attend_item), so
// it is shared evenly whatever the lengths; but the kernel, and whether there is a second launch, go by what the table can
// hold, so a table much wider than its sequences costs (16384 tokens of table against an exact one, 16 heads of 128 over 4: a
// round of 56 rows after 500 tokens 21.2 / 9.1 us, after 1000 18.5 / 11.4, after 4007 20.8 / 17.8; 64 tokens after 1000 20.1 /
// 14.8, after up to 8191 the same; 1 token after 499, 8 heads of 64, 9.3 / 6.7; 512 rows after 1500 the same). `grid` bounds
// the workgroups that any lengths can ask for: one per group and as many more as the work is cut into.
inline AttendPlan attend_plan(int64_t kv_heads, int64_t page, int64_t head_dim, int64_t heads, int64_t total, int64_t seqs,
                              int64_t max_rows, int64_t table_width, int64_t window, int64_t sinks, bool mask, bool e8) {
  AttendPlan p{};
  const int64_t group = heads / kv_heads, chunks = (head_dim + 63) / 64;
  const int64_t most = max_rows * group;
  // What a tile of columns sees at most: all the table holds, or with a window the rows' own span of it.
  const int64_t far = int64_t{1} << 30;
  const auto seen = [&](int64_t columns) {
    const int64_t all = (table_width * page + kStep - 1) / kStep, span = mask ? max_rows : std::min(max_rows, columns / group + 2);
    return window > 0 ? std::min(all, (std::min(window, far) + std::min(sinks, far) + span) / kStep + 3) : all;
  };
  // Tiles of 16 columns, whose four wavefronts take different tokens, are done soonest while all of a call's are short of
  // work for the device; wider ones need less of it. (Rounds of 56 rows over 500 / 4007 / 16000 tokens, 16 heads over 4:
  // 10.0 / 18.4 / 35 us against 18.7 / 21.3 / 34; four sequences' over 2000, 32 heads over 8, 41.5 against 40.5.) Up to
  // 96 tokens there is nothing to take apart. 128 columns need half the loads and conversions of 64, once there are tiles
  // of them for all CUs (4096 rows after 4096 tokens: 266 against 340 us on the same card); short walks end more evenly in
  // smaller tiles (prompts through a window of 512: 42 us in 128 columns, 40 in 64).
  const int64_t narrow = kv_heads * (seqs + total * group / 16);
  const bool many = most > 256 && kv_heads * (total * group / 128) >= (seen(128) < 24 ? 2048 : 256);
  if (most <= 16 || (seen(16) > 3 && narrow * seen(16) <= kNarrowWork)) p.columns = 16;
  else if (chunks <= 2 && most <= 32) p.columns = 32;
  else p.columns = chunks <= 2 && many ? 128 : 64;
  p.groups = kv_heads * (seqs + total * group / p.columns);
  // Ranges are joined by a second launch and each has a walk's beginning and end: 5 to 8 us that a cut has to win back.
  // A step of 32 tokens takes a quarter of about 0.8 us (up to 32 columns, a step per wavefront) or half of 1.2 us.
  p.least = p.columns <= 32 ? 16 : 8;
  p.whole = p.columns <= 32 ? 32 : 20;
  const int64_t steps = seen(p.columns);
  // Workgroups that fill a CU take groups of middling length whole, with a wavefront's steps and the joining launch saved,
  // where all find a CU of the 256: the last few would start behind the others otherwise. (`groups` counts a sequence's last
  // tile twice; rows without row_starts are known exactly. Wide / not, one past the other's side of the rule: 304 groups of
  // 59 steps 58 / 56 us, 280 of 20 21 / 14, 260 of 32 19.8 / 18.4, 264 of 29 at heads of 256 42 / 32; 240 that `groups`
  // takes for 480 13.8 / 17, of 79 steps 21 / 30.) One CU reads about 60 GB/s from memory: few groups
  // of many steps or bytes are cut instead, but for those whose tiles share them. (Wide / not: 16 tokens after 1000, 16
  // heads of 128 over 4 in 8 bits, 10.7 / 14.8 us, 64 after 1000 14.4 / 17, 64 after up to 3000 26 / 30; a round of 56 rows
  // after 1000 11.7 / 14.4, after 2500 16.5 / 17.7, four of 42 through a window of 777 12.2 / 14.8. One token after 3000, 8
  // key heads, 20.7 / 15.6; 8 after 2000 in 16 bits 23.7 / 17.4; a round after 4007 22.5 / 18; up to 16 steps 8.7 / 8.4.)
  const int64_t bytes = steps * kStep * chunks * (e8 ? 128 : 256);  // of a group's keys and values
  const int64_t real = std::min(p.groups, kv_heads * seqs * ((most + p.columns - 1) / p.columns));
  p.wide = p.columns == 16 && attend_wide(e8, static_cast<int>(chunks)) > kWaves && real <= kWideGroups &&
           steps > 4 * kWaves && steps <= kWideSteps &&
           (most > 16 || p.groups >= 128 || (steps <= kWideAlone && bytes <= kWideBytes));
  // Not cut: what is short, a single sequence's groups, which are alike, where they fill the device, and groups that do
  // and cannot be much unlike. (Cut / not: two sequences of 131004 tokens 50 / 1029 us, 64 of 4500 on average 60 / 88, a
  // round over 4007 18 / 33; 32 windows of 1024 53 / 49, a prompt of 4096 rows 250 / 242, through a window 48 / 41.)
  const bool full = p.groups - kv_heads >= 256;
  p.target = !p.wide && steps > p.whole && !(full && (seqs == 1 || steps <= 4 * p.least)) ? 512 : 0;
  p.grid = p.groups + p.target;
  // There are 2 * target ranges of groups of several at most: a cut sequence has less than twice load / chunk of
  // them, and a chunk is load / target at least. Such a group has two at least.
  if (p.target > 0) {
    p.groups = std::min<int64_t>(p.groups, p.target);
    p.bytes = 2 * p.target * attend_slot_floats(p.columns, static_cast<int>(64 * chunks)) * 4;
  }
  return p;
}

}  // namespace plm

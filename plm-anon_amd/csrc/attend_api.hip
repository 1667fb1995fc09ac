// C ABI of the attention over the paged cache (plm_attend), declared in include/plm_amd.h.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attend.h"
#include "plm_amd.h"

namespace plm {
namespace {

constexpr int64_t kNarrowWork = 24000;  // groups of 16 columns times steps
constexpr int64_t kWideGroups = 320, kWideSteps = 100, kWideAlone = 56, kWideBytes = 448 * 1024;

struct AttendPlan {
  int columns;        // of a workgroup's tile
  int target, least, whole, wide;  // AttendArgs
  int64_t grid, groups, bytes;
};

// The launch of a call, from what the host knows: sizes, never the lengths. The work is cut on the device
// (attend_item), so a wide table costs nothing; `grid` bounds the workgroups that any lengths can ask for:
// one per group and as many more as the work is cut into.
AttendPlan attend_plan(int64_t kv_heads, int64_t page, int64_t head_dim, int64_t heads, int64_t total, int64_t seqs,
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
  // where all find a CU (`groups` counts a sequence's last tile twice). One CU reads about 60 GB/s from memory: few groups
  // of many steps or bytes are cut instead, but for those whose tiles share them. (Wide / not: 16 tokens after 1000, 16
  // heads of 128 over 4 in 8 bits, 10.7 / 14.8 us, 64 after 1000 14.4 / 17, 64 after up to 3000 26 / 30; a round of 56 rows
  // after 1000 11.7 / 14.4, after 2500 16.5 / 17.7, four of 42 through a window of 777 12.2 / 14.8. One token after 3000, 8
  // key heads, 20.7 / 15.6; 8 after 2000 in 16 bits 23.7 / 17.4; a round after 4007 22.5 / 18; up to 16 steps 8.7 / 8.4.)
  const int64_t bytes = steps * kStep * chunks * (e8 ? 128 : 256);  // of a group's keys and values
  p.wide = p.columns == 16 && attend_wide(e8, static_cast<int>(chunks)) > kWaves && p.groups <= kWideGroups &&
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

// The plan of a call whose numbers go together; false where they do not.
bool attend_of(const plm_attend_call* call, AttendArgs& a, AttendPlan& p) {
  if (call == nullptr) return false;
  const plm_attend_call& h = *call;
  if (!kv_cache_of(h.cache, a.cache) || !kv_type_fits(h.cache, h.dtype) || !kv_rows_of(a.cache, h.rows, a.rows)) return false;
  const int64_t heads = a.cache.heads;
  if (h.heads < heads || h.heads > 4096 || h.heads % heads != 0 || h.rows.total * (h.heads / heads) >= (int64_t{1} << 30))
    return false;
  // The kernels multiply scores by the scale times log2 e times a page's scale (2^-64 at least) in fp32: what is masked
  // would be NaN if that were zero or infinite.
  if (h.window < 0 || h.sinks < 0 || !(h.scale >= 0x1p-62 && h.scale <= 0x1p126)) return false;
  if (h.mask != nullptr && (h.mask_rows < 1 || h.mask_words < 1 || h.mask_rows >= (1 << 28) || h.mask_words >= (1 << 24)))
    return false;
  p = attend_plan(heads, a.cache.page, a.cache.dim, h.heads, h.rows.total, h.rows.seqs, h.rows.max_rows, h.rows.table_width,
                  h.window, h.sinks, h.mask != nullptr, h.cache->type == PLM_CACHE_E4M3);
  if (h.rows.row_starts != nullptr) p.grid += 1;  // a workgroup without work, for rows without a sequence (attend_clear)
  return p.grid < (int64_t{1} << 31);
}

}  // namespace
}  // namespace plm

extern "C" {

size_t plm_attend_workspace_bytes(const plm_attend_call* call) {
  plm::AttendArgs a{};
  plm::AttendPlan p{};
  return plm::attend_of(call, a, p) ? static_cast<size_t>(p.bytes) : 0;
}

int plm_attend(const plm_attend_call* call, void* workspace, size_t workspace_bytes, void* stream) {
  plm::AttendArgs a{};
  plm::AttendPlan p{};
  if (!plm::attend_of(call, a, p)) return PLM_ERR_ARGUMENT;
  const plm_attend_call& h = *call;
  if (h.q == nullptr || h.out == nullptr) return PLM_ERR_ARGUMENT;
  if (h.q_row % 8 != 0 || h.q_head % 8 != 0) return PLM_ERR_ALIGNMENT;
  for (const void* x : {h.q, static_cast<const void*>(h.out), static_cast<const void*>(a.cache.k),
                        static_cast<const void*>(a.cache.v), static_cast<const void*>(workspace)})
    if (!plm::aligned16_ptr(x)) return PLM_ERR_ALIGNMENT;
  if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.bytes))) return PLM_ERR_WORKSPACE;
  constexpr int64_t far = int64_t{1} << 30;
  a.q = static_cast<const uint16_t*>(h.q);
  a.out = static_cast<uint16_t*>(h.out);
  a.q_row = h.q_row;
  a.q_head = h.q_head;
  a.positions = h.positions;
  a.mask = h.mask;
  a.partials = static_cast<float*>(workspace);
  a.scale = static_cast<float>(h.scale * 1.44269504088896340736);
  a.heads = static_cast<int>(h.heads);
  a.group = a.heads / a.cache.heads;
  a.window = h.window;
  a.sinks = static_cast<int>(std::min(h.sinks, far));
  a.mask_rows = static_cast<int>(h.mask_rows);
  a.mask_words = static_cast<int>(h.mask_words);
  a.target = p.target;
  a.per_target = p.target > 0 ? 1.001f / static_cast<float>(p.target) : 0.0f;
  a.least = p.least;
  a.whole = p.whole;
  a.wide = p.wide;
  const unsigned grid = static_cast<unsigned>(p.grid);
  const int32_t dtype = static_cast<int32_t>(h.dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool e8 = h.cache->type == PLM_CACHE_E4M3;
  hipError_t err;
  if (dtype == PLM_BF16) err = e8 ? plm::attend_bf16_e4m3(a, p.columns, grid, s) : plm::attend_bf16_model(a, p.columns, grid, s);
  else err = e8 ? plm::attend_f16_e4m3(a, p.columns, grid, s) : plm::attend_f16_model(a, p.columns, grid, s);
  if (err == hipSuccess && p.target > 0) err = plm::attend_join(dtype, a, p.columns, p.groups, s);
  return err == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

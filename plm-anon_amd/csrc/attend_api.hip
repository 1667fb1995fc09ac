// C ABI of the attention over the paged cache (plm_attend), declared in include/plm_amd.h.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attend.h"
#include "plm_amd.h"

namespace plm {
namespace {

struct AttendPlan {
  int columns;        // of a workgroup's tile
  int target, least;  // AttendArgs
  int64_t grid, groups, bytes;
};

// The launch of a call, from what the host knows: sizes, never the lengths. The work is cut on the device
// (attend_item), so a wide table costs nothing; `grid` bounds the workgroups that any lengths can ask for:
// one per group and as many more as the work is cut into.
AttendPlan attend_plan(int64_t kv_heads, int64_t page, int64_t head_dim, int64_t heads, int64_t total, int64_t seqs,
                       int64_t max_rows, int64_t table_width) {
  AttendPlan p{};
  const int64_t group = heads / kv_heads, chunks = (head_dim + 63) / 64;
  const int64_t most = max_rows * group;
  p.columns = most <= 16 ? 16 : chunks > 2 ? 64 : most <= 32 ? 32 : most <= 256 ? 64 : 128;
  p.groups = kv_heads * (seqs + total * group / p.columns);
  const int64_t capacity = (table_width * page + kStep - 1) / kStep;
  p.least = p.columns <= 32 ? 16 : 8;
  // A single sequence's groups are alike: where they fill the device there is nothing to even out.
  p.target = capacity > p.least && !(seqs == 1 && p.groups >= 256) ? 512 : 0;
  p.grid = p.groups + p.target;
  // There are 2 * target ranges of groups of several at most: a cut sequence has less than twice load / chunk of
  // them, and a chunk is load / target at least. Such a group has two at least.
  if (p.target > 0) {
    p.groups = std::min<int64_t>(p.groups, p.target);
    p.bytes = 2 * p.target * attend_slot_floats(p.columns, static_cast<int>(64 * chunks)) * 4;
  }
  return p;
}

bool attend_sizes(int64_t kv_heads, int64_t page, int64_t head_dim, int64_t heads, int64_t total, int64_t seqs,
                  int64_t max_rows, int64_t table_width) {
  return kv_heads >= 1 && kv_heads <= 1024 && heads >= kv_heads && heads <= 4096 && heads % kv_heads == 0 &&
         (page == 16 || page == 32 || page == 64 || page == 128) && head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0 &&
         seqs >= 1 && seqs <= (1 << 20) && max_rows >= 1 && max_rows <= total && total < (1 << 28) &&
         total * (heads / kv_heads) < (int64_t{1} << 30) && table_width >= 1 && table_width * page <= (int64_t{1} << 29);
}

}  // namespace
}  // namespace plm

extern "C" {

size_t plm_attend_workspace_bytes(int32_t kv_heads, int32_t page, int32_t head_dim, int32_t heads, int64_t total,
                                  int64_t seqs, int64_t max_rows, int64_t table_width) {
  if (!plm::attend_sizes(kv_heads, page, head_dim, heads, total, seqs, max_rows, table_width)) return 0;
  return static_cast<size_t>(plm::attend_plan(kv_heads, page, head_dim, heads, total, seqs, max_rows, table_width).bytes);
}

int plm_attend(int32_t dtype, const plm_kv_cache* cache, const void* q, int64_t q_row, int64_t q_head, int32_t heads,
               void* out, int64_t total, int64_t seqs, int64_t max_rows, const int32_t* table, int64_t table_stride,
               int64_t table_width, const int64_t* lengths, const int64_t* row_starts, int64_t window, int64_t sinks,
               const uint32_t* mask, int64_t mask_rows, int64_t mask_words, const int64_t* positions, float scale,
               void* workspace, size_t workspace_bytes, void* stream) {
  plm::AttendArgs a{};
  if (!plm::kv_cache_of(cache, a.cache) || !plm::kv_type_fits(cache, dtype)) return PLM_ERR_ARGUMENT;
  if (!plm::attend_sizes(cache->kv_heads, cache->page, cache->head_dim, heads, total, seqs, max_rows, table_width))
    return PLM_ERR_ARGUMENT;
  if (!plm::kv_rows_of(a.cache, total, seqs, max_rows, table, table_stride, table_width, lengths, row_starts, a.rows))
    return PLM_ERR_ARGUMENT;
  if (q == nullptr || out == nullptr || window < 0 || sinks < 0) return PLM_ERR_ARGUMENT;
  if (mask != nullptr && (mask_rows < 1 || mask_words < 1 || mask_rows >= (1 << 28) || mask_words >= (1 << 24)))
    return PLM_ERR_ARGUMENT;
  if (q_row % 8 != 0 || q_head % 8 != 0) return PLM_ERR_ALIGNMENT;
  for (const void* p : {q, static_cast<const void*>(out), static_cast<const void*>(cache->k),
                        static_cast<const void*>(cache->v), static_cast<const void*>(workspace)})
    if (!plm::aligned16_ptr(p)) return PLM_ERR_ALIGNMENT;
  const plm::AttendPlan p =
      plm::attend_plan(cache->kv_heads, cache->page, cache->head_dim, heads, total, seqs, max_rows, table_width);
  if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(p.bytes))) return PLM_ERR_WORKSPACE;
  if (p.grid >= (int64_t{1} << 31)) return PLM_ERR_ARGUMENT;
  constexpr int64_t far = int64_t{1} << 30;
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_row = q_row;
  a.q_head = q_head;
  a.positions = positions;
  a.mask = mask;
  a.partials = static_cast<float*>(workspace);
  a.scale = scale * 1.44269504088896340736f;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.window = static_cast<int>(window < far ? window : 0);  // longer than any cache: no window
  a.sinks = static_cast<int>(std::min(sinks, far));
  a.mask_rows = static_cast<int>(mask_rows);
  a.mask_words = static_cast<int>(mask_words);
  a.target = p.target;
  a.per_target = p.target > 0 ? 1.001f / static_cast<float>(p.target) : 0.0f;
  a.least = p.least;
  const unsigned grid = static_cast<unsigned>(p.grid);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool e8 = cache->type == PLM_CACHE_E4M3;
  hipError_t err;
  if (dtype == PLM_BF16) err = e8 ? plm::attend_bf16_e4m3(a, p.columns, grid, s) : plm::attend_bf16_model(a, p.columns, grid, s);
  else err = e8 ? plm::attend_f16_e4m3(a, p.columns, grid, s) : plm::attend_f16_model(a, p.columns, grid, s);
  if (err == hipSuccess && p.target > 0)
    err = plm::attend_join(dtype, a, p.columns, p.groups, s);
  return err == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

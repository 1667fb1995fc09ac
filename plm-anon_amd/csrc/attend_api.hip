// C ABI of the attention over the paged cache (plm_attend), declared in include/plm_amd.h.
#include <hip/hip_runtime.h>

#include "attend.h"
#include "plm_amd.h"

namespace plm {
namespace {

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
  a.walkers = static_cast<int>(std::min(p.grid, (int64_t{1} << 31) - 1));
  p.grid += kv_clear_groups(a.rows, h.heads * (a.cache.dim / 8));
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

// C ABI of the products over e4m3 rows (plm_fp8_linear), declared in include/plm_amd.h.
#include <hip/hip_runtime.h>

#include "fp8_gemm.h"

namespace plm {
namespace {

struct Fp8Plan {
  bool tile, round;   // round: rows of 16 bits first, by a launch of their own
  Fp8TileKind kind;
  Fp8Narrow narrow;
  size_t codes, scales, bytes;   // of a workspace's rounded rows and, behind them, all of it with the partial sums
};

// The plan of a call whose numbers go together; false where they do not.
bool linear_of(const plm_fp8_linear_call* call, Fp8Gemm& a, Fp8Plan& p) {
  if (call == nullptr) return false;
  const plm_fp8_linear_call& h = *call;
  const bool act = h.act != 0;
  if (h.m < 1 || h.m > PLM_FP8_MOST || h.n < 1 || h.n > PLM_FP8_MOST || plm_fp8_codes_bytes(h.n, h.k) == 0 || (act && h.n % 32 != 0))
    return false;
  if (h.ldy < (act ? h.n / 2 : h.n) || h.out < PLM_FP8_BF16 || h.out > PLM_FP8_F32) return false;
  if (h.x_type < PLM_FP8_CODES || h.x_type > PLM_FP8_ROWS_F16) return false;
  const bool in16 = h.x_type != PLM_FP8_CODES;
  if (in16 && (h.x_row < 0 || plm_fp8_codes_bytes(h.m, h.k) == 0)) return false;
  // Up to 16 rows every workgroup rounds for itself, which saves a launch (2048 x 2048 over one row 3.7 us for 6); not several
  // for each of an LM head's many workgroups (50257 x 2048 over 16 rows 28 us for 26).
  p.round = in16 && (h.m > 16 || (h.m > 4 && h.n > 16384));
  a.ldy = h.ldy;
  a.x_row = h.x_row;
  a.m = static_cast<int>(h.m);
  a.n = static_cast<int>(h.n);
  a.k = static_cast<int>(h.k);
  a.blocks = static_cast<int>(fp8_blocks(h.k));
  a.x_frags = static_cast<int>(fp8_frags(h.m));
  a.w_frags = static_cast<int>(fp8_frags(h.n));
  a.x_type = p.round ? static_cast<int>(PLM_FP8_CODES) : static_cast<int>(h.x_type);
  a.out = static_cast<int>(h.out);
  p.narrow = narrow_plan(a.x_frags, a.w_frags, a.blocks, act, a.x_type != PLM_FP8_CODES);
  const bool exact = h.out == PLM_FP8_F32;
  const Fp8TilePlan t = tile_plan(a.x_frags, a.w_frags, a.blocks, exact);
  // Results in fp32 are a fifth to a half slower the narrow way (128 x 8192 x 2048 11.5 us for 9.2, 256 19 for 14.6).
  p.tile = a.x_frags >= kFp8TileFrags && t.us < (exact ? 1.25 : 1.0) * p.narrow.us;
  p.kind = t.kind;
  p.codes = p.round ? plm_fp8_codes_bytes(h.m, h.k) : 0;
  p.scales = p.round ? plm_fp8_scales_bytes(h.m, h.k) : 0;
  p.bytes = p.codes + p.scales;
  if (!p.tile && p.narrow.ranges > 1) p.bytes += static_cast<size_t>(p.narrow.ranges) * a.x_frags * a.w_frags * 1024;
  return true;
}

}  // namespace
}  // namespace plm

extern "C" {

size_t plm_fp8_linear_workspace_bytes(const plm_fp8_linear_call* call) {
  plm::Fp8Gemm a{};
  plm::Fp8Plan p{};
  return plm::linear_of(call, a, p) ? p.bytes : 0;
}

int plm_fp8_linear(const plm_fp8_linear_call* call, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace plm;
  Fp8Gemm a{};
  Fp8Plan p{};
  if (!linear_of(call, a, p)) return PLM_ERR_ARGUMENT;
  const plm_fp8_linear_call& h = *call;
  const bool codes = h.x_type == PLM_FP8_CODES;
  if (h.x == nullptr || (codes && h.x_scales == nullptr) || h.w == nullptr || h.w_scales == nullptr || h.y == nullptr)
    return PLM_ERR_ARGUMENT;
  for (const void* at : {h.x, h.x_scales, h.w, h.w_scales, static_cast<const void*>(workspace)})
    if (!aligned16_ptr(at)) return PLM_ERR_ALIGNMENT;
  if (!codes && h.x_row % 8 != 0) return PLM_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(h.y) % (h.out == PLM_FP8_F32 ? 4 : 2) != 0) return PLM_ERR_ALIGNMENT;
  if (p.bytes > 0 && (workspace == nullptr || workspace_bytes < p.bytes)) return PLM_ERR_WORKSPACE;
  a.x = static_cast<const uint8_t*>(h.x);
  a.x_scales = static_cast<const uint8_t*>(h.x_scales);
  a.w = static_cast<const uint8_t*>(h.w);
  a.w_scales = static_cast<const uint8_t*>(h.w_scales);
  a.y = h.y;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t err = hipSuccess;
  uint8_t* space = static_cast<uint8_t*>(workspace);
  if (p.round) {
    err = fp8_round(h.x_type == PLM_FP8_ROWS_BF16 ? PLM_BF16 : PLM_F16, h.x, h.x_row, h.m, h.k, space, space + p.codes, s);
    a.x = space;
    a.x_scales = space + p.codes;
  }
  if (err != hipSuccess) return PLM_ERR_LAUNCH;
  a.partials = reinterpret_cast<f32x4*>(space + p.codes + p.scales);
  err = p.tile ? fp8_tile(a, p.kind, h.act != 0, s) : fp8_narrow(a, p.narrow, h.act != 0, s);
  return err == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

// C ABI of the products over e4m3 rows (plm_fp8_linear), declared in include/plm_amd.h.
#include <hip/hip_runtime.h>

#include "fp8_gemm.h"

extern "C" {

int plm_fp8_linear(const plm_fp8_linear_call* call, void* stream) {
  using namespace plm;
  if (call == nullptr) return PLM_ERR_ARGUMENT;
  const plm_fp8_linear_call& h = *call;
  const bool act = h.act != 0;
  const int64_t columns = act ? h.n / 2 : h.n;
  if (plm_fp8_codes_bytes(h.m, h.k) == 0 || plm_fp8_codes_bytes(h.n, h.k) == 0 || (act && h.n % 32 != 0)) return PLM_ERR_ARGUMENT;
  // The second dimension of a grid has 65535 workgroups of 64 rows at least.
  if (h.m > (int64_t{1} << 21) || h.ldy < columns || h.out < PLM_FP8_BF16 || h.out > PLM_FP8_F32) return PLM_ERR_ARGUMENT;
  if (h.x == nullptr || h.x_scales == nullptr || h.w == nullptr || h.w_scales == nullptr || h.y == nullptr) return PLM_ERR_ARGUMENT;
  for (const void* p : {h.x, h.x_scales, h.w, h.w_scales})
    if (!aligned16_ptr(p)) return PLM_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(h.y) % (h.out == PLM_FP8_F32 ? 4 : 2) != 0) return PLM_ERR_ALIGNMENT;
  Fp8Gemm a{};
  a.x = static_cast<const uint8_t*>(h.x);
  a.x_scales = static_cast<const uint8_t*>(h.x_scales);
  a.w = static_cast<const uint8_t*>(h.w);
  a.w_scales = static_cast<const uint8_t*>(h.w_scales);
  a.y = h.y;
  a.ldy = h.ldy;
  a.m = static_cast<int>(h.m);
  a.n = static_cast<int>(h.n);
  a.blocks = static_cast<int>(fp8_blocks(h.k));
  a.x_frags = static_cast<int>(fp8_frags(h.m));
  a.w_frags = static_cast<int>(fp8_frags(h.n));
  a.out = static_cast<int>(h.out);
  return fp8_narrow(a, act, static_cast<hipStream_t>(stream)) == hipSuccess ? PLM_OK : PLM_ERR_LAUNCH;
}

}  // extern "C"

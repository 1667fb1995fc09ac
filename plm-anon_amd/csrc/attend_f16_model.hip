// Attention over 16-bit pages, f16 rows: the kernels of attend.h, a translation unit of its own so that
// the build compiles them in parallel.
#include "attend_pick.h"

namespace plm {

hipError_t attend_f16_model(const AttendArgs& a, int columns, unsigned grid, hipStream_t s) {
  return attend_pick<DT_F16, false>(a, columns, grid, s);
}

}  // namespace plm

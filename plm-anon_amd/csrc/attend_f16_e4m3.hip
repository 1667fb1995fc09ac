// Attention over e4m3 pages, f16 rows: the kernels of attend.h, a translation unit of its own so that
// the build compiles them in parallel.
#include "attend_pick.h"

namespace plm {

hipError_t attend_f16_e4m3(const AttendArgs& a, int columns, unsigned grid, hipStream_t s) {
  return attend_pick<DT_F16, true>(a, columns, grid, s);
}

}  // namespace plm

// Down products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4>
static void by_rows(const MxLaunch& l, int rows) {
  if (rows == 128)
    launch_mx_tile<false, FP4, 2>(l);
  else
    launch_mx_tile<false, FP4, 1>(l);
}
void launch_mx_down(const MxLaunch& l, bool fp4, int rows) { fp4 ? by_rows<true>(l, rows) : by_rows<false>(l, rows); }
}  // namespace kmoe_mx

// Down products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4>
static void by_rows(const MxLaunch& l, int mi) {
  if (mi == 4)
    launch_mx_tile<false, FP4, 4, 4>(l);
  else if (mi == 2)
    launch_mx_tile<false, FP4, 2, 4>(l);
  else
    launch_mx_tile<false, FP4, 1, 4>(l);
}
void launch_mx_down(const MxLaunch& l, bool fp4, int mi) { fp4 ? by_rows<true>(l, mi) : by_rows<false>(l, mi); }
}  // namespace kmoe_mx

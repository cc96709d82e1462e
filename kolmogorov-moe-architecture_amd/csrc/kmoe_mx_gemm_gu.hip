// Gate/up products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4, bool SAVE>
static void by_rows(const MxLaunch& l, int mi) {
  if (mi == 4)
    launch_mx_tile<true, FP4, 4, 4, SAVE>(l);
  else if (mi == 2)
    launch_mx_tile<true, FP4, 2, 4, SAVE>(l);
  else
    launch_mx_tile<true, FP4, 1, 4, SAVE>(l);
}
void launch_mx_gate_up(const MxLaunch& l, bool fp4, int mi) {
  if (fp4)
    l.g.gu ? by_rows<true, true>(l, mi) : by_rows<true, false>(l, mi);
  else
    l.g.gu ? by_rows<false, true>(l, mi) : by_rows<false, false>(l, mi);
}
}  // namespace kmoe_mx

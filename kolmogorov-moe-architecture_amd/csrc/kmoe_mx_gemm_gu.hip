// Gate/up products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4, bool SAVE>
static void by_rows(const MxLaunch& l, int rows) {
  if (rows == 128)
    launch_mx_tile<true, FP4, 2, SAVE>(l);
  else
    launch_mx_tile<true, FP4, 1, SAVE>(l);
}
void launch_mx_gate_up(const MxLaunch& l, bool fp4, int rows) {
  if (fp4)
    l.g.gu ? by_rows<true, true>(l, rows) : by_rows<true, false>(l, rows);
  else
    l.g.gu ? by_rows<false, true>(l, rows) : by_rows<false, false>(l, rows);
}
}  // namespace kmoe_mx

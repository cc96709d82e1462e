// Gate/up products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4, bool SAVE>
static void by_tile(const MxLaunch& l, MxTileSize t) {
  if (t == MxTileSize::R128xC256)
    launch_mx_tile<true, FP4, 2, 4, SAVE>(l);
  else if (t == MxTileSize::R64xC256)
    launch_mx_tile<true, FP4, 1, 4, SAVE>(l);
  else
    launch_mx_tile<true, FP4, 1, 2, SAVE>(l);
}
void launch_mx_gate_up(const MxLaunch& l, bool fp4, MxTileSize t) {
  if (fp4)
    l.g.gu ? by_tile<true, true>(l, t) : by_tile<true, false>(l, t);
  else
    l.g.gu ? by_tile<false, true>(l, t) : by_tile<false, false>(l, t);
}
}  // namespace kmoe_mx

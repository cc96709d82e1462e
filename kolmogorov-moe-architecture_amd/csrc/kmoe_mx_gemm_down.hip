// Down products over microscaled rows, see kmoe_mx_gemm.h.
#include "kmoe_mx_gemm.h"

namespace kmoe_mx {
template <bool FP4>
static void by_tile(const MxLaunch& l, MxTileSize t) {
  if (t == MxTileSize::R128xC256)
    launch_mx_tile<false, FP4, 2, 4>(l);
  else if (t == MxTileSize::R64xC256)
    launch_mx_tile<false, FP4, 1, 4>(l);
  else
    launch_mx_tile<false, FP4, 1, 2>(l);
}
void launch_mx_down(const MxLaunch& l, bool fp4, MxTileSize t) { fp4 ? by_tile<true>(l, t) : by_tile<false>(l, t); }
}  // namespace kmoe_mx

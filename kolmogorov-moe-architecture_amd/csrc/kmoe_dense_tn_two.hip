// Weight gradients in two parts: few rows with what their roundings lost.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_wgrad_two(const Args& g, hipStream_t s) { return launch_tile<64, 128, 2, 3, true, true, EPI_TWO, false>(g, s); }
}  // namespace kmoe_dense

// Weight gradients: products along the rows of both operands.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_wgrad(const Args& g, hipStream_t s) { return launch_any<true, true, EPI_PLAIN>(g, s); }
}  // namespace kmoe_dense

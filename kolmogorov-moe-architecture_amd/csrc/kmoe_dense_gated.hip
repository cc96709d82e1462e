// Products with two Linear weights: the gate and up projections with their activation.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_gated(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_GATED>(g, s); }
}  // namespace kmoe_dense

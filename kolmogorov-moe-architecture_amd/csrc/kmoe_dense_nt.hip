// Products with a Linear weight: the gate and up projections with their activation, and one projection.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_gated(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_GATED>(g, s); }
int launch_linear(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_PLAIN>(g, s); }
}  // namespace kmoe_dense

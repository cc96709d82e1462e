// The gate and up projections with adapters.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_gated_adapt(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_GATED, true>(g, s); }
}  // namespace kmoe_dense

// Products with a Linear weight: one projection.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_linear(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_PLAIN>(g, s); }
int launch_linear_adapt(const Args& g, hipStream_t s) { return launch_any<false, false, EPI_PLAIN, true>(g, s); }
int launch_linear_runs(const Args& g, hipStream_t s) { return launch_tile<64, 64, 2, 4, false, false, EPI_PLAIN, false>(g, s); }
int launch_linear_runs_adapt(const Args& g, hipStream_t s) {
  return launch_tile<64, 64, 2, 4, false, false, EPI_PLAIN, true>(g, s);
}
}  // namespace kmoe_dense

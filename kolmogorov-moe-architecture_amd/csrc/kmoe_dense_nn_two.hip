// The backward's products with a Linear weight as it lies: of the block's input, and with adapters.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_dx_two(const Args& g, hipStream_t s) { return launch_any<false, true, EPI_TWO>(g, s); }
int launch_dx_adapt(const Args& g, hipStream_t s) { return launch_any<false, true, EPI_PLAIN, true>(g, s); }
}  // namespace kmoe_dense

// The backward's products with a Linear weight as it lies: of the hidden values and of a projection's input.
#include "kmoe_dense_launch.h"

namespace kmoe_dense {
int launch_dh(const Args& g, hipStream_t s) { return launch_any<false, true, EPI_DH>(g, s); }
int launch_dx(const Args& g, hipStream_t s) { return launch_any<false, true, EPI_PLAIN>(g, s); }
}  // namespace kmoe_dense

// The group norm's kernels of the second derivative for one element type.
#include "group_norm_launch.h"

namespace ictc {
template void group_norm_bwd2<__bf16>(const GroupNormCall&);
}  // namespace ictc

// The group norm's forward and gradient kernels for one element type.
#include "group_norm_launch.h"

namespace ictc {
template void group_norm_fwd<float>(const GroupNormCall&);
template void group_norm_bwd<float>(const GroupNormCall&);
}  // namespace ictc

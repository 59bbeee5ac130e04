// The group norm's kernels for one element type.
#include "group_norm.h"

namespace ictc {
template void group_norm_fwd<float>(const GroupNormCall&);
template void group_norm_bwd<float>(const GroupNormCall&);
template void group_norm_bwd2<float>(const GroupNormCall&);
}  // namespace ictc

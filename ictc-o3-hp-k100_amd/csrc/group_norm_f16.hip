// The group norm's kernels for one element type.
#include "group_norm.h"

namespace ictc {
template void group_norm_fwd<_Float16>(const GroupNormCall&);
template void group_norm_bwd<_Float16>(const GroupNormCall&);
template void group_norm_bwd2<_Float16>(const GroupNormCall&);
}  // namespace ictc

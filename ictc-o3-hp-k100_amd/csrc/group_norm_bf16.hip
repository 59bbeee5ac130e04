// The group norm's kernels for one element type.
#include "group_norm.h"

namespace ictc {
template void group_norm_fwd<__bf16>(const GroupNormCall&);
template void group_norm_bwd<__bf16>(const GroupNormCall&);
template void group_norm_bwd2<__bf16>(const GroupNormCall&);
}  // namespace ictc

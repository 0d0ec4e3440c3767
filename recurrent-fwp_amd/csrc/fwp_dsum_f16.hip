// The decayed sum rule's kernels for rows of half elements, in a translation unit of their own.
#include "fwp_dsum.hpp"

namespace fwp {
FWP_DSUM_INSTANCES(half_t)
}  // namespace fwp

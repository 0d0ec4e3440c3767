// The decayed sum rule's kernels for rows of float elements, in a translation unit of their own.
#include "fwp_dsum.hpp"

namespace fwp {
FWP_DSUM_INSTANCES(float)
}  // namespace fwp

// The decayed sum rule's kernels for rows of bf16 elements, in a translation unit of their own.
#include "fwp_dsum.hpp"

namespace fwp {
FWP_DSUM_INSTANCES(bf16_t)
}  // namespace fwp

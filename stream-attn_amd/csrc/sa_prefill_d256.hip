// The kernels of a prompt's attention over the paged cache for a padded head_dim of 256.
#include "sa_prefill_kernel.h"

namespace sa {
hipError_t launch_prefill_d256(const PrefillLaunch& l) { return launch_prefill<256>(l); }
}  // namespace sa

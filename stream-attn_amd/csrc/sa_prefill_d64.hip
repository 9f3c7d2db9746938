// The kernels of a prompt's attention over the paged cache for a padded head_dim of 64.
#include "sa_prefill_kernel.h"

namespace sa {
hipError_t launch_prefill_d64(const PrefillLaunch& l) { return launch_prefill<64>(l); }
}  // namespace sa

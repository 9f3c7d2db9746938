// The decoding attention's kernels for a padded head_dim of 256.
#include "sa_decode_kernel.h"

namespace sa {
void launch_decode_d256(const DecodeLaunch& l) { l.bf16 ? launch_decode<Bf16, 256>(l) : launch_decode<Fp16, 256>(l); }
}  // namespace sa

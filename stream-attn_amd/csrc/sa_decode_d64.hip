// The decoding attention's kernels for a padded head_dim of 64.
#include "sa_decode_kernel.h"

namespace sa {
void launch_decode_d64(const DecodeLaunch& l) { l.bf16 ? launch_decode<Bf16, 64>(l) : launch_decode<Fp16, 64>(l); }
}  // namespace sa

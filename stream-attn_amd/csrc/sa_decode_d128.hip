// The decoding attention's kernels for a padded head_dim of 128.
#include "sa_decode_kernel.h"

namespace sa {
void launch_decode_d128(const DecodeLaunch& l) { l.bf16 ? launch_decode<Bf16, 128>(l) : launch_decode<Fp16, 128>(l); }
}  // namespace sa

// The shared-prefix attention kernels of head dim 64.
#include "prefix_attn_kernel.h"

namespace bc {
template void prefix_launch<64>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
}  // namespace bc

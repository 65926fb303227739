// The shared-prefix attention kernels of head dim 128.
#include "prefix_attn_kernel.h"

namespace bc {
template void prefix_launch<128>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
}  // namespace bc

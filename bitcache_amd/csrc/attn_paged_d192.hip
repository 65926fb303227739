// The paged matrix-core attention kernels of head dim 192.
#include "attn_mfma_kernel.h"

namespace bc {
template void paged_launch<192>(int, int, const AttnArgs&, dim3, hipStream_t);
template int paged_occupancy<192>(int, int);
}  // namespace bc

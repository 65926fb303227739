// The paged matrix-core attention kernels of head dim 160.
#include "attn_mfma_kernel.h"

namespace bc {
template void paged_launch<160>(int, int, const AttnArgs&, dim3, hipStream_t);
template int paged_occupancy<160>(int, int);
}  // namespace bc

// The paged matrix-core attention kernels of head dim 224.
#include "attn_mfma_kernel.h"

namespace bc {
template void paged_launch<224>(int, int, const AttnArgs&, dim3, hipStream_t);
template int paged_occupancy<224>(int, int);
}  // namespace bc

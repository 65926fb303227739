// The paged matrix-core attention kernels of head dim 32.
#include "attn_mfma_kernel.h"

namespace bc {
template void paged_launch<32>(int, int, const AttnArgs&, dim3, hipStream_t);
template int paged_occupancy<32>(int, int);
}  // namespace bc

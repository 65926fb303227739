// The paged matrix-core attention kernels of head dim 128.
#include "attn_mfma_kernel.h"

namespace bc {
template void paged_launch<128>(int, int, const AttnArgs&, dim3, hipStream_t);
template int paged_occupancy<128>(int, int);
}  // namespace bc

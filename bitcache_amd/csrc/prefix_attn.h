// Host face of the shared-prefix attention kernel (prefix_attn_kernel.h).
#pragma once

#include "attn.h"

namespace bc {

struct PrefixArgs {
    float* ws;        // [splits][B * Hq][D + 2] partials: m (log2 domain), l, acc[D]
    int tiles;        // 64-key tiles of the prefix (tables' first row)
    int tiles_per;    // tiles of a split
    int row_waves;    // row blocks of a workgroup: 1, 2, 4 or 8
};

// Head dims with instances, and the rows of a row block there (in sixteens)
constexpr bool prefix_dim(int d) { return d % 64 == 0; }
// grid.x splits, grid.y kv heads times row-block groups
template <int D>
int prefix_launch(bool res, int nc, const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st);

}  // namespace bc

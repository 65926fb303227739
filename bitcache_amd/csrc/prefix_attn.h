// Host face of the shared-prefix attention kernel (prefix_attn_kernel.h).
#pragma once

#include "attn.h"

namespace bc {

struct PrefixArgs {
    float* ws;        // [splits][B * Hq][D + 2] partials: m (log2 domain), l, acc[D]
    int tiles;        // 64-key tiles of the prefix (tables' first row)
    int tiles_per;    // tiles of a split
};

// Head dims with instances, and a workgroup's rows there at most (in sixteens):
// what holds the rows' operands and sums in registers at two waves per SIMD
constexpr bool prefix_dim(int d) { return d % 64 == 0; }
constexpr int prefix_columns(int d) { return d <= 128 ? 4 : 2; }
// Workgroups per CU (one wave of each per SIMD) of an instance: few rows need few
// registers and wait for memory
constexpr int prefix_waves(int d, int nc, bool res) {
    return nc == 1 && d <= 128 ? (res ? 3 : 4) : !res && d <= 128 && nc == 2 ? 3 : 2;
}
// nc 1, 2 or 4 (at most prefix_columns): 16 nc rows per workgroup; grid.x splits,
// grid.y kv heads times groups of rows
template <int D>
void prefix_launch(bool res, int nc, const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st);

}  // namespace bc

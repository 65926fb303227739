// Decode attention over a paged compressed cache, a length per sequence: host side
// and merge.  The attention itself is attn_mfma_kernel.h's paged instances over
// work units that the device cuts from the lengths (attn.h, PagedUnit).
#include <math.h>

#include "attn.h"
#include "prefix_attn.h"

namespace bc {
extern template void prefix_launch<64>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
extern template void prefix_launch<128>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
extern template void prefix_launch<192>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
extern template void prefix_launch<256>(bool, int, const AttnArgs&, const PrefixArgs&, dim3, hipStream_t);
}  // namespace bc

namespace {
using bc::AttnArgs;
using bc::PrefixArgs;
using bc::MODE_BINARY;
using bc::MODE_COMP;

// The merge of a sequence's units, and of the shared prefix's splits (prefix:
// `splits` partials per row): one workgroup per (sequence, query head), the
// partials spread over its 256 / D groups of threads (one of at least D).
template <int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(AttnArgs a, uint16_t* out, const float* prefix, int splits) {
    constexpr int P = 256 / D;
    __shared__ float fac[256];
    __shared__ float red[P * D];
    __shared__ float wmax[4], wsum[4];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bc::PagedUnits u = bc::paged_units(a, b, lane);
    const int64_t own_step = (int64_t)a.Hq * (D + 2), prefix_step = own_step * a.B;
    const float* own = a.ws + (int64_t)u.first * own_step + (int64_t)h * (D + 2);
    const float* shared = prefix + ((int64_t)b * a.Hq + h) * (D + 2);
    const int total = splits + u.count;
    auto partial = [&](int s) { return s < splits ? shared + s * prefix_step : own + (s - splits) * own_step; };
    const int part = tid / D, e = tid % D;
    // online over blocks of 256 partials
    float M = -INFINITY, L = 0.0f, acc = 0.0f;
    for (int s0 = 0; s0 < total; s0 += 256) {
        const int n = min(256, total - s0);
        const float* const p = partial(s0 + min(tid, n - 1));
        const float m = tid < n ? p[0] : -INFINITY;
        const float l = tid < n ? p[1] : 0.0f;
        const float mw = wave_max(m);
        if (lane == 0) wmax[wave] = mw;
        __syncthreads();
        const float mn = fmaxf(fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3])), M);
        const float f = m == -INFINITY ? 0.0f : exp2f(m - mn);
        fac[tid] = f;
        // (a NaN sum marks a bad page: it stays one at any factor)
        const float lw = wave_sum(l == l ? f * l : l);
        if (lane == 0) wsum[wave] = lw;
        __syncthreads();
        const float old = M == -INFINITY ? 0.0f : exp2f(M - mn);
        L = L * old + ((wsum[0] + wsum[1]) + (wsum[2] + wsum[3]));
        acc *= old;
        if (part < P) {
#pragma unroll 8
            for (int s = part; s < n; s += P) acc += fac[s] * partial(s0 + s)[2 + e];
        }
        M = mn;
        __syncthreads();
    }
    if (part < P) red[part * D + e] = acc;
    __syncthreads();
    if (tid < D) {
        float o = red[tid];
#pragma unroll
        for (int q = 1; q < P; q++) o += red[q * D + tid];
        // (NaN where the length is out of bounds)
        o = bc::paged_bad_len(a, a.lens[b]) ? __builtin_nanf("") : L == 0.0f ? 0.0f : o * (1.0f / L);
        out[((int64_t)b * a.Hq + h) * D + tid] = a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)o) : f2h(o);
    }
}

struct PagedPlan {
    int G, groups;     // query heads of a workgroup, workgroups per sequence and unit
    int unit_tiles, unit_target;
    int units;         // at most
    // the shared prefix's kernel (splits 0: the prefix is attended as own keys)
    int splits, tiles_per, nc, row_groups;
    size_t own_bytes, bytes;   // of the units' partials, and with the prefix's
};

// The shared prefix: groups of 16 nc query rows, and two workgroups per CU.
void plan_prefix(PagedPlan& p, int batch, int n_heads, int n_kv_heads, int shared_len, int d) {
    const int64_t rows = (int64_t)batch * (n_heads / n_kv_heads);
    if (shared_len == 0 || batch < 2 || !bc::prefix_dim(d)) return;
    p.nc = rows <= 16 ? 1 : rows <= 32 ? 2 : bc::prefix_columns(d);
    p.row_groups = (int)((rows + 16 * p.nc - 1) / (16 * p.nc));
    const int tiles = shared_len / 64;
    int64_t splits = 2LL * bc::device_cu_count() / ((int64_t)n_kv_heads * p.row_groups);
    if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4;
    if (splits < 1) splits = 1;
    p.tiles_per = (int)((tiles + splits - 1) / splits);
    p.splits = (tiles + p.tiles_per - 1) / p.tiles_per;
}

PagedPlan plan(int mode, int batch, int n_heads, int n_kv_heads, int max_seq_len, int shared_len, int d) {
    PagedPlan p{};
    plan_prefix(p, batch, n_heads, n_kv_heads, shared_len, d);
    if (p.splits > 0) max_seq_len -= shared_len;   // (units hold the keys after it)
    p.G = bc::attention_group(n_heads / n_kv_heads, d, mode);
    p.groups = n_kv_heads * (n_heads / n_kv_heads / p.G);
    const int64_t tiles = ((int64_t)max_seq_len + 63) / 64;
    const int cu = bc::device_cu_count();
    int fit = bc::paged_wgs_per_cu(mode, d, p.G);
    if (fit <= 0) fit = 3;
    p.unit_target = (int)((2LL * fit * cu + p.groups - 1) / p.groups);
    // (at least two tiles a wave, one where that leaves CUs idle)
    p.unit_tiles = (int64_t)batch * p.groups * ((tiles + 7) / 8) < cu ? 4 : 8;
    if (tiles <= p.unit_tiles && p.splits == 0) {
        p.unit_tiles = 0;
        p.units = batch;
        return p;
    }
    const int64_t most = (int64_t)batch * ((tiles + p.unit_tiles - 1) / p.unit_tiles);
    const int64_t capped = ((int64_t)batch * tiles + bc::kUnitTiles - 1) / bc::kUnitTiles;
    int64_t units = (capped > p.unit_target ? capped : p.unit_target) + batch;
    if (units > most) units = most;
    p.units = (int)units;
    p.own_bytes = (size_t)units * n_heads * (d + 2) * sizeof(float);
    p.bytes = p.own_bytes + (size_t)p.splits * batch * n_heads * (d + 2) * sizeof(float);
    return p;
}

int validate(int batch, int n_heads, int n_kv_heads, int max_seq_len, int shared_len, int d) {
    BC_REQUIRE(bc::head_dim_ok(d), BC_ERR_UNSUPPORTED,
               "head_dim must be a multiple of 32 in [32, 256], got %d", d);
    BC_REQUIRE(batch >= 0 && n_heads >= 0 && n_kv_heads > 0 && max_seq_len >= 0 && shared_len >= 0,
               BC_ERR_INVALID_ARGUMENT, "invalid dims batch=%d n_heads=%d n_kv_heads=%d max_seq_len=%d shared_len=%d",
               batch, n_heads, n_kv_heads, max_seq_len, shared_len);
    BC_REQUIRE(n_heads % n_kv_heads == 0, BC_ERR_INVALID_ARGUMENT,
               "n_heads (%d) must be a multiple of n_kv_heads (%d)", n_heads, n_kv_heads);
    BC_REQUIRE(shared_len <= max_seq_len, BC_ERR_INVALID_ARGUMENT, "shared_len (%d) above max_seq_len (%d)",
               shared_len, max_seq_len);
    BC_REQUIRE(shared_len % 64 == 0, BC_ERR_INVALID_ARGUMENT, "shared_len (%d) must be whole pages", shared_len);
    BC_REQUIRE(batch <= 65535, BC_ERR_UNSUPPORTED, "batch above 65535");
    BC_REQUIRE(n_heads <= 65535, BC_ERR_UNSUPPORTED, "n_heads above 65535");
    BC_REQUIRE((int64_t)batch * (max_seq_len / 64 + 1) <= INT32_MAX, BC_ERR_UNSUPPORTED,
               "batch * max_seq_len above 2^37");
    return BC_OK;
}

}  // namespace

extern "C" int bc_paged_attention_workspace_size(int batch, int n_heads, int n_kv_heads, int max_seq_len,
                                                 int shared_len, int head_dim, size_t* bytes) {
    BC_REQUIRE(bytes != nullptr, BC_ERR_INVALID_ARGUMENT, "null pointer");
    const int rc = validate(batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim);
    if (rc != BC_OK) return rc;
    *bytes = 0;
    if ((int64_t)batch * n_heads == 0) return BC_OK;
    for (int mode : {MODE_BINARY, MODE_COMP}) {
        const size_t n = plan(mode, batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim).bytes;
        if (n > *bytes) *bytes = n;
    }
    return BC_OK;
}

extern "C" int bc_paged_attention(const void* q, const void* k_bin, const void* k_res, const void* v_bin,
                                  const void* v_res, const int32_t* block_tables, int table_width,
                                  const int32_t* seq_lens, void* out, int batch, int n_heads, int n_kv_heads,
                                  int n_pages, int page_size, int max_seq_len, int shared_len, int head_dim,
                                  int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = validate(batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim);
    if (rc != BC_OK) return rc;
    BC_REQUIRE(dtype == BC_FP16 || dtype == BC_BF16, BC_ERR_UNSUPPORTED, "dtype must be BC_FP16 or BC_BF16");
    BC_REQUIRE(n_pages >= 0 && page_size > 0 && page_size % 64 == 0, BC_ERR_INVALID_ARGUMENT,
               "page_size must be a multiple of 64, got %d (n_pages %d)", page_size, n_pages);
    BC_REQUIRE((int64_t)n_pages * page_size <= INT32_MAX, BC_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    // (a tile's place among the pool's tiles is an int)
    BC_REQUIRE((int64_t)n_pages * (page_size / 64) * n_kv_heads <= INT32_MAX, BC_ERR_UNSUPPORTED,
               "more than 2^37 vectors in the pool");
    BC_REQUIRE(table_width >= 0, BC_ERR_INVALID_ARGUMENT, "negative table width");
    BC_REQUIRE(shared_len % page_size == 0 && shared_len / page_size <= table_width, BC_ERR_INVALID_ARGUMENT,
               "shared_len (%d) must be whole pages of %d slots within the tables", shared_len, page_size);
    BC_REQUIRE((k_res == nullptr) == (v_res == nullptr), BC_ERR_INVALID_ARGUMENT,
               "k_res and v_res must both be given or both be null");
    if ((int64_t)batch * n_heads == 0) return BC_OK;
    BC_REQUIRE(q && out && seq_lens && (table_width == 0 || block_tables) && (n_pages == 0 || (k_bin && v_bin)),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    const int mode = k_res ? MODE_COMP : MODE_BINARY;
    const PagedPlan p = plan(mode, batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim);
    BC_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes), BC_ERR_WORKSPACE,
               "workspace of %zu bytes required, got %zu", p.bytes, workspace_bytes);
    BC_REQUIRE(p.groups <= 65535 && (int64_t)n_kv_heads * p.row_groups <= 65535, BC_ERR_UNSUPPORTED, "more than 65535 head groups");
    const int64_t cap = (int64_t)n_pages * n_kv_heads * page_size;
    hipStream_t st = (hipStream_t)stream;
    AttnArgs a{};
    a.q = (const uint16_t*)q;
    a.kb = bin_planes(k_bin, cap, head_dim);
    a.vb = bin_planes(v_bin, cap, head_dim);
    if (k_res) a.kr = res_planes(k_res, cap, head_dim);
    if (v_res) a.vr = res_planes(v_res, cap, head_dim);
    a.B = batch;
    a.Hq = n_heads;
    a.Hkv = n_kv_heads;
    a.ws = (float*)workspace;
    a.lens = seq_lens;
    a.tables = block_tables;
    a.width = table_width;
    a.n_pages = n_pages;
    a.page_tiles = page_size / 64;
    a.max_len = n_pages > 0 ? max_seq_len : 0;   // (without pages no length but zero is right)
    a.unit_tiles = p.unit_tiles;
    a.unit_target = p.unit_target;
    a.bf16 = dtype == BC_BF16;
    float* const prefix_ws = (float*)((uint8_t*)workspace + p.own_bytes);
    // (a pool without pages holds no length but zero: nothing to attend)
    const int splits = n_pages > 0 ? p.splits : 0;
    if (p.splits > 0) a.key0 = shared_len;
    if (splits > 0) {
        const PrefixArgs x{prefix_ws, shared_len / 64, p.tiles_per};
        const dim3 grid(p.splits, n_kv_heads * p.row_groups);
        switch (head_dim) {
#define BC_CASE(DD) case DD: bc::prefix_launch<DD>(k_res != nullptr, p.nc, a, x, grid, st); break;
            BC_CASE(64) BC_CASE(128) BC_CASE(192) BC_CASE(256)
#undef BC_CASE
            default: return bc::set_error(BC_ERR_UNSUPPORTED, "head_dim %d", head_dim);
        }
        const int prefix_rc = bc::check_launch("prefix attention");
        if (prefix_rc != BC_OK) return prefix_rc;
    }
    if (p.unit_tiles == 0) a.out = (uint16_t*)out;
    if (p.units > 0)
        BC_REQUIRE(bc::launch_paged_split(mode, head_dim, p.G, a, dim3(p.units, p.groups), st), BC_ERR_UNSUPPORTED,
                   "head_dim %d", head_dim);
    const int launched = bc::check_launch("paged attention");
    if (launched != BC_OK || p.unit_tiles == 0) return launched;
    const dim3 grid(n_heads, batch);
    switch (head_dim) {
#define BC_CASE(DD) \
    case DD: hipLaunchKernelGGL((paged_combine_kernel<DD>), grid, dim3(256), 0, st, a, (uint16_t*)out, prefix_ws, splits); break;
        BC_CASE(32) BC_CASE(64) BC_CASE(96) BC_CASE(128) BC_CASE(160) BC_CASE(192) BC_CASE(224) BC_CASE(256)
#undef BC_CASE
        default: return bc::set_error(BC_ERR_UNSUPPORTED, "head_dim %d", head_dim);
    }
    return bc::check_launch("paged attention merge");
}

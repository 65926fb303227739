// Decode attention over a paged compressed cache, a length per sequence: host side
// and merge.  The attention itself is attn_mfma_kernel.h's paged instances over
// work units that the device cuts from the lengths (attn.h, PagedUnit).
#include <math.h>
#include <stdlib.h>

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

// The merge of a sequence's units, and of the shared prefix's `splits` partials per
// row: PARTS waves per (sequence, query head), each over every PARTS-th partial
// (lane = partial for the factors, lanes = dims for the sums), joined in LDS.
// Bound: the latency of its three loads in turn (units, maxima, sums): 5 us for 256
// to 2048 rows of 5 to 10 partials, 7 with the prefix's.
template <int D, int PARTS>
__global__ __launch_bounds__(256) void paged_combine_kernel(AttnArgs a, uint16_t* out, const float* prefix, int splits) {
    constexpr int N = (D + 63) / 64;     // dims of a lane
    constexpr int ROWS = 4 / PARTS;      // rows of a workgroup
    __shared__ float join[PARTS > 1 ? 4 : 1][D + 2];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int part = wave % PARTS;
    const int64_t row = (int64_t)blockIdx.x * ROWS + wave / PARTS;
    const bool live = row < (int64_t)a.B * a.Hq;
    const int b = live ? (int)(row / a.Hq) : 0, h = live ? (int)(row - (int64_t)b * a.Hq) : 0;
    // (without units: all keys are the prefix's)
    const int len = a.lens[b];
    int2 u = make_int2(0, 0);
    if (a.unit_each > 0) u = make_int2(b * a.unit_each, (bc::paged_tiles(a, len) + bc::kUnitTiles - 1) / bc::kUnitTiles);
    else if (a.unit_most > 0) u = a.units[b];
    const int64_t own_step = (int64_t)a.Hq * (D + 2), prefix_step = own_step * a.B;
    const float* const own = a.ws + (int64_t)u.x * own_step + (int64_t)h * (D + 2);
    const float* const shared = prefix + ((int64_t)b * a.Hq + h) * (D + 2);
    const int total = live ? splits + u.y : 0;
    // (s-th partial of this wave)
    auto partial = [&](int s) {
        s = s * PARTS + part;
        return s < splits ? shared + s * prefix_step : own + (s - splits) * own_step;
    };
    const int mine = (total - part + PARTS - 1) / PARTS;
    float M = -INFINITY, L = 0.0f, acc[N];
#pragma unroll
    for (int n = 0; n < N; n++) acc[n] = 0.0f;
    for (int s0 = 0; s0 < mine; s0 += 64) {
        const int cnt = min(64, mine - s0);
        const float* const p = partial(s0 + min(lane, cnt - 1));
        const float m = lane < cnt ? p[0] : -INFINITY, l = lane < cnt ? p[1] : 0.0f;
        const float mn = fmaxf(wave_max(m), M);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float old = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - mn);
        // (a NaN sum marks a bad page: it stays one at any factor)
        L = L * old + wave_sum(l == l ? f * l : l);
        M = mn;
#pragma unroll
        for (int n = 0; n < N; n++) acc[n] *= old;
#pragma unroll 8
        for (int s = 0; s < cnt; s++) {
            const float* const q = partial(s0 + s) + 2 + lane;
            const float fs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), s));
#pragma unroll
            for (int n = 0; n < N; n++)
                if (D % 64 == 0 || n < N - 1 || lane < 32) acc[n] = fmaf(fs, q[64 * n], acc[n]);
        }
    }
    if constexpr (PARTS > 1) {
#pragma unroll
        for (int n = 0; n < N; n++)
            if (64 * n + lane < D) join[wave][64 * n + lane] = acc[n];
        if (lane == 0) {
            join[wave][D] = M;
            join[wave][D + 1] = L;
        }
        __syncthreads();
        if (part != 0) return;
        const int w0 = wave;
        float m[PARTS], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < PARTS; w++) {
            m[w] = join[w0 + w][D];
            top = fmaxf(top, m[w]);
        }
        L = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) acc[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < PARTS; w++) {
            const float f = m[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[w] - top), l = join[w0 + w][D + 1];
            L += l == l ? f * l : l;
#pragma unroll
            for (int n = 0; n < N; n++)
                if (64 * n + lane < D) acc[n] = fmaf(f, join[w0 + w][64 * n + lane], acc[n]);
        }
    }
    if (!live) return;
    const bool bad = bc::paged_bad_len(a, len);   // (NaN where the length is out of bounds)
    const float inv = bad ? __builtin_nanf("") : L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int n = 0; n < N; n++)
        if (64 * n + lane < D) {
            const float o = acc[n] * inv;
            out[row * D + 64 * n + lane] = a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)o) : f2h(o);
        }
}

struct PagedPlan {
    int G, groups;     // query heads of a workgroup, workgroups per sequence and unit
    int unit_tiles, unit_slots, unit_each;
    int units;         // at most
    // the shared prefix's kernel (splits 0: the prefix is attended as own keys)
    int splits, tiles_per, nc, row_groups;
    size_t own_bytes, bytes;   // of the units' notes and partials, and with the prefix's
};

// What notes every sequence's units
size_t note_bytes(int batch) { return ((size_t)batch * sizeof(int2) + 15) & ~(size_t)15; }

// Whether the shared prefix has its own kernel: where the sequences would read 192 MB
// or more of it.  Less, and its launch and its partials cost more than the bytes
// (whole calls, 200 keys more per sequence, us without and with it; residual
// planes, 32/8 heads of 128: 32768 keys, 4 sequences 34 and 42, 8 50 and 43, 32 144
// and 75; 8192 keys, 16 sequences 33 and 43, 32 48 and 49; 32/32 heads, 2048 keys, 8
// sequences 20 and 25, 32 43 and 37; signs only, 32/8 heads, 32768 keys, 16
// sequences 37 and 48, 32 58 and 56).  BITCACHE_SHARED=1 and =0 choose it always and never (tuning).
bool prefix_pays(int mode, int64_t batch, int n_kv_heads, int64_t shared_len, int d) {
    if (const char* e = getenv("BITCACHE_SHARED")) return e[0] == '1';
    const int64_t pair = 2 * (mode == MODE_BINARY ? d / 8 + 2 : d / 8 + 2 + d / 2 + 2);
    return batch * shared_len * n_kv_heads * pair >= 192ll << 20;
}

// Its plan: groups of 16 nc query rows, and as many workgroups as the CUs hold.
void plan_prefix(PagedPlan& p, int mode, int batch, int n_heads, int n_kv_heads, int shared_len, int d) {
    const int64_t rows = (int64_t)batch * (n_heads / n_kv_heads);
    if (shared_len == 0 || batch < 2 || !bc::prefix_dim(d) || !prefix_pays(mode, batch, n_kv_heads, shared_len, d)) return;
    p.nc = rows <= 16 ? 1 : rows <= 32 ? 2 : bc::prefix_columns(d);
    p.row_groups = (int)((rows + 16 * p.nc - 1) / (16 * p.nc));
    const int tiles = shared_len / 64;
    int64_t splits = (int64_t)bc::prefix_waves(d, p.nc, mode != MODE_BINARY) * bc::device_cu_count() / ((int64_t)n_kv_heads * p.row_groups);
    if (splits > (tiles + 3) / 4) splits = (tiles + 3) / 4;
    if (splits < 1) splits = 1;
    p.tiles_per = (int)((tiles + splits - 1) / splits);
    p.splits = (tiles + p.tiles_per - 1) / p.tiles_per;
}

PagedPlan plan(int mode, int batch, int n_heads, int n_kv_heads, int max_seq_len, int shared_len, int d) {
    PagedPlan p{};
    plan_prefix(p, mode, batch, n_heads, n_kv_heads, shared_len, d);
    if (p.splits > 0) max_seq_len -= shared_len;   // (units hold the keys after it)
    p.G = bc::attention_group(n_heads / n_kv_heads, d, mode);
    p.groups = n_kv_heads * (n_heads / n_kv_heads / p.G);
    const int64_t tiles = ((int64_t)max_seq_len + 63) / 64;
    // short sequences: one unit each, and no merge (4 sequences of 100 to 1024 keys:
    // 12 us, 18.7 us in units)
    if (tiles <= 16 && p.splits == 0) {
        p.units = batch;
        return p;
    }
    const int cu = bc::device_cu_count();
    int fit = bc::paged_wgs_per_cu(mode, d, p.G);
    if (fit <= 0) fit = 3;
    // (two workgroups a CU keep the memory busy with residual planes, four with signs
    // alone, and a round of more cuts sequences finer: residual planes, 64 sequences of
    // 500 to 16000 keys, 32/8 heads of 64, 50 us, 55 with 3 or 4; 64 of 6144 keys of 128,
    // 90 and 96; signs, 64 of 8192 keys, 32/8 heads of 128, 41 us, with 3 49, with 2 52)
    const int most_fit = mode == MODE_BINARY ? 4 : 2;
    if (fit > most_fit) fit = most_fit;
    p.unit_slots = (int)(((int64_t)fit * cu + p.groups - 1) / p.groups);
    // (at least two tiles a wave, one where that leaves CUs idle)
    p.unit_tiles = (int64_t)batch * p.groups * ((tiles + 7) / 8) < cu ? 4 : 8;
    const int64_t most = (int64_t)batch * ((tiles + p.unit_tiles - 1) / p.unit_tiles);
    int64_t units = bc::paged_unit_most(p.unit_slots, batch, batch * tiles);
    if (units > most) units = most;
    // A large batch is even enough by itself, and its lengths take each wave long to go
    // through: equal units of every sequence instead (us by the lengths and in equal units,
    // 500 to 4000 keys, 32/8 heads of 128: 128 sequences 77 and 77, 400 215 and 186, 1024 585
    // and 418; 100 to 8000 keys, 8/2 heads: 128 sequences 33 and 67, 700 121 and 116, 1024
    // 173 and 145; signs, 64 to 20000 keys, 32/8 heads: 256 98 and 147, 700 296 and 328, 1024
    // 499 and 444).
    // (as far as a launch holds them)
    const int64_t each = (tiles + bc::kUnitTiles - 1) / bc::kUnitTiles;
    if ((batch > 4 * p.unit_slots || batch > 640) && units > 0 && batch * each <= 65535) {
        p.unit_each = (int)each;
        units = batch * each;
    }
    p.units = (int)units;
    p.own_bytes = note_bytes(batch) + (size_t)units * n_heads * (d + 2) * sizeof(float);
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
    // (planes start where their vectors are whole 16 bytes, after 64 and more of them)
    BC_REQUIRE((((uintptr_t)k_bin | (uintptr_t)k_res | (uintptr_t)v_bin | (uintptr_t)v_res | (uintptr_t)workspace) & 15) == 0,
               BC_ERR_INVALID_ARGUMENT, "blobs and workspace must be 16-byte aligned");
    const int mode = k_res ? MODE_COMP : MODE_BINARY;
    const PagedPlan p = plan(mode, batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim);
    BC_REQUIRE(p.units <= 65535, BC_ERR_UNSUPPORTED, "more than 65535 work units");
    BC_REQUIRE(p.bytes == 0 || (workspace != nullptr && workspace_bytes >= p.bytes), BC_ERR_WORKSPACE,
               "workspace of %zu bytes required, got %zu", p.bytes, workspace_bytes);
    BC_REQUIRE((int64_t)n_kv_heads * p.row_groups <= 65535, BC_ERR_UNSUPPORTED, "more than 65535 head and row groups");
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
    a.ws = (float*)((uint8_t*)workspace + note_bytes(batch));
    a.lens = seq_lens;
    a.tables = block_tables;
    a.width = table_width;
    a.n_pages = n_pages;
    a.page_tiles = page_size / 64;
    a.max_len = n_pages > 0 ? max_seq_len : 0;   // (without pages no length but zero is right)
    a.unit_tiles = p.unit_tiles;
    a.unit_slots = p.unit_slots;
    a.unit_most = p.units;
    a.unit_each = p.unit_each;
    // (the workspace: the sequences' units, their partials, the prefix's)
    a.units = (int2*)workspace;
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
        BC_REQUIRE(bc::launch_paged_split(mode, head_dim, p.G, a, dim3(p.groups, p.units), st), BC_ERR_UNSUPPORTED,
                   "head_dim %d", head_dim);
    const int launched = bc::check_launch("paged attention");
    if (launched != BC_OK || p.unit_tiles == 0) return launched;
    // (four waves a row while the device's wave slots hold them: 2.4 and 2.1 us less
    // over 512 and 2048 rows of 30 partials)
    const int64_t rows = (int64_t)batch * n_heads;
    const bool four = rows < 16LL * bc::device_cu_count();
    const dim3 grid((unsigned)(four ? rows : (rows + 3) / 4));
    switch (head_dim) {
#define BC_CASE(DD)                                                                                                   \
    case DD:                                                                                                          \
        if (four)                                                                                                     \
            hipLaunchKernelGGL((paged_combine_kernel<DD, 4>), grid, dim3(256), 0, st, a, (uint16_t*)out, prefix_ws, splits); \
        else                                                                                                          \
            hipLaunchKernelGGL((paged_combine_kernel<DD, 1>), grid, dim3(256), 0, st, a, (uint16_t*)out, prefix_ws, splits); \
        break;
        BC_CASE(32) BC_CASE(64) BC_CASE(96) BC_CASE(128) BC_CASE(160) BC_CASE(192) BC_CASE(224) BC_CASE(256)
#undef BC_CASE
        default: return bc::set_error(BC_ERR_UNSUPPORTED, "head_dim %d", head_dim);
    }
    return bc::check_launch("paged attention merge");
}

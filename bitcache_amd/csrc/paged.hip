// Decode attention over a paged compressed cache, a length per sequence.
//
// Simple form: a workgroup per (sequence, query head), its four waves take
// 64-key tiles in turn.  Scores: lane = key.  Values: lane = dimension, one key
// after the other.  Online softmax per wave, merged over the waves at the end.
#include <math.h>

#include "attn.h"

namespace {
using bc::kLog2e;

struct PagedArgs {
    const uint16_t* q;
    BinPlanes kb, vb;
    ResPlanes kr, vr;
    const int32_t* tables;
    const int32_t* lens;
    uint16_t* out;
    int Hq, Hkv, n_pages, page_size, width, max_len;
};

template <bool BF>
__device__ __forceinline__ float q_f(uint16_t h) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)h << 16);
    return h2f(h);
}

__device__ __forceinline__ float nibble(uint32_t w, int i) { return (float)((int)(w << (28 - 4 * i)) >> 28); }

template <int D, bool BF, bool RES>
__global__ __launch_bounds__(256) void paged_kernel(PagedArgs a) {
    constexpr int N = (D + 63) / 64;
    __shared__ float qf[D];
    __shared__ uint32_t qs[D / 32];
    __shared__ float acc_w[4][D], m_w[4], l_w[4];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int hkv = h / (a.Hq / a.Hkv);
    const int64_t row = (int64_t)b * a.Hq + h;
    const int len = a.lens[b];
    const bool bad_len = len > a.max_len || (int64_t)len > (int64_t)a.width * a.page_size;
    if (tid < D) qf[tid] = q_f<BF>(a.q[row * D + tid]);
    __syncthreads();
    if (tid < D / 32) {
        uint32_t w = 0;
        for (int i = 0; i < 32; i++) w |= (qf[32 * tid + i] >= 0.0f ? 1u : 0u) << i;
        qs[tid] = w;
    }
    float scale_q = 0.0f;
    for (int i = 0; i < D; i++) scale_q += fabsf(qf[i]);
    scale_q /= (float)D;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[N];
    for (int n = 0; n < N; n++) acc[n] = 0.0f;
    bool bad = bad_len;
    for (int t0 = wave * 64; t0 < len && !bad; t0 += 256) {
        const int page = a.tables[(int64_t)b * a.width + t0 / a.page_size];
        if (page < 0 || page >= a.n_pages) {
            bad = true;
            break;
        }
        const int64_t v0 = ((int64_t)page * a.Hkv + hkv) * a.page_size + t0 % a.page_size;
        const int n_keys = min(64, len - t0);
        float sc = -INFINITY;
        if (lane < n_keys) {
            const int64_t v = v0 + lane;
            int pc = 0;
            for (int w = 0; w < D / 32; w++) pc += __builtin_popcount(~(qs[w] ^ ((const uint32_t*)(a.kb.signs + v * (D / 8)))[w]));
            float s = scale_q * h2f(a.kb.scales[v]) * (float)(2 * pc - D);
            if constexpr (RES) {
                float r = 0.0f;
                for (int w = 0; w < D / 8; w++) {
                    const uint32_t c = ((const uint32_t*)(a.kr.codes + v * (D / 2)))[w];
                    for (int i = 0; i < 8; i++) r = fmaf(qf[8 * w + i], nibble(c, i), r);
                }
                s = fmaf(r, h2f(a.kr.scales[v]) * (1.0f / 7.0f), s);
            }
            sc = s * ((1.0f / sqrtf((float)D)) * kLog2e);
        }
        const float mn = fmaxf(m, wave_max(sc));
        const float f = m == -INFINITY ? 0.0f : exp2f(m - mn);
        const float p = lane < n_keys ? exp2f(sc - mn) : 0.0f;
        l = l * f + p;
        for (int n = 0; n < N; n++) acc[n] *= f;
        m = mn;
        for (int k = 0; k < n_keys; k++) {
            const float pk = __shfl(p, k);
            const int64_t v = v0 + k;
            const float sv = h2f(a.vb.scales[v]);
            float rv = 0.0f;
            if constexpr (RES) rv = h2f(a.vr.scales[v]) * (1.0f / 7.0f);
            for (int n = 0; n < N; n++) {
                const int e = 64 * n + lane;
                if (e >= D) continue;
                float x = (a.vb.signs[v * (D / 8) + e / 8] >> (e % 8)) & 1 ? sv : -sv;
                if constexpr (RES) x += rv * nibble(a.vr.codes[v * (D / 2) + e / 2], e & 1);
                acc[n] = fmaf(pk, x, acc[n]);
            }
        }
    }
    for (int n = 0; n < N; n++)
        if (64 * n + lane < D) acc_w[wave][64 * n + lane] = acc[n];
    const float lw = wave_sum(l);
    if (lane == 0) {
        m_w[wave] = m;
        l_w[wave] = bad ? __builtin_nanf("") : lw;
    }
    __syncthreads();
    for (int e = tid; e < D; e += 256) {
        float M = -INFINITY, L = 0.0f, x = 0.0f;
        for (int w = 0; w < 4; w++) M = fmaxf(M, m_w[w]);
        for (int w = 0; w < 4; w++) {
            if (l_w[w] != l_w[w]) L = x = l_w[w];
            if (m_w[w] == -INFINITY) continue;
            const float f = exp2f(m_w[w] - M);
            L += f * l_w[w];
            x += f * acc_w[w][e];
        }
        const float o = L == 0.0f ? 0.0f : x / L;
        if constexpr (BF) a.out[row * D + e] = __builtin_bit_cast(uint16_t, (__bf16)o);
        else a.out[row * D + e] = f2h(o);
    }
}

template <int D>
void launch(const PagedArgs& a, int batch, bool bf, bool res, hipStream_t st) {
    const dim3 grid(a.Hq, batch);
    if (bf && res) hipLaunchKernelGGL((paged_kernel<D, true, true>), grid, dim3(256), 0, st, a);
    else if (bf) hipLaunchKernelGGL((paged_kernel<D, true, false>), grid, dim3(256), 0, st, a);
    else if (res) hipLaunchKernelGGL((paged_kernel<D, false, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_kernel<D, false, false>), grid, dim3(256), 0, st, a);
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
    BC_REQUIRE(batch <= 65535, BC_ERR_UNSUPPORTED, "batch above 65535");
    return BC_OK;
}

}  // namespace

extern "C" int bc_paged_attention_workspace_size(int batch, int n_heads, int n_kv_heads, int max_seq_len,
                                                 int shared_len, int head_dim, size_t* bytes) {
    BC_REQUIRE(bytes != nullptr, BC_ERR_INVALID_ARGUMENT, "null pointer");
    const int rc = validate(batch, n_heads, n_kv_heads, max_seq_len, shared_len, head_dim);
    if (rc != BC_OK) return rc;
    *bytes = 0;
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
    BC_REQUIRE(table_width >= 0, BC_ERR_INVALID_ARGUMENT, "negative table width");
    BC_REQUIRE(shared_len % page_size == 0 && shared_len / page_size <= table_width, BC_ERR_INVALID_ARGUMENT,
               "shared_len (%d) must be whole pages of %d slots within the tables", shared_len, page_size);
    BC_REQUIRE((k_res == nullptr) == (v_res == nullptr), BC_ERR_INVALID_ARGUMENT,
               "k_res and v_res must both be given or both be null");
    if ((int64_t)batch * n_heads == 0) return BC_OK;
    BC_REQUIRE(q && out && seq_lens && (table_width == 0 || block_tables) && (n_pages == 0 || (k_bin && v_bin)),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    const int64_t cap = (int64_t)n_pages * n_kv_heads * page_size;
    PagedArgs a{};
    a.q = (const uint16_t*)q;
    a.kb = bin_planes(k_bin, cap, head_dim);
    a.vb = bin_planes(v_bin, cap, head_dim);
    if (k_res) a.kr = res_planes(k_res, cap, head_dim);
    if (v_res) a.vr = res_planes(v_res, cap, head_dim);
    a.tables = block_tables;
    a.lens = seq_lens;
    a.out = (uint16_t*)out;
    a.Hq = n_heads;
    a.Hkv = n_kv_heads;
    a.n_pages = n_pages;
    a.page_size = page_size;
    a.width = table_width;
    a.max_len = max_seq_len;
    const bool bf = dtype == BC_BF16, res = k_res != nullptr;
    hipStream_t st = (hipStream_t)stream;
    switch (head_dim) {
#define BC_CASE(DD) case DD: launch<DD>(a, batch, bf, res, st); break;
        BC_CASE(32) BC_CASE(64) BC_CASE(96) BC_CASE(128) BC_CASE(160) BC_CASE(192) BC_CASE(224) BC_CASE(256)
#undef BC_CASE
        default: return bc::set_error(BC_ERR_UNSUPPORTED, "head_dim %d", head_dim);
    }
    return bc::check_launch("paged attention");
}

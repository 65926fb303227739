// Norms of query and key heads with the position rotation, and the paged append:
// new tokens' queries, keys and values (rows of fp16 or bf16) in one launch.
//
// A row x of a head: y = x w / sqrt(mean x^2 + eps) (without weights y = x), then
// the pairs (i, i + R/2), or (2i, 2i + 1), of its first R elements turn by the
// token's position: z1 = y1 c - y2 s, z2 = y2 c + y1 s.  Queries (and keys
// without a cache) are written as rows; keys and values with a cache are
// encoded into their slots as bc_online_encode_kv encodes them.
//
// Products and sums are in 64 bits and rounded to the rows' type once.  The
// encoder has borders (the sign at zero, half steps between codes), so a value
// next to one has to come out the same wherever it is computed; a rounding of
// fp16 from 32-bit products differs in one element of some thousands.  The
// vector ALUs take 64-bit products at the rate of 32-bit ones.
//
// A wave takes eight tokens of one head at a time, eight lanes a row (the
// column encoder's layout: lane j holds elements 64k + 8j .. 64k + 8j + 7), and
// goes through several heads with the tokens' cosines and sines in registers: a
// row's factors are twice its own bytes.
#include <math.h>

#include "common.h"
#include "encode_columns.h"

namespace {
using bc::EncodeDst;
using bc::FastDiv;

// One of a call's sources: n heads of every token.
struct RotaryRows {
    const uint16_t* src;       // [T, heads, D], strides in elements
    int64_t token_stride, head_stride;
    const uint16_t* weight;    // [D], or null: no norm
    uint16_t* out;             // [T, heads, D]; null: into the cache planes
    int heads;
    int rotate;
    int wide;                  // rows start 16-byte aligned
    EncodeDst dst;
};

struct RotaryArgs {
    RotaryRows rows[3];
    const int64_t* positions;  // [T]
    const float* cos;          // [table, R / 2]
    const float* sin;
    int64_t table;
    const int64_t* slots;      // [T]
    int64_t n_slots;
    FastDiv page;              // slots per page
    double eps;
    int T, R, total_heads, heads_per_wave, kv_heads;
};

// How a lane finds the partner of an element: in its own slices (half pairs of
// whole heads, d = 128 and 256), in another slice of the row, read again (half
// pairs elsewhere), or beside it.
enum Pairing : int { PAIR_OWN = 0, PAIR_ROW = 1, PAIR_NEXT = 2 };

template <bool BF>
__device__ __forceinline__ float to_f(uint16_t h) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)h << 16);
    return h2f(h);
}
// (the empty asm: the compiler would join the roundings to 32 and to 16 bits into
// a conversion from 64, some thirty instructions that give another value for
// every 2^13th element)
template <bool BF>
__device__ __forceinline__ uint16_t from_f(float f) {
    asm volatile("" : "+v"(f));
    if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)f);
    return f2h(f);
}

// Eight elements at p as they are stored
__device__ __forceinline__ bc_v4u load_eight(const uint16_t* p, bool wide) {
    if (wide) return *(const bc_v4u*)p;
    bc_v4u r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return r;
}

template <bool BF>
__device__ __forceinline__ float element(const bc_v4u r, int e) {
    return to_f<BF>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
}

// The sum over the eight lanes of a row, in every one of them
__device__ __forceinline__ double sum_eight(double v) {
    auto move = [](double x, auto step) {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        constexpr int CTRL = decltype(step)::value;
        const uint32_t lo = dpp_u<CTRL>((uint32_t)u), hi = dpp_u<CTRL>((uint32_t)(u >> 32));
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    v += move(v, std::integral_constant<int, 0xB1>{});    // quad 1,0,3,2
    v += move(v, std::integral_constant<int, 0x4E>{});    // quad 2,3,0,1
    v += move(v, std::integral_constant<int, 0x141>{});   // half mirror
    return v;
}

// 1 / sqrt(a) to the last bits of 64: the instruction's estimate r0 and one step
// of third order, r0 + r0 e (1/2 + 3/8 e) with e = 1 - a r0^2 (error e^3)
__device__ __forceinline__ double inv_sqrt(double a) {
    const double r0 = __builtin_amdgcn_rsq(a);
    const double e = fma(-a * r0, r0, 1.0);
    return fma(r0 * e, fma(e, 0.375, 0.5), r0);
}

template <int D, bool BF, int PAIR>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    constexpr int K = (D + 63) / 64;
    constexpr int NC = PAIR == PAIR_OWN ? K / 2 : K;          // slices with factors of their own
    constexpr int NE = PAIR == PAIR_NEXT ? 4 : 8;             // ... and factors of a slice
    const int lane = threadIdx.x & 63, sub = lane >> 3, j = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * 8;
    if (first >= a.T) return;
    const bool token_live = first + sub < a.T;
    const int64_t t = token_live ? first + sub : a.T - 1;
    const int R = a.R;
    // the half slice past d (d % 64 == 32)
    auto inside = [&](int k) { return D % 64 == 0 || k < K - 1 || j < 4; };

    // the token's factors; a position outside the table turns by NaN
    float c[NC][NE], s[NC][NE];
    if (a.positions != nullptr) {
        const int64_t pos = a.positions[t];
        const bool known = pos >= 0 && pos < a.table;
        const int64_t row = (known ? pos : 0) * (R / 2);
#pragma unroll
        for (int k = 0; k < NC; k++) {
            const int e0 = 64 * k + 8 * j;
            const int i0 = PAIR == PAIR_NEXT ? e0 / 2 : (e0 < R / 2 ? e0 : e0 - R / 2);
            const bool in = e0 < R;
#pragma unroll
            for (int e = 0; e < NE; e++) {
                c[k][e] = known && in ? a.cos[row + i0 + e] : __builtin_nanf("");
                s[k][e] = known && in ? a.sin[row + i0 + e] : __builtin_nanf("");
            }
        }
    }
    // the token's slot
    bool slot_live = false;
    int64_t page = 0;
    int offset = 0;
    if (a.slots != nullptr) {
        const int64_t slot = a.slots[t];
        slot_live = token_live && slot >= 0 && slot < a.n_slots;
        const uint32_t u = slot_live ? (uint32_t)slot : 0u;
        page = bc::fast_div(u, a.page);
        offset = (int)(u - (uint32_t)page * a.page.d);
    }

    const int h_first = blockIdx.y * a.heads_per_wave;
    const int h_last = min(a.total_heads, h_first + a.heads_per_wave);
    int base = 0;
#pragma unroll 1
    for (int part = 0; part < 3; part++) {
        const RotaryRows& P = a.rows[part];
        const int h0 = max(h_first - base, 0), h1 = min(h_last - base, P.heads);
        base += P.heads;
        if (h0 >= h1) continue;
        const bool wide = P.wide != 0, norm = P.weight != nullptr;
        const uint16_t* row = P.src + t * P.token_stride;
        // the element where slice k's partners start
        auto partner = [&](int k) {
            const int e0 = 64 * k + 8 * j;
            return e0 < R / 2 ? e0 + R / 2 : e0 < R ? e0 - R / 2 : e0;
        };
        bc_v4u w[K], wp[PAIR == PAIR_ROW ? K : 1];
        if (norm) {
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int e0 = inside(k) ? 64 * k + 8 * j : 0;
                w[k] = load_eight(P.weight + e0, false);
                if constexpr (PAIR == PAIR_ROW) wp[k] = load_eight(P.weight + (inside(k) ? partner(k) : 0), false);
            }
        }
#pragma unroll 1
        for (int h = h0; h < h1; h++) {
            const uint16_t* x0 = row + (int64_t)h * P.head_stride;
            bc_v4u raw[K], rawp[PAIR == PAIR_ROW ? K : 1];
            const bc_v4u zero = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int k = 0; k < K; k++) {
                raw[k] = inside(k) ? load_eight(x0 + 64 * k + 8 * j, wide) : zero;
                if constexpr (PAIR == PAIR_ROW)
                    rawp[k] = inside(k) && P.rotate ? load_eight(x0 + partner(k), wide) : zero;
            }
            float z[K][8];
            if (P.rotate || norm) {
                double f = 1.0;
                if (norm) {
                    double sq = 0.0;
#pragma unroll
                    for (int k = 0; k < K; k++)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const double x = element<BF>(raw[k], e);
                            sq = fma(x, x, sq);
                        }
                    f = inv_sqrt(sum_eight(sq) * (1.0 / D) + a.eps);
                }
                auto value = [&](const bc_v4u r, const bc_v4u wt, int e) {
                    const double x = element<BF>(r, e);
                    return norm ? x * f * (double)element<BF>(wt, e) : x;
                };
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        // (slices past the rotated dims keep y)
                        const bool turns = P.rotate && (PAIR == PAIR_OWN || 64 * k + 8 * j < R);
                        double v;
                        if constexpr (PAIR == PAIR_OWN) {
                            if (k >= K / 2) continue;
                            const double x = value(raw[k], w[k], e), y = value(raw[k + K / 2], w[k + K / 2], e);
                            z[k + K / 2][e] = (float)(turns ? fma(y, (double)c[k][e], x * (double)s[k][e]) : y);
                            v = turns ? fma(x, (double)c[k][e], -(y * (double)s[k][e])) : x;
                        } else if constexpr (PAIR == PAIR_NEXT) {
                            if (e & 1) continue;
                            const double x = value(raw[k], w[k], e), y = value(raw[k], w[k], e + 1);
                            z[k][e + 1] = (float)(turns ? fma(y, (double)c[k][e / 2], x * (double)s[k][e / 2]) : y);
                            v = turns ? fma(x, (double)c[k][e / 2], -(y * (double)s[k][e / 2])) : x;
                        } else {
                            v = value(raw[k], w[k], e);
                            if (turns) {
                                const double y = value(rawp[k], wp[k], e) * (double)s[k][e];
                                v = fma(v, (double)c[k][e], 64 * k + 8 * j < R / 2 ? -y : y);
                            }
                        }
                        z[k][e] = (float)v;
                    }
            } else {
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) z[k][e] = element<BF>(raw[k], e);
            }
            if (P.out != nullptr) {
                uint16_t* o = P.out + (t * P.heads + h) * D;
#pragma unroll
                for (int k = 0; k < K; k++) {
                    bc_v4u r;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        r[i] = (uint32_t)from_f<BF>(z[k][2 * i]) | ((uint32_t)from_f<BF>(z[k][2 * i + 1]) << 16);
                    if (token_live && inside(k)) *(bc_v4u*)(o + 64 * k + 8 * j) = r;
                }
            } else {
                // (the rows that a cache of unfused calls would be given)
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) z[k][e] = inside(k) ? to_f<BF>(from_f<BF>(z[k][e])) : 0.0f;
                const int64_t dv = (page * a.kv_heads + h) * (int64_t)a.page.d + offset;
                bc::encode_row_columns<D, bc::ENC_FUSED_FP32>(z, j, slot_live, P.dst, dv);
            }
        }
    }
}

template <int D, bool BF>
void launch_rotary(const RotaryArgs& a, int pair, dim3 grid, hipStream_t st) {
    if constexpr (D % 128 == 0) {
        if (pair == PAIR_OWN) {
            hipLaunchKernelGGL((rotary_kernel<D, BF, PAIR_OWN>), grid, dim3(256), 0, st, a);
            return;
        }
    }
    if (pair == PAIR_NEXT)
        hipLaunchKernelGGL((rotary_kernel<D, BF, PAIR_NEXT>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((rotary_kernel<D, BF, PAIR_ROW>), grid, dim3(256), 0, st, a);
}

// The tables' side of a call: checks, and the arguments that all rows share.
int rotary_setup(RotaryArgs& a, const int64_t* positions, const float* cos, const float* sin, int64_t table_len,
                 int rot_dim, double eps, int64_t n_tokens, int head_dim) {
    BC_REQUIRE(bc::head_dim_ok(head_dim), BC_ERR_UNSUPPORTED,
               "head_dim must be a multiple of 32 in [32, 256], got %d", head_dim);
    BC_REQUIRE(n_tokens >= 0 && n_tokens <= INT32_MAX, BC_ERR_INVALID_ARGUMENT, "n_tokens must be 0 to 2^31 - 1");
    a.T = (int)n_tokens;
    a.eps = eps;
    if (positions != nullptr || cos != nullptr || sin != nullptr) {
        BC_REQUIRE(positions && cos && sin, BC_ERR_INVALID_ARGUMENT, "positions, cos and sin: all or none");
        BC_REQUIRE(rot_dim > 0 && rot_dim <= head_dim && rot_dim % 16 == 0, BC_ERR_UNSUPPORTED,
                   "rot_dim must be a multiple of 16 up to head_dim, got %d", rot_dim);
        BC_REQUIRE(table_len > 0, BC_ERR_INVALID_ARGUMENT, "table_len must be > 0");
        a.positions = positions;
        a.cos = cos;
        a.sin = sin;
        a.table = table_len;
        a.R = rot_dim;
    }
    return BC_OK;
}

RotaryRows source(const void* src, int64_t token_stride, int64_t head_stride, const void* weight, int heads,
                  bool rotate) {
    RotaryRows r{};
    r.src = (const uint16_t*)src;
    r.token_stride = token_stride;
    r.head_stride = head_stride;
    r.weight = (const uint16_t*)weight;
    r.heads = heads;
    r.rotate = rotate;
    r.wide = ((uintptr_t)src | (uint64_t)(token_stride * 2) | (uint64_t)(head_stride * 2)) % 16 == 0;
    return r;
}

EncodeDst planes_of(void* bin, void* res, int64_t cap, int d) {
    return EncodeDst{(uint8_t*)bin, (uint16_t*)((uint8_t*)bin + cap * (d / 8)), (uint8_t*)res,
                     res ? (uint16_t*)((uint8_t*)res + cap * (d / 2)) : nullptr};
}

int launch(RotaryArgs& a, int head_dim, int interleaved, int dtype, hipStream_t st) {
    a.total_heads = a.rows[0].heads + a.rows[1].heads + a.rows[2].heads;
    if (a.T == 0 || a.total_heads == 0) return BC_OK;
    const int pair = interleaved ? PAIR_NEXT : (a.R == head_dim && head_dim % 128 == 0) || a.R == 0 && head_dim % 128 == 0 ? PAIR_OWN : PAIR_ROW;
    a.heads_per_wave = a.total_heads;
    const int64_t blocks = ((int64_t)a.T + 31) / 32;
    while (a.heads_per_wave > 1 && blocks * 4 * ((a.total_heads + a.heads_per_wave - 1) / a.heads_per_wave) < 4096)
        a.heads_per_wave = (a.heads_per_wave + 1) / 2;
    const dim3 grid((unsigned)blocks, (a.total_heads + a.heads_per_wave - 1) / a.heads_per_wave);
#define BC_CASE(DD)                                                        \
    case DD:                                                               \
        if (dtype == BC_BF16) launch_rotary<DD, true>(a, pair, grid, st);  \
        else launch_rotary<DD, false>(a, pair, grid, st);                  \
        break;
    switch (head_dim) {
        BC_CASE(32) BC_CASE(64) BC_CASE(96) BC_CASE(128) BC_CASE(160) BC_CASE(192) BC_CASE(224) BC_CASE(256)
        default: return bc::set_error(BC_ERR_UNSUPPORTED, "head_dim %d unsupported", head_dim);
    }
#undef BC_CASE
    return bc::check_launch("rotary");
}

}  // namespace

extern "C" int bc_norm_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                              int64_t k_token_stride, int64_t k_head_stride, const int64_t* positions,
                              const float* cos, const float* sin, int64_t table_len, const void* q_weight,
                              const void* k_weight, double eps, void* q_out, void* k_out, int64_t n_tokens,
                              int n_heads, int n_kv_heads, int head_dim, int rot_dim, int interleaved, int dtype,
                              void* stream) {
    RotaryArgs a{};
    const int rc = rotary_setup(a, positions, cos, sin, table_len, rot_dim, eps, n_tokens, head_dim);
    if (rc != BC_OK) return rc;
    BC_REQUIRE(dtype == BC_FP16 || dtype == BC_BF16, BC_ERR_UNSUPPORTED, "dtype must be BC_FP16 or BC_BF16");
    BC_REQUIRE(n_heads >= 0 && n_kv_heads >= 0, BC_ERR_INVALID_ARGUMENT, "negative head count");
    BC_REQUIRE(n_tokens == 0 || ((n_heads == 0 || (q && q_out)) && (n_kv_heads == 0 || (k && k_out))),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    a.rows[0] = source(q, q_token_stride, q_head_stride, q_weight, n_heads, positions != nullptr);
    a.rows[1] = source(k, k_token_stride, k_head_stride, k_weight, n_kv_heads, positions != nullptr);
    a.rows[0].out = (uint16_t*)q_out;
    a.rows[1].out = (uint16_t*)k_out;
    return launch(a, head_dim, interleaved, dtype, (hipStream_t)stream);
}

extern "C" int bc_paged_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* v,
                               int64_t v_token_stride, int64_t v_head_stride, const int64_t* positions,
                               const float* cos, const float* sin, int64_t table_len, const void* q_weight,
                               const void* k_weight, double eps, void* q_out, const int64_t* slots, void* k_bin,
                               void* k_res, void* v_bin, void* v_res, int n_pages, int page_size,
                               int64_t n_tokens, int n_heads, int n_kv_heads, int head_dim, int rot_dim,
                               int interleaved, int dtype, void* stream) {
    RotaryArgs a{};
    const int rc = rotary_setup(a, positions, cos, sin, table_len, rot_dim, eps, n_tokens, head_dim);
    if (rc != BC_OK) return rc;
    BC_REQUIRE(dtype == BC_FP16 || dtype == BC_BF16, BC_ERR_UNSUPPORTED, "dtype must be BC_FP16 or BC_BF16");
    BC_REQUIRE(n_heads >= 0 && n_kv_heads >= 0, BC_ERR_INVALID_ARGUMENT, "negative head count");
    BC_REQUIRE(n_pages >= 0 && page_size > 0 && page_size % 64 == 0, BC_ERR_INVALID_ARGUMENT,
               "page_size must be a multiple of 64, got %d (n_pages %d)", page_size, n_pages);
    BC_REQUIRE((int64_t)n_pages * page_size <= INT32_MAX, BC_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    BC_REQUIRE((k_res == nullptr) == (v_res == nullptr), BC_ERR_INVALID_ARGUMENT,
               "k_res and v_res must both be given or both be null");
    BC_REQUIRE(q_weight == nullptr || n_heads > 0, BC_ERR_INVALID_ARGUMENT, "q_weight without queries");
    BC_REQUIRE(n_tokens == 0 || n_heads == 0 || (q && q_out), BC_ERR_INVALID_ARGUMENT, "null pointer");
    BC_REQUIRE(n_tokens == 0 || n_kv_heads == 0 || (k && v && slots && (n_pages == 0 || (k_bin && v_bin))),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    a.slots = slots;
    a.n_slots = (int64_t)n_pages * page_size;
    a.page = bc::make_fastdiv((uint32_t)page_size);
    a.kv_heads = n_kv_heads;
    const int64_t cap = a.n_slots * n_kv_heads;
    a.rows[0] = source(q, q_token_stride, q_head_stride, q_weight, n_heads, positions != nullptr);
    a.rows[0].out = (uint16_t*)q_out;
    a.rows[1] = source(k, k_token_stride, k_head_stride, k_weight, n_kv_heads, positions != nullptr);
    a.rows[1].dst = planes_of(k_bin, k_res, cap, head_dim);
    a.rows[2] = source(v, v_token_stride, v_head_stride, nullptr, n_kv_heads, false);
    a.rows[2].dst = planes_of(v_bin, v_res, cap, head_dim);
    return launch(a, head_dim, interleaved, dtype, (hipStream_t)stream);
}

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
// row's factors are twice its own bytes.  Bound: memory, with some 150
// instructions per row and lane beside it, so the next row's load is in flight
// under them, and nothing that they need is held in 64 bits over the rows (104
// registers in place of 212: 80 us against 92).
//
// 16384 tokens of 32 and 8 heads of 128 (bf16, 344 MB): 68 us, 5.0 TB/s, where a
// copy of as many bytes takes 65; 5001 of 64 heads of 96, a third of them turned
// (fp16, 124 MB): 29 us, 4.3 TB/s; 4 tokens 5.4 us.  With the append: 16383 tokens
// (bf16, 366 MB) 80 us, 4.6 TB/s; signs of 4096 tokens of 3 x 32 heads of 64 (fp16,
// 71 MB) 17 us, 4.2 TB/s; 32 tokens 5.4 us.  Half pairs read again (PAIR_ROW) cost
// their conversions twice: 16384 tokens of 64 heads of 96 124 us, 86 in neighbours.
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
    int stream;                // read past the caches
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
    FastDiv inner;             // workgroups are (outer, inner) of token blocks and head groups
    double eps;
    int T, R, total_heads, heads_per_wave, kv_heads;
    int heads_first;           // inner is the head group
};

// How a lane finds the partner of an element: in its own slices (half pairs of
// whole heads, d = 128 and 256); in a lane beside it (half pairs of 16, 32 or 64
// dims); in another slice of the row, read again (half pairs elsewhere); or beside
// it.  (Heads of 64, normed and turned, 268 MB in and
// out: 57 us by lanes, 64 read again.)
enum Pairing : int { PAIR_OWN = 0, PAIR_ROW = 1, PAIR_NEXT = 2, PAIR_LANE = 3 };

template <bool BF>
__device__ __forceinline__ float to_f(uint16_t h) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)h << 16);
    return h2f(h);
}
// Two rounded elements.  (The empty asm: the compiler would join the roundings to
// 32 and to 16 bits into a conversion from 64, some thirty instructions that give
// another value for every 2^13th element.)
template <bool BF>
__device__ __forceinline__ uint32_t from_two(float f0, float f1) {
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
    asm volatile("" : "+v"(f0), "+v"(f1));
    if constexpr (BF) return __builtin_bit_cast(uint32_t, b2_t{(__bf16)f0, (__bf16)f1});
    return __builtin_bit_cast(uint32_t, h2_t{(_Float16)f0, (_Float16)f1});
}

// Eight elements at p as they are stored (rows start at any element: a load of 16
// bytes needs no alignment)
__device__ __forceinline__ bc_v4u load_eight(const uint16_t* p) {
    typedef uint32_t Eight __attribute__((ext_vector_type(4), aligned(2)));
    return *(const Eight*)p;
}
// The value is there from here on, and nothing made of it before is kept
__device__ __forceinline__ void settle(bc_v4u& r) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t w = r[i];
        asm volatile("" : "+v"(w));
        r[i] = w;
    }
}

// In 64 bits, converted here: a float, and an element of stored ones.  (The compiler
// would hold a loop's constants in 64 bits, which takes the registers of half the
// waves.)
__device__ __forceinline__ double here(float f) {
    double d;
    asm volatile("v_cvt_f64_f32 %0, %1" : "=v"(d) : "v"(f));
    return d;
}
template <bool BF>
__device__ __forceinline__ double here(const bc_v4u r, int e) {
    const uint32_t w = r[e >> 1];
    float f;
    if constexpr (BF) {
        if (e & 1) asm volatile("v_and_b32 %0, 0xffff0000, %1" : "=v"(f) : "v"(w));
        else asm volatile("v_lshlrev_b32 %0, 16, %1" : "=v"(f) : "v"(w));
    } else {
        if (e & 1)
            asm volatile("v_cvt_f32_f16_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1" : "=v"(f) : "v"(w));
        else asm volatile("v_cvt_f32_f16 %0, %1" : "=v"(f) : "v"(w));
    }
    return here(f);
}

template <bool BF>
__device__ __forceinline__ float element(const bc_v4u r, int e) {
    const uint32_t w = r[e >> 1];   // (by value: a vector's element)
    if constexpr (BF) return __builtin_bit_cast(float, e & 1 ? w & 0xFFFF0000u : w << 16);
    return to_f<BF>((uint16_t)(w >> (16 * (e & 1))));
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
    constexpr int NC = PAIR == PAIR_OWN ? K / 2 : PAIR == PAIR_LANE ? 1 : K;          // slices with factors of their own
    constexpr int NE = PAIR == PAIR_NEXT ? 4 : 8;             // ... and factors of a slice
    const int lane = threadIdx.x & 63, sub = lane >> 3, j = lane & 7;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t outer = bc::fast_div(blockIdx.x, a.inner), inner = blockIdx.x - outer * a.inner.d;
    const uint32_t block = a.heads_first ? outer : inner, group = a.heads_first ? inner : outer;
    const int64_t first = ((int64_t)block * (blockDim.x >> 6) + wave) * 8;
    if (first >= a.T) return;
    const bool token_live = first + sub < a.T;
    const int64_t t = token_live ? first + sub : a.T - 1;
    const int R = a.R;
    // the half slice past d (d % 64 == 32)
    auto inside = [&](int k) { return D % 64 == 0 || k < K - 1 || j < 4; };
    // elements of slice k turn in this lane, in any lane
    auto turning = [&](int k) { return 64 * k + 8 * j < R; };
    auto any_turning = [&](int k) { return PAIR == PAIR_LANE ? k == 0 : 64 * k < R; };

    // the value in the partner's lane
    const int other = 4 * (lane ^ R >> 4);
    auto from_lane = [&](double v) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_ds_bpermute(other, (int)(uint32_t)u), hi = __builtin_amdgcn_ds_bpermute(other, (int)(u >> 32));
        return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
    };
    // the token's row of the tables
    bool known = false;
    int64_t turn = 0;
    if (a.positions != nullptr) {
        const int64_t pos = a.positions[t];
        known = pos >= 0 && pos < a.table;
        turn = (known ? pos : 0) * (R / 2);
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

    const int h_first = (int)group * a.heads_per_wave;
    const int h_last = min(a.total_heads, h_first + a.heads_per_wave);
    int base = 0;
#pragma unroll 1
    for (int part = 0; part < 3; part++) {
        const RotaryRows P = a.rows[part];
        const int h0 = max(h_first - base, 0), h1 = min(h_last - base, P.heads);
        base += P.heads;
        if (h0 >= h1) continue;
        const bool norm = P.weight != nullptr, rotate = P.rotate != 0;
        const uint16_t* row = P.src + t * P.token_stride;
        // the element where slice k's partners start
        auto partner = [&](int k) {
            const int e0 = 64 * k + 8 * j;
            return e0 < R / 2 ? e0 + R / 2 : e0 < R ? e0 - R / 2 : e0;
        };
        const bc_v4u zero = {0u, 0u, 0u, 0u};
        bc_v4u next[K], nextp[PAIR == PAIR_ROW ? K : 1];
        // (a builtin of its own where the rows are read past the caches: of two plain loads
        // the compiler would make one)
        const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(P.src + first * P.token_stride), (short)0, INT32_MAX, 0x00020000);
        const int mine = (int)(t - first) * (int)P.token_stride * 2 + 16 * j;
        const bool stream = P.stream != 0;
        auto load = [&](int h) {
            const uint16_t* const x0 = row + (int64_t)h * P.head_stride;
            if (stream) {
                const int at = h * (int)P.head_stride * 2;
#pragma unroll
                for (int k = 0; k < K; k++)
                    next[k] = __builtin_amdgcn_raw_buffer_load_b128(rows, inside(k) ? mine + 128 * k : INT32_MAX, at, 2);
            } else {
#pragma unroll
                for (int k = 0; k < K; k++) next[k] = load_eight(x0 + (inside(k) ? 64 * k + 8 * j : 0));
            }
            // (zeros for lanes that do not turn)
            if constexpr (PAIR == PAIR_ROW)
#pragma unroll
                for (int k = 0; k < K; k++) {
                    nextp[k] = zero;
                    if (rotate && any_turning(k) && turning(k)) nextp[k] = load_eight(x0 + partner(k));
                }
        };
        load(h0);
        // the weights, and the token's factors; a position outside the table turns by NaN
        const uint32_t two = BF ? 0x3F803F80u : 0x3C003C00u;   // (1, 1)
        const bc_v4u ones = {two, two, two, two};
        bc_v4u w[K], wp[PAIR == PAIR_ROW ? K : 1];
#pragma unroll
        for (int k = 0; k < K; k++) {
            w[k] = ones;
            if constexpr (PAIR == PAIR_ROW) wp[k] = ones;
            if (norm) {
                w[k] = load_eight(P.weight + (inside(k) ? 64 * k + 8 * j : 0));
                if constexpr (PAIR == PAIR_ROW) wp[k] = load_eight(P.weight + (inside(k) ? partner(k) : 0));
            }
        }
        float c[NC][NE], s[NC][NE];
        if (rotate) {
#pragma unroll
            for (int k = 0; k < NC; k++) {
                const int e0 = 64 * k + 8 * j;
                const int i0 = PAIR == PAIR_NEXT ? e0 / 2 : (e0 < R / 2 ? e0 : e0 - R / 2);
                const bool in = known && e0 < R;
                const float* const pc = a.cos + turn + (in ? i0 : 0);
                const float* const ps = a.sin + turn + (in ? i0 : 0);
#pragma unroll
                for (int e = 0; e < NE; e++) {
                    c[k][e] = pc[e];
                    s[k][e] = ps[e];
                }
#pragma unroll
                for (int e = 0; e < NE; e++) {
                    c[k][e] = in ? c[k][e] : __builtin_nanf("");
                    s[k][e] = in ? s[k][e] : __builtin_nanf("");
                    // (the first half turns against its partner, the second with it)
                    if ((PAIR == PAIR_ROW || PAIR == PAIR_LANE) && e0 < R / 2) s[k][e] = -s[k][e];
                }
            }
        }
        // one row: turned and scaled
        auto turned = [&](int h, bc_v4u (&raw)[K]) {
            bc_v4u rawp[PAIR == PAIR_ROW ? K : 1];
#pragma unroll
            for (int k = 0; k < K; k++) {
                raw[k] = inside(k) ? next[k] : zero;
                if constexpr (PAIR == PAIR_ROW) rawp[k] = nextp[k];
            }
            if (h + 1 < h1) load(h + 1);
            if (!rotate && !norm) return;
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
            // (converted again, and in small steps, for the registers)
#pragma unroll
            for (int k = 0; k < K; k++) settle(raw[k]);
            // dword i of slice k (PAIR_OWN: and of its pair): turned, only scaled, or as the lane
            // needs it
            auto step = [&](int k, int i, auto turn, auto scale) {
                constexpr bool TURN = decltype(turn)::value, SCALE = decltype(scale)::value;
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (PAIR == PAIR_OWN) {
                    float z0[2], z1[2];
#pragma unroll
                    for (int o = 0; o < 2; o++) {
                        const int e = 2 * i + o;
                        const double x = f * (double)element<BF>(raw[k], e) * here<BF>(w[k], e);
                        const double y = f * (double)element<BF>(raw[k + K / 2], e) * here<BF>(w[k + K / 2], e);
                        z0[o] = (float)x;
                        z1[o] = (float)y;
                        if constexpr (TURN) {
                            const double ct = here(c[k][e]), st = here(s[k][e]);
                            z0[o] = (float)fma(x, ct, -(y * st));
                            z1[o] = (float)fma(y, ct, x * st);
                        }
                    }
                    raw[k][i] = from_two<BF>(z0[0], z0[1]);
                    raw[k + K / 2][i] = from_two<BF>(z1[0], z1[1]);
                } else {
                    uint32_t scaled = raw[k][i];
                    const double x = f * (double)element<BF>(raw[k], 2 * i) * here<BF>(w[k], 2 * i);
                    const double y = f * (double)element<BF>(raw[k], 2 * i + 1) * here<BF>(w[k], 2 * i + 1);
                    if constexpr (SCALE) scaled = from_two<BF>((float)x, (float)y);
                    if constexpr (TURN) {
                        uint32_t turned;
                        if constexpr (PAIR == PAIR_NEXT) {
                            const double ct = here(c[k][i]), st = here(s[k][i]);
                            turned = from_two<BF>((float)fma(x, ct, -(y * st)), (float)fma(y, ct, x * st));
                        } else if constexpr (PAIR == PAIR_LANE) {
                            const double xp = from_lane(x), yp = from_lane(y);
                            turned = from_two<BF>((float)fma(x, here(c[k][2 * i]), xp * here(s[k][2 * i])),
                                                  (float)fma(y, here(c[k][2 * i + 1]), yp * here(s[k][2 * i + 1])));
                        } else {
                            const double xp = f * (double)element<BF>(rawp[k], 2 * i) * here<BF>(wp[k], 2 * i);
                            const double yp = f * (double)element<BF>(rawp[k], 2 * i + 1) * here<BF>(wp[k], 2 * i + 1);
                            turned = from_two<BF>((float)fma(x, here(c[k][2 * i]), xp * here(s[k][2 * i])),
                                                  (float)fma(y, here(c[k][2 * i + 1]), yp * here(s[k][2 * i + 1])));
                        }
                        scaled = turning(k) ? turned : scaled;
                    }
                    raw[k][i] = scaled;
                }
            };
            auto slice = [&](int k, auto turn, auto scale) {
#pragma unroll
                for (int i = 0; i < 4; i++) step(k, i, turn, scale);
            };
#pragma unroll
            for (int k = 0; k < (PAIR == PAIR_OWN ? K / 2 : K); k++) {
                if (rotate && any_turning(k)) {
                    if (PAIR == PAIR_OWN || !norm || 64 * k + 64 <= R) slice(k, std::true_type{}, std::false_type{});
                    else slice(k, std::true_type{}, std::true_type{});
                } else if (norm) {
                    slice(k, std::false_type{}, std::true_type{});
                }
                // (a slice that neither turns nor is scaled stays as it is)
            }
        };
        if (P.out != nullptr) {
            // (buffer stores, which drop tokens past the last one and the half slice past d
            // by themselves: around a branch, the wait for the next row would be one for
            // these stores too)
            const __amdgpu_buffer_rsrc_t o = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(P.out + first * P.heads * D), (short)0, (int)min((int64_t)8, a.T - first) * P.heads * (D * 2), 0x00020000);
            const int at = sub * P.heads * (D * 2) + 16 * j;
#pragma unroll 1
            for (int h = h0; h < h1; h++) {
                bc_v4u raw[K];
                turned(h, raw);
#pragma unroll
                for (int k = 0; k < K; k++)
                    __builtin_amdgcn_raw_buffer_store_b128(raw[k], o, inside(k) ? at + h * (D * 2) + 128 * k : INT32_MAX, 0, 0);
            }
        } else {
#pragma unroll 1
            for (int h = h0; h < h1; h++) {
                bc_v4u raw[K];
                turned(h, raw);
                // (the rows that a cache of unfused calls would be given)
                float z[K][8];
#pragma unroll
                for (int k = 0; k < K; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) z[k][e] = element<BF>(raw[k], e);
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
    if (pair == PAIR_LANE)
        hipLaunchKernelGGL((rotary_kernel<D, BF, PAIR_LANE>), grid, dim3(256), 0, st, a);
    else if (pair == PAIR_NEXT)
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
    return r;
}

EncodeDst planes_of(void* bin, void* res, int64_t cap, int d) {
    return EncodeDst{(uint8_t*)bin, (uint16_t*)((uint8_t*)bin + cap * (d / 8)), (uint8_t*)res,
                     res ? (uint16_t*)((uint8_t*)res + cap * (d / 2)) : nullptr};
}

int launch(RotaryArgs& a, int head_dim, int interleaved, int dtype, hipStream_t st) {
    a.total_heads = a.rows[0].heads + a.rows[1].heads + a.rows[2].heads;
    if (a.T == 0 || a.total_heads == 0) return BC_OK;
    const int pair = interleaved                                            ? PAIR_NEXT
                     : head_dim % 128 == 0 && (a.R == head_dim || a.R == 0) ? PAIR_OWN
                     : a.R == 64 || a.R == 32 || a.R == 16 || a.R == 0      ? PAIR_LANE
                                                                            : PAIR_ROW;
    // Rows that the caches cannot hold: read past them, which leaves them to the outputs,
    // and in the order of their addresses, all heads of a block of tokens beside each
    // other and few heads a wave, so that the workgroups of a moment lie close together
    // in memory: 16384 tokens of 40 heads of 128 86 us without either, 84 read past the
    // caches, 68 in order too; with the append 102 and 80.  Fewer rows, just written or
    // soon read again, are better left there (25 to 63 MB 1 to 2 us less of 14 to 30),
    // and more heads a wave then share its factors (4096 tokens of 96 heads of 64,
    // appended: 16.6 us, 20.7 in order).
    constexpr int64_t kStreamBytes = 80 << 20;
    int64_t bytes = 0;
    for (const RotaryRows& r : a.rows) bytes += (int64_t)a.T * r.heads * head_dim * 2;
    const bool stream = bytes > kStreamBytes;
    // (offsets within a wave's eight tokens are 31 bits)
    for (RotaryRows& r : a.rows) {
        const int64_t ts = r.token_stride * 2, hs = r.head_stride * 2, limit = 1 << 27;
        r.stream = stream && ((uintptr_t)r.src | (uint64_t)ts | (uint64_t)hs) % 16 == 0 && ts >= 0 && ts < limit &&
                   hs >= 0 && hs < limit && hs * r.heads < 1 << 30;
    }
    // heads of a wave: all, or as few as give every CU 24 waves (40; 32 and 48 2 us more)
    const int64_t octets = ((int64_t)a.T + 7) / 8, blocks = (octets + 3) / 4;
    const int64_t want = (int64_t)(stream ? 40 : 24) * bc::device_cu_count();
    int64_t groups = (want + octets - 1) / octets;
    if (groups > a.total_heads) groups = a.total_heads;
    a.heads_per_wave = (int)((a.total_heads + groups - 1) / groups);
    groups = (a.total_heads + a.heads_per_wave - 1) / a.heads_per_wave;
    a.heads_first = stream;
    a.inner = bc::make_fastdiv((uint32_t)(stream ? groups : blocks));
    const dim3 grid((unsigned)(blocks * groups));
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
    BC_REQUIRE(n_heads <= 65535 && n_kv_heads <= 65535, BC_ERR_UNSUPPORTED, "more than 65535 heads");
    BC_REQUIRE(((uintptr_t)q_out & 15) == 0, BC_ERR_INVALID_ARGUMENT, "q_out must be 16-byte aligned");
    BC_REQUIRE(n_tokens == 0 || ((n_heads == 0 || (q && q_out)) && (n_kv_heads == 0 || (k && k_out))),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    BC_REQUIRE(((uintptr_t)k_out & 15) == 0, BC_ERR_INVALID_ARGUMENT, "k_out must be 16-byte aligned");
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
    BC_REQUIRE(n_heads <= 65535 && n_kv_heads <= 65535, BC_ERR_UNSUPPORTED, "more than 65535 heads");
    BC_REQUIRE(((uintptr_t)q_out & 15) == 0, BC_ERR_INVALID_ARGUMENT, "q_out must be 16-byte aligned");
    BC_REQUIRE(n_pages >= 0 && page_size > 0 && page_size % 64 == 0, BC_ERR_INVALID_ARGUMENT,
               "page_size must be a multiple of 64, got %d (n_pages %d)", page_size, n_pages);
    BC_REQUIRE((int64_t)n_pages * page_size <= INT32_MAX, BC_ERR_UNSUPPORTED, "more than 2^31 - 1 slots");
    BC_REQUIRE((k_res == nullptr) == (v_res == nullptr), BC_ERR_INVALID_ARGUMENT,
               "k_res and v_res must both be given or both be null");
    BC_REQUIRE(q_weight == nullptr || n_heads > 0, BC_ERR_INVALID_ARGUMENT, "q_weight without queries");
    BC_REQUIRE(n_tokens == 0 || n_heads == 0 || (q && q_out), BC_ERR_INVALID_ARGUMENT, "null pointer");
    BC_REQUIRE(n_tokens == 0 || n_kv_heads == 0 || (k && v && slots && (n_pages == 0 || (k_bin && v_bin))),
               BC_ERR_INVALID_ARGUMENT, "null pointer");
    BC_REQUIRE((((uintptr_t)k_bin | (uintptr_t)k_res | (uintptr_t)v_bin | (uintptr_t)v_res) & 15) == 0,
               BC_ERR_INVALID_ARGUMENT, "blobs must be 16-byte aligned");
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

// Attention of a whole batch over a prefix that its sequences share, on the
// matrix cores (gfx950): each key and value of the prefix is read once for the
// M = batch * (query heads per kv head) query rows of its kv head.
//
// With many rows the products are matrix products of two compressed operands:
//   scores   S1 = sgn q . sgn k as fp4 (+-1: one 16x16x128 MFMA per 128 dims,
//            exact), S2 = q . n as fp16 (q whole, the INT4 code n + 8 as an exact
//            fp16 subnormal: its nibble masked in place, odd dims 16 times larger
//            with 1/16 in q; -8 sum q is where the accumulator starts);
//            s = (mean|q| sk S1 + rk S2 / 7) / sqrt d
//   values   out = sum a (2 bit - 1) + sum (b / 7) n, a = p sv and b = p rv rounded
//            to fp16 (2^-12 of each weight on average, of signs that differ from
//            key to key: below the rounding of the output), bits and codes as
//            above; the offsets sum a + 8 / 7 sum b come from the rounded weights by
//            the same MFMAs, so they cancel exactly.
// Keys are rows of the score products and query rows columns, so a lane holds 16
// keys of one query: its softmax needs no other lane until a maximum moves,
// its factors are one register, and its weights are the operand of the value
// product as they lie (the transposed reads give the keys of a dimension in the
// same order).
//
// A workgroup of 8 waves takes a range of the prefix and WR row blocks of 16 NC
// rows each: waves share out the row blocks, and the 8 / WR waves of a block the
// range's 64-key tiles in turn; the block's waves are merged at the end.  Waves
// run without barriers in between: a tile is read again by the waves of other
// row blocks, out of the first cache level.  Bound: the vector ALU (unpacking, about
// ten operations a score of which the exponential takes four times the others).
#pragma once

#include "attn_mfma_kernel.h"
#include "prefix_attn.h"

namespace {

using bc::PrefixArgs;

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

// (by value: a __builtin_bit_cast of a vector's element takes its first one)
__device__ __forceinline__ h2_t as_h2(uint32_t w) { return __builtin_bit_cast(h2_t, w); }
__device__ __forceinline__ uint32_t as_u(h2_t h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ h8_t as_h8(const uint32_t (&w)[4]) {
    return __builtin_bit_cast(h8_t, v4u_t{w[0], w[1], w[2], w[3]});
}

template <int D, int NC, bool RES>
struct PrefixLds {
    static constexpr int kSteps = D / 32;              // fp16 score MFMAs of 16 keys
    static constexpr int kSigns = (D + 127) / 128;     // fp4 score MFMAs of 16 keys
    static constexpr int kStage = (RES ? 32 * D : 0) + (8 * D + 1023) / 1024 * 1024;
    // per row block: operands, then (mean |q|, q's unit, accumulator start, keys) of its rows
    static constexpr int kQ16 = RES ? NC * kSteps * 1024 : 0;
    static constexpr int kQ4 = NC * kSigns * 1024;
    static constexpr int kRow = NC * 16 * 16;
    static constexpr int kBlock = kQ16 + kQ4 + kRow;
    // per wave: V staging, then the tile's scales (K's as floats, V's as fp16 pairs)
    static constexpr int kScales = 64 * (4 + 4 + 2 + 2);
    static constexpr int kWave = kStage + kScales;
    // the end: sums of 16 NC rows per wave, and (m, l)
    static constexpr int kEnd = NC * 16 * (D + 2) * 4;
    static constexpr int bytes(int wr) {
        const int loop = wr * kBlock + 8 * kWave, end = 8 * kEnd;
        return loop > end ? loop : end;
    }
};

// K operands of one tile in registers: lane l holds, of block kb, the row l % 16 =
// key 16 (r / 4) + 4 kb + r % 4, its quarter l / 16 of the codes and the sign words
template <int D, bool RES>
struct PrefixK {
    static constexpr int W = D / 32, NS = (D + 127) / 128;
    uint32_t code[RES ? 4 : 1][RES ? W : 1];
    uint32_t sign[4][NS];
    uint16_t sk, rk, sv, rv;    // of key = lane
};

template <int D, int NC, bool RES>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_attn_kernel(AttnArgs a, PrefixArgs x) {
    using L = PrefixLds<D, NC, RES>;
    constexpr int SB = D / 8, CB = D / 2, NB = D / 16, NH = D / 64, W = D / 32, NS = L::kSigns;
    constexpr int Q = D / 32;    // 16-byte pieces per code row
    constexpr bool Q_POW2 = (Q & (Q - 1)) == 0;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g4 = lane >> 4, lj = lane & 15;
    const int wr = x.row_waves, wk = 8 / wr;            // row blocks, and waves of each
    const int rb = wave % wr, kw = wave / wr;
    const int group = a.Hq / a.Hkv, rows = a.B * group;
    const int hkv = blockIdx.y % a.Hkv;
    const int block0 = (blockIdx.y / a.Hkv) * wr;       // first row block
    const int64_t cap = (int64_t)a.n_pages * a.Hkv * a.page_tiles * 64;
    uint8_t* const blk = lds + rb * L::kBlock;
    uint8_t* const mine = lds + wr * L::kBlock + wave * L::kWave;

    // the wave's tiles: where the i-th lies, in lane i (as in attn_mfma_kernel.h)
    const int first = blockIdx.x * x.tiles_per;
    const int tiles = min(x.tiles_per, x.tiles - first);
    const int n = (tiles - kw + wk - 1) / wk;           // (the host: at most 64)
    int tile_at = 0;
    bool bad_page = false;
    if (lane < n) {
        const int tile = first + kw + wk * lane;
        const int page = a.tables[tile / a.page_tiles];
        bad_page = page < 0 || page >= a.n_pages;
        tile_at = ((bad_page ? 0 : page) * a.Hkv + hkv) * a.page_tiles + tile % a.page_tiles;
    }
    const uint64_t bad_tiles = __ballot(bad_page);

    // ---------------- the rows' operands: 16 lanes per row, a 16-byte piece each
    for (int r0 = wave * 4; r0 < wr * NC * 16; r0 += 32) {
        const int r = r0 + g4, row = (block0 * NC) * 16 + r;
        const bool live = row < rows;
        const int b = live ? row / group : 0;
        const uint16_t* src = a.q + ((int64_t)b * a.Hq + hkv * group + (live ? row % group : 0)) * D;
        constexpr int N = (D + 127) / 128;   // pieces of a lane
        float v[N][8];
        float sum = 0.0f, top = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int u = lj + 16 * i;
            bc_v4u raw = {0u, 0u, 0u, 0u};
            if (live && u < D / 8) raw = *(const bc_v4u*)(src + 8 * u);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint16_t h = (uint16_t)(raw[e >> 1] >> (16 * (e & 1)));
                v[i][e] = a.bf16 ? __builtin_bit_cast(float, (uint32_t)h << 16) : h2f(h);
                sum += fabsf(v[i][e]);
                top = fmaxf(top, fabsf(v[i][e]));
            }
        }
        auto row16 = [](float t, auto op) {
            t = op(t, dpp_f<0x128>(t));
            t = op(t, dpp_f<0x124>(t));
            t = op(t, dpp_f<0x122>(t));
            return op(t, dpp_f<0x121>(t));
        };
        sum = row16(sum, [](float p, float q) { return p + q; });
        top = row16(top, [](float p, float q) { return fmaxf(p, q); });
        // q 2^e with the largest element in [2^13, 2^14): every element exact in fp16
        // down to 2^-27 of it (odd dims carry another 1/16)
        const int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
        const int e = ex > 0 && ex < 255 ? 13 - (ex - 127) : 0;
        uint8_t* const dst = lds + (r / (NC * 16)) * L::kBlock;
        const int c = r / 16 % NC, col = r % 16;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int u = lj + 16 * i;
            uint32_t byte = 0;
            float t[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                byte |= (v[i][k] >= 0.0f ? 0u : 1u) << k;
                t[k] = ldexpf(v[i][k], e);
                total += t[k];
            }
            if (u < D / 8) {
                const int g = u / W, s = u % W;
                if constexpr (RES) {
                    // slots of a step: dims 0, 4, 1, 5, 2, 6, 3, 7
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float f = k & 1 ? 0.0625f : 1.0f;
                        w[k] = (uint32_t)f2h(t[k] * f) | ((uint32_t)f2h(t[k + 4] * f) << 16);
                    }
                    *(v4u_t*)(dst + ((c * W + s) * 64 + 16 * g + col) * 16) = v4u_t{w[0], w[1], w[2], w[3]};
                }
                // sign word u / 4 of the row, byte u % 4 (expanded below)
                dst[L::kQ16 + ((c * NS + u / 16) * 64 + 16 * (u / 4 % 4) + col) * 16 + u % 4] = (uint8_t)byte;
            }
        }
        total = row16(total, [](float p, float q) { return p + q; });
        if (lj == 0) {
            constexpr float isd2 = kLog2e;
            const int len = live ? a.lens[b] : 0;
            float* const rc = (float*)(dst + L::kQ16 + L::kQ4 + (c * 16 + col) * 16);
            rc[0] = sum * (1.0f / (float)D) * (isd2 / sqrtf((float)D));
            rc[1] = ldexpf(isd2 / sqrtf((float)D) * (1.0f / 7.0f), 24 - e);
            rc[2] = ldexpf(-8.0f * total, -24);
            // (padding rows and rows of a bad length, whose sums nobody reads, mask nothing)
            ((int*)rc)[3] = !live || bc::paged_bad_len(a, len) ? x.tiles * 64 : len;
        }
    }
    __syncthreads();
    // a sign word as fp4: +1.0 = 0x2, -1.0 = 0xA; register p holds dims 4 i + p
    auto fp4 = [](uint32_t w, int p) { return ((w << (3 - p)) & 0x88888888u) | 0x22222222u; };
    for (int i = threadIdx.x; i < wr * NC * NS * 64; i += 512) {
        const int j = i % (NC * NS * 64);
        uint8_t* const at = lds + i / (NC * NS * 64) * L::kBlock + L::kQ16 + j * 16;
        const int word = 4 * (j / 64 % NS) + j % 64 / 16;
        const uint32_t w = *(const uint32_t*)at;
        v4u_t o = {fp4(w, 0), fp4(w, 1), fp4(w, 2), fp4(w, 3)};
        if (word >= D / 32) o = v4u_t{0u, 0u, 0u, 0u};   // (past the dims: 0 times anything)
        *(v4u_t*)at = o;
    }
    __syncthreads();

    float rho1[NC], rho2[NC], start[NC];
    int limit[NC], least = 0x7FFFFFFF;   // keys of the lane's rows, of the wave's shortest
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const float* rc = (const float*)(blk + L::kQ16 + L::kQ4 + (c * 16 + lj) * 16);
        rho1[c] = rc[0];
        rho2[c] = rc[1];
        start[c] = rc[2];
        limit[c] = ((const int*)rc)[3];
        least = min(least, limit[c]);
    }
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) least = min(least, __shfl_xor(least, k));
    least = __builtin_amdgcn_readfirstlane(least);

    f4_t cs[NH][4][NC];                  // sign part: rows = dims 64 h + 4 m + p
    f4_t cn[RES ? NB : 1][NC];           // residual part: rows = dims 16 db + m
    f4_t co[NC];                         // row 0 of 4: sum p, row 1: 7 sum a + 8 sum b
#pragma unroll
    for (int c = 0; c < NC; c++) {
        co[c] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int p = 0; p < 4; p++) cs[h][p][c] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < (RES ? NB : 1); d++) cn[d][c] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    // constant operands of the sums: (1 1 ..) in the rows = 0 mod 4, 7 and 8 (times 16
    // for odd keys, whose weights carry 1/16) in the rows = 1 mod 4
    auto rows_of = [&](int r, float even, float odd) {
        const uint32_t on = (lane & 3) == r ? 0xFFFFFFFFu : 0u;
        const uint32_t e = (uint32_t)f2h(even) * 0x10001u & on, o = (uint32_t)f2h(odd) * 0x10001u & on;
        return __builtin_bit_cast(h8_t, v4u_t{e, o, e, o});
    };
    const h8_t one_op = rows_of(0, 1.0f, 1.0f), a_op = rows_of(1, 7.0f, 112.0f), b_op = rows_of(1, 8.0f, 128.0f);

    // the softmax reference per row, lowered lazily: weights stay <= 2^kTau
    constexpr float kTau = 8.0f;
    constexpr float kNone = -1e30f;
    float m[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) m[c] = kNone;
    // V scales enter as fp16 times 2^we, the largest in [2^5, 2^6): a weight stays
    // below 2^14 and keeps its bits down to 2^-28 of the largest
    int we = 0;
    bool have_we = false;
    float wlim = 0.0f;

    auto rsrc = [&](const uint8_t* plane, int rb_, int i) {
        const int64_t v = (int64_t)(uint32_t)__builtin_amdgcn_readlane(tile_at, i & 63) * 64;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(plane + v * rb_), (short)0, i < n ? 64 * rb_ : 0, kBufWord3);
    };
    PrefixK<D, RES> k;
    auto load_k = [&](int i) {
        const int row = 16 * (lj >> 2) + (lj & 3);
        const __amdgpu_buffer_rsrc_t r_s = rsrc(a.kb.signs, SB, i);
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const int w = min(4 * s + g4, D / 32 - 1);
                k.sign[kb][s] = __builtin_amdgcn_raw_buffer_load_b32(r_s, (row + 4 * kb) * SB + 4 * w, 0, 0);
            }
        const __amdgpu_buffer_rsrc_t r_ks = rsrc(a.kb.signs + cap * SB, 2, i), r_vs = rsrc(a.vb.signs + cap * SB, 2, i);
        k.sk = __builtin_amdgcn_raw_buffer_load_b16(r_ks, lane * 2, 0, 0);
        k.sv = __builtin_amdgcn_raw_buffer_load_b16(r_vs, lane * 2, 0, 0);
        if constexpr (RES) {
            const __amdgpu_buffer_rsrc_t r_c = rsrc(a.kr.codes, CB, i);
#pragma unroll
            for (int kb = 0; kb < 4; kb++) {
                const int at = (row + 4 * kb) * CB + g4 * (CB / 4);
#pragma unroll
                for (int w = 0; w + 4 <= W; w += 4) {
                    const v4u_t t = __builtin_amdgcn_raw_buffer_load_b128(r_c, at + 4 * w, 0, 0);
                    k.code[kb][w] = t[0]; k.code[kb][w + 1] = t[1]; k.code[kb][w + 2] = t[2]; k.code[kb][w + 3] = t[3];
                }
                if constexpr (W % 4 == 2) {
                    const v2u_t t = __builtin_amdgcn_raw_buffer_load_b64(r_c, at + 4 * (W - 2), 0, 0);
                    k.code[kb][W - 2] = t[0]; k.code[kb][W - 1] = t[1];
                }
            }
            const __amdgpu_buffer_rsrc_t r_kr = rsrc(a.kr.codes + cap * CB, 2, i), r_vr = rsrc(a.vr.codes + cap * CB, 2, i);
            k.rk = __builtin_amdgcn_raw_buffer_load_b16(r_kr, lane * 2, 0, 0);
            k.rv = __builtin_amdgcn_raw_buffer_load_b16(r_vr, lane * 2, 0, 0);
        } else {
            k.rk = k.rv = 0;
        }
    };
    // V tile to LDS: codes in linear rows with their pieces swizzled, then signs
    auto load_v = [&](int i) {
        uint8_t* const signs = mine + (RES ? 32 * D : 0);
        const __amdgpu_buffer_rsrc_t r_s = rsrc(a.vb.signs, SB, i);
#pragma unroll
        for (int c = 0; c < SB / 16; c++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_s, LDS_PTR(void, signs + c * 1024), 16, 16 * lane + c * 1024, 0, 0, 0);
        if constexpr (SB % 16 != 0)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_s, LDS_PTR(void, signs + SB / 16 * 1024), 16,
                                                     16 * (lane & 31) + SB / 16 * 1024, 0, 0, 0);
        if constexpr (RES) {
            const __amdgpu_buffer_rsrc_t r_c = rsrc(a.vr.codes, CB, i);
#pragma unroll
            for (int c = 0; c < Q; c++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    r_c, LDS_PTR(void, mine + c * 1024), 16,
                    c * 1024 + 16 * (Q_POW2 ? lane ^ ((4 * c + (lane >> 4)) & (Q - 1)) : lane), 0, 0, 0);
        }
    };
    const int vsw = Q_POW2 ? ((lane * CB) >> 8) & (Q - 1) : 0;
    float* const s_k = (float*)(mine + L::kStage);          // [64] sk, [64] rk
    uint16_t* const s_v = (uint16_t*)(s_k + 128);           // [64] sv, [64] rv in weight pairs

    load_k(0);
    load_v(0);
    for (int i = 0; i < n; i++) {
        // ---------------- scales of the tile, by key
        {
            float sk = h2f(k.sk);
            const float sv = h2f(k.sv), rv = h2f(k.rv);
            if (bad_tiles >> i & 1) sk = __builtin_nanf("");
            // (a scale that is not finite takes no part in the plan)
            const float wa = fabsf(sv), wr_ = fabsf(rv);
            const float wb = fmaxf(wa < INFINITY ? wa : 0.0f, wr_ < INFINITY ? wr_ : 0.0f);
            if (__ballot(wb >= wlim && wb > 0.0f) != 0ull) {
                const float mx = wave_max(wb);
                // (subnormal fp16 scales included: their floats are normal)
                const int e = 5 - ((int)(__builtin_bit_cast(uint32_t, mx) >> 23) - 127);
                if (have_we) {
                    const float f = ldexpf(1.0f, e - we);
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        co[c][1] *= f;
#pragma unroll
                        for (int h = 0; h < NH; h++)
#pragma unroll
                            for (int p = 0; p < 4; p++) cs[h][p][c] *= f;
#pragma unroll
                        for (int d = 0; d < (RES ? NB : 1); d++) cn[d][c] *= f;
                    }
                }
                we = e;
                have_we = true;
                wlim = ldexpf(1.0f, 6 - e);
            }
            s_k[lane] = sk;
            if constexpr (RES) s_k[64 + lane] = h2f(k.rk);
            // weight pairs of a run of 8 keys: (0, 4), (1, 5), (2, 6), (3, 7); odd keys 1/16
            const int at = (lane & ~7) + 2 * (lane & 3) + (lane >> 2 & 1);
            const float unit = ldexpf(lane & 1 ? 0.0625f : 1.0f, we);
            s_v[at] = f2h(sv * unit);
            if constexpr (RES) s_v[64 + at] = f2h(rv * unit);
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");

        // ---------------- scores and weights, 32 keys (8 a lane) at a time
        const int t0 = (first + kw + wk * i) * 64;
        const bool whole = t0 + 64 <= least;
        uint32_t wa[NC][2][4], wb[RES ? NC : 1][2][4];
#pragma unroll
        for (int mh = 0; mh < 2; mh++) {
            f4_t s1[2][NC], s2[2][NC];
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                const int kb = 2 * mh + kk;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    s1[kk][c] = f4_t{0.f, 0.f, 0.f, 0.f};
                    s2[kk][c] = f4_t{start[c], start[c], start[c], start[c]};
                }
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const uint32_t w = ~k.sign[kb][s];
                    const v8i_t av = {(int)fp4(w, 0), (int)fp4(w, 1), (int)fp4(w, 2), (int)fp4(w, 3), 0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        const v4i_t b4 = *(const v4i_t*)(blk + L::kQ16 + ((c * NS + s) * 64 + lane) * 16);
                        const v8i_t bv = {b4[0], b4[1], b4[2], b4[3], 0, 0, 0, 0};
                        s1[kk][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, s1[kk][c], 4, 4, 0, 0x7F7F7F7F,
                                                                                     0, 0x7F7F7F7F);
                    }
                }
                if constexpr (RES) {
#pragma unroll
                    for (int s = 0; s < W; s++) {
                        const uint32_t w = k.code[kb][s] ^ 0x88888888u, y = w >> 8;
                        const h8_t av = __builtin_bit_cast(h8_t, v4u_t{w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu,
                                                                       y & 0x00F000F0u});
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            const h8_t bv = *(const h8_t*)(blk + ((c * W + s) * 64 + lane) * 16);
                            s2[kk][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, bv, s2[kk][c], 0, 0, 0);
                        }
                    }
                }
            }
            // the lane's 8 keys: 16 g4 + 8 mh + 4 kk + j
            f4_t fk[2], fr[2];
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
                fk[kk] = *(const f4_t*)&s_k[16 * g4 + 8 * mh + 4 * kk];
                if constexpr (RES) fr[kk] = *(const f4_t*)&s_k[64 + 16 * g4 + 8 * mh + 4 * kk];
            }
            const v4u_t pa = *(const v4u_t*)&s_v[16 * g4 + 8 * mh];
            v4u_t pb = {0u, 0u, 0u, 0u};
            if constexpr (RES) pb = *(const v4u_t*)&s_v[64 + 16 * g4 + 8 * mh];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                float z[2][4], top = -INFINITY;
#pragma unroll
                for (int kk = 0; kk < 2; kk++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float t = -m[c];
                        if constexpr (RES) t = fmaf(s2[kk][c][j] * fr[kk][j], rho2[c], t);
                        z[kk][j] = fmaf(s1[kk][c][j] * fk[kk][j], rho1[c], t);
                        if (!whole && t0 + 16 * g4 + 8 * mh + 4 * kk + j >= limit[c]) z[kk][j] = -INFINITY;
                        top = fmaxf(top, z[kk][j]);
                    }
                if (__ballot(top > kTau) != 0ull) {
                    // a row's largest score over its four lanes
                    float t = fmaxf(top, __shfl_xor(top, 16));
                    t = fmaxf(t, __shfl_xor(t, 32));
                    const bool moves = t > kTau;
                    // (the new reference from the scores themselves: next to kNone they
                    // have no bits left)
                    float raw[2][4], hi = -INFINITY;
#pragma unroll
                    for (int kk = 0; kk < 2; kk++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            float v = 0.0f;
                            if constexpr (RES) v = (s2[kk][c][j] * fr[kk][j]) * rho2[c];
                            raw[kk][j] = fmaf(s1[kk][c][j] * fk[kk][j], rho1[c], v);
                            if (!whole && t0 + 16 * g4 + 8 * mh + 4 * kk + j >= limit[c]) raw[kk][j] = -INFINITY;
                            hi = fmaxf(hi, raw[kk][j]);
                        }
                    hi = fmaxf(hi, __shfl_xor(hi, 16));
                    hi = fmaxf(hi, __shfl_xor(hi, 32));
                    const float mn = moves ? hi : m[c];
                    const float alpha = __builtin_amdgcn_exp2f(m[c] - mn);
                    m[c] = mn;
                    co[c] *= alpha;
#pragma unroll
                    for (int h = 0; h < NH; h++)
#pragma unroll
                        for (int p = 0; p < 4; p++) cs[h][p][c] *= alpha;
#pragma unroll
                    for (int d = 0; d < (RES ? NB : 1); d++) cn[d][c] *= alpha;
                    if (mh == 1) {
                        // the weights of the first half, formed from the old reference
                        const h2_t f = {(_Float16)alpha, (_Float16)alpha};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            wa[c][0][j] = as_u(as_h2(wa[c][0][j]) * f);
                            if constexpr (RES) wb[c][0][j] = as_u(as_h2(wb[c][0][j]) * f);
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < 2; kk++)
#pragma unroll
                        for (int j = 0; j < 4; j++) z[kk][j] = raw[kk][j] - mn;
                }
                uint32_t p[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float lo = __builtin_amdgcn_exp2f(z[0][j]), hi = __builtin_amdgcn_exp2f(z[1][j]);
                    p[j] = as_u(h2_t{(_Float16)lo, (_Float16)hi});
                    wa[c][mh][j] = as_u(as_h2(p[j]) * as_h2(pa[j]));
                    if constexpr (RES) wb[c][mh][j] = as_u(as_h2(p[j]) * as_h2(pb[j]));
                }
                if (!whole) {
                    // (a masked key adds nothing whatever its scales are)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = t0 + 16 * g4 + 8 * mh + j;
                        const uint32_t in = (key < limit[c] ? 0xFFFFu : 0u) | (key + 4 < limit[c] ? 0xFFFF0000u : 0u);
                        wa[c][mh][j] &= in;
                        if constexpr (RES) wb[c][mh][j] &= in;
                    }
                }
                co[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one_op, as_h8(p), co[c], 0, 0, 0);
            }
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int mh = 0; mh < 2; mh++) {
                co[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a_op, as_h8(wa[c][mh]), co[c], 0, 0, 0);
                if constexpr (RES) co[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b_op, as_h8(wb[c][mh]), co[c], 0, 0, 0);
            }

        // ---------------- the tile's V data is in LDS; the next tile's K loads fly
        // during the value products, its V loads during the next scores
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0);
        __builtin_amdgcn_wave_barrier();
        load_k(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t* const signs = mine + (RES ? 32 * D : 0);
        const int row_key = 16 * g4 + lj;
        v2i_t wsg[NH], wrs[RES ? NB : 1];
#pragma unroll
        for (int h = 0; h < NH; h++)
            wsg[h] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(LDS_PTR(v2i_t, signs + SB * row_key + 8 * h));
        if constexpr (RES) {
#pragma unroll
            for (int db = 0; db < NB; db++)
                wrs[db] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                    LDS_PTR(v2i_t, mine + CB * row_key + 16 * ((db >> 1) ^ vsw) + 8 * (db & 1)));
        }
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int mh = 0; mh < 2; mh++) {
                const uint32_t w = (uint32_t)(mh ? wsg[h].y : wsg[h].x), y = w >> 8;
#pragma unroll
                for (int p = 0; p < 4; p++) {
                    const h8_t av = __builtin_bit_cast(h8_t, v4u_t{w & (0x00010001u << p), w & (0x00100010u << p),
                                                                   y & (0x00010001u << p), y & (0x00100010u << p)});
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        cs[h][p][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, as_h8(wa[c][mh]), cs[h][p][c], 0, 0, 0);
                }
            }
        if constexpr (RES) {
#pragma unroll
            for (int db = 0; db < NB; db++)
#pragma unroll
                for (int mh = 0; mh < 2; mh++) {
                    const uint32_t w = (uint32_t)(mh ? wrs[db].y : wrs[db].x) ^ 0x88888888u, y = w >> 8;
                    const h8_t av = __builtin_bit_cast(h8_t, v4u_t{w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu,
                                                                   y & 0x00F000F0u});
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        cn[db][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, as_h8(wb[c][mh]), cn[db][c], 0, 0, 0);
                }
        }
        // the staging buffer's reads retire before it is refilled
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
        load_v(i + 1);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();

    // ---------------- the end: every wave's rows in LDS ([row][D] then m, l), the
    // waves of a row block merged, one partial per row and split
    constexpr int RS = D + 2;
    float* const end = (float*)lds + wave * (NC * 16 * RS);
    const float unit = ldexpf(1.0f, have_we ? -we : 0);
#pragma unroll
    for (int c = 0; c < NC; c++) {
        float* const o = end + (c * 16 + lj) * RS;
        // (row 1 of every lane group's rows holds the offset, row 0 the sum)
        const float off = co[c][1] * (1.0f / 7.0f);
#pragma unroll
        for (int h = 0; h < NH; h++)
#pragma unroll
            for (int p = 0; p < 4; p++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[64 * h + 4 * (4 * g4 + j) + p] = (cs[h][p][c][j] * (33554432.0f / (float)(1 << p)) - off) * unit;
        if (g4 == 0) {
            o[D] = m[c];
            o[D + 1] = co[c][0];
        }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if constexpr (RES) {
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int db = 0; db < NB; db++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float* const o = end + (c * 16 + lj) * RS + 16 * db + 4 * g4 + j;
                    *o += cn[db][c][j] * (16777216.0f / 7.0f) * unit;
                }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < wr * NC * 16 * D; i += 512) {
        const int r = i / D, e = i % D, row = block0 * NC * 16 + r;
        if (row >= rows) break;
        const float* p = (const float*)lds + (r / (NC * 16)) * (NC * 16 * RS) + r % (NC * 16) * RS;
        float M = kNone, Ls = 0.0f, acc = 0.0f;
        for (int w = 0; w < wk; w++) M = fmaxf(M, p[w * wr * (NC * 16 * RS) + D]);
        for (int w = 0; w < wk; w++) {
            const float* t = p + w * wr * (NC * 16 * RS);
            const float f = __builtin_amdgcn_exp2f(t[D] - M);
            // (a wave without keys of the row has sums of zero)
            Ls += t[D + 1] * f;
            acc += t[e] * f;
        }
        const int b = row / group, h = hkv * group + row % group;
        float* dst = x.ws + (((int64_t)blockIdx.x * a.B + b) * a.Hq + h) * RS;
        dst[2 + e] = acc;
        if (e == 0) {
            dst[0] = M;
            dst[1] = Ls;
        }
    }
}

}  // namespace

namespace bc {

template <int D, int NC, bool RES>
static int prefix_go(const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st) {
    const int bytes = PrefixLds<D, NC, RES>::bytes(x.row_waves);
    const hipError_t e = hipFuncSetAttribute((const void*)prefix_attn_kernel<D, NC, RES>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return set_error(BC_ERR_HIP, "prefix attention: %s", hipGetErrorString(e));
    hipLaunchKernelGGL((prefix_attn_kernel<D, NC, RES>), grid, dim3(512), bytes, st, a, x);
    return check_launch("prefix attention");
}

template <int D>
int prefix_launch(bool res, int nc, const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st) {
    if constexpr (D <= 128) {
        if (nc == 2) return res ? prefix_go<D, 2, true>(a, x, grid, st) : prefix_go<D, 2, false>(a, x, grid, st);
    }
    return res ? prefix_go<D, 1, true>(a, x, grid, st) : prefix_go<D, 1, false>(a, x, grid, st);
}

}  // namespace bc

// One vector of the column encoder: eight lanes per vector, any head dim.  The
// row encoders (encode.hip) and the paged append (rotary.hip) run it.
#pragma once

#include "common.h"
#include "encode_row.h"

namespace bc {

// Unsigned 32-bit division by an invariant divisor 1 <= d <= 2^31 (the
// round-up method of Granlund and Montgomery, "Division by invariant integers
// using multiplication", 1994): with l = ceil(log2 d) and
// m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(m, n) + n) >> l for every
// 32-bit n (the sum taken in 64 bits).
struct FastDiv {
    uint32_t d, m;
    int l;
};

inline FastDiv make_fastdiv(uint32_t d) {
    FastDiv f{d, 0u, 0};
    while ((1ull << f.l) < d) f.l++;
    f.m = (uint32_t)(((1ull << 32) * ((1ull << f.l) - d)) / d + 1ull);
    return f;
}

__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) {
    return (uint32_t)(((uint64_t)__umulhi(n, f.m) + n) >> f.l);
}

// Eight codes of finite y (|y| < 7.5) as a dword: y + 12582920 rounded to an
// integer (1.5 * 2^23 + 8, even: ties as in rint) has rint(y) + 8 in its low
// byte; xor 0x8 per nibble turns the offset code into two's complement.
__device__ __forceinline__ uint32_t pack_codes(const float* y) {
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; k++) c[k] = __builtin_bit_cast(uint32_t, y[k] + 12582920.0f);
    const uint32_t p0 = (c[1] << 4) | c[0], p1 = (c[3] << 4) | c[2];
    const uint32_t p2 = (c[5] << 4) | c[4], p3 = (c[7] << 4) | c[6];
    const uint32_t t0 = __builtin_amdgcn_perm(p1, p0, 0x0C0C0400u);   // p0.b0, p1.b0
    const uint32_t t1 = __builtin_amdgcn_perm(p3, p2, 0x0C0C0400u);   // p2.b0, p3.b0
    return __builtin_amdgcn_perm(t1, t0, 0x05040100u) ^ 0x88888888u;
}

// Eight lanes per vector, lane j holding elements 64k + 8j .. 64k + 8j + 7 of every
// 64-element block k as floats (x is overwritten; the last block of d % 64 == 32
// is half: lanes 4..7 hold zeros there, whose terms are exact +0.0).  The
// reference's thread t sums |x_t| + |x_{t+128}|, its s = 64 step pairs t with
// t + 64: in-lane adds over the blocks; s = 32, 16, 8 pair lane j with j + 4, 2, 1
// and s = 4, 2, 1 are in-lane: the reference tree's association exactly.  One
// wave per vector (the kernel that ran the head dims other than 64, 128 and 256,
// shuffles and 2-byte loads) took 4.7 times as long: 524288 vectors of d = 96
// 139.7 -> 42.1 us (3.2 TB/s).
template <int D, int MODE>
__device__ __forceinline__ void encode_row_columns(float (&x)[(D + 63) / 64][8], int j, bool live,
                                                   const EncodeDst& dst, int64_t dv) {
    constexpr int K = (D + 63) / 64;
    constexpr bool HALF = D % 64 != 0;
    bool pos[K][8];   // x >= 0: +-0 -> 1, NaN -> 0 (src/binary_encode.cu:36)
    uint32_t bytes[K];
    // (a lane past the last block's elements)
    const bool pad = HALF && j >= 4;
    float s;
    if constexpr (MODE == ENC_RESIDUAL_ONLY) {
        const uint8_t* sp = dst.sign_plane + dv * (D / 8);
#pragma unroll
        for (int k = 0; k < K; k++) {
            bytes[k] = (k == K - 1 && pad) ? 0u : sp[8 * k + j];
#pragma unroll
            for (int e = 0; e < 8; e++) pos[k][e] = (bytes[k] >> e) & 1u;
        }
        s = h2f(dst.scale_plane[dv]);
    } else {
#pragma unroll
        for (int k = 0; k < K; k++) {
            bytes[k] = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                pos[k][e] = x[k][e] >= 0.0f;
                bytes[k] |= (pos[k][e] ? 1u : 0u) << e;
            }
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float pa = fabsf(x[0][e]), pb = 0.0f;
            if constexpr (K > 2) pa = pa + fabsf(x[2][e]);
            if constexpr (K > 1) pb = fabsf(x[1][e]);
            if constexpr (K > 3) pb = pb + fabsf(x[3][e]);
            p[e] = pa + pb;                                                  // s = 64
        }
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = p[e] + dpp_f<0x104>(p[e]);       // s = 32
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = p[e] + dpp_f<0x102>(p[e]);       // s = 16
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = p[e] + dpp_f<0x101>(p[e]);       // s = 8
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = p[e] + p[e + 4];                  // s = 4
        p[0] = p[0] + p[2];
        p[1] = p[1] + p[3];                                                   // s = 2
        p[0] = p[0] + p[1];                                                   // s = 1
        const float mean = swz_f<0x18>(p[0]) / (float)D;   // (lane 0 of the eight)
        if constexpr (MODE == ENC_FUSED_FP16) s = h2f(f2h(mean));
        else s = mean;
        // sign bytes of four lanes -> one dword
#pragma unroll
        for (int k = 0; k < K; k++) {
            const uint32_t w = bytes[k] | (dpp_u<0x101>(bytes[k]) << 8) | (dpp_u<0x102>(bytes[k]) << 16) |
                               (dpp_u<0x103>(bytes[k]) << 24);
            if (live && (j & 3) == 0 && !(k == K - 1 && pad))
                *(uint32_t*)(dst.sign_plane + dv * (D / 8) + 8 * k + j) = w;
        }
        if (live && j == 0) dst.scale_plane[dv] = f2h(mean);
    }
    if constexpr (MODE != ENC_BINARY) {
        if (dst.code_plane == nullptr) return;
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[k][e] = x[k][e] - (pos[k][e] ? s : -s);   // the residual
                // fmaxf ignores NaN and is order independent (src/residual.cu:30-53)
                if (!(k == K - 1 && pad)) m = fmaxf(m, fabsf(x[k][e]));
            }
        // (non-negative and never NaN: the integer order is the float order)
        uint32_t mb = __builtin_bit_cast(uint32_t, m);
        mb = max(mb, dpp_u<0x141>(mb));   // half mirror
        mb = max(mb, dpp_u<0x4E>(mb));
        mb = max(mb, dpp_u<0xB1>(mb));
        const float absmax = __builtin_bit_cast(float, mb);
        const float inv = absmax > 0.0f ? 7.0f / absmax : 0.0f;
        // (as in encode_two_slices: the mean is finite only if each element is;
        // against a stored scale, 0 * residual summed is 0 only then)
        float probe = s;
        if constexpr (MODE == ENC_RESIDUAL_ONLY) {
            probe = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++)
#pragma unroll
                for (int e = 0; e < 8; e++) probe = fmaf(x[k][e], 0.0f, probe);
        }
        const bool exact = __ballot(!__builtin_isfinite(probe) || !__builtin_isfinite(inv)) != 0ull;
#pragma unroll
        for (int k = 0; k < K; k++) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = x[k][e] * inv;
            uint32_t word = 0;
            if (!exact) {
                word = pack_codes(y);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) word |= ((uint32_t)quant7(y[e]) & 0xFu) << (4 * e);
            }
            if (live && !(k == K - 1 && pad)) ((uint32_t*)(dst.code_plane + dv * (D / 2)))[8 * k + j] = word;
        }
        if (live && j == 0) dst.rscale_plane[dv] = f2h(absmax);
    }
}

}  // namespace bc

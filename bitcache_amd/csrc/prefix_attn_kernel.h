// Attention of a whole batch over a prefix that its sequences share, on the
// matrix cores (gfx950): each key and value of the prefix is read and unpacked
// once for up to 64 of the M = batch * (query heads per kv head) query rows of
// its kv head.
//
// With many rows the products are matrix products of two compressed operands:
//   scores   S1 = sgn q . sgn k as fp4 (+-1: one 16x16x128 MFMA per 128 dims,
//            exact), S2 = q . n as fp16 (q whole, the INT4 code n + 8 as an exact
//            fp16 subnormal: its nibble masked in place, odd dims 16 times larger
//            with 1/16 in q; -8 sum q is where the accumulator starts);
//            s = (mean|q| sk S1 + rk S2 / 7) / sqrt d
//   values   out = sum a (+-1) + sum (b / 7) n, a = p sv and b = p rv rounded to
//            fp16 once (errors of signs that differ from key to key: 1.7e-4 of the
//            output, its own rounding to fp16 is 2.1e-4), signs and codes as exact
//            fp16 values.  (Bits and codes + 8 with the offsets taken off at the end
//            take an operation less per pair, but the sums then carry what cancels,
//            up to 200 times the output, and the matrix cores drop its last bits:
//            3.6e-4 of the output in all, so 2.7e-4.)
//
// A workgroup of four waves takes 16 NC rows and a range of the prefix, a
// 64-key tile at a time.  Scores: each wave takes 16 of the tile's keys against
// all rows (keys are the rows of the products and query rows their columns, so
// a lane's four scores are of one query row), and leaves the weights in LDS as
// the value product's operands.  Values, after the tile's one barrier: two waves
// take the sign part and two the residual part, half of the dims each, of all
// rows.  No operand is unpacked twice in a workgroup.  Bound: the vector ALU
// (eleven operations a score, of which the exponential counts as four, against
// 2 D / 1024 cycles of matrix core a score and wave).  2048 query rows over 32768
// keys (64 sequences, 32/8 heads of 128): 105 us, 69 GFLOP; 142 with 16 rows of its
// own and all 64 keys for each wave, which unpacks every operand four times.
//
// The softmax reference of a row is shared by the four waves and moves rarely:
// weights stay below 2^kTau; a tile that would pass it (and one with a V scale
// larger than the weights' unit holds) is formed again after the reference
// moved.  The next tile's loads fly during the value products; V tiles go to LDS
// directly, in two buffers.
#pragma once

#include "attn_mfma_kernel.h"
#include "prefix_attn.h"

namespace {

using bc::PrefixArgs;

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t as_u(h2_t h) { return __builtin_bit_cast(uint32_t, h); }

// a 32-element sign word (set: negative) as fp4, +1.0 = 0x2 and -1.0 = 0xA:
// register p holds elements 4 i + p
__device__ __forceinline__ uint32_t fp4_signs(uint32_t w, int p) { return ((w << (3 - p)) & 0x88888888u) | 0x22222222u; }

template <int D, int NC, bool RES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(bc::prefix_waves(D, NC, RES), bc::prefix_waves(D, NC, RES))))
void prefix_attn_kernel(AttnArgs a, PrefixArgs x) {
    constexpr int SB = D / 8, CB = D / 2, NB = D / 16, W = D / 32, NS = (D + 127) / 128;
    constexpr int Q = D / 32;    // 16-byte pieces per code row
    constexpr bool Q_POW2 = (Q & (Q - 1)) == 0;
    constexpr int R = 16 * NC;   // rows
    // 16-dim blocks of a wave's value products: waves 0, 1 (binary: all) the sign
    // part, waves 2, 3 the residual part
    constexpr int NBW = RES ? NB / 2 : NB / 4;
    constexpr int kSignBytes = 64 * SB, kCodeBytes = RES ? 64 * CB : 0;
    constexpr int kP = (RES ? 2 : 1) * NC * 2 * 1024;         // one tile's weights
    // the rows' operands: fp16 ones of many rows stay in LDS (their registers would
    // be spilled), the others are read from there once
    constexpr bool QL = RES && NC * W >= 16;
    constexpr int kQ = NC * (W + NS) * 1024;
    constexpr int RS = D + 1;                                 // row of the sums at the end
    constexpr int kLoop = QL ? 2 * kP + kQ : 2 * kP;
    constexpr int kRaw = 4 * NC * ((D + 127) / 128) * 1024;   // the rows as they came
    constexpr bool kRawIn = QL && NC * NS * 1024 + kRaw <= 2 * kP;   // in the weights' place
    constexpr int kRawAt = kRawIn ? NC * NS * 1024 : QL ? 2 * kP + kQ : kQ;
    constexpr int kStart = kRawIn ? 2 * kP + kQ : kRawAt + kRaw;
    constexpr int kEnd = R * RS * 4;
    constexpr int kBuf = ((kLoop > kStart ? kLoop : kStart) > kEnd ? (kLoop > kStart ? kLoop : kStart) : kEnd) + 15 & ~15;
    __shared__ __attribute__((aligned(16))) uint8_t stage0[kCodeBytes + kSignBytes];
    __shared__ __attribute__((aligned(16))) uint8_t stage1[kCodeBytes + kSignBytes];
    __shared__ __attribute__((aligned(16))) uint8_t buf[kBuf];
    __shared__ __attribute__((aligned(16))) float scal[4][64];   // per wave: sk, rk, sv, rv of its 16 keys
    __shared__ __attribute__((aligned(16))) int flags[2][4];
    __shared__ float rmax[4][R], vmax[4], lsums[4][R], qtop[4];
    // per row: mean |q| in the exponent's unit, where the score product starts, its keys
    __shared__ __attribute__((aligned(16))) float row_const[R][4];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int g4 = lane >> 4, lj = lane & 15;
    const int group = a.Hq / a.Hkv, rows = a.B * group;
    const int hkv = blockIdx.y % a.Hkv;
    const int row0 = (blockIdx.y / a.Hkv) * R;
    const int64_t cap = (int64_t)a.n_pages * a.Hkv * a.page_tiles * 64;

    // ---------------- the tiles' places, and the first tile's loads
    const int first = blockIdx.x * x.tiles_per;
    const int n = min(x.tiles_per, x.tiles - first);
    // (a block of 64 tiles at a time, tile 64 b + i in lane i; a bad page reads the
    // pool's first, with NaN for its keys' scales)
    int tile_at = 0;
    uint64_t bad_tiles = 0;
    auto place = [&](int t) {
        bool bad = false;
        tile_at = 0;
        if (t + lane < n) {
            const int tile = first + t + lane;
            const int page = a.tables[tile / a.page_tiles];
            bad = page < 0 || page >= a.n_pages;
            tile_at = ((bad ? 0 : page) * a.Hkv + hkv) * a.page_tiles + tile % a.page_tiles;
        }
        bad_tiles = __ballot(bad);
    };
    auto rsrc = [&](const uint8_t* plane, int rb, int t) {
        const int64_t v = (int64_t)(uint32_t)__builtin_amdgcn_readlane(tile_at, t & 63) * 64;
        return __builtin_amdgcn_make_buffer_rsrc((void*)(plane + v * rb), (short)0, t < n ? 64 * rb : 0, kBufWord3);
    };
    // the key of row i of the wave's score block: lane group g's four keys, in the
    // order in which a value operand takes them (0, 4, 1, 5 or 2, 6, 3, 7 of a
    // run of 8)
    const int run = 8 * (wave >> 1) + 2 * (wave & 1);
    auto key_of = [&](int i) { return 16 * (i >> 2) + run + 4 * (i & 1) + (i >> 1 & 1); };
    // K of the wave's 16 keys: the lane's row's quarter g4 of the codes, its sign
    // words; scales of key lj, plane g4 (K signs, K codes, V signs, V codes)
    // (two sets: a tile's loads have the tile before it to land)
    struct KRegs2 {
        uint32_t code[RES ? W : 1], sign[NS];
        uint16_t scale;
        bool bad;
    };
    KRegs2 k_even, k_odd;
    const uint16_t* const scale_base =
        (const uint16_t*)(g4 == 0   ? a.kb.signs + cap * SB
                          : g4 == 1 ? (RES ? a.kr.codes + cap * CB : a.kb.signs + cap * SB)
                          : g4 == 2 ? a.vb.signs + cap * SB
                                    : (RES ? a.vr.codes + cap * CB : a.vb.signs + cap * SB)) + key_of(lj);
    auto load_k = [&](KRegs2& k, int t) {
        const int key = key_of(lj);
        const __amdgpu_buffer_rsrc_t r_s = rsrc(a.kb.signs, SB, t);
#pragma unroll
        for (int s = 0; s < NS; s++)
            k.sign[s] = __builtin_amdgcn_raw_buffer_load_b32(r_s, key * SB + 4 * min(4 * s + g4, D / 32 - 1), 0, 0);
        if constexpr (RES) {
            const __amdgpu_buffer_rsrc_t r_c = rsrc(a.kr.codes, CB, t);
            const int at = key * CB + g4 * (CB / 4);
#pragma unroll
            for (int w = 0; w + 4 <= W; w += 4) {
                const v4u_t c = __builtin_amdgcn_raw_buffer_load_b128(r_c, at + 4 * w, 0, 0);
                k.code[w] = c[0]; k.code[w + 1] = c[1]; k.code[w + 2] = c[2]; k.code[w + 3] = c[3];
            }
            if constexpr (W % 4 == 2) {
                const v2u_t c = __builtin_amdgcn_raw_buffer_load_b64(r_c, at + 4 * (W - 2), 0, 0);
                k.code[W - 2] = c[0]; k.code[W - 1] = c[1];
            }
        }
        // (past the range the last tile's again)
        const int last = min(t, n - 1);
        k.scale = scale_base[(int64_t)(uint32_t)__builtin_amdgcn_readlane(tile_at, last & 63) * 64];
        k.bad = bad_tiles >> (t & 63) & 1;
    };
    // the V tile: linear rows of codes with their pieces swizzled, then of signs; a
    // quarter of each by every wave
    auto load_v = [&](uint8_t* st, int t) {
        const __amdgpu_buffer_rsrc_t r_s = rsrc(a.vb.signs, SB, t);
        constexpr int kPart = kSignBytes / 4;    // 128, 256, 384 or 512 bytes
#pragma unroll
        for (int c = 0; c < (kPart + 255) / 256; c++) {
            const int at = wave * kPart + c * 256;
            // (lanes past the part repeat its last words into the next part's place
            // with that part's own bytes)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_s, LDS_PTR(void, st + kCodeBytes + min(at, kSignBytes - 256)), 4,
                                                     min(at, kSignBytes - 256) + 4 * lane, 0, 0, 0);
        }
        if constexpr (RES) {
            const __amdgpu_buffer_rsrc_t r_c = rsrc(a.vr.codes, CB, t);
#pragma unroll
            for (int i = 0; i < (Q + 3) / 4; i++) {
                const int c = min(wave + 4 * i, Q - 1);   // (Q = 2, 6: two waves load the last KiB)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    r_c, LDS_PTR(void, st + c * 1024), 16,
                    c * 1024 + 16 * (Q_POW2 ? lane ^ ((4 * c + (lane >> 4)) & (Q - 1)) : lane), 0, 0, 0);
            }
        }
    };

    // ---------------- the rows' operands: a wave takes 4 NC rows, 16 lanes per row and
    // a 16-byte piece each; all loads first
    constexpr int N = (D + 127) / 128;   // pieces of a lane
    bc_v4u raw[NC][N];
    int len[NC];
    bool live[NC];
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int row = row0 + 4 * (wave + 4 * i) + g4;
        live[i] = row < rows;
        const int b = live[i] ? row / group : 0;
        const uint16_t* src = a.q + ((int64_t)b * a.Hq + hkv * group + (live[i] ? row - b * group : 0)) * D;
        len[i] = a.lens[b];
#pragma unroll
        for (int k = 0; k < N; k++) {
            raw[i][k] = bc_v4u{0u, 0u, 0u, 0u};
            // (rows start at any element)
            typedef uint32_t Eight __attribute__((ext_vector_type(4), aligned(2)));
            if (live[i] && lj + 16 * k < D / 8) raw[i][k] = *(const Eight*)(src + 8 * (lj + 16 * k));
        }
    }
    place(0);
    load_k(k_even, 0);
    load_v(stage0, 0);
    load_k(k_odd, 1);
    // (past the weights' buffers where it stays, else past the sign words, in their place)
    uint8_t* const q_lds = buf + (QL ? 2 * kP : NC * NS * 1024);
    // (the rows wait in LDS: the loops over them stay rolled, since straight-line code
    // that runs once is fetched for as long as it takes)
    bc_v4u* const q_raw = (bc_v4u*)(buf + kRawAt) + wave * (NC * N * 64);
    float top = 0.0f;
    auto row16 = [](float t, auto op) {
        t = op(t, dpp_f<0x128>(t));
        t = op(t, dpp_f<0x124>(t));
        t = op(t, dpp_f<0x122>(t));
        return op(t, dpp_f<0x121>(t));
    };
    // (the type by a mask: a choice per element became a branch per element)
    const uint32_t bf = a.bf16 ? 0xFFFFFFFFu : 0u;
    auto value = [&](const bc_v4u& w, int e) { return bc::half_f((uint16_t)(w[e >> 1] >> (16 * (e & 1))), bf); };
#pragma unroll
    for (int i = 0; i < NC; i++)
#pragma unroll
        for (int k = 0; k < N; k++)
            if (lj + 16 * k < D / 8) q_raw[(i * N + k) * 64 + lane] = raw[i][k];
    // limits of the rows (those past the batch and those of a bad length, whose sums
    // nobody reads, mask nothing)
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int r = 4 * (wave + 4 * i) + g4;
        if (lj == 0) ((int*)row_const[r])[2] = !live[i] || bc::paged_bad_len(a, len[i]) ? 0x7FFFFFFF : len[i];
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll 1
    for (int i = 0; i < NC * N; i++) {
        if (lj + 16 * (i % N) >= D / 8) continue;
        const bc_v4u w = q_raw[i * 64 + lane];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float t = fabsf(value(w, e));
            top = fmaxf(top, t < INFINITY ? t : 0.0f);
        }
    }
    top = wave_max(top);
    if (lane == 0) qtop[wave] = top;
    for (int i = threadIdx.x; i < 4 * R; i += 256) (&rmax[0][0])[i] = -INFINITY;
    if (threadIdx.x < 4) vmax[threadIdx.x] = 0.0f;
    lds_barrier();
    // q 2^ex with the largest element of all rows in [2^13, 2^14): exact in fp16 down
    // to 2^-27 of it (odd dims carry another 1/16)
    top = fmaxf(fmaxf(qtop[0], qtop[1]), fmaxf(qtop[2], qtop[3]));
    const int field = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
    const int ex = __builtin_amdgcn_readfirstlane(field > 0 ? 140 - field : 0);
    const float isd2 = kLog2e / sqrtf((float)D);
    const float res_unit = ldexpf(isd2 * (1.0f / 7.0f), 24 - ex);
#pragma unroll 1
    for (int i = 0; i < NC; i++) {
        const int r = 4 * (wave + 4 * i) + g4, c = r >> 4, col = r & 15;
        float sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int u = lj + 16 * k;
            if (u >= D / 8) continue;
            const bc_v4u w = q_raw[(i * N + k) * 64 + lane];
            uint32_t byte = 0;
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = value(w, e);
                byte |= (v >= 0.0f ? 0u : 1u) << e;
                sum += fabsf(v);
                t[e] = ldexpf(v, ex);
                total += t[e];
            }
            const int g = u / W, s = u % W;
            if constexpr (RES) {
                // slots of a step: dims 0, 4, 1, 5, 2, 6, 3, 7
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f = e & 1 ? 0.0625f : 1.0f;
                    h[e] = (uint32_t)f2h(t[e] * f) | ((uint32_t)f2h(t[e + 4] * f) << 16);
                }
                *(v4u_t*)(q_lds + ((c * W + s) * 64 + 16 * g + col) * 16) = v4u_t{h[0], h[1], h[2], h[3]};
            }
            // sign word u / 4 of the row, byte u % 4 (expanded when it is read)
            buf[((c * NS + u / 16) * 64 + 16 * (u / 4 % 4) + col) * 16 + u % 4] = (uint8_t)byte;
        }
        sum = row16(sum, [](float p, float q) { return p + q; });
        total = row16(total, [](float p, float q) { return p + q; });
        if (lj == 0) {
            row_const[r][0] = sum * (1.0f / (float)D) * isd2;
            row_const[r][1] = ldexpf(-8.0f * total, -24);
        }
    }
    lds_barrier();
    h8_t q16[RES && !QL ? NC : 1][RES && !QL ? W : 1];
    v4i_t q4[NC][NS];
    float m[NC], l[NC];
    int least = 0x7FFFFFFF;   // keys of the workgroup's shortest row
    constexpr float kTau = 8.0f, kNone = -1e30f;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        if constexpr (RES && !QL) {
#pragma unroll
            for (int s = 0; s < W; s++) q16[c][s] = *(const h8_t*)(q_lds + ((c * W + s) * 64 + lane) * 16);
        }
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const uint32_t w = *(const uint32_t*)(buf + ((c * NS + s) * 64 + lane) * 16);
            // (past the dims: 0 times anything)
            q4[c][s] = 4 * s + g4 < D / 32 ? v4i_t{(int)fp4_signs(w, 0), (int)fp4_signs(w, 1), (int)fp4_signs(w, 2),
                                                   (int)fp4_signs(w, 3)}
                                           : v4i_t{0, 0, 0, 0};
        }
        // (all waves hold the same)
        if (QL && wave == 0) {
#pragma unroll
            for (int s = 0; s < NS; s++) *(v4i_t*)(q_lds + ((NC * W + c * NS + s) * 64 + lane) * 16) = q4[c][s];
        }
        least = min(least, ((const int*)row_const[16 * c + lj])[2]);
        m[c] = kNone;
        l[c] = 0.0f;
    }
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) least = min(least, __shfl_xor(least, k));
    least = __builtin_amdgcn_readfirstlane(least);
    lds_barrier();   // (the operands have been read: the weights take their place)

    // ---------------- the value products: blocks of 16 dims, the sign part's block
    // 4 h + p holds dims 64 h + 4 i + p, the residual part's dims 16 b + i
    const bool res_wave = RES && wave >= 2;
    const int block0 = (res_wave ? wave - 2 : wave) * NBW;
    f4_t acc[NBW][NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
#pragma unroll
        for (int i = 0; i < NBW; i++) acc[i][c] = f4_t{0.f, 0.f, 0.f, 0.f};
    }
    // V scales enter as floats times 2^we, the largest in [2^4, 2^5): weights stay
    // below 2^14 and keep their bits down to 2^-28 of the largest
    int we = 0;
    float wlim = 0.0f;

    // one tile: st its V data, at the other buffer, t its number
    auto tile = [&](KRegs2& k, uint8_t* st, uint8_t* next, int parity, int t) {
        uint8_t* const pb = buf + parity * kP;
        const int t0 = (first + t) * 64;
        const bool whole = t0 + 64 <= least;
        float sums[NC];
        for (;;) {
            // ------------ the wave's scales: lane = (plane g4, key lj)
            const float raw_scale = h2f(k.scale);
            float sv = raw_scale;
            if (g4 == 0 && k.bad) sv = __builtin_nanf("");
            if (g4 == 1) sv *= res_unit;
            if (g4 >= 2) sv = ldexpf(sv, we);
            // (a scale that is not finite takes no part in the plan)
            const float big = g4 >= 2 && fabsf(raw_scale) < INFINITY ? fabsf(raw_scale) : 0.0f;
            const bool grow = __ballot(big >= wlim && big > 0.0f) != 0ull;
            scal[wave][lane] = sv;
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            const f4_t sk = *(const f4_t*)&scal[wave][4 * g4], rk = *(const f4_t*)&scal[wave][16 + 4 * g4];
            const f4_t fa = *(const f4_t*)&scal[wave][32 + 4 * g4], fb = *(const f4_t*)&scal[wave][48 + 4 * g4];
            v8i_t k4[NS];
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const uint32_t w = ~k.sign[s];
                k4[s] = v8i_t{(int)fp4_signs(w, 0), (int)fp4_signs(w, 1), (int)fp4_signs(w, 2), (int)fp4_signs(w, 3), 0, 0, 0, 0};
            }
            h8_t k16[RES ? W : 1];
            if constexpr (RES) {
#pragma unroll
                for (int s = 0; s < W; s++) {
                    const uint32_t w = k.code[s] ^ 0x88888888u, y = w >> 8;
                    k16[s] = __builtin_bit_cast(h8_t, v4u_t{w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u});
                }
            }
            bool moves = false;
            // the products of the next sixteen rows run under the softmax of these (the
            // barriers keep the compiler from fetching all rows' operands at once)
            f4_t s1[2], s2[2];
            auto products = [&](int c) {
                const float from = row_const[16 * c + lj][1];
                f4_t& u1 = s1[c & 1];
                f4_t& u2 = s2[c & 1];
                u1 = f4_t{0.f, 0.f, 0.f, 0.f};
                u2 = f4_t{from, from, from, from};
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    v4i_t t;
                    if constexpr (QL) t = *(const v4i_t*)(q_lds + ((NC * W + c * NS + s) * 64 + lane) * 16);
                    else t = q4[c][s];
                    const v8i_t q = {t[0], t[1], t[2], t[3], 0, 0, 0, 0};
                    u1 = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k4[s], q, u1, 4, 4, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
                }
                if constexpr (RES) {
#pragma unroll
                    for (int s = 0; s < W; s++) {
                        h8_t q;
                        if constexpr (QL) q = *(const h8_t*)(q_lds + ((c * W + s) * 64 + lane) * 16);
                        else q = q16[c][s];
                        u2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k16[s], q, u2, 0, 0, 0);
                    }
                }
            };
            products(0);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                __builtin_amdgcn_sched_barrier(0);
                if (c + 1 < NC) products(c + 1);
                const float rho = row_const[16 * c + lj][0];
                const int limit = ((const int*)row_const[16 * c + lj])[2];
                const f4_t &u1 = s1[c & 1], &u2 = s2[c & 1];
                float p[4];
                auto scores = [&](float from) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float z = from;
                        if constexpr (RES) z = fmaf(u2[j], rk[j], z);
                        p[j] = fmaf(u1[j] * sk[j], rho, z);
                    }
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 4; j++) p[j] = t0 + key_of(4 * g4 + j) < limit ? p[j] : -INFINITY;
                    }
                };
                scores(-m[c]);
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] = __builtin_amdgcn_exp2f(p[j]);
                const float sum = (p[0] + p[1]) + (p[2] + p[3]);
                sums[c] = sum;
                // weights as operands: keys (j = 0, 1) and (2, 3) of the lane share a dword
                auto weights = [&](const f4_t& f) {
                    h2_t w0, w1;
                    w0[0] = (_Float16)(p[0] * f[0]); w0[1] = (_Float16)(p[1] * f[1]);
                    w1[0] = (_Float16)(p[2] * f[2]); w1[1] = (_Float16)(p[3] * f[3]);
                    return v2u_t{as_u(w0), as_u(w1)};
                };
                v2u_t wa = weights(fa), wb = {0u, 0u};
                if constexpr (RES) wb = weights(fb);
                if (!whole) {
                    // (a masked key adds nothing whatever its scales are)
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        const uint32_t in = (t0 + key_of(4 * g4 + j) < limit ? 0x0000FFFFu : 0u) |
                                            (t0 + key_of(4 * g4 + j + 1) < limit ? 0xFFFF0000u : 0u);
                        wa[j >> 1] &= in;
                        wb[j >> 1] &= in;
                    }
                }
                uint8_t* const at = pb + ((c * 2 + (wave >> 1)) * 64 + lane) * 16 + 8 * (wave & 1);
                *(v2u_t*)at = wa;
                if constexpr (RES) *(v2u_t*)(at + NC * 2 * 1024) = wb;
                // a row whose weights pass 2^kTau: its largest score, over the lane groups
                if (__ballot(sum > 256.0f) != 0ull) {
                    scores(0.0f);
                    float hi = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
                    hi = fmaxf(hi, __shfl_xor(hi, 16));
                    hi = fmaxf(hi, __shfl_xor(hi, 32));
                    // (moved only to a reference above the old one: the tile's next form
                    // passes 2^kTau no more)
                    if (g4 == 0 && hi > m[c]) rmax[wave][16 * c + lj] = hi;
                    moves |= __ballot(hi > m[c]) != 0ull;
                }
            }
            if (grow) {
                const float v = wave_max(big);
                if (lane == 0) vmax[wave] = v;
            }
            if (lane == 0) flags[parity][wave] = moves || grow;
            // this tile's V data has landed, and the weights are in LDS
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const v4i_t fl = *(const v4i_t*)flags[parity];
            if (__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) == 0) break;
            // ------------ the references move, and the weights' unit
            const float v = fmaxf(fmaxf(vmax[0], vmax[1]), fmaxf(vmax[2], vmax[3]));
            const int vf = __builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, v) >> 23));
            float unit = 1.0f;
            if (vf > 0) {
                const int e = 4 + 127 - vf;
                if (wlim > 0.0f) unit = ldexpf(1.0f, e - we);
                we = e;
                wlim = ldexpf(1.0f, 5 - e);
            }
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const int r = 16 * c + lj;
                const float to = fmaxf(fmaxf(fmaxf(rmax[0][r], rmax[1][r]), fmaxf(rmax[2][r], rmax[3][r])), m[c]);
                const float f = __builtin_amdgcn_exp2f(m[c] - to);
                m[c] = to;
                l[c] *= f;
                const float fu = f * unit;
#pragma unroll
                for (int i = 0; i < NBW; i++) acc[i][c] *= fu;
            }
            lds_barrier();   // (everyone has read them)
#pragma unroll
            for (int c = 0; c < NC; c++) rmax[wave][16 * c + lj] = -INFINITY;
            if (lane == 0) vmax[wave] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < NC; c++) l[c] += sums[c];
        // ---------------- the next tile's loads
        __builtin_amdgcn_sched_barrier(0);
        load_v(next, t + 1);
        if (((t + 2) & 63) == 0 && t + 2 < n) place(t + 2);
        load_k(k, t + 2);
        __builtin_amdgcn_sched_barrier(0);
        // ---------------- values
        const uint8_t* const pw = pb + (res_wave ? NC * 2 * 1024 : 0);
        h8_t w[NC][2];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int mh = 0; mh < 2; mh++) w[c][mh] = *(const h8_t*)(pw + ((c * 2 + mh) * 64 + lane) * 16);
        const int row_key = lane;   // (key 16 g4 + lj)
        const int vsw = Q_POW2 ? ((lane * CB) >> 8) & (Q - 1) : 0;
        v2i_t bits[NBW];
#pragma unroll
        for (int i = 0; i < NBW; i++) {
            const int b = block0 + i;
            const uint8_t* at = st + (res_wave ? CB * row_key + 16 * ((b >> 1) ^ vsw) + 8 * (b & 1)
                                               : kCodeBytes + SB * row_key + 8 * (b >> 2));
            bits[i] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(LDS_PTR(v2i_t, at));
        }
        auto products = [&](int i, int mh, const uint32_t (&u)[4]) {
            const h8_t av = __builtin_bit_cast(h8_t, v4u_t{u[0], u[1], u[2], u[3]});
#pragma unroll
            for (int c = 0; c < NC; c++) acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, w[c][mh], acc[i][c], 0, 0, 0);
        };
        // nibble r of a word is key r's: pairs (0, 4), (1, 5), (2, 6), (3, 7) as halves
        if (res_wave) {
            const h2_t one = {(_Float16)1.0f, (_Float16)1.0f}, sixteenth = one * (_Float16)0.0625f;
            const h2_t off_lo = one * (_Float16)-1032.0f, off_hi = one * (_Float16)-72.0f;
#pragma unroll
            for (int i = 0; i < NBW; i++)
#pragma unroll
                for (int mh = 0; mh < 2; mh++) {
                    // the code + 8 in the last bits of 1024 + ..: in the low nibble as it is,
                    // in the next one sixteen times
                    const uint32_t v = (uint32_t)(mh ? bits[i].y : bits[i].x) ^ 0x88888888u, y = v >> 8;
                    uint32_t u[4] = {(v & 0x000F000Fu) | 0x64006400u, (v & 0x00F000F0u) | 0x64006400u,
                                     (y & 0x000F000Fu) | 0x64006400u, (y & 0x00F000F0u) | 0x64006400u};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const h2_t h = __builtin_bit_cast(h2_t, u[j]);
                        u[j] = as_u(j & 1 ? __builtin_elementwise_fma(h, sixteenth, off_hi) : h + off_lo);
                    }
                    products(i, mh, u);
                }
        } else {
#pragma unroll
            for (int i = 0; i < NBW; i++) {
                const int p = (block0 + i) & 3;
#pragma unroll
                for (int mh = 0; mh < 2; mh++) {
                    // the sign bit is the value's bit p (so -1 where the value is positive:
                    // turned at the end)
                    const uint32_t v = (uint32_t)(mh ? bits[i].y : bits[i].x);
                    uint32_t u[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) u[j] = ((v << (15 - 4 * j - p)) & 0x80008000u) | 0x3C003C00u;
                    products(i, mh, u);
                }
            }
        }
    };
    for (int t = 0; t < n; t += 2) {
        tile(k_even, stage0, stage1, 0, t);
        if (t + 1 >= n) break;
        tile(k_odd, stage1, stage0, 1, t + 1);
    }
    __builtin_amdgcn_s_waitcnt(0);   // (the last prefetch)
    __syncthreads();

    // ---------------- the end: the sign part's sums in LDS, the residual part's on
    // them, one partial per row
    float* const o = (float*)buf;
    const float unit = wlim > 0.0f ? ldexpf(1.0f, -we) : 1.0f;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        float t = l[c];
        t += __shfl_xor(t, 16);
        t += __shfl_xor(t, 32);
        if (g4 == 0) lsums[wave][16 * c + lj] = t;
        // (every wave's rows: the references are the same)
        if (wave == 0 && g4 == 0) row_const[16 * c + lj][0] = m[c];
    }
    auto put = [&](bool res) {
#pragma unroll
        for (int i = 0; i < NBW; i++) {
            const int b = block0 + i, p = b & 3;
            const float k = res ? unit * (1.0f / 7.0f) : -unit;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int d = res ? 16 * b + 4 * g4 + j : 64 * (b >> 2) + 4 * (4 * g4 + j) + p;
                    float* const at = o + (16 * c + lj) * RS + d;
                    const float v = acc[i][c][j] * k;
                    *at = res ? *at + v : v;
                }
        }
    };
    if (!res_wave) put(false);
    __syncthreads();
    if (RES) {
        if (res_wave) put(true);
        __syncthreads();
    }
    // (a wave a row; where row r goes in lane r)
    int64_t place_of = 0;
    if (lane < R && row0 + lane < rows) {
        const int b = (row0 + lane) / group, h = hkv * group + (row0 + lane) - b * group;
        place_of = (((int64_t)blockIdx.x * a.B + b) * a.Hq + h) * (D + 2);
    }
    const int last_row = min(R, rows - row0);
#pragma unroll 4
    for (int r = wave; r < last_row; r += 4) {
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)place_of, r);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)place_of >> 32), r);
        float* const dst = x.ws + (int64_t)((uint64_t)hi << 32 | lo);
#pragma unroll
        for (int e = 0; e < D; e += 64) dst[2 + e + lane] = o[r * RS + e + lane];
        if (lane == 0) {
            dst[0] = row_const[r][0];
            dst[1] = (lsums[0][r] + lsums[1][r]) + (lsums[2][r] + lsums[3][r]);
        }
    }
}

}  // namespace

namespace bc {

template <int D, int NC>
static void prefix_go(bool res, const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st) {
    if (res) hipLaunchKernelGGL((prefix_attn_kernel<D, NC, true>), grid, dim3(256), 0, st, a, x);
    else hipLaunchKernelGGL((prefix_attn_kernel<D, NC, false>), grid, dim3(256), 0, st, a, x);
}

template <int D>
void prefix_launch(bool res, int nc, const AttnArgs& a, const PrefixArgs& x, dim3 grid, hipStream_t st) {
    if constexpr (prefix_columns(D) == 4) {
        if (nc == 4) return prefix_go<D, 4>(res, a, x, grid, st);
    }
    if (nc == 2) return prefix_go<D, 2>(res, a, x, grid, st);
    prefix_go<D, 1>(res, a, x, grid, st);
}

}  // namespace bc

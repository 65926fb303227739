// Shared declarations of the split-KV attention kernels (attention.hip,
// attn_mfma_kernel.h).
#pragma once

#include "common.h"

namespace bc {

constexpr float kLog2e = 1.4426950408889634f;

// MODE_MIXED: compensated data flow, each (b, query head) adding its residual
// (score and value) or not as head_mode says: per-head binary / compensated
// dispatch in one launch.
enum AttnMode : int { MODE_BINARY = 0, MODE_COMP = 1, MODE_ADAPTIVE = 2, MODE_MIXED = 3 };

struct AttnArgs {
    const uint16_t* q;  // [B, Hq, D] fp16
    BinPlanes kb, vb;
    ResPlanes kr, vr;
    int B, Hq, Hkv, S, kv_stride;
    int n_splits, chunk;  // chunk: keys per split (multiple of 64)
    float* ws;            // [B*Hq][n_splits][D + 2]: m (log2 domain), l, acc[D]
    // adaptive selection (MODE_ADAPTIVE)
    const uint32_t* thresh;      // [B*Hq] ordered key threshold
    const int32_t* cutoff;       // [B*Hq] keys equal to the threshold are taken up to
                                 // this key index (-1: none)
    uint8_t* selected;           // optional [B, Hq, S]
    const void* pcs;             // adaptive: [B*Hq/G][pcs_stride(S)] PcPack<PcT<D>, G>
                                 // popcounts of the selection passes (G = the kernel's
                                 // head group)
    // in-place append (binary and compensated modes, one query-head group per
    // kv head): the new K and V vectors [B*Hkv, D] fp16 are encoded into cache
    // position app_slot of every (b, kv head) row before the row is attended
    // (null: no append)
    const uint16_t* app_k;
    const uint16_t* app_v;
    int app_slot;
    // MODE_MIXED: [B*Hq] 0 = binary attention for that head, else compensated
    const uint8_t* head_mode;
    // per-head modes run as two launches (binary kernel, mixed kernel), each
    // over the query-head groups of its kind: grid row y takes group
    // group_list[y] while y < *group_count, and returns otherwise (lists in
    // the workspace, written by a compaction launch; null: row y is group y)
    const int32_t* group_list;
    const int32_t* group_count;
    // one split per group (n_splits == 1): when set, the kernel writes the
    // normalised output [B, Hq, D] fp16 here instead of its partial, and no
    // merge launch follows
    uint16_t* out;
    // paged caches: sequence b's keys are the first lens[b] of the pages
    // tables[b * width + i], page_tiles 64-key tiles each (a null lens: no
    // pages).  Keys before key0 (a shared prefix) are attended elsewhere.
    const int32_t* lens;
    const int32_t* tables;
    int width, n_pages, page_tiles, key0, max_len;
    int unit_tiles;   // see PagedUnit; 0: one unit per sequence
    int unit_slots, unit_most;
    int unit_each;    // units of every sequence, kUnitTiles each; 0: cut by the lengths
    int2* units;      // each sequence's first unit and how many it has
    int bf16;         // queries and outputs are bf16
};

// Work units of a paged call.  A sequence's tiles after key0 are cut into units of
// equal size, as many as bring a unit to at most `chunk` tiles; the device
// chooses chunk from the lengths, so that the launch is planned without knowing
// them and a captured call follows them.  unit_slots units (times the head
// groups) run at once.  Eight candidates aim at half to two rounds of them, and
// the cheapest is taken (the fixed work of a unit, its query preparation, merge and
// first loads, counts as kUnitFixed tiles), as far as its units fit the launched
// ones (unit_most); chunk is at least unit_tiles and at most kUnitTiles (a wave
// holds its tiles' places in one register), which always fits.  unit_tiles = 0:
// unit b is sequence b; unit_each: unit b unit_each + i is the i-th of sequence b (a
// large batch, whose lengths would take each wave too long to go through).  Each wave finds its unit by itself, and one notes the
// sequences' units for the merge.  (64 sequences of 128 to 32768 keys, 32/8 heads,
// 478 MB: 93 us; by rounds times the mean unit 111, since few units of unequal
// length leave a tail; 64 of 6144 keys, 528 MB, 90 and 104.  One equal range of
// tiles per slot, across sequences, took 40 us more than units: two segments in
// most ranges, each with the fixed work and none beside another's loop.)
constexpr int kUnitTiles = 256, kUnitFixed = 6, kUnitRounds = 2;
struct PagedUnit {
    int b, len;        // (b < 0: no such unit)
    int first, tiles;  // the unit's tiles, counted from key0
};
// A length that no bound or table holds
__host__ __device__ inline bool paged_bad_len(const AttnArgs& a, int len) {
    return len > a.max_len || (int64_t)len > (int64_t)a.width * a.page_tiles * 64;
}
__device__ __forceinline__ int paged_tiles(const AttnArgs& a, int len) {
    return len <= a.key0 || paged_bad_len(a, len) ? 0 : (len - a.key0 + 63) / 64;
}
// Inclusive sum over the wave's lanes
__device__ __forceinline__ int wave_scan_add(int v) {
#define BC_SCAN_STEP(CTRL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
    BC_SCAN_STEP(0x111, 0xF)   // row_shr 1, 2, 4, 8
    BC_SCAN_STEP(0x112, 0xF)
    BC_SCAN_STEP(0x114, 0xF)
    BC_SCAN_STEP(0x118, 0xF)
    BC_SCAN_STEP(0x142, 0xA)   // row broadcasts into the rows after
    BC_SCAN_STEP(0x143, 0xC)
#undef BC_SCAN_STEP
    return v;
}
// Units at most, of a batch of `tiles` tiles at most
__host__ __device__ inline int64_t paged_unit_most(int slots, int batch, int64_t tiles) {
    const int64_t full = (int64_t)kUnitRounds * slots, capped = (tiles + kUnitTiles - 1) / kUnitTiles + batch;
    return capped > full ? capped : full;
}
// Tiles of a unit at most.  own: the tiles of sequence `lane` (0 past the batch).
__device__ __forceinline__ int paged_chunk(const AttnArgs& a, int lane, int& own) {
    own = lane < a.B ? paged_tiles(a, a.lens[lane]) : 0;
    int n = own;
    for (int i = lane + 64; i < a.B; i += 64) n += paged_tiles(a, a.lens[i]);
    const int total = __builtin_amdgcn_readlane(wave_scan_add(n), 63);
    // lane = (candidate, eighth of the sequences); candidates in 16ths of a round
    const int cand = lane & 7;
    const int sixteenths = (int)(0x20181410'0F0E0C08ull >> (8 * cand)) & 0xFF;
    const float even = ceilf(16.0f * (float)total / ((float)a.unit_slots * (float)sixteenths));
    const int chunk = max((int)fminf(even, (float)kUnitTiles), a.unit_tiles);
    const float inv = 1.0f / (float)chunk;
    int units = 0;
    for (int i0 = 0; i0 < a.B; i0 += 64) {
        const int t = i0 == 0 ? own : i0 + lane < a.B ? paged_tiles(a, a.lens[i0 + lane]) : 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            // (the quotient within one, then exact: the launch holds the units)
            const int x = __builtin_amdgcn_ds_bpermute(4 * (8 * k + (lane >> 3)), t), n = (int)((float)x * inv);
            const int rest = x - n * chunk;
            units += n + (rest > 0) + (rest > chunk);
        }
    }
    // (the eighths: lanes 8, 16 and 32 apart)
    units += __builtin_amdgcn_ds_swizzle(units, 0x201F);
    units += __builtin_amdgcn_ds_swizzle(units, 0x401F);
    units += __builtin_amdgcn_ds_bpermute(4 * (lane ^ 32), units);
    // (one round: its longest unit; more: the slots' share, and half a unit at the end)
    const float tiles = units <= a.unit_slots
                            ? (float)(chunk + kUnitFixed)
                            : ((float)total + (float)kUnitFixed * (float)units) / (float)a.unit_slots + 0.5f * (float)chunk;
    uint32_t cost[1] = {~((uint32_t)fminf(16.0f * tiles, 268435455.0f) << 3 | (uint32_t)cand)};
    if (units > a.unit_most) cost[0] = 0;
    wave_umax(cost);
    const uint32_t best = __builtin_amdgcn_readfirstlane(cost[0]);
    return best == 0 ? kUnitTiles : __builtin_amdgcn_readlane(chunk, (int)(~best & 7));
}
// tells: the caller is the wave that notes every sequence's units (with unit 0)
__device__ __forceinline__ PagedUnit paged_unit(const AttnArgs& a, int unit, int lane, bool tells) {
    if (a.unit_tiles == 0) {
        const int len = __builtin_amdgcn_readfirstlane(a.lens[unit]);
        return PagedUnit{unit, len, 0, paged_tiles(a, len)};
    }
    if (a.unit_each > 0) {
        const int b = unit / a.unit_each, first = (unit - b * a.unit_each) * kUnitTiles;
        const int len = __builtin_amdgcn_readfirstlane(a.lens[b]), tiles = paged_tiles(a, len);
        if (first >= tiles) return PagedUnit{-1, 0, 0, 0};
        return PagedUnit{b, len, first, min(tiles - first, kUnitTiles)};
    }
    int own;
    const int chunk = paged_chunk(a, lane, own);
    if (unit == 0 && tells) {
        int base = 0;
        for (int i0 = 0; i0 < a.B; i0 += 64) {
            const int tiles = i0 == 0 ? own : i0 + lane < a.B ? paged_tiles(a, a.lens[i0 + lane]) : 0;
            const int n = (tiles + chunk - 1) / chunk, incl = wave_scan_add(n);
            if (i0 + lane < a.B) a.units[i0 + lane] = make_int2(base + incl - n, n);
            base += __builtin_amdgcn_readlane(incl, 63);
        }
    }
    int base = 0;
    for (int i0 = 0; i0 < a.B; i0 += 64) {
        const int tiles = i0 == 0 ? own : i0 + lane < a.B ? paged_tiles(a, a.lens[i0 + lane]) : 0;
        const int n = (tiles + chunk - 1) / chunk;
        const int incl = wave_scan_add(n), last = __builtin_amdgcn_readlane(incl, 63);
        if (unit - base < last) {
            const int at = __builtin_ctzll(__ballot(incl > unit - base));
            const int mine = __builtin_amdgcn_readlane(tiles, at), count = __builtin_amdgcn_readlane(n, at);
            const int split = unit - base - (__builtin_amdgcn_readlane(incl, at) - count);
            const int per = (mine + count - 1) / count;
            return PagedUnit{i0 + at, __builtin_amdgcn_readfirstlane(a.lens[i0 + at]), split * per, max(0, min(per, mine - split * per))};
        }
        base += last;
    }
    return PagedUnit{-1, 0, 0, 0};
}
// Packs per row of the stored popcounts: S rounded up to 16, so that every
// row starts 16-byte aligned and eight-key runs load whole.
__host__ __device__ inline int pcs_stride(int S) { return (S + 15) & ~15; }

// Stored popcount of one (query head, key): 8 bits, 16 for d = 256 (popcount
// up to 256).  A pack holds the G heads of a query-head group for one key.
template <bool WIDE> struct PcSel { typedef uint8_t type; };
template <> struct PcSel<true> { typedef uint16_t type; };
template <int D> using PcT = typename PcSel<(D > 255)>::type;
template <typename P, int G>
struct __attribute__((aligned(G * sizeof(P)))) PcPack {
    P v[G];
};

// MFMA value-phase kernels (attn_mfma_kernel.h): true if (D, G, mode) is
// handled there and the launch was issued.
bool launch_mfma_split(int mode, int D, int G, const AttnArgs& a, dim3 grid, hipStream_t st, int nw = 4);
// The instances of one head dim (one translation unit each, attn_mfma_d*.hip).
template <int D>
bool mfma_launch(int mode, int G, const AttnArgs& a, dim3 grid, hipStream_t st, int nw);
template <int D>
int mfma_occupancy(int mode, int G);
// Query-head groups per kv head that the MFMA kernels' packed plan argument holds.
constexpr int kMaxHeadGroups = (1 << 13) - 1;
// True if the MFMA kernels handle head_dim D with splits of `chunk` keys and
// `head_groups` query-head groups per kv head.
bool mfma_split_ok(int D, int64_t chunk, int64_t head_groups);
// Head dims whose kernels append a token in place (the one-slice row encoder
// of encode_row.h takes power-of-two lane groups).
__host__ __device__ constexpr bool append_dim(int D) { return D == 64 || D == 128 || D == 256; }
// The paged instances (binary and compensated modes): grid.x kv heads times
// query-head groups of a kv head, grid.y units (those past the batch's last one,
// which leave at once, come last); the partial of unit u and query
// head h goes to ws[(u * Hq + h) * (D + 2)], or the outputs to a.out (one unit per
// sequence).
template <int D>
void paged_launch(int mode, int G, const AttnArgs& a, dim3 grid, hipStream_t st);
template <int D>
int paged_occupancy(int mode, int G);
bool launch_paged_split(int mode, int D, int G, const AttnArgs& a, dim3 grid, hipStream_t st);
int paged_wgs_per_cu(int mode, int D, int G);
// Resident workgroups per CU of the MFMA kernel of (mode, D, G) on the current
// device (0 when no MFMA kernel handles it).
int mfma_wgs_per_cu(int mode, int D, int G);

// An fp16 value, or a bf16 one where bf is all ones (0 else)
__device__ __forceinline__ float half_f(uint16_t h, uint32_t bf) {
    return __builtin_bit_cast(float, ((uint32_t)h << 16 & bf) | (__builtin_bit_cast(uint32_t, h2f(h)) & ~bf));
}

// Query heads that one workgroup attends for, of the `group` that share a kv head.
int attention_group(int group, int D, int mode);

// New K/V token encoded into cache position `slot` by the attention launch
// itself (see AttnArgs::app_k).
struct AppendArgs {
    const void* k;   // [B*Hkv, D] fp16
    const void* v;
    int slot;
};

// Split partials + combine (attention.hip), shared by the public entry points
// and the adaptive driver (adaptive.hip).  app: append the token first (the
// caller has checked that the MFMA kernel runs with one query-head group per
// kv head).
int run_attention(int mode, const void* q, const void* k_bin, const void* k_res, const void* v_bin,
                  const void* v_res, void* out, int batch, int n_heads, int n_kv_heads,
                  int seq_len, int kv_stride, int head_dim, void* workspace,
                  size_t workspace_bytes, hipStream_t st, const uint32_t* thresh,
                  const int32_t* cutoff, uint8_t* selected, const void* pcs,
                  const AppendArgs* app = nullptr, const uint8_t* head_mode = nullptr);
size_t attention_ws_bytes(int batch, int n_heads, int n_kv_heads, int seq_len, int d);
}  // namespace bc

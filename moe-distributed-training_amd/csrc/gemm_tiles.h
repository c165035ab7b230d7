// What the matrix-core grouped GEMMs of both element widths (grouped_gemm_kernel.h, int8_gemm_kernel.h) share: direct-to-LDS loads, and the
// plan that gives every workgroup its output tile, or K part of one.
#pragma once
#include "common.h"

namespace {

constexpr int NXCD = 8;
constexpr int INTERLEAVE_MIN_ROUNDS = 8;    // launches with at least this many rounds of tiles deal them to the XCDs in chunks
constexpr int CONTIGUOUS_MIN_ROUNDS = 4;    // ... and so do launches of fewer rounds than this; those in between give every XCD one contiguous range

// 16 bytes per lane, global -> LDS without passing through VGPRs: lane l's data lands at lds_addr + 16*l.  The source
// is a raw buffer (base address in a scalar resource descriptor) plus a 32-bit per-lane byte offset plus a scalar byte
// offset, so advancing along K costs no vector instructions.  Issued through inline assembly so that the compiler's
// wait-count insertion does not serialise the prefetch against the fragment reads of the other stage; completion is
// awaited with explicit s_waitcnt vmcnt(n) below.
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4_t make_buffer(const void* base, uint32_t num_records = 0xFFFFFFFFu)
{
    const uint64_t a = (uint64_t)base;
    i32x4_t r;
    r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));   // stride field (bits 16..29 of this word) = 0: raw buffer
    r.z = (int)num_records;                                           // a per-lane offset at or above this is out of range (loads return zeros); real offsets are checked on the host
    r.w = 0x00020000;                                                 // 32-bit data format
    return r;
}
// NT: non-temporal, for data that nobody else will read again.
template <bool NT = false>
__device__ __forceinline__ void load_to_lds_16(i32x4_t rsrc, uint32_t lane_off, uint32_t uniform_off, uint32_t lds_addr)
{
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" ::"s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(lane_off), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(uniform_off)) : "memory", "m0");
    else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(lane_off), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(uniform_off)) : "memory", "m0");
}

// logistic function through the hardware exponential and reciprocal (about 1 ulp each; the results are rounded to bf16)
__device__ __forceinline__ float sigmoid_f(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// ---- work item of a workgroup -> (expert, n tile, m tile, K part).  One workgroup per work item; the hardware dispatcher
// hands the next item to whichever compute unit of the XCD frees up first (blockIdx round-robins over the 8 XCDs), which
// balances ragged (cheaper) row tiles inside an XCD by itself; between XCDs work cannot migrate.
struct WorkItem {
    bool valid;
    int expert, nt;            // expert, n tile
    int64_t row0, row1;        // rows of the m tile
    int part, nparts;          // K part of a split tile (0 of 1: whole tile)
    int split_item;            // exchange slot of this part (the slots of a tile are consecutive, in part order)
    int split_tile;            // counter of the split tile
    bool only_tile;            // the group fits in this one row tile
    int mtile;                 // number of the row tile among all row tiles (experts in order)
};

// Rows of row tile mt of a group's mte tiles: the group's 16-row blocks are dealt evenly to its tiles (mte = the number of
// tiles of BM rows the group needs; the figures are of 256 rows).  Measured per round of tiles at K=4096: 99 us with 16 row blocks, 87 with 13, and a tail
// of 1-3 blocks behind full tiles about as much as a full one (its waves wait for the same weight tiles), so 1060 rows run
// as five tiles of 13-14 blocks instead of four of 16 and one of 3.  8192 rows over 8 experts: gate/up launch 1630 -> 1556 us,
// the layer's forward and backward 5029 -> 4950 us.
__device__ __forceinline__ void even_rows(int64_t start, int64_t end, uint32_t mt, uint32_t mte, int64_t* row0, int64_t* row1)
{
    const uint32_t blocks = (uint32_t)((end - start + 15) >> 4), per = blocks / mte, more = blocks - per * mte;
    const uint32_t b0 = mt * per + (mt < more ? mt : more);
    *row0 = start + (int64_t)b0 * 16;
    const int64_t r1 = *row0 + (int64_t)(per + (mt < more ? 1 : 0)) * 16;
    *row1 = r1 < end ? r1 : end;
}

template <int BM, int MIN_PART_KTILES>
__device__ __forceinline__ WorkItem decode_work_item(const void* offsets, int off64, int E, int ntiles_n, int ktiles,
                                                     int max_split, int ncu)
{
    // 32-bit throughout (a launch has fewer than 2^31 tiles): six 64-bit divisions and the shuffles of 64-bit scans made this lookup
    // 1.6 us of every tile, 4.0 where the kernel is cold; now 0.85 and 1.3 (the four launches of a 512-token step with d=256: 92 -> 85 us)
    WorkItem w = {};
    ExpertScan sc = scan_expert_tiles_from(offsets, off64, E, BM, 0);   // every wave sees 64 expert groups at once
    uint32_t mtiles = __builtin_amdgcn_readlane(sc.tiles_through, 63);
    for (int base = 64; base < E; base += 64) mtiles += __builtin_amdgcn_readlane(scan_expert_tiles_from(offsets, off64, E, BM, base).tiles_through, 63);
    const uint32_t T = mtiles * (uint32_t)ntiles_n;
    const uint32_t xcd = blockIdx.x % NXCD, q = blockIdx.x / NXCD;
    const uint32_t CH = (uint32_t)ncu / NXCD;   // compute units per XCD
    uint32_t t = 0;                             // output tile in the list (expert, n tile, m tile fastest)
    {
        // The T tiles are cut into F = (T / #CU) * #CU tiles that fill whole rounds of compute units and a remainder; the
        // remainder tiles' K ranges are split 2 or 4 ways (when that many parts still fit in one round), so that the
        // last round is a half or a quarter as long instead of leaving most compute units idle.  Whole-round tiles, few
        // rounds: each XCD takes one contiguous range of the tile list (for evenly sized groups that is one expert per
        // XCD, whose row tiles it re-reads from nearby caches).  Many rounds: consecutive chunks of one XCD's worth of
        // tiles go to consecutive XCDs instead -- a chunk still runs side by side on its XCD (its tiles share weight and
        // row tiles in that L2), but every XCD sees every part of the list, which evens out the cheaper tiles of ragged
        // groups (measured: the gate/up launch, 16 rounds, 3 % faster dealt out in chunks, the 9-round launches of a
        // skewed 16384-token batch 8 %).  Launches of two or three rounds are dealt out the same way: over eight routing
        // draws of 8192 rows their two N-contiguous launches run 1-2 % faster than with contiguous ranges (0.4 % of the
        // layer's GEMM time on average, 1 % on the default draw, and no slower with evenly sized groups), while the
        // 7-round launch with the SwiGLU-backward epilogue measured 1.5 % slower dealt out and keeps its ranges.  Measured and
        // dropped for launches of few rounds: XCD ranges cut by the running cost of the tiles (32-row blocks, at
        // least half a tile) instead of by their number -- 4-7 % slower, with either way of splitting the last tiles.
        const uint32_t F = T / (uint32_t)ncu * (uint32_t)ncu;
        const int rem = (int)(T - F);
        int split = 1, lg = 0;
        while (split * 2 <= max_split && rem * split * 2 <= ncu && (ktiles >> (lg + 1)) >= MIN_PART_KTILES) { split *= 2; ++lg; }
        const uint32_t S = (uint32_t)rem * split;        // items of the last round
        const uint32_t Fx = F / NXCD;
        const uint32_t Sx = (S + NXCD - 1) / NXCD;
        if (q < Fx) {
            const bool deal = F >= (uint32_t)(INTERLEAVE_MIN_ROUNDS * ncu) || F < (uint32_t)(CONTIGUOUS_MIN_ROUNDS * ncu);
            if (deal) { const uint32_t c = q / CH; t = (c * NXCD + xcd) * CH + (q - c * CH); }
            else t = xcd * Fx + q;
        } else {
            const uint32_t j = xcd * Sx + (q - Fx);
            if (q - Fx >= Sx || j >= S) return w;
            t = F + (j >> lg);
            w.part = (int)(j & (split - 1));
            w.nparts = split;
            w.split_item = (int)j;
            w.split_tile = (int)(j >> lg);
        }
    }
    if (w.nparts == 0) w.nparts = 1;
    uint32_t before_block = 0;   // row tiles of the experts before `base`
    for (int base = 0; base < E; base += 64) {
        if (base > 0) sc = scan_expert_tiles_from(offsets, off64, E, BM, base);
        const uint32_t tl = t - before_block * (uint32_t)ntiles_n;
        const unsigned long long hit = __ballot(tl >= (uint32_t)sc.tiles_before * (uint32_t)ntiles_n && tl < (uint32_t)sc.tiles_through * (uint32_t)ntiles_n);
        if (hit == 0) { before_block += __builtin_amdgcn_readlane(sc.tiles_through, 63); continue; }
        // everything derived from the item is uniform and belongs in scalar registers
        const int hl = __ffsll(hit) - 1;
        const int64_t start = readlane_i64(sc.start, hl), end = readlane_i64(sc.end, hl);
        const uint32_t before = __builtin_amdgcn_readlane(sc.tiles_before, hl), mte = __builtin_amdgcn_readlane(sc.tiles_through, hl) - before;
        const uint32_t local = tl - before * (uint32_t)ntiles_n, nt = local / mte, mt = local - nt * mte;
        int64_t row0, row1;
        even_rows(start, end, mt, mte, &row0, &row1);
        w.expert = __builtin_amdgcn_readfirstlane(base + hl);
        w.nt = __builtin_amdgcn_readfirstlane((int)nt);
        w.row0 = uniform_i64(row0);
        w.row1 = uniform_i64(row1);
        w.mtile = __builtin_amdgcn_readfirstlane((int)(before_block + before + mt));
        w.only_tile = __builtin_amdgcn_readfirstlane((int)(mte == 1)) != 0;
        w.valid = true;
        break;
    }
    w.part = __builtin_amdgcn_readfirstlane(w.part);
    w.nparts = __builtin_amdgcn_readfirstlane(w.nparts);
    w.split_item = __builtin_amdgcn_readfirstlane(w.split_item);
    w.split_tile = __builtin_amdgcn_readfirstlane(w.split_tile);
    return w;
}

}  // namespace

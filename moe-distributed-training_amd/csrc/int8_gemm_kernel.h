// Grouped product of 8-bit codes over ragged expert groups on the gfx950 matrix cores (signed 8-bit in, exact 32-bit sums):
//
//   Y[out_row(m)][n] = x_scale[in_row(m)] * w_scale[e(m)][n] * sum_seg sum_k X[in_row(m)][seg][k] W_seg[e(m)][k][n]
//
// The structure is that of grouped_gemm_kernel.h: a K tile of 128 codes is a row of 128 bytes, as 64 bf16 values are, and a 16x16x64 step of
// 8-bit integers takes the same 16 bytes per lane and the same cycles as a 16x16x32 step of bf16.  So the same images, rings and waits carry twice
// the products.  Tiles of 256 x 256 (8 waves of 128 x 64, one workgroup per compute unit) or 128 x 128 (4 waves of 64 x 64, two).
//   - X tiles (two stages) and W tiles (three) come HBM -> LDS by direct 16-byte loads; XOR-swizzled images, ds_read_b128 fragments where the
//     operand is contiguous along k, ds_read_b64_tr_b8 where W is contiguous along n.
//   - Codes of X rows are padded with zeros to whole K tiles, so what stands in W's image behind K does not matter; only addresses do (KTAIL).
//   - The sums are integers: K parts of a tile may be added in any order, with one result.
//   - Epilogues: the scaled product in the output's type; the same as 24-bit integers with a scale per 32 columns (for the next product's codes);
//     or SwiGLU of a gate and an up product in that form.
//
// Included by one translation unit per tile size (MOE_I8_TILE: 256 or 128).
#pragma once
#include "gemm_tiles.h"
#include "kernels.h"

namespace {

constexpr int BM = MOE_I8_TILE, BN = MOE_I8_TILE, BK = MOE_I8_KTILE;
constexpr int NWAVES = BM / 32, NTHREADS = NWAVES * 64;
constexpr int WGS_PER_CU = 256 / BM;
constexpr int WAVES_N = NWAVES / 2;
constexpr int WTM = BM / 2, WTN = BN / WAVES_N;     // a wave's rows and columns: 128 or 64, 64
constexpr int MB = WTM / 16, NB = WTN / 16, NBH = NB / 2, MBH = MB / 2;
constexpr int LPT = BM / 8 / NWAVES;                // direct-to-LDS load instructions per wave, operand and K tile
constexpr int A_STAGE_BYTES = BM * BK, B_STAGE_BYTES = BN * BK;
constexpr int B_REGION = 2 * A_STAGE_BYTES;
constexpr int LDS_BYTES = B_REGION + 3 * B_STAGE_BYTES;   // 160 or 80 KiB
// Row and scale tables borrow the third weight stage: it is empty before the main loop's first tile, and behind the epilogue's staging after the last.
constexpr int TABLE_OFF = B_REGION + 2 * B_STAGE_BYTES;
static_assert(TABLE_OFF >= NWAVES * WTM * WTN * 2, "epilogue staging must not reach the tables");
constexpr int MIN_PART_KTILES = MOE_I8_MIN_PART;    // K tiles of a split tile's part, at least
static_assert(NTHREADS == BM + BN && WTN == 2 * MOE_SEG_COLS, "a thread brings one row's or one column's scale; a wave holds two segments per row");

typedef int i8frag_t __attribute__((ext_vector_type(4)));   // 16 codes of a lane
typedef int i32x2_t __attribute__((ext_vector_type(2)));

// NN: W contiguous along n.  KTAIL: K is no multiple of the K tile.
template <bool NN, int EPI, bool KTAIL>
__global__ void __launch_bounds__(NTHREADS, 2) i8_gemm_kernel(const MoeI8Gemm p)
{
    constexpr bool PAIR = EPI == MOE_I8_SWIGLU, TWO_SEG = EPI == MOE_I8_STORE;
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    int64_t* s_row = (int64_t*)(smem + TABLE_OFF);      // input rows before the loop, output rows after it
    float* s_xscale = (float*)(s_row + BM);
    float* s_wscale = s_xscale + BM;
    int* s_arrival = (int*)(s_wscale + BN);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;
    const int ntiles_n = PAIR ? (int)((p.N + BN / 2 - 1) / (BN / 2)) : (int)((p.N + BN - 1) / BN);
    const int ktiles_seg = (int)((p.K + BK - 1) / BK);
    const int ktiles = TWO_SEG ? ktiles_seg * p.nseg : ktiles_seg;
    const WorkItem item = decode_work_item<BM, MIN_PART_KTILES>(p.offsets, p.off64, p.E, ntiles_n, ktiles, p.max_split, p.num_cus);
    if (!item.valid) return;
    const int expert = item.expert, nt = item.nt, part = item.part, nparts = item.nparts;
    const int64_t row0 = item.row0;
    const int nrows = (int)(item.row1 - row0);
    // the two rows of waves share the tile's 16-row blocks
    const int nblocks = (nrows + 15) / 16, wrow0 = __builtin_amdgcn_readfirstlane(wm * ((nblocks + 1) / 2) * 16);
    const int wrows = __builtin_amdgcn_readfirstlane(wm == 0 ? (nrows < ((nblocks + 1) / 2) * 16 ? nrows : ((nblocks + 1) / 2) * 16) : (nrows > wrow0 ? nrows - wrow0 : 0));
    const int64_t n0 = (int64_t)nt * (PAIR ? BN / 2 : BN);

    // input rows; a thread of the first half also holds its row's scale until the epilogue, one of the second half a column's
    float my_scale = 1.f;
    if (tid < BM) {
        const int64_t m = row0 + (tid < nrows ? tid : nrows - 1);   // rows past the group re-read its last row
        const int64_t in_row = p.x_grouped ? m : load_idx(p.pos, m, p.pos64) / p.fan_out;
        s_row[tid] = in_row;
        my_scale = p.x_scale[in_row];
    } else {
        const int c = tid - BM;
        int64_t n = PAIR ? n0 + (c & (BN / 2 - 1)) : n0 + c;
        if (n >= p.N) n = p.N - 1;
        const float* ws = PAIR && c >= BN / 2 ? p.w_scale[1] : p.w_scale[0];
        if (ws) my_scale = ws[(int64_t)expert * p.N + n];
    }
    __syncthreads();

    // ---- per-lane offsets of the direct-to-LDS loads (the K tile's offset is added per tile).  Image of a K-contiguous operand: row r at r*128 bytes, its
    // 16-byte chunk c at slot c ^ ((r >> 1) & 7): the 16 rows of a fragment read meet 16 different bank groups.  Wave w's instruction j fills rows [(j*NWAVES + w)*8, +8).
    // SEGMENTS: the columns of a wave's blocks 2 s and 2 s + 1 are dealt to their MFMA rows so that a lane ends up with 8 consecutive columns of a
    // 32-column segment: row i of block b is column 8 (i >> 2) + 4 b + (i & 3).  W's image is swizzled for that set of rows instead.
    constexpr bool SEGMENTS = EPI != MOE_I8_STORE;
    static_assert(!NN || !SEGMENTS, "segments are written for K-contiguous weights");
    auto b_swizzle = [](int r) { return SEGMENTS ? ((r >> 1) & 1) | (((r >> 3) & 3) << 1) : (r >> 1) & 7; };
    const int64_t a_row_base = p.x_grouped ? row0 : 0;
    uint32_t a_off[LPT], b_off[LPT];
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
        const int r = (j * NWAVES + wave) * 8 + (lane >> 3);
        a_off[j] = (uint32_t)((s_row[r] - a_row_base) * p.ldx + ((lane & 7) ^ ((r >> 1) & 7)) * 16);
    }
    // (a masked load of KTAIL has an offset at or above the descriptor's range: zeros come back and memory is not touched)
    constexpr uint32_t LOAD_RANGE = KTAIL ? 0x80000000u : 0xFFFFFFFFu, OUT_OF_RANGE = 0xFFFFFFF0u;
    const i32x4_t a_buf = make_buffer(p.X + a_row_base * p.ldx);
    const i32x4_t b_buf0 = make_buffer(p.W[0] + (int64_t)expert * p.swe, LOAD_RANGE);
    const i32x4_t b_buf1 = make_buffer(((TWO_SEG && p.nseg > 1) || PAIR ? p.W[1] : p.W[0]) + (int64_t)expert * p.swe, LOAD_RANGE);
    constexpr int NCH = BN / 16, KROWS = 64 / NCH;   // N-contiguous image [128 k][BN n]: 16-byte chunks and rows of an instruction
    // ... chunk (k, c) at slot c ^ x(k).  A transposing fragment read touches rows 16 g + 0..7 (g = 0..3) of one chunk column; 256 bytes span the 64 banks, one row
    // of 256 columns or two of 128, and x sends those 32 pieces to every 16-byte bank group twice, as few times as 512 bytes allow.
    auto nn_swizzle = [](int k) { return BN == 256 ? (k & 7) | (((k >> 4) & 1) << 3) : ((k >> 1) & 3) | (((k >> 4) & 1) << 2); };
#pragma unroll
    for (int j = 0; j < LPT; ++j) {
        if (!NN) {
            const int r = (j * NWAVES + wave) * 8 + (lane >> 3);
            int64_t n = PAIR ? n0 + (r & (BN / 2 - 1)) : n0 + r;
            if (n >= p.N) n = p.N - 1;
            b_off[j] = (uint32_t)(n * p.ldw + ((lane & 7) ^ b_swizzle(r)) * 16);
        } else {
            const int k = (j * NWAVES + wave) * KROWS + lane / NCH;
            int64_t n = n0 + ((lane & (NCH - 1)) ^ nn_swizzle(k)) * 16;
            if (n >= p.N) n = 0;
            b_off[j] = (uint32_t)((int64_t)k * p.ldw + n);
        }
    }

    // ---- per-lane LDS fragment offsets.  A 16x16x64 operand: lane l holds row (l & 15), codes 16 * (l >> 4) .. + 15 of a 64-wide step, one chunk.
    int a_frag_off[2], b_frag_off[NN ? NB : 2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) a_frag_off[ks] = (wrow0 + (lane & 15)) * 128 + (((ks * 4 + (lane >> 4)) ^ ((lane >> 1) & 7)) << 4);
    if (!NN) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int r = SEGMENTS ? 8 * ((lane & 15) >> 2) + (lane & 3) : lane & 15;
            b_frag_off[ks] = r * 128 + (((ks * 4 + (lane >> 4)) ^ b_swizzle(r)) << 4);
        }
    } else {
        // transposing reads: of a group g of 16 lanes, lane i fetches 8 columns (half i & 1 of the block's 16) at k row 16 g + (i >> 1), a second read 8 rows further
        // down; the hardware hands lane i the 8 codes of column i
        const int g = lane >> 4, i = lane & 15, krow = 16 * g + (i >> 1);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) b_frag_off[nb] = (krow * NCH + ((wn * (WTN / 16) + nb) ^ nn_swizzle(krow))) * 16 + (i & 1) * 8;
    }

    i8frag_t acc[MB][NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = (i8frag_t){0, 0, 0, 0};
    const int mb_cnt = __builtin_amdgcn_readfirstlane((wrows + 15) / 16);   // 16-row blocks of this wave that hold a row (scalar: selects the copy of the loop)
    const int kb = ktiles * part / nparts, ke = ktiles * (part + 1) / nparts;

    const uint32_t smem_u = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(smem) + wave * 1024);   // this wave's 1 KiB of the image that a round of load instructions fills
    const int live_rows = (nrows + 31) / 32 * 32;
    const uint32_t tail_k = (uint32_t)(((lane & 7) ^ b_swizzle(wave * 8 + (lane >> 3))) * 16);   // k of this lane's chunk within W's K-contiguous image (the same for every instruction)
    // Only tile of its group: K tiles are walked from a start that differs between output tiles, so that all workgroups' pieces do not lie on a few memory
    // channels; and the weight loads are non-temporal (nobody else reads them).
    const int krot = __builtin_amdgcn_readfirstlane((int)((uint32_t)(nt + expert * 8) % (uint32_t)(ke - kb)));
    auto tile_of = [&](int kt, auto once) {
        kt = __builtin_amdgcn_readfirstlane(kt < ke ? kt : ke - 1);   // tiles past the end re-read the last one, into a stage that nobody reads any more
        if constexpr (decltype(once)::value) {
            kt += krot;
            if (kt >= ke) kt -= ke - kb;
        }
        return kt;
    };
    auto issue_a = [&](int kt, int j, int stage, bool ragged, auto once) {
        kt = tile_of(kt, once);
        if (!ragged || (j * NWAVES + wave) * 8 < live_rows)
            load_to_lds_16(a_buf, a_off[j], (uint32_t)kt * BK, smem_u + stage * A_STAGE_BYTES + j * (NWAVES * 1024));
    };
    auto issue_b = [&](int kt, int j, int stage, auto once) {
        constexpr bool NT = decltype(once)::value;
        kt = tile_of(kt, once);
        const int seg = TWO_SEG && kt >= ktiles_seg ? 1 : 0;
        const uint32_t k0 = (uint32_t)(kt - seg * ktiles_seg) * BK;
        const bool second = PAIR ? j >= LPT / 2 : seg != 0;
        uint32_t voff = b_off[j], soff = NN ? k0 * (uint32_t)p.ldw : k0;
        if constexpr (KTAIL) {
            if (k0 + BK > (uint32_t)p.K) {
                const bool in = NN ? k0 + (uint32_t)((j * NWAVES + wave) * KROWS + lane / NCH) < (uint32_t)p.K : k0 + tail_k < (uint32_t)p.K;
                voff = in ? voff + soff : OUT_OF_RANGE;
                soff = 0;
            }
        }
        load_to_lds_16<NT>(second ? b_buf1 : b_buf0, voff, soff, smem_u + B_REGION + stage * B_STAGE_BYTES + j * (NWAVES * 1024));
    };
    // The weight fragment is the MFMA's first operand: a lane ends up with 4 consecutive output columns of one row.
    auto read_b1 = [&](const uint8_t* b_lds, int ks, int nb, i8frag_t* bfrag) {
        if (!NN) {
            const int b = SEGMENTS ? (nb % NBH) * 4 : (nb % NBH) * 16;
            const int brow = (PAIR ? (nb / NBH) * (BN / 2) + wn * (WTN / 2) : wn * WTN + (nb / NBH) * (WTN / 2)) + b;
            bfrag[nb] = *(const i8frag_t*)(b_lds + brow * 128 + b_frag_off[ks]);
        } else {
            const uint8_t* bp = b_lds + b_frag_off[nb] + ks * 64 * BN;
            const i32x2_t lo = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)LDS_PTR(bp));
            const i32x2_t hi = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)LDS_PTR(bp + 8 * BN));
            bfrag[nb] = (i8frag_t){lo.x, lo.y, hi.x, hi.y};
        }
    };
    auto read_a1 = [&](const uint8_t* a_lds, int ks, int mh, int mb, i8frag_t* afrag) { afrag[mb] = *(const i8frag_t*)(a_lds + (mh * MBH + mb) * 16 * 128 + a_frag_off[ks]); };

    // Software pipeline, as in grouped_gemm_kernel.h (measurements there): a K tile in four half steps (64 codes x half the rows), fragments fetched one half step
    // ahead, the tile's barrier before the last half step, whose MFMAs cover the next tile's first reads; loads and reads spread between the MFMAs.  X tile kt lives in X
    // stage (kt - kb) % 2, W tile kt in W stage (kt - kb) % 3; the half step behind a barrier requests X tile kt+2, the next two W tile kt+3, and the barrier
    // leaves the youngest LPT loads, W's, in flight.  NBLK: the wave's 16-row blocks that take part; FULL: X loads of rows past the tile are issued all the same.
    constexpr int MFMAS_PER_STEP = MBH * NB, READ_GAP = MFMAS_PER_STEP / 8, A_LOAD_GAP = MFMAS_PER_STEP / 4, B_LOAD_GAP = MFMAS_PER_STEP / 2;
    static_assert((NB + MBH) * READ_GAP <= MFMAS_PER_STEP && LPT * A_LOAD_GAP <= MFMAS_PER_STEP && LPT * B_LOAD_GAP <= 3 * MFMAS_PER_STEP, "reads and loads are issued inside their half steps");
    auto mainloop = [&](auto nblk_tag, auto full_tag, auto once) {
        constexpr int NBLK = decltype(nblk_tag)::value;
        constexpr bool FULL = decltype(full_tag)::value;
#pragma unroll
        for (int i = 0; i < LPT; ++i) issue_a(kb, i, 0, !FULL, once);
#pragma unroll
        for (int i = 0; i < LPT; ++i) issue_b(kb, i, 0, once);
#pragma unroll
        for (int i = 0; i < LPT; ++i) issue_a(kb + 1, i, 1, !FULL, once);
#pragma unroll
        for (int i = 0; i < LPT; ++i) issue_b(kb + 1, i, 1, once);
        // tile kb has landed (without FULL the number of X loads varies: those of tile kb+1 are waited for)
        __builtin_amdgcn_s_waitcnt(0x0F70 | (FULL ? 2 * LPT : LPT));
        __syncthreads();                            // (also: every wave has read the row table that shares W stage 2)
        i8frag_t af[2][MBH], bf[2][NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) read_b1(smem + B_REGION, 0, nb, bf[0]);
#pragma unroll
        for (int mb = 0; mb < MBH; ++mb) read_a1(smem, 0, 0, mb, af[0]);
        int bs = 0;
        for (int kt = kb; kt < ke; ++kt) {
            const int as = (kt - kb) & 1;
            const int bs1 = bs == 2 ? 0 : bs + 1, bs2 = bs1 == 2 ? 0 : bs1 + 1;
            const uint8_t* a_lds = smem + as * A_STAGE_BYTES;
            const uint8_t* b_lds = smem + B_REGION + bs * B_STAGE_BYTES;
#pragma unroll
            for (int hs = 0; hs < 4; ++hs) {
                const int cur_a = hs & 1, cur_b = hs >> 1, mh = hs & 1, nhs = (hs + 1) & 3;
                if (hs == 3) {
                    __builtin_amdgcn_s_waitcnt(0x0F70 | LPT);   // all but the youngest LPT loads: tile kt+1 has landed
                    __syncthreads();                            // for every wave, and every wave is done reading tile kt
                }
                const uint8_t* ra = hs == 3 ? smem + (as ^ 1) * A_STAGE_BYTES : a_lds;
                const uint8_t* rb = hs == 3 ? smem + B_REGION + bs1 * B_STAGE_BYTES : b_lds;
                __builtin_amdgcn_sched_barrier(0);
                // (of the two waves of a SIMD the one that is behind issues first)
                if (nhs == 0) __builtin_amdgcn_s_setprio(3);
                else if (nhs == 1) __builtin_amdgcn_s_setprio(2);
                else if (nhs == 2) __builtin_amdgcn_s_setprio(1);
                else __builtin_amdgcn_s_setprio(0);
#pragma unroll
                for (int m = 0; m < MFMAS_PER_STEP; ++m) {
                    const int mb = m / NB, nb = (mb & 1) ? NB - 1 - m % NB : m % NB;   // from one MFMA to the next only one operand changes
                    if (m % READ_GAP == 0) {
                        const int nbr = (nhs & 1) == 0 ? NB : 0, q = m / READ_GAP;
                        if (q < nbr) { if (NBLK > 0) read_b1(rb, nhs >> 1, q, bf[cur_b ^ 1]); __builtin_amdgcn_sched_barrier(0); }
                        else if (q - nbr < MBH) { if ((nhs & 1) * MBH + (q - nbr) < NBLK) read_a1(ra, nhs >> 1, nhs & 1, q - nbr, af[cur_a ^ 1]); __builtin_amdgcn_sched_barrier(0); }
                    }
                    if (hs == 3 && m % A_LOAD_GAP == 0 && m / A_LOAD_GAP < LPT) {
                        issue_a(kt + 2, m / A_LOAD_GAP, as, !FULL, once);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    const int gb = hs * MFMAS_PER_STEP + m;
                    if (hs < 3 && gb % B_LOAD_GAP == 0 && gb / B_LOAD_GAP < LPT) {
                        issue_b(kt + 2, gb / B_LOAD_GAP, bs2, once);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if (mh * MBH + mb < NBLK)
                        acc[mh * MBH + mb][nb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[cur_b][nb], af[cur_a][mb], acc[mh * MBH + mb][nb], 0, 0, 0);
                }
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            bs = bs1;
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);   // loads past the last tile must not land in the epilogue's staging
        __syncthreads();
    };
    using T_ = std::true_type;
    using F_ = std::false_type;
    if (nblocks > MB || !item.only_tile) {   // more than half a tile, or one of several tiles of a group, whose rows are dealt evenly
        if (item.only_tile) {
            if (MB == 8 && mb_cnt <= 6) mainloop(std::integral_constant<int, MB * 3 / 4>{}, T_{}, T_{});
            else mainloop(std::integral_constant<int, MB>{}, T_{}, T_{});
        } else if (mb_cnt == MB) mainloop(std::integral_constant<int, MB>{}, T_{}, F_{});
        else if (mb_cnt == MB - 1) mainloop(std::integral_constant<int, MB - 1>{}, T_{}, F_{});
        else if (MB == 8 && mb_cnt == 6) mainloop(std::integral_constant<int, MB * 3 / 4>{}, T_{}, F_{});
        else if (MB == 8 && mb_cnt == 5) mainloop(std::integral_constant<int, MB / 2 + 1>{}, T_{}, F_{});
        else mainloop(std::integral_constant<int, MBH>{}, T_{}, F_{});
    } else if (mb_cnt > 2) mainloop(std::integral_constant<int, MBH>{}, F_{}, T_{});
    else if (mb_cnt == 2) mainloop(std::integral_constant<int, 2>{}, F_{}, T_{});
    else if (mb_cnt == 1) mainloop(std::integral_constant<int, 1>{}, F_{}, T_{});
    else mainloop(std::integral_constant<int, 0>{}, F_{}, T_{});

    // ---- K parts of a split tile; nobody waits for anybody.
    // Tiles of 128: every part adds its sums to the launch's (zeroed) matrix of sums by device-scope atomics and then bumps the tile's counter; the part that finds
    // all others counted takes the complete sums out, leaving zeros for the next launch.  Integers: the order does not matter.  Data and counter move by
    // relaxed atomics alone, each awaited before the next: no fence, which writes back and empties whole L2 caches (with the parts in slots and fences as below, h W2 of
    // one token, 512 parts: 46 us).  Only rows that exist are moved.
    // Tiles of 256: a part's sums are too many for atomics; they go to a slot of their own by device-scope stores, and the last part adds the others' to its own.
    if (nparts > 1) {
        if constexpr (BM == 128) {
            const int g = lane >> 4;
            const int64_t m0 = row0 + wrow0 + (lane & 15);
            auto each = [&](auto fn) {   // (sum, where it lies) of every element of this lane that exists
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
                    if (mb * 16 + (lane & 15) < wrows)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const int half = nb / NBH, b = nb % NBH;
                            const int64_t n = n0 + (PAIR ? wn * (WTN / 2) : wn * WTN + half * (WTN / 2)) + (EPI != MOE_I8_STORE ? g * 8 + b * 4 : b * 16 + g * 4);
                            int* at = p.sk_partials + ((PAIR && half ? p.rows : 0) + m0 + mb * 16) * p.N + n;
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (n + r < p.N) fn(mb, nb, r, at + r);
                        }
            };
            each([&](int mb, int nb, int r, int* at) { (void)__hip_atomic_fetch_add(at, acc[mb][nb][r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's sums have been added
            __syncthreads();                                   // ... and every wave's
            if (tid == 0) *s_arrival = __hip_atomic_fetch_add(&p.sk_counters[item.split_tile], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (*s_arrival != nparts - 1) return;
            if (tid == 0) __hip_atomic_store(&p.sk_counters[item.split_tile], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("" ::: "memory");
            each([&](int mb, int nb, int r, int* at) { acc[mb][nb][r] = __hip_atomic_exchange(at, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); });
        } else {
        constexpr int DEVICE_SCOPE = 16;
        const __amdgpu_buffer_rsrc_t xbuf = __builtin_amdgcn_make_buffer_rsrc(p.sk_partials, 0, (int)0x80000000u, 0x00020000);
        auto slot = [&](int x) { return (uint32_t)(item.split_item - part + x) * (uint32_t)(BM * BN * sizeof(int)); };
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
            if (mb < mb_cnt)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[mb][nb]), xbuf, slot(part) + (uint32_t)(((mb * NB + nb) * NTHREADS + tid) * 16), 0, DEVICE_SCOPE);
        __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's stores are acknowledged
        __syncthreads();                      // ... and every wave's
        if (tid == 0) *s_arrival = __hip_atomic_fetch_add(&p.sk_counters[item.split_tile], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (*s_arrival != nparts - 1) return;
        if (tid == 0) __hip_atomic_store(&p.sk_counters[item.split_tile], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // clean for the next launch
        for (int x = 0; x < nparts; ++x) {
            if (x == part) continue;
            const uint32_t at = slot(x);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if (mb < mb_cnt) {
                    u32x4_t v[NB];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) v[nb] = __builtin_amdgcn_raw_buffer_load_b128(xbuf, at + (uint32_t)(((mb * NB + nb) * NTHREADS + tid) * 16), 0, DEVICE_SCOPE);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) acc[mb][nb] += __builtin_bit_cast(i8frag_t, v[nb]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        }
    }

    // ---- epilogue: acc[mb][nb][r] is (row mb*16 + lane%16, column nb*16 + (lane/16)*4 + r) of the wave's sub-tile; SEGMENTS: column (lane/16)*8 + (nb%2)*4 + r of
    // segment nb/2
    if (tid < BM) {
        s_xscale[tid] = my_scale;
        if (!p.y_grouped) s_row[tid] = load_idx(p.pos, row0 + (tid < nrows ? tid : nrows - 1), p.pos64);
    } else s_wscale[tid - BM] = my_scale;
    __syncthreads();
    if constexpr (SEGMENTS) {
        const int64_t segs = p.N / MOE_SEG_COLS;
        const int g = lane >> 4;
        // The tile's scales are gathered in LDS and written behind the codes, whole pieces of a row: one by one they made a third of the launch's store requests.
        constexpr int SEGS = (PAIR ? BN / 2 : BN) / MOE_SEG_COLS;   // per row and output
        float* s_seg = (float*)smem;
        static_assert(3 * BM * SEGS * 4 <= TABLE_OFF, "segment scales lie in front of the tables");
        // Segment h of the wave's rows in block mb (value(i): element i of this lane's 8, times row_scale): four lanes hold a row's 32 values, whose
        // maximum gives the scale; a lane stores the upper 16 bits of its 8 codes and then their lower 8, the four lanes of a row side by side.
        auto put_segment = [&](int mb, auto value, float row_scale, uint8_t* out, float* scales, int seg) {
            const int64_t ncol = n0 + seg * MOE_SEG_COLS;
            if (ncol >= p.N) return;
            float v[8];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                v[i] = value(i);
                v[i + 1] = value(i + 1);
                top = max(max(__float_as_uint(v[i]) & 0x7fffffffu, __float_as_uint(v[i + 1]) & 0x7fffffffu), top);   // (bits: NaN above infinity above every number)
            }
            auto pair = __builtin_amdgcn_permlane16_swap(top, top, false, false);
            top = max(pair[0], pair[1]);
            pair = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = max(pair[0], pair[1]);
            float amax = __uint_as_float(top), inv = MOE_SEG_LEVELS * __builtin_amdgcn_rcpf(amax);
            if (__any(top - 0x1f800000u > 0x5f800000u - 0x1f800000u)) {   // not 2^-64 .. 2^64
                // (magnitudes whose steps per unit would leave fp32's range are multiplied by a power of two first; zeros; a segment that is not finite: its scale says NaN)
                const bool fine = top < 0x7f800000u;
                const float by = amax > 0x1p64f ? 0x1p-64f : amax < 0x1p-64f ? 0x1p64f : 1.f;
                inv = fine && amax > 0.f ? MOE_SEG_LEVELS * __builtin_amdgcn_rcpf(amax * by) : 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fine ? v[i] * by : 0.f;
                amax = fine ? amax : __uint_as_float(0x7fc00000u);
            }
            int q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = (int)rintf(v[i] * inv);
            u32x4_t hi;
            uint2 lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) hi[i] = __builtin_amdgcn_perm((uint32_t)q[2 * i + 1], (uint32_t)q[2 * i], 0x06050201u);
            lo.x = __builtin_amdgcn_perm((uint32_t)q[1], (uint32_t)q[0], 0x0c0c0400u) | __builtin_amdgcn_perm((uint32_t)q[3], (uint32_t)q[2], 0x04000c0cu);
            lo.y = __builtin_amdgcn_perm((uint32_t)q[5], (uint32_t)q[4], 0x0c0c0400u) | __builtin_amdgcn_perm((uint32_t)q[7], (uint32_t)q[6], 0x04000c0cu);
            const int m = mb * 16 + (lane & 15);
            if (m < wrows) {
                const int64_t at = (row0 + wrow0 + m) * segs + ncol / MOE_SEG_COLS;
                uint8_t* to = out + at * MOE_SEG_BYTES;
                *(u32x4_t*)(to + g * 16) = hi;
                *(uint2*)(to + 64 + g * 8) = lo;
                if (g == 0) scales[(wrow0 + m) * SEGS + seg] = amax * row_scale;   // (zeros of a row whose scale is NaN are NaN)
            }
        };
        auto xs = [&](int mb) { return s_xscale[wrow0 + mb * 16 + (lane & 15)]; };
        if (EPI == MOE_I8_SEG) {   // (without column scales: the maximum of the sums themselves)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if (mb >= mb_cnt) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h)   // (both segments of a row block together: their 192 bytes meet in the cache)
                    put_segment(mb, [&](int i) { return (float)acc[mb][2 * h + i / 4][i % 4]; }, xs(mb), p.S[0], s_seg, wn * 2 + h);
            }
        } else {   // SwiGLU: gate = acc[mb][b], up = acc[mb][NBH + b] at the same row and column
            float wg[8], wu[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                wg[i] = s_wscale[wn * (WTN / 2) + g * 8 + i];
                wu[i] = s_wscale[BN / 2 + wn * (WTN / 2) + g * 8 + i];
            }
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if (mb >= mb_cnt) continue;
                const float x = xs(mb);
                // (the hardware's exponential and reciprocal, off by 1 in the last place each: beside the roundings of a, u and the segment)
                put_segment(mb, [&](int i) {
                    const float a = (float)acc[mb][i / 4][i % 4] * x * wg[i], u = (float)acc[mb][NBH + i / 4][i % 4] * x * wu[i];
                    return a * __builtin_amdgcn_rcpf(1.f + __expf(-a)) * u;
                }, 1.f, p.S[0], s_seg, wn);
                if (p.S[1]) {
                    put_segment(mb, [&](int i) { return (float)acc[mb][i / 4][i % 4] * wg[i]; }, x, p.S[1], s_seg + BM * SEGS, wn);
                    put_segment(mb, [&](int i) { return (float)acc[mb][NBH + i / 4][i % 4] * wu[i]; }, x, p.S[2], s_seg + 2 * BM * SEGS, wn);
                }
            }
        }
        __syncthreads();
        const int64_t seg0 = n0 / MOE_SEG_COLS;
#pragma unroll
        for (int out = 0; out < (PAIR ? 3 : 1); ++out) {
            if (!p.SS[out]) continue;
            for (int i = tid; i < nrows * (SEGS / 2); i += NTHREADS) {   // (segments come in pairs: N is a multiple of 64)
                const int r = i / (SEGS / 2), c = i % (SEGS / 2) * 2;
                if (seg0 + c < segs) *(float2*)(p.SS[out] + (row0 + r) * segs + seg0 + c) = *(const float2*)(s_seg + (out * BM + r) * SEGS + c);
            }
        }
        return;
    }
    const int mrow = lane & 15, nq = (lane >> 4) * 4;
    uint8_t* stg = smem + wave * (WTM * WTN * 2);   // 16-bit values of the wave's sub-tile
    auto swz = [](int sw, int m, int c) { return c ^ ((m / (sw >= 128 ? 1 : 128 / sw)) & (sw / 8 - 1)); };
    auto stage_put = [&](int sw, int m, int ncol, uint2 v) { *(uint2*)(stg + m * (sw * 2) + (swz(sw, m, ncol >> 3) << 4) + ((ncol >> 2) & 1) * 8) = v; };
    // the staged sub-tile of sw columns to grouped rows, or rows of the table, of a 16-bit matrix: 16 bytes per lane, whole row segments
    auto stage_flush = [&](int sw, uint16_t* Y, int64_t ld, bool scattered, int64_t ncol0, bool vec) {
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): this wave's staging writes have landed
        const int lpr = sw / 8, rows_per_it = 64 / lpr, slot = lane % lpr;
        const int iters = (wrows + rows_per_it - 1) / rows_per_it;
        for (int it = 0; it < iters; ++it) {
            const int m = it * rows_per_it + lane / lpr;
            const u32x4_t v = *(const u32x4_t*)(stg + m * (sw * 2) + slot * 16);
            const int64_t n = ncol0 + swz(sw, m, slot) * 8;
            if (m >= wrows || n >= p.N) continue;
            uint16_t* y = Y + (scattered ? s_row[wrow0 + m] : row0 + wrow0 + m) * ld + n;
            if (vec) *(u32x4_t*)y = v;
            else
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (n + i < p.N) y[i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
        }
        __builtin_amdgcn_s_waitcnt(0xC07F);   // reads done before the slice is reused
    };
    auto column_scales = [&](int nb, float* w) {   // of this lane's four columns of block nb
        const float4 v = *(const float4*)(s_wscale + wn * WTN + nb * 16 + nq);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    };
    {
        float w[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) column_scales(nb, w[nb]);
        const int64_t ncol0 = n0 + wn * WTN;
        // Sum times row scale times column scale.  FAR: where the first product could leave fp32's range (rows of 2^71 on) the row scale comes 2^40 times smaller, and what
        // it comes to is as much larger again: powers of two round nothing.  (A copy of its own for waves that have such rows: as a branch or a select around each product
        // the products of 64 narrow experts took 110 -> 115 us.)
        auto write = [&](auto far_tag) {
            constexpr bool FAR = decltype(far_tag)::value;
            auto values = [&](int mb, int nb, float xs, float* v) {
                const bool much = FAR && xs > 0x1p64f;
                const float x = much ? xs * 0x1p-40f : xs;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = (float)acc[mb][nb][r] * x * w[nb][r];
                    if (FAR) v[r] = much ? v[r] * 0x1p40f : v[r];
                }
            };
            if (p.ydtype == MOE_F32) {
                const bool vec = p.y_vec;
#pragma unroll
                for (int mb = 0; mb < MB; ++mb) {
                    const int m = mb * 16 + mrow;
                    if (mb >= mb_cnt || m >= wrows) continue;
                    const float xs = s_xscale[wrow0 + m];
                    float* y = (float*)p.Y + (p.y_grouped ? row0 + wrow0 + m : s_row[wrow0 + m]) * p.ldy;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const int64_t n = ncol0 + nb * 16 + nq;
                        float v[4];
                        values(mb, nb, xs, v);
                        if (vec && n < p.N) *(float4*)(y + n) = make_float4(v[0], v[1], v[2], v[3]);
                        else
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (n + r < p.N) y[n + r] = v[r];
                    }
                }
                return;
            }
            const bool f16 = p.ydtype == MOE_F16;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if (mb >= mb_cnt) continue;
                const float xs = s_xscale[wrow0 + mb * 16 + mrow];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float v[4];
                    values(mb, nb, xs, v);
                    uint2 o;
                    if (f16) { o.x = NumF16::pack2(v[0], v[1]); o.y = NumF16::pack2(v[2], v[3]); }
                    else { o.x = NumBf16::pack2(v[0], v[1]); o.y = NumBf16::pack2(v[2], v[3]); }
                    stage_put(WTN, mb * 16 + mrow, nb * 16 + nq, o);
                }
            }
            stage_flush(WTN, (uint16_t*)p.Y, p.ldy, !p.y_grouped, ncol0, p.y_vec);
        };
        bool far = false;
#pragma unroll
        for (int i = 0; i < WTM; i += 64) far = far || s_xscale[wrow0 + i + lane] > 0x1p64f;   // (rows behind the wave's own are in the table as well)
        if (__builtin_expect(__any(far), 0)) write(T_{});
        else write(F_{});
    }
}

int64_t plan_grid(int64_t R, int E, int ntiles_n, int ncu)
{
    const int64_t grid = (R / BM + E) * ntiles_n + ncu;   // an upper bound on the tiles, and a round for the split items; surplus workgroups leave at once
    return (grid + NXCD - 1) / NXCD * NXCD;
}

template <bool NN, int EPI, bool KTAIL> int launch_typed(const MoeI8Gemm& p, int64_t R, hipStream_t stream)
{
    static std::atomic<bool> attr_set[MOE_MAX_DEVICES];
    auto kern = i8_gemm_kernel<NN, EPI, KTAIL>;
    const int dev = moe_current_device();
    if (!attr_set[dev]) {
        if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES) != hipSuccess) return MOE_ERR_LAUNCH;
        attr_set[dev] = true;
    }
    MoeI8Gemm q = p;
    q.num_cus = WGS_PER_CU * p.num_cus;
    const int cols = EPI == MOE_I8_SWIGLU ? BN / 2 : BN;
    const int64_t grid = plan_grid(R, p.E, (int)((p.N + cols - 1) / cols), q.num_cus);
    if (!moe_grid_fits(grid, NTHREADS)) return MOE_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(NTHREADS), LDS_BYTES, stream, q);
    return moe_launch_status();
}

template <bool NN, int EPI> int launch_tail(const MoeI8Gemm& p, int64_t R, hipStream_t stream)
{
    return p.K % BK ? launch_typed<NN, EPI, true>(p, R, stream) : launch_typed<NN, EPI, false>(p, R, stream);
}

int launch_epilogue(const MoeI8Gemm& p, int64_t R, hipStream_t stream)
{
    if (p.epi == MOE_I8_STORE) return p.nn ? launch_tail<true, MOE_I8_STORE>(p, R, stream) : launch_tail<false, MOE_I8_STORE>(p, R, stream);
    if (p.nn) return MOE_ERR_UNSUPPORTED;
    return p.epi == MOE_I8_SEG ? launch_tail<false, MOE_I8_SEG>(p, R, stream) : launch_tail<false, MOE_I8_SWIGLU>(p, R, stream);
}

}  // namespace

// Grouped product of 16-bit rows with 4-bit weights (fp4.h) on the matrix cores, both directions, tiles of 128 (or 112, or 96) rows x 256 columns:
//
//   forward:   Y[out_row(m)][n]  = sum_k X[in_row(m)][k] W[e(m)][n][k]
//   backward:  Y[out_row(m)][k] = c[m] sum_n X[in_row(m)][n] W[e(m)][n][k]      (X: gradient rows, c: their gate weights or 1)
//
// Four waves of 128 x 64, two workgroups per compute unit, which cover each other's barriers and first loads.  Rows of X and codes come HBM -> LDS by direct 16-byte loads, two stages of 64
// contraction steps each; codes stay 4-bit in LDS, a quarter of the weights' usual traffic there, and become operands on their way into the matrix instructions: one conversion
// per pair, 64 weights a wave and step of 32 against 32 matrix instructions.
//   Forward, codes run along the contraction: a lane reads 8 bytes of its column (16 inputs of one scale) per 64 steps; its inputs are 16 g + 8 j .. + 7, and so are those of the row operand.
//   Backward, the contraction runs over n, so a lane's 8 weights lie in 8 rows with a scale each: it reads two bytes of each (four columns), converts, and two moves of 16-bit
//   halves per pair of rows make four operands of it.
// Measured: 8192 rows of 8 experts x 4096 x 14336 forward 770 to 830 us by card = 1.16 to 1.25 PFLOP/s (matrix cores busy in 64 % of the cycles at 1.96 GHz; the library's dense product of
// these sizes runs at 1.52), 3000 rows of 4096 x 4096 forward 120 us, backward 125 us: 416 and 512 tiles on 512 places, so compute units hold two or one of them.
// Columns are dealt to the matrix instructions so that a lane ends up with 16 consecutive ones of a row.  Sums, gate weights and the rows that the caller sums further are fp32.
#include "fp4.h"
#include "gemm_tiles.h"
#include "kernels.h"

namespace {

constexpr int BM = 128, BN = 256, BK = 64, WAVES = 4, THREADS = WAVES * 64, WGS_PER_CU = 2;
constexpr int MB = BM / 16, NB = 4;
constexpr uint32_t RANGE = 0x80000000u;              // of the buffers, and an offset outside of them: 2 GiB (checked on the host)
constexpr int A_STAGE = BM * BK * 2;                 // 16 KiB: rows of 128 bytes
constexpr int B_STAGE = 16384;                       // forward: 256 columns x 64 bytes (128 inputs); backward: 64 rows x 128 bytes, half of it
constexpr int S_STAGE = 1024;                        // scales: forward 256 columns x 4, backward 64 rows x 8
constexpr int B_OFF = 2 * A_STAGE, S_OFF = B_OFF + 2 * B_STAGE, LDS_BYTES = S_OFF + 2 * S_STAGE;

// Which places of its eight a row's pieces are dealt to: place = piece ^ turn(row).  A 16-byte read of LDS takes lanes 0 .. 3, 12 .. 15 with 20 .. 27 and the like at a time, rows of one piece
// with those of the next lane group's: turn() gives {0, 1, 6, 7} and {2, 3, 4, 5} halves of their own, which neighbours one (backward) or two (forward) pieces apart keep.  (turn = row >> 1:
// every forward read in two passes, 17 % of a compute unit's cycles.)
__device__ __forceinline__ int turn(int row) { const int x = (row >> 1) & 7; return x ^ ((x & 2) << 1); }

// four bytes per lane, global -> LDS at lds_addr + 4 * lane (load_to_lds_16 otherwise)
__device__ __forceinline__ void load_to_lds_4(i32x4_t rsrc, uint32_t lane_off, uint32_t uniform_off, uint32_t lds_addr)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(lane_off), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(uniform_off)) : "memory", "m0");
}

// sixteen consecutive values of a row, `live` of which exist
__device__ __forceinline__ void store16(void* Y, int64_t at, int dtype, const float* v, int live, bool vec)
{
    if (dtype == MOE_F32) {
        float* y = (float*)Y + at;
        if (vec && live >= 16)
#pragma unroll
            for (int i = 0; i < 16; i += 4) *(float4*)(y + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        else
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i < live) y[i] = v[i];
        return;
    }
    uint16_t* y = (uint16_t*)Y + at;
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = dtype == MOE_BF16 ? NumBf16::pack2(v[2 * i], v[2 * i + 1]) : NumF16::pack2(v[2 * i], v[2 * i + 1]);
    if (vec && live >= 16)
#pragma unroll
        for (int i = 0; i < 8; i += 4) *(fp4_u32x4_t*)(y + 2 * i) = (fp4_u32x4_t){o[i], o[i + 1], o[i + 2], o[i + 3]};
    else
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < live) y[i] = (uint16_t)(o[i / 2] >> (16 * (i & 1)));
}

template <class Num, bool BWD, int ROWS>
__global__ void __launch_bounds__(THREADS, 2) fp4_tile_kernel(const MoeFp4Gemm p)
{
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, q = lane >> 4;
    const int64_t cols = BWD ? p.K : p.N;                       // of Y
    const int len = BWD ? (int)p.N : p.K;                       // of the contraction
    const int G = (p.K + FP4_GROUP - 1) / FP4_GROUP;
    const int ntiles_n = (int)((cols + BN - 1) / BN), ktiles = (len + BK - 1) / BK;
    const WorkItem item = decode_work_item<ROWS, 1>(p.offsets, p.off64, p.E, ntiles_n, ktiles, 1, p.num_cus);
    if (!item.valid) return;
    const int e = item.expert, nrows = (int)(item.row1 - item.row0), nblocks = (nrows + 15) / 16;
    const int64_t row0 = item.row0, n0 = (int64_t)item.nt * BN;

    // ---- where this lane's pieces of the images come from.  X: rows of 128 bytes, 16-byte piece c of row r at place c ^ turn(r); instruction j of wave w fills rows (4 j + w) * 8 ..
    const int64_t base = p.x_grouped ? row0 : 0;
    uint32_t a_off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = (4 * j + wave) * 8 + (lane >> 3);
        const int64_t m = row0 + (r < nrows ? r : nrows - 1);   // rows past the tile re-read its last one
        a_off[j] = (uint32_t)(((p.x_grouped ? m : load_idx(p.pos, m, p.pos64) / p.fan_out) - base) * p.ldx) * 2 + ((lane & 7) ^ turn(r)) * 16;
    }
    const int a_k = ((lane & 7) ^ turn(8 * wave + (lane >> 3))) * 8;   // this lane's first input within a stage (the same for every j)
    const i32x4_t a_buf = make_buffer((const uint16_t*)p.X + base * p.ldx, RANGE);
    const i32x4_t b_buf = make_buffer(p.w.codes + e * p.w.sce, RANGE), s_buf = make_buffer(p.w.scales + e * p.w.sse, RANGE);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(smem));
    const int live_rows = __builtin_amdgcn_readfirstlane((nrows + 31) / 32 * 32);   // an instruction of all waves fills 32 rows
    auto issue_a = [&](int kt, int stage) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (32 * j < live_rows) load_to_lds_16(a_buf, kt * BK + a_k < len ? a_off[j] : RANGE, kt * (BK * 2), lds0 + stage * A_STAGE + (4 * j + wave) * 1024);
    };
    // Forward: a wave's own 64 columns, piece c (one group of 32 inputs) of column x at place c ^ ((x >> 2) & 3); columns in the order of the matrix instructions.  Backward: 64 rows, piece c (32
    // columns) of row n at place c ^ 2 ((n >> 3) & 3); instruction j of wave w fills rows (4 j + w) * 8 ..
    uint32_t b_off[4], s_off;
    int b_piece, s_piece = 0;
    if constexpr (!BWD) {
        auto column = [&](int x) {   // x = 16 nb + c: column c of the wave's block nb
            const int64_t n = n0 + wave * 64 + ((x & 15) >> 2) * 16 + (x >> 4) * 4 + (x & 3);
            return n < p.N ? n : p.N - 1;
        };
        b_piece = (lane & 3) ^ (lane >> 4);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) b_off[nb] = (uint32_t)(column(16 * nb + (lane >> 2)) * p.w.scn) + b_piece * FP4_GROUP_BYTES;
        s_off = (uint32_t)(column(lane) * p.w.ssn);
    } else {
        b_piece = (int)(n0 / FP4_GROUP) + ((lane & 7) ^ (2 * (wave & 3)));
#pragma unroll
        for (int j = 0; j < 2; ++j) b_off[j] = (uint32_t)(((4 * j + wave) * 8 + (lane >> 3)) * p.w.scn) + b_piece * FP4_GROUP_BYTES;
        s_piece = (int)(n0 / FP4_GROUP) + (lane & 1) * 4;
        s_off = (uint32_t)(((wave & 1) * 32 + (lane >> 1)) * p.w.ssn) + s_piece;
    }
    // forward: unit u of 128 inputs; backward: stage kt of 64 rows
    auto issue_b = [&](int u, int stage) {
        if constexpr (!BWD) {
            const bool in = 4 * u + b_piece < G;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) load_to_lds_16(b_buf, in ? b_off[nb] : RANGE, u * 64, lds0 + B_OFF + stage * B_STAGE + (wave * 4 + nb) * 1024);
            load_to_lds_4(s_buf, s_off, u * 4, lds0 + S_OFF + stage * S_STAGE + wave * 256);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool in = b_piece < G && u * BK + (4 * j + wave) * 8 + (lane >> 3) < len;
                load_to_lds_16(b_buf, in ? b_off[j] + (uint32_t)(u * BK) * (uint32_t)p.w.scn : RANGE, 0, lds0 + B_OFF + stage * B_STAGE + (4 * j + wave) * 1024);
            }
            if (wave < 2) {
                const bool in = s_piece < G && u * BK + wave * 32 + (lane >> 1) < len;
                load_to_lds_4(s_buf, in ? s_off + (uint32_t)(u * BK) * (uint32_t)p.w.ssn : RANGE, 0, lds0 + S_OFF + stage * S_STAGE + wave * 256);
            }
        }
    };

    f32x4_t acc[MB][NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

    auto mainloop = [&](auto nblk) {
        constexpr int NBLK = decltype(nblk)::value;
        issue_a(0, 0);
        issue_b(0, 0);
        for (int kt = 0; kt < ktiles; ++kt) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // stage kt has landed
            __syncthreads();                                   // for every wave, and every wave is done with the stage before
            const int as = kt & 1, bs = BWD ? kt & 1 : (kt >> 1) & 1;
            if (kt + 1 < ktiles) issue_a(kt + 1, as ^ 1);
            if (BWD) { if (kt + 1 < ktiles) issue_b(kt + 1, bs ^ 1); }
            else if ((kt & 1) == 0 && kt + 2 < ktiles) issue_b((kt >> 1) + 1, bs ^ 1);
            __builtin_amdgcn_sched_barrier(0);
            const uint8_t *a_lds = smem + as * A_STAGE, *b_lds = smem + B_OFF + bs * B_STAGE, *s_lds = smem + S_OFF + bs * S_STAGE;
            uint2 codes[NB];
            float scale[NB];
            if constexpr (!BWD) {
                // inputs 16 q .. + 15 of this half of the unit: half a group
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const int piece = 2 * (kt & 1) + (q >> 1);
                    codes[nb] = *(const uint2*)(b_lds + (wave * 4 + nb) * 1024 + i * 64 + (piece ^ (i >> 2)) * 16 + (q & 1) * 8);
                    scale[nb] = fp4_scale(*(const uint32_t*)(s_lds + wave * 256 + (nb * 16 + i) * 4) >> (8 * piece) & 0xff);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8_t b[NB];
                if constexpr (!BWD) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) b[nb] = fp4_expand8<Num>(j ? codes[nb].y : codes[nb].x, scale[nb]);
                } else {
                    uint32_t v[8][2];   // columns 4 i, 4 i + 1 and 4 i + 2, 4 i + 3 of rows 32 j + 8 q + t
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const int n = 32 * j + 8 * q + t;
                        const uint32_t c = *(const uint16_t*)(b_lds + n * 128 + ((2 * wave + (i >> 3)) ^ (2 * q)) * 16 + (i & 7) * 2);
                        const float s = fp4_scale(s_lds[n * 8 + 2 * wave + (i >> 3)]);
                        v[t][0] = fp4_pair<Num, 0>(c, s);
                        v[t][1] = fp4_pair<Num, 1>(c, s);
                    }
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        fp4_u32x4_t w;
#pragma unroll
                        for (int t = 0; t < 4; ++t) w[t] = __builtin_amdgcn_perm(v[2 * t + 1][nb / 2], v[2 * t][nb / 2], nb & 1 ? 0x07060302u : 0x05040100u);
                        b[nb] = __builtin_bit_cast(bf16x8_t, w);
                    }
                }
                const int chunk = BWD ? 4 * j + q : 2 * q + j;
#pragma unroll
                for (int mb = 0; mb < NBLK; ++mb) {
                    const bf16x8_t a = *(const bf16x8_t*)(a_lds + (mb * 16 + i) * 128 + (chunk ^ turn(i)) * 16);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = Num::mfma(b[nb], a, acc[mb][nb]);
                }
            }
        }
    };
    if (ROWS > 96 && nblocks > 6) mainloop(std::integral_constant<int, ROWS == 112 ? 7 : 8>{});
    else if (nblocks > 4) mainloop(std::integral_constant<int, 6>{});
    else if (nblocks > 2) mainloop(std::integral_constant<int, 4>{});
    else mainloop(std::integral_constant<int, 2>{});

    // ---- forward: acc[mb][nb][r] is column 16 q + 4 nb + r of the wave's 64, backward 16 q + 4 r + nb
    const int64_t n = n0 + wave * 64 + q * 16;
    if (n >= cols) return;
    const int live = cols - n < 16 ? (int)(cols - n) : 16;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int r = mb * 16 + i;
        if (r >= nrows) continue;
        const int64_t m = row0 + r;
        const int64_t flat = p.y_grouped && !p.gates ? m : load_idx(p.pos, m, p.pos64);
        const float c = p.gates ? load_gate(p.gates, flat, p.gates_dtype) : 1.f;
        float v[16];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int x = 0; x < 4; ++x) v[BWD ? 4 * x + nb : 4 * nb + x] = p.gates ? acc[mb][nb][x] * c : acc[mb][nb][x];
        store16(p.Y, (p.y_grouped ? m : flat) * p.ldy + n, p.ydtype, v, live, p.y_vec);
    }
}

template <class Num, bool BWD, int ROWS> int launch_rows(MoeFp4Gemm p, int64_t R, hipStream_t stream)
{
    static std::atomic<bool> attr_set[MOE_MAX_DEVICES];
    auto kern = fp4_tile_kernel<Num, BWD, ROWS>;
    const int dev = moe_current_device();
    if (!attr_set[dev]) {
        if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES) != hipSuccess) return MOE_ERR_LAUNCH;
        attr_set[dev] = true;
    }
    p.num_cus = WGS_PER_CU * moe_device_cus();
    const int64_t cols = BWD ? p.K : p.N, ntiles = (cols + BN - 1) / BN;
    // an upper bound on the tiles (a tile holds a row at least), and a round for the last, partial one; surplus workgroups leave at once
    const int64_t most = R / ROWS + p.E, grid = ((most < R ? most : R) * ntiles + p.num_cus + NXCD - 1) / NXCD * NXCD;
    if (!moe_grid_fits(grid, THREADS)) return MOE_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(THREADS), LDS_BYTES, stream, p);
    return moe_launch_status();
}

template <class Num, bool BWD> int launch_typed(const MoeFp4Gemm& p, int64_t R, hipStream_t stream)
{
    // Rows of a tile: by the tiles that fall to a compute unit and their rows, half a tile more for each expert than its rows fill.  A launch of a few tiles per compute unit gains by smaller ones that
    // come out even; backward 112 rows too (forward their odd number of blocks cost what they gained).  128 rows / the choice, us, 8 experts, forward and backward: 2000 rows of 4096 x 4096 97 / 84 and 104 /
    // 94, 3000 120 / 120 and 129 / 125, 4000 155 / 138 and 176 / 152, 8192 270 / 264 and 278 / 259; 4096 of 2048 x 2048 52 / 44 and 57 / 50; 800 of 4096 x 4096 64 / 57 and 79 / 69.  (96 rows where 128 are chosen:
    // 3000 rows 140 and 160.)
    const int64_t used = p.E < R ? p.E : R, ntiles = ((BWD ? p.K : p.N) + BN - 1) / BN, rows = (R + used - 1) / used, cus = moe_device_cus();
    auto time = [&](int bm) {
        const double tiles = (double)R / bm + 0.5 * used;
        return ceil((tiles > used ? tiles : used) * ntiles / cus) * (rows < bm ? (rows + 31) / 32 * 32 : bm);
    };
    if (time(96) < 0.95 * time(128) && (!BWD || time(96) <= time(112))) return launch_rows<Num, BWD, 96>(p, R, stream);
    if constexpr (BWD)
        if (time(112) < 0.95 * time(128)) return launch_rows<Num, BWD, 112>(p, R, stream);
    return launch_rows<Num, BWD, 128>(p, R, stream);
}

}  // namespace

int moe_launch_fp4_tiles(MoeFp4Gemm p, int64_t R, bool backward, hipStream_t stream)
{
    p.y_vec = p.ydtype == MOE_F32 ? p.ldy % 4 == 0 && (uintptr_t)p.Y % 16 == 0 : p.ldy % 8 == 0 && (uintptr_t)p.Y % 16 == 0;
    if (backward) return p.f16 ? launch_typed<NumF16, true>(p, R, stream) : launch_typed<NumBf16, true>(p, R, stream);
    return p.f16 ? launch_typed<NumF16, false>(p, R, stream) : launch_typed<NumBf16, false>(p, R, stream);
}

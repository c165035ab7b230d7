// Grouped product of fp32 rows with 4-bit weights (fp4.h), both directions, tiles of 64 rows x 64 columns on the fp32 matrix instructions:
//
//   forward:   Y[out_row(m)][n] = sum_k X[in_row(m)][k] W[e(m)][n][k]
//   backward:  Y[out_row(m)][k] = c[m] sum_n X[in_row(m)][n] W[e(m)][n][k]      (X: gradient rows, c: their gate weights or 1)
//
// Four waves of 32 x 32.  Both operands pass through LDS as fp32, contraction by contraction step of 32: the codes become numbers on their way there, eight of a thread, so no weight is
// written to memory as fp32 and only the experts that hold a row are read.  A step is 32 matrix instructions of 32 cycles a wave against 8 reads of LDS, so the matrix cores bound it; the next
// step's global loads are in registers meanwhile.  v_mfma_f32_16x16x4_f32 multiplies and adds in fp32; a lane reads four contraction steps at once, and which four of a group of 16 is free as
// long as both operands agree.
// Measured, eight experts: 8192 rows of 4096 x 4096 forward 2552 us (108 TFLOP/s; an fp32 copy of the weights and a product over it 6151), 512 rows of 1024 x 1024 33 (87), two rows of 4096 x
// 4096 81 (866).
#include "fp4.h"
#include "kernels.h"

namespace {

constexpr int BM = 64, BN = 64, BK = 32, THREADS = 256, PITCH = BK + 4;   // (rows 144 bytes apart: 16 of them meet all banks)

template <bool BWD>
__global__ void __launch_bounds__(THREADS) fp4_f32_kernel(const MoeFp4Gemm p)
{
    __shared__ __attribute__((aligned(16))) float xs[2][BM][PITCH], ws[2][BN][PITCH];   // rows, and columns of the result, by contraction step
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, q = lane >> 4;
    const int64_t cols = BWD ? p.K : p.N, len = BWD ? p.N : p.K, G = (p.K + FP4_GROUP - 1) / FP4_GROUP;
    const uint32_t ncb = (uint32_t)p.col_blocks, tile = blockIdx.x / ncb, cb = blockIdx.x - tile * ncb;
    RowTile t;
    if (!find_row_tile(p.offsets, p.off64, p.E, BM, tile, &t)) return;
    const int64_t row0 = uniform_i64(t.row0), n0 = (int64_t)cb * BN;
    const int nrows = __builtin_amdgcn_readfirstlane((int)(t.row1 - t.row0)), e = __builtin_amdgcn_readfirstlane(t.expert);

    // ---- this thread's part of a step: eight values of a row, eight codes
    const int xr = tid >> 2, x_at = (tid & 3) * 8;
    const bool row = xr < nrows;
    const int64_t m0 = row0 + (row ? xr : 0);
    const float* x = (const float*)p.X + (p.x_grouped ? m0 : load_idx(p.pos, m0, p.pos64) / p.fan_out) * p.ldx;
    // forward: column tid >> 2, inputs 8 (tid & 3) on; backward: row tid >> 3 of the step, columns 8 (tid & 7) on
    const int wr = BWD ? tid >> 3 : tid >> 2, w_at = BWD ? (tid & 7) * 8 : (tid & 3) * 8;
    const int64_t w_group = BWD ? (n0 + w_at) / FP4_GROUP : 0, wn = n0 + wr < p.N ? n0 + wr : p.N - 1;
    const uint8_t* codes = p.w.codes + e * p.w.sce + (BWD ? w_group * FP4_GROUP_BYTES + (w_at & (FP4_GROUP - 1)) / 2 : wn * p.w.scn + w_at / 2);
    const uint8_t* scales = p.w.scales + e * p.w.sse + (BWD ? w_group : wn * p.w.ssn);
    float xv[8];
    uint32_t code, scale;
    auto fetch = [&](int64_t k0) {
        const int64_t k = k0 + x_at;
        if (p.x_vec && k + 8 <= len) {
            const float4 a = *(const float4*)(x + k), b = *(const float4*)(x + k + 4);
            xv[0] = a.x; xv[1] = a.y; xv[2] = a.z; xv[3] = a.w; xv[4] = b.x; xv[5] = b.y; xv[6] = b.z; xv[7] = b.w;
        } else
#pragma unroll
            for (int v = 0; v < 8; ++v) xv[v] = k + v < len ? x[k + v] : 0.f;
        code = 0;
        scale = 0;
        if constexpr (!BWD) {
            code = *(const uint32_t*)(codes + k0 / 2);
            scale = scales[k0 / FP4_GROUP];
        } else if (k0 + wr < len && w_group < G) {
            code = *(const uint32_t*)(codes + (k0 + wr) * p.w.scn);
            scale = scales[(k0 + wr) * p.w.ssn];
        }
    };
    auto store = [&](int b, int64_t k0) {
#pragma unroll
        for (int v = 0; v < 8; ++v) xv[v] = row ? xv[v] : 0.f;
        *(float4*)&xs[b][xr][x_at] = make_float4(xv[0], xv[1], xv[2], xv[3]);
        *(float4*)&xs[b][xr][x_at + 4] = make_float4(xv[4], xv[5], xv[6], xv[7]);
        const float s = fp4_scale(scale);
        const float2 v0 = fp4_pair_f32<0>(code, s), v1 = fp4_pair_f32<1>(code, s), v2 = fp4_pair_f32<2>(code, s), v3 = fp4_pair_f32<3>(code, s);
        float w[8] = {v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
        if constexpr (!BWD) {
#pragma unroll
            for (int v = 0; v < 8; ++v) w[v] = k0 + w_at + v < len ? w[v] : 0.f;   // (what codes behind the last input stand for meets no number)
            *(float4*)&ws[b][wr][w_at] = make_float4(w[0], w[1], w[2], w[3]);
            *(float4*)&ws[b][wr][w_at + 4] = make_float4(w[4], w[5], w[6], w[7]);
        } else
#pragma unroll
            for (int v = 0; v < 8; ++v) ws[b][w_at + v][wr] = w[v];
    };

    const int wm = (wave >> 1) * 32, wc = (wave & 1) * 32;
    f32x4_t acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc[a][c] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    fetch(0);
    store(0, 0);
    int b = 0;
    for (int64_t k0 = 0; k0 < len; k0 += BK, b ^= 1) {
        __syncthreads();   // this step is there, and nobody reads the one before any more
        const bool more = k0 + BK < len;
        if (more) fetch(k0 + BK);
#pragma unroll
        for (int s = 0; s < BK; s += 16) {
            f32x4_t xa[2], wa[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) xa[a] = *(const f32x4_t*)&xs[b][wm + 16 * a + i][s + 4 * q];
#pragma unroll
            for (int c = 0; c < 2; ++c) wa[c] = *(const f32x4_t*)&ws[b][wc + 16 * c + i][s + 4 * q];
#pragma unroll
            for (int a = 0; a < 2; ++a)
                if (wm + 16 * a < nrows)
#pragma unroll
                    for (int v = 0; v < 4; ++v)
#pragma unroll
                        for (int c = 0; c < 2; ++c) acc[a][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(wa[c][v], xa[a][v], acc[a][c], 0, 0, 0);
        }
        if (more) store(b ^ 1, k0 + BK);
    }
    // ---- a lane holds columns 4 q .. + 3 of row i
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int r = wm + 16 * a + i;
        if (r >= nrows) continue;
        const int64_t m = row0 + r, flat = p.y_grouped && !p.gates ? m : load_idx(p.pos, m, p.pos64);
        const float g = p.gates ? load_gate(p.gates, flat, p.gates_dtype) : 1.f;
        float* y = (float*)p.Y + (p.y_grouped ? m : flat) * p.ldy;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int64_t n = n0 + wc + 16 * c + 4 * q;
            const f32x4_t v = p.gates ? acc[a][c] * g : acc[a][c];
            if (p.y_vec && n + 4 <= cols) *(float4*)(y + n) = make_float4(v[0], v[1], v[2], v[3]);
            else
#pragma unroll
                for (int z = 0; z < 4; ++z)
                    if (n + z < cols) y[n + z] = v[z];
        }
    }
}

}  // namespace

int moe_launch_fp4_f32(MoeFp4Gemm p, int64_t R, bool backward, hipStream_t stream)
{
    const int64_t most = R / BM + p.E, tiles = most < R ? most : R;   // (a tile holds a row at least)
    p.col_blocks = ((backward ? p.K : p.N) + BN - 1) / BN;
    p.x_vec = p.ldx % 4 == 0 && (uintptr_t)p.X % 16 == 0;
    p.y_vec = p.ldy % 4 == 0 && (uintptr_t)p.Y % 16 == 0;
    if (!moe_grid_fits(tiles * p.col_blocks, THREADS)) return MOE_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(tiles * p.col_blocks));
    if (backward) hipLaunchKernelGGL((fp4_f32_kernel<true>), grid, dim3(THREADS), 0, stream, p);
    else hipLaunchKernelGGL((fp4_f32_kernel<false>), grid, dim3(THREADS), 0, stream, p);
    return moe_launch_status();
}

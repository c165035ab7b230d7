// Grouped product of 8-bit codes over ragged expert groups:
//   Y[out_row(m)][n] = x_scale[in_row(m)] * w_scale[e(m)][n] * sum_k X[in_row(m)][k] W[e(m)][k][n]
// The sum of K < 2^17 products of 8-bit integers is exact in 32 bits.  One workgroup per 64 x 64 output tile, operands through LDS as dwords of four
// codes along k, v_dot4 on 4 x 4 outputs per thread.
#include "common.h"
#include "kernels.h"

namespace {

constexpr int TM = 64, TN = 64, TK = 64;

template <bool PAIR>
__global__ void __launch_bounds__(256) i8_gemm_simple_kernel(const MoeI8Gemm p, int64_t kp)
{
    __shared__ uint32_t xs[TM][TK / 4 + 1];
    __shared__ uint32_t ws[PAIR ? 2 : 1][TN][TK / 4 + 1];
    __shared__ float ys[TM][TN + 1];
    RowTile t;
    if (!find_row_tile(p.offsets, p.off64, p.E, TM, blockIdx.y, &t)) return;
    const int nrows = (int)(t.row1 - t.row0);
    const int64_t n0 = (int64_t)blockIdx.x * TN;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[PAIR ? 2 : 1][4][4] = {};
    auto in_row = [&](int r) {
        const int64_t m = t.row0 + (r < nrows ? r : nrows - 1);
        return p.x_grouped ? m : load_idx(p.pos, m, p.pos64) / p.fan_out;
    };
    for (int seg = 0; seg < p.nseg; ++seg)
        for (int64_t k0 = 0; k0 < p.K; k0 += TK) {
            for (int i = threadIdx.x; i < TM * TK / 4; i += 256) {
                const int r = i / (TK / 4), c = i % (TK / 4);
                xs[r][c] = *(const uint32_t*)(p.X + in_row(r) * p.ldx + seg * kp + k0 + c * 4);
                const int64_t n = n0 + r;
#pragma unroll
                for (int h = 0; h < (PAIR ? 2 : 1); ++h) {
                    const int8_t* W = p.W[PAIR ? h : seg] + (int64_t)t.expert * p.swe;
                    uint32_t v = 0;
                    for (int b = 0; b < 4; ++b) {
                        const int64_t k = k0 + c * 4 + b;
                        if (k < p.K && n < p.N) v |= (uint32_t)(uint8_t)(p.nn ? W[k * p.ldw + n] : W[n * p.ldw + k]) << (8 * b);
                    }
                    ws[h][r][c] = v;
                }
            }
            __syncthreads();
            for (int c = 0; c < TK / 4; ++c)
#pragma unroll
                for (int h = 0; h < (PAIR ? 2 : 1); ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[h][i][j] = __builtin_amdgcn_sdot4((int)xs[ty * 4 + i][c], (int)ws[h][tx * 4 + j][c], acc[h][i][j], false);
            __syncthreads();
        }
    float v[PAIR ? 2 : 1][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float xs_ = p.x_scale[in_row(ty * 4 + i)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx * 4 + j < p.N ? n0 + tx * 4 + j : p.N - 1;
#pragma unroll
            for (int h = 0; h < (PAIR ? 2 : 1); ++h)
                v[h][i][j] = (float)acc[h][i][j] * xs_ * (p.w_scale[h] ? p.w_scale[h][(int64_t)t.expert * p.N + n] : 1.f);
        }
    }
    if (p.epi == MOE_I8_STORE) {
        for (int i = 0; i < 4; ++i) {
            const int r = ty * 4 + i;
            if (r >= nrows) continue;
            const int64_t m = t.row0 + r, o = p.y_grouped ? m : load_idx(p.pos, m, p.pos64);
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + tx * 4 + j;
                if (n >= p.N) continue;
                if (p.ydtype == MOE_F32) ((float*)p.Y)[o * p.ldy + n] = v[0][i][j];
                else if (p.ydtype == MOE_BF16) ((uint16_t*)p.Y)[o * p.ldy + n] = NumBf16::from_f32(v[0][i][j]);
                else ((uint16_t*)p.Y)[o * p.ldy + n] = NumF16::from_f32(v[0][i][j]);
            }
        }
        return;
    }
    for (int s = 0; s < 3; ++s) {
        if (!p.S[s]) continue;
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const float g = v[0][i][j], u = v[PAIR ? 1 : 0][i][j];
                ys[ty * 4 + i][tx * 4 + j] = !PAIR || s == 1 ? g : s == 2 ? u : g / (1.f + __expf(-g)) * u;
            }
        __syncthreads();
        for (int q = threadIdx.x; q < TM * (TN / MOE_SEG_COLS); q += 256) {
            const int r = q / (TN / MOE_SEG_COLS), c0 = q % (TN / MOE_SEG_COLS) * MOE_SEG_COLS;
            if (r >= nrows || n0 + c0 >= p.N) continue;
            uint32_t top = 0;
            for (int c = 0; c < MOE_SEG_COLS; ++c) top = max(top, __float_as_uint(ys[r][c0 + c]) & 0x7fffffffu);
            const float amax = __uint_as_float(top), inv = top > 0 && top < 0x7f800000u ? 32767.f / amax : 0.f;
            for (int c = 0; c < MOE_SEG_COLS; ++c) p.S[s][(t.row0 + r) * p.N + n0 + c0 + c] = inv > 0.f ? (int16_t)rintf(ys[r][c0 + c] * inv) : (int16_t)0;
            p.SS[s][((t.row0 + r) * p.N + n0 + c0) / MOE_SEG_COLS] = top < 0x7f800000u ? amax / 32767.f : __uint_as_float(0x7fc00000u);
        }
        __syncthreads();
    }
}

}  // namespace

bool moe_i8_weights_ok(const void* W, int64_t swe, int64_t ldw) { return (uintptr_t)W % 16 == 0 && swe % 16 == 0 && ldw % 16 == 0; }
bool moe_i8_gemm_supported(const MoeI8Gemm& p, int64_t R, int64_t x_rows)
{
    (void)R;
    return x_rows * p.ldx < ((int64_t)1 << 32) && (p.nn ? p.K : p.N) * p.ldw < ((int64_t)1 << 32);
}
size_t moe_i8_exchange_bytes(int64_t, int, int64_t, int64_t, bool) { return 256; }
int moe_launch_i8_gemm(const MoeI8Gemm& p, int64_t R, hipStream_t stream)
{
    if (R == 0 || p.N == 0) return MOE_OK;
    const dim3 grid((unsigned)((p.N + TN - 1) / TN), (unsigned)(R / TM + p.E));
    if (p.epi == MOE_I8_SWIGLU) hipLaunchKernelGGL(i8_gemm_simple_kernel<true>, grid, dim3(256), 0, stream, p, moe_i8_pitch(p.K));
    else hipLaunchKernelGGL(i8_gemm_simple_kernel<false>, grid, dim3(256), 0, stream, p, moe_i8_pitch(p.K));
    return moe_launch_status();
}

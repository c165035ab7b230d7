// Weights of 16 or 32 bits into 4-bit codes with a scale per 32 inputs (fp4.h), once per weight; and copies of rows and scales that the 16-bit products do not take as they lie.
#include "fp4.h"
#include "kernels.h"

namespace {

// A group's power of two is the least p that leaves its largest magnitude a at 7 * 2^p or below: 7 is half way between the largest code, 6, and the next number of the same
// precision, 8, so no weight loses more than half a step of its own binade.  (Error of normally distributed weights, root of the mean square over the deviation: 0.1118; with a at
// 6 * 2^p or below 0.1154, below 8 * 2^p 0.1149, and with the better power chosen for every group 0.1115.)  Weights become the nearest code, the even one of two.
// A group of zeros gets the scale 0 (2^-127), one that holds an infinity or a NaN the scale 255 (NaN) and codes 0.
template <typename T>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(const T* W, int64_t swe, int64_t swk, int64_t swn, int64_t K, int64_t N, int64_t G, int64_t total, int n_first,
                                                           uint8_t* codes, int64_t sce, int64_t scn, uint8_t* scales, int64_t sse, int64_t ssn)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;   // neighbours read neighbouring weights: next group of the same column, or the same group of the next column
    if (i >= total) return;
    const int64_t e = i / (N * G), j = i - e * N * G;
    const int64_t n = n_first ? j % N : j / G, g = n_first ? j / N : j % G;
    const T* w = W + e * swe + n * swn + g * FP4_GROUP * swk;
    const int live = K - g * FP4_GROUP < FP4_GROUP ? (int)(K - g * FP4_GROUP) : FP4_GROUP;
    float v[FP4_GROUP];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < FP4_GROUP; ++k) {
        v[k] = k < live ? Elem<T>::ld(w + k * swk) : 0.f;
        const uint32_t m = __float_as_uint(v[k]) & 0x7fffffffu;   // (bits: NaN above infinity above every number)
        top = m > top ? m : top;
    }
    const bool fine = top < 0x7f800000u;
    int p = 0;
    const float mantissa = frexpf(__uint_as_float(fine ? top : 0u), &p);
    p -= mantissa > 0.875f ? 2 : 3;
    p = p < -127 ? -127 : p;
    if (top == 0) p = -127;
    fp4_u32x4_t out;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t word = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float t = fine ? ldexpf(fabsf(v[c * 8 + k]), -p) : 0.f;
            // steps of a half below 2, of one below 4, of two above; a code counts those steps
            uint32_t code = t < 2.f ? (uint32_t)rintf(2.f * t) : t < 4.f ? 2u + (uint32_t)rintf(t) : 4u + (uint32_t)rintf(0.5f * t);
            code = code > 7u ? 7u : code;
            if (v[c * 8 + k] < 0.f && fine) code |= 8u;
            word |= code << (4 * k);
        }
        out[c] = word;
    }
    *(fp4_u32x4_t*)(codes + e * sce + n * scn + g * FP4_GROUP_BYTES) = out;
    scales[e * sse + n * ssn + g] = fine ? (uint8_t)(p + 127) : 255;
}

// Rows that 16-byte loads do not take, in the order of the product and padded to whole pieces.  (Rows behind the last group are left alone: their positions may be anything.)
__global__ void __launch_bounds__(256) fp4_pack_rows_kernel(const uint16_t* X, int64_t ldx, const void* pos, int pos64, int fan_out, const void* offsets, int off64, int E, int64_t K,
                                                            uint16_t* out, int64_t ldo)
{
    const int64_t m = blockIdx.x;
    if (m >= load_idx(offsets, E - 1, off64)) return;
    const uint16_t* x = X + (pos ? load_idx(pos, m, pos64) / fan_out : m) * ldx;
    for (int64_t c = threadIdx.x; c < ldo; c += 256) out[m * ldo + c] = c < K ? x[c] : (uint16_t)0;
}

// Scales that 4-byte loads do not take, in rows of whole fours.
__global__ void __launch_bounds__(256) fp4_pack_scales_kernel(const uint8_t* scales, int64_t sse, int64_t ssn, int64_t N, int64_t G, uint8_t* out, int64_t ldo, int64_t total)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / ldo, g = i - row * ldo, e = row / N, n = row - e * N;
    out[i] = g < G ? scales[e * sse + n * ssn + g] : (uint8_t)0;
}

}  // namespace

int moe_launch_fp4_pack_scales(const uint8_t* scales, int64_t sse, int64_t ssn, int E, int64_t N, int64_t G, uint8_t* out, int64_t ldo, hipStream_t stream)
{
    const int64_t total = E * N * ldo;
    if (!moe_grid_fits((total + 255) / 256, 256)) return MOE_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(fp4_pack_scales_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, stream, scales, sse, ssn, N, G, out, ldo, total);
    return moe_launch_status();
}

int moe_launch_fp4_pack_rows(const void* X, int64_t ldx, const void* pos, int pos64, int fan_out, const void* offsets, int off64, int E, int64_t R, int64_t K, void* out, int64_t ldo,
                             hipStream_t stream)
{
    if (!moe_grid_fits(R, 256)) return MOE_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(fp4_pack_rows_kernel, dim3((unsigned)R), dim3(256), 0, stream, (const uint16_t*)X, ldx, pos, pos64, fan_out, offsets, off64, E, K, (uint16_t*)out,
                       ldo);
    return moe_launch_status();
}

int moe_launch_fp4_quantize(const void* W, int64_t swe, int64_t swk, int64_t swn, int dtype, int E, int64_t K, int64_t N, uint8_t* codes, int64_t sce, int64_t scn, uint8_t* scales,
                            int64_t sse, int64_t ssn, hipStream_t stream)
{
    const int64_t G = (K + FP4_GROUP - 1) / FP4_GROUP, total = E * N * G;
    if (!moe_grid_fits((total + 255) / 256, 256)) return MOE_ERR_UNSUPPORTED;
    MOE_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((fp4_quantize_kernel<T>), dim3((unsigned)((total + 255) / 256)), dim3(256), 0, stream, (const T*)W, swe, swk, swn, K, N, G, total,
                                                 swn < swk, codes, sce, scn, scales, sse, ssn));
    return moe_launch_status();
}

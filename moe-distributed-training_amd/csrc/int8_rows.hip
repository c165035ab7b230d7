// Rows of the 8-bit expert products: activations and gradients into codes with a scale per row, the interims between two products, and
// weights in an order that the product kernel can read.
//
// A row v becomes codes q[c] = rne(127 v[c] / a) with a = max |v| and the scale a / 127: the quotient is rounded as it is, not as some fp32 value of
// it comes out (ties are common: half the maximum is 63.5 for every row of a 2-byte type), so the codes are the same on every path and in any
// precision that a checker takes.  q is guessed with one multiplication by 127 / a and put right from its remainder 127 v - q a, which fp32 holds
// exactly for 2-byte types (at most 19 bits: values below a / 254 have q = 0) and fp64 for fp32 values.  A row that holds an infinity or a NaN gets the
// scale NaN and codes 0, so that every product of it is NaN and no other row changes; a row of zeros the scale 0.
//
// Interims (h, the saved gate and up, dh) travel as 24-bit integers with a scale for each 32 columns of a row: 3 bytes per value, 2^-24 of the segment's maximum
// off.  Every value that a rounding on the way carries over a border of the 8-bit codes costs a whole step, so this noise falls with the root of
// the rounding only: with 16 bits 1 code in 700 changed and the MLP's error against 64 bits was 1.5e-3 of its result's norm (bf16 rows would be off by four
// times that), with 24 it is that of fp32 arithmetic, at three quarters of an fp32 tensor's bytes.
#include "common.h"
#include "kernels.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = fmax(v, __shfl_xor(v, m));
    return v;
}

// Largest value of a workgroup and whether any thread saw something that is not finite (both in every thread).
template <typename C> __device__ __forceinline__ C block_max(C v, bool& bad)
{
    __shared__ C s_max[16];
    __shared__ int s_bad[16];
    v = wave_max(v);
    const bool b = __any(bad);
    const int wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) { s_max[wave] = v; s_bad[wave] = b; }
    __syncthreads();
    v = s_max[0];
    int any = s_bad[0];
    for (int w = 1; w < nw; ++w) { v = v > s_max[w] ? v : s_max[w]; any |= s_bad[w]; }
    bad = any != 0;
    return v;
}

__device__ __forceinline__ float mag(float v) { return fabsf(v); }
__device__ __forceinline__ double mag(double v) { return fabs(v); }
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
__device__ __forceinline__ bool finite(double v) { return fabs(v) <= 1.7976931348623157e308; }
__device__ __forceinline__ float near_int(float v) { return rintf(v); }
__device__ __forceinline__ double near_int(double v) { return rint(v); }
__device__ __forceinline__ float mul_add(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double mul_add(double a, double b, double c) { return fma(a, b, c); }

// What a row's values are multiplied by before they meet its maximum, so that 127 v and 127 / a stay inside fp32's range (fp64: 1; a value that the factor
// makes subnormal is far below half a step).
__device__ __forceinline__ float row_factor(float a) { return a > 0x1p64f ? 0x1p-64f : a < 0x1p-64f ? 0x1p64f : 1.f; }
__device__ __forceinline__ double row_factor(double) { return 1.0; }

template <typename C> struct RowCoder {
    C f, a, inv;
    float scale;
    __device__ __forceinline__ RowCoder(C amax, bool bad)
    {
        f = row_factor(amax);
        a = amax * f;
        inv = !bad && a > 0 ? (C)127 / a : (C)0;
        if (inv == (C)0) f = 0;   // every code 0
        scale = bad ? __uint_as_float(0x7fc00000u) : (float)(amax / (C)127);
    }
    __device__ __forceinline__ int code(C v) const
    {
        const C x = f == (C)0 ? (C)0 : v * f;
        C q = near_int(x * inv);
        const C r = mul_add(-q, a, (C)127 * x), d = 2 * mag(r);
        if (d > a || (d == a && ((int)q & 1))) q += r < 0 ? (C)-1 : (C)1;
        return (int)q;
    }
};

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d)
{
    return (uint32_t)(a & 0xff) | (uint32_t)(b & 0xff) << 8 | (uint32_t)(c & 0xff) << 16 | (uint32_t)d << 24;
}

// the expert that grouped row m belongs to (E or more: none)
__device__ __forceinline__ int expert_of_row(const void* offsets, int off64, int E, int64_t m)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int base = 0; base < E; base += 64) {
        const int e = base + lane;
        n += __popcll(__ballot(e < E && load_idx(offsets, e < E ? e : E - 1, off64) <= m));
    }
    return __builtin_amdgcn_readfirstlane(n);
}

template <typename T> struct Loader;   // 8 consecutive elements as fp32
template <> struct Loader<float> {
    static __device__ __forceinline__ void ld8(const float* p, float* v)
    {
        const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <> struct Loader<__hip_bfloat16> {
    static __device__ __forceinline__ void ld8(const __hip_bfloat16* p, float* v)
    {
        const u32x4_t w = *(const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};
template <> struct Loader<__half> {
    static __device__ __forceinline__ void ld8(const __half* p, float* v)
    {
        const u32x4_t w = *(const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = NumF16::to_f32((uint16_t)w[i]); v[2 * i + 1] = NumF16::to_f32((uint16_t)(w[i] >> 16)); }
    }
};

// One workgroup per row.  KEEP: a thread holds its KEEP pieces of 8 columns between the two passes (0: the row is read twice).  SCALED: row m is row
// pos[m] / fan_out of src times coeff[pos[m]] and, column by column, col_scale[expert of m] (a gradient on its way through the weights' scales).
// Those products, and fp32 rows, are worked through in fp64 throughout: the quotient that is rounded is that of the exact values to 2^-50.
template <typename T, bool SCALED, int KEEP>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const MoeQuantizeRows p)
{
    typedef std::conditional_t<SCALED || std::is_same_v<T, float>, double, float> C;
    const int64_t m = blockIdx.x;
    int64_t src_row = m;
    C coeff = 1;
    const float* cs = nullptr;
    if (SCALED) {
        int64_t at = m;
        if (p.pos) {
            at = load_idx(p.pos, m, p.pos64);
            src_row = at / p.fan_out;
        }
        if (p.coeff) coeff = (C)load_gate(p.coeff, at, p.coeff_dtype);
        if (p.col_scale) {
            const int e = expert_of_row(p.offsets, p.off64, p.E, m);
            if (e >= p.E) return;   // behind the last group: no product reads the row
            cs = p.col_scale + (int64_t)e * p.cols;
        }
    }
    const T* row = (const T*)p.src + src_row * p.lds;
    const int nt = blockDim.x;
    auto load = [&](int64_t c0, C* v) {
        float x[8];
        if (p.vec && c0 + 8 <= p.cols) Loader<T>::ld8(row + c0, x);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = c0 + i < p.cols ? Elem<T>::ld(row + c0 + i) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = (C)x[i];
            if (SCALED) {
                v[i] *= coeff;
                if (cs) v[i] *= c0 + i < p.cols ? (C)cs[c0 + i] : (C)0;
            }
        }
    };
    C keep[KEEP ? KEEP : 1][8];
    C amax = 0;
    bool bad = false;
    auto look = [&](const C* v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bad |= !finite(v[i]);
            amax = mag(v[i]) > amax ? mag(v[i]) : amax;
        }
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int64_t c0 = ((int64_t)j * nt + threadIdx.x) * 8;
            if (c0 < p.ldc) { load(c0, keep[j]); look(keep[j]); }
        }
    } else {
        for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < p.ldc; c0 += (int64_t)nt * 8) { load(c0, keep[0]); look(keep[0]); }
    }
    amax = block_max(amax, bad);
    const RowCoder<C> rc(amax, bad);
    int8_t* out = p.codes + m * p.ldc;
    auto store = [&](int64_t c0, const C* v) {
        uint2 w;
        w.x = pack4(rc.code(v[0]), rc.code(v[1]), rc.code(v[2]), rc.code(v[3]));
        w.y = pack4(rc.code(v[4]), rc.code(v[5]), rc.code(v[6]), rc.code(v[7]));
        *(uint2*)(out + c0) = w;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int64_t c0 = ((int64_t)j * nt + threadIdx.x) * 8;
            if (c0 < p.ldc) store(c0, keep[j]);
        }
    } else {
        for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < p.ldc; c0 += (int64_t)nt * 8) { load(c0, keep[0]); store(c0, keep[0]); }
    }
    if (threadIdx.x == 0) p.scale[m] = rc.scale;
}

// columns c0 .. c0 + 7 of a row of segments, times s
__device__ __forceinline__ void ld8_seg(const uint8_t* row, int64_t c0, float s, float* v)
{
    const uint8_t* seg = row + c0 / MOE_SEG_COLS * MOE_SEG_BYTES;
    const int c = (int)(c0 % MOE_SEG_COLS);
    const u32x4_t hi = *(const u32x4_t*)(seg + c * 2);
    const uint2 lo = *(const uint2*)(seg + 64 + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t l = (i < 2 ? lo.x : lo.y) >> (16 * (i & 1));
        v[2 * i] = (float)(((int)(hi[i] << 16) >> 8) | (int)(l & 0xff)) * s;
        v[2 * i + 1] = (float)(((int)(hi[i] & 0xffff0000u) >> 8) | (int)((l >> 8) & 0xff)) * s;
    }
}

// Rows of segments -> codes: the maximum of a row is that of its segments, whose largest integer is MOE_SEG_LEVELS.
__global__ void __launch_bounds__(1024) requantize_rows_kernel(const uint8_t* src, const float* seg, int64_t cols, int8_t* codes, int64_t ldc, float* scale)
{
    const int64_t m = blockIdx.x;
    const int64_t nseg = cols / MOE_SEG_COLS;
    float top = 0.f;
    bool bad = false;
    for (int64_t i = threadIdx.x; i < nseg; i += blockDim.x) {
        const float s = seg[m * nseg + i];
        bad |= !finite(s);
        top = fmaxf(top, s);
    }
    top = block_max(top, bad);
    const float amax = top * (float)MOE_SEG_LEVELS;
    bad |= !finite(amax);
    const float f = row_factor(amax);
    const float inv = !bad && amax > 0.f ? 127.f / (amax * f) : 0.f;
    for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < ldc; c0 += (int64_t)blockDim.x * 8) {
        uint2 w = {0u, 0u};
        if (c0 < cols && inv > 0.f) {
            float v[8];
            ld8_seg(src + m * nseg * MOE_SEG_BYTES, c0, seg[m * nseg + c0 / MOE_SEG_COLS] * f * inv, v);
            int q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = (int)rintf(fminf(fmaxf(v[i], -127.f), 127.f));
            w.x = pack4(q[0], q[1], q[2], q[3]);
            w.y = pack4(q[4], q[5], q[6], q[7]);
        }
        *(uint2*)(codes + m * ldc + c0) = w;
    }
    if (threadIdx.x == 0) scale[m] = bad ? __uint_as_float(0x7fc00000u) : amax / 127.f;
}

// SwiGLU's backward pass and the codes of the joint row [dgate * s1 | dup * s3] in one pass over dh, gate and up:
//   dgate = dh up sig(g) (1 + g (1 - sig(g))),  dup = dh g sig(g).
// One scale for both halves, so that the product behind it is one sum over 2 f codes.
template <int KEEP>
__global__ void __launch_bounds__(1024) swiglu_bwd_codes_kernel(const MoeSwigluBwdCodes p)
{
    const int64_t m = blockIdx.x;
    const int e = expert_of_row(p.offsets, p.off64, p.E, m);
    if (e >= p.E) return;
    const float *c1 = p.s1 + (int64_t)e * p.f, *c3 = p.s3 + (int64_t)e * p.f;
    const int64_t nseg = p.f / MOE_SEG_COLS;
    auto load = [&](int64_t c0, float* a, float* b) {
        float dh[8], g[8], u[8];
        const int64_t s = m * nseg + c0 / MOE_SEG_COLS;
        ld8_seg(p.dh + m * nseg * MOE_SEG_BYTES, c0, p.dh_seg[s], dh);
        ld8_seg(p.gate + m * nseg * MOE_SEG_BYTES, c0, p.gate_seg[s], g);
        ld8_seg(p.up + m * nseg * MOE_SEG_BYTES, c0, p.up_seg[s], u);
        float x1[8], x3[8];
        Loader<float>::ld8(c1 + c0, x1);
        Loader<float>::ld8(c3 + c0, x3);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sg = __builtin_amdgcn_rcpf(1.f + __expf(-g[i]));
            a[i] = dh[i] * u[i] * sg * (1.f + g[i] * (1.f - sg)) * x1[i];
            b[i] = dh[i] * g[i] * sg * x3[i];
        }
    };
    float a[KEEP ? KEEP : 1][8], b[KEEP ? KEEP : 1][8], amax = 0.f;
    bool bad = false;
    auto look = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bad |= !finite(v[i]);
            amax = fmaxf(amax, fabsf(v[i]));
        }
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int64_t c0 = ((int64_t)j * blockDim.x + threadIdx.x) * 8;
            if (c0 < p.f) { load(c0, a[j], b[j]); look(a[j]); look(b[j]); }
        }
    } else {
        for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < p.f; c0 += (int64_t)blockDim.x * 8) { load(c0, a[0], b[0]); look(a[0]); look(b[0]); }
    }
    amax = block_max(amax, bad);
    const RowCoder<float> rc(amax, bad);
    int8_t* out = p.codes + m * 2 * p.ldc;
    auto store = [&](int8_t* at, const float* v) {
        uint2 w;
        w.x = pack4(rc.code(v[0]), rc.code(v[1]), rc.code(v[2]), rc.code(v[3]));
        w.y = pack4(rc.code(v[4]), rc.code(v[5]), rc.code(v[6]), rc.code(v[7]));
        *(uint2*)at = w;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) {
            const int64_t c0 = ((int64_t)j * blockDim.x + threadIdx.x) * 8;
            if (c0 < p.f) { store(out + c0, a[j]); store(out + p.ldc + c0, b[j]); }
        }
    } else {
        for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < p.f; c0 += (int64_t)blockDim.x * 8) {
            load(c0, a[0], b[0]);
            store(out + c0, a[0]);
            store(out + p.ldc + c0, b[0]);
        }
    }
    for (int64_t c0 = p.f + (int64_t)threadIdx.x * 8; c0 < p.ldc; c0 += (int64_t)blockDim.x * 8) {   // zeros up to whole K tiles
        *(uint2*)(out + c0) = (uint2){0u, 0u};
        *(uint2*)(out + p.ldc + c0) = (uint2){0u, 0u};
    }
    if (threadIdx.x == 0) p.scale[m] = rc.scale;
}

// Expert matrices of any strides -> [E][N][ldo], contiguous along the contraction, zeros from K on.  64 x 64 tiles through LDS: the loads run along
// whichever dimension is contiguous, the stores along the contraction.
__global__ void __launch_bounds__(256) pack_codes_kernel(const int8_t* W, int64_t swe, int64_t swk, int64_t swn, int64_t K, int64_t N, int8_t* out, int64_t ldo)
{
    __shared__ int8_t tile[64][68];
    const int64_t k0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64, e = blockIdx.z;
    const int lane = threadIdx.x & 63, r0 = threadIdx.x >> 6;
    const bool along_n = swn <= swk;
    for (int r = r0; r < 64; r += 4) {
        const int64_t k = k0 + (along_n ? r : lane), n = n0 + (along_n ? lane : r);
        tile[along_n ? lane : r][along_n ? r : lane] = k < K && n < N ? W[e * swe + k * swk + n * swn] : (int8_t)0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i >> 4, c = (i & 15) * 4;
        if (n0 + r < N && k0 + c < ldo) *(uint32_t*)(out + (e * N + n0 + r) * ldo + k0 + c) = *(const uint32_t*)&tile[r][c];
    }
}

// Weights (E, K, N) of a 2- or 4-byte type, any strides -> codes of the same orientation and the scale of every output column.  Two passes over the matrix:
// the maxima of 256 columns by slices of K (an atomic maximum of the magnitudes' bits, whose order of arrival does not matter), then the codes.
// NaN's bits lie above those of every number: a column that holds one, or an infinity, ends with the scale NaN and codes 0.
template <typename T>
__global__ void __launch_bounds__(256) weight_max_kernel(const T* W, int64_t swe, int64_t swk, int64_t swn, int64_t K, int64_t N, uint32_t* top)
{
    const int64_t e = blockIdx.z;
    const bool along_n = swn <= swk;
    uint32_t best = 0;
    if (along_n) {   // a thread per column, a slice of 256 k per workgroup
        const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x, k0 = (int64_t)blockIdx.y * 256;
        if (n >= N) return;
        for (int64_t k = k0; k < k0 + 256 && k < K; ++k) {
            const uint32_t b = __float_as_uint(Elem<T>::ld(W + e * swe + k * swk + n * swn)) & 0x7fffffffu;
            best = b > best ? b : best;
        }
        atomicMax(top + e * N + n, best);
    } else {         // a wave per column
        const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (n >= N) return;
        for (int64_t k = threadIdx.x & 63; k < K; k += 64) {
            const uint32_t b = __float_as_uint(Elem<T>::ld(W + e * swe + k * swk + n * swn)) & 0x7fffffffu;
            best = b > best ? b : best;
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)best, s); best = o > best ? o : best; }
        if ((threadIdx.x & 63) == 0) top[e * N + n] = best;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) weight_codes_kernel(const T* W, int64_t swe, int64_t swk, int64_t swn, int64_t K, int64_t N, const uint32_t* top,
                                                           int8_t* codes, int64_t sce, int64_t sck, int64_t scn, float* scale)
{
    typedef std::conditional_t<std::is_same_v<T, float>, double, float> C;
    const int64_t e = blockIdx.z;
    const bool along_n = swn <= swk;
    const int64_t inner = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t j = (int64_t)blockIdx.y * 16; j < (int64_t)blockIdx.y * 16 + 16; ++j) {
        const int64_t k = along_n ? j : inner, n = along_n ? inner : j;
        if (k >= K || n >= N) continue;
        const float a = __uint_as_float(top[e * N + n]);
        const RowCoder<C> rc((C)a, !finite(a));
        codes[e * sce + k * sck + n * scn] = (int8_t)rc.code((C)Elem<T>::ld(W + e * swe + k * swk + n * swn));
        if (k == 0) scale[e * N + n] = rc.scale;
    }
}

__global__ void zero_u32_kernel(uint32_t* p, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

template <typename T, bool SCALED> int launch_quantize_t(const MoeQuantizeRows& p, int64_t rows, hipStream_t stream)
{
    // pieces of 8 columns: one to four of them a thread
    const int64_t pieces = (p.ldc + 7) / 8;
    const int nt = pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 1024 ? 256 : pieces <= 2048 ? 512 : 1024;
    const int64_t keep = (pieces + nt - 1) / nt;
    if (keep <= 1) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 1>), dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else if (keep <= 2) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 2>), dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else if (keep <= 4) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 4>), dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 0>), dim3((unsigned)rows), dim3(nt), 0, stream, p);
    return moe_launch_status();
}

}  // namespace

int moe_launch_quantize_rows(const MoeQuantizeRows& p_, int dtype, int64_t rows, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    MoeQuantizeRows p = p_;
    const bool scaled = p.pos || p.coeff || p.col_scale;
    MOE_DISPATCH_DTYPE(dtype, {
        p.vec = (uintptr_t)p.src % 16 == 0 && (p.lds * sizeof(T)) % 16 == 0;
        return scaled ? launch_quantize_t<T, true>(p, rows, stream) : launch_quantize_t<T, false>(p, rows, stream);
    });
}

int moe_launch_requantize_rows(const uint8_t* src, const float* seg, int64_t rows, int64_t cols, int8_t* codes, int64_t ldc, float* scale, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    const int nt = ldc / 8 <= 64 ? 64 : ldc / 8 <= 128 ? 128 : 256;
    hipLaunchKernelGGL(requantize_rows_kernel, dim3((unsigned)rows), dim3(nt), 0, stream, src, seg, cols, codes, ldc, scale);
    return moe_launch_status();
}

int moe_launch_swiglu_bwd_codes(const MoeSwigluBwdCodes& p, int64_t rows, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    const int64_t pieces = p.f / 8;
    const int nt = pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 512 ? 256 : pieces <= 1024 ? 512 : 1024;
    const int64_t keep = (pieces + nt - 1) / nt;
    if (keep <= 1) hipLaunchKernelGGL(swiglu_bwd_codes_kernel<1>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else if (keep <= 2) hipLaunchKernelGGL(swiglu_bwd_codes_kernel<2>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else hipLaunchKernelGGL(swiglu_bwd_codes_kernel<0>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    return moe_launch_status();
}

int moe_launch_pack_codes(const int8_t* W, int64_t swe, int64_t swk, int64_t swn, int E, int64_t K, int64_t N, int8_t* out, int64_t ldo, hipStream_t stream)
{
    hipLaunchKernelGGL(pack_codes_kernel, dim3((unsigned)((ldo + 63) / 64), (unsigned)((N + 63) / 64), (unsigned)E), dim3(256), 0, stream, W, swe, swk, swn, K, N, out, ldo);
    return moe_launch_status();
}

int moe_launch_quantize_weights(const void* W, int64_t swe, int64_t swk, int64_t swn, int dtype, int E, int64_t K, int64_t N, int8_t* codes, int64_t sce,
                                int64_t sck, int64_t scn, float* scale, uint32_t* top, hipStream_t stream)
{
    const bool along_n = swn <= swk;
    const int64_t total = (int64_t)E * N;
    hipLaunchKernelGGL(zero_u32_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, stream, top, total);
    const dim3 g1 = along_n ? dim3((unsigned)((N + 255) / 256), (unsigned)((K + 255) / 256), (unsigned)E) : dim3((unsigned)((N + 3) / 4), 1, (unsigned)E);
    const dim3 g2((unsigned)(((along_n ? N : K) + 255) / 256), (unsigned)(((along_n ? K : N) + 15) / 16), (unsigned)E);
    MOE_DISPATCH_DTYPE(dtype, {
        hipLaunchKernelGGL(weight_max_kernel<T>, g1, dim3(256), 0, stream, (const T*)W, swe, swk, swn, K, N, top);
        hipLaunchKernelGGL(weight_codes_kernel<T>, g2, dim3(256), 0, stream, (const T*)W, swe, swk, swn, K, N, top, codes, sce, sck, scn, scale);
        return moe_launch_status();
    });
}

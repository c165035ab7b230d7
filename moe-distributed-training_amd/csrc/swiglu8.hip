// SwiGLU that keeps its inputs for the backward pass in 8 bits:  h = silu(gate) * up  of the inputs as they are;  kept are, of either, the codes rne(127 v / a) of blocks of 64
// columns of a row and the blocks' scales a / 127 (a: the block's largest magnitude), 1.0625 bytes a value;  and with g, u = codes * scale, s = 1 / (1 + exp(-g))
//   dgate = dh u s (1 + g (1 - s)),   dup = dh g s.
// A block that holds an infinity or a NaN gets the scale NaN: gradients of it are NaN, those of other blocks what they were.
//
// Both kernels are bound by memory: 6 bytes a value and 2.1 more of codes forward (16-bit types), 2.1 and 6 backward, each moved once.  Eight lanes share a block, eight values
// each: one 16-byte load per lane and tensor of a 16-bit type, the maximum in three exchanges between lanes, 8-byte stores of codes.
// Measured, 8192 x 14336 in bf16: forward 164 us, backward 161 us, 5.8 and 5.9 TB/s.
#include "codes8.h"
#include "kernels.h"

namespace {

constexpr int THREADS = 256;
constexpr int BLOCK = MOE_KEPT_BLOCK, PER_LANE = 8, LANES = BLOCK / PER_LANE;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T> struct Values;   // eight values of a lane, in 16-byte pieces
template <> struct Values<float> {
    static __device__ __forceinline__ void load(const float* p, float* v)
    {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float* v)
    {
        ((float4*)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4*)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    // (fp32 keeps the library's exponential: the hardware's loses |x| roundings)
    static __device__ __forceinline__ float sigmoid(float g) { return 1.f / (1.f + expf(-g)); }
};
template <typename T, class Num> struct Values16 {
    static __device__ __forceinline__ void load(const T* p, float* v)
    {
        const u32x4_t w = *(const u32x4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = Num::to_f32((uint16_t)w[i]); v[2 * i + 1] = Num::to_f32((uint16_t)(w[i] >> 16)); }
    }
    static __device__ __forceinline__ void store(T* p, const float* v)
    {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = Num::pack2(v[2 * i], v[2 * i + 1]);
        *(u32x4_t*)p = w;
    }
    static __device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }
};
template <> struct Values<__hip_bfloat16> : Values16<__hip_bfloat16, NumBf16> {};
template <> struct Values<__half> : Values16<__half, NumF16> {};

// where a lane's eight values lie; live: how many of them exist (VEC: all or none)
struct Place { uint32_t row, block, col; int live; };
template <bool VEC> __device__ __forceinline__ bool place(const MoeSwiglu8& p, Place* at)
{
    const uint32_t i = (blockIdx.x * THREADS + threadIdx.x) / LANES;   // (blocks are counted in 32 bits: checked on the host)
    if (i >= p.nblocks) return false;
    at->row = i / p.row_blocks;
    at->block = i - at->row * p.row_blocks;
    at->col = at->block * BLOCK + (threadIdx.x % LANES) * PER_LANE;
    const int64_t left = p.cols - at->col;
    at->live = left < 0 ? 0 : left < PER_LANE ? (int)left : PER_LANE;
    return true;
}
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* row, const Place& at, float* v)
{
    if (VEC) {
        if (at.live) Values<T>::load(row + at.col, v);
        else
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) v[i] = 0.f;
    } else
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) v[i] = i < at.live ? Elem<T>::ld(row + at.col + i) : 0.f;
}
template <typename T, bool VEC> __device__ __forceinline__ void store8(T* row, const Place& at, const float* v)
{
    if (VEC) {
        if (at.live) Values<T>::store(row + at.col, v);
    } else
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (i < at.live) Elem<T>::st(row + at.col + i, v[i]);
}

// the block's codes of this lane; its scale from the block's first lane
__device__ __forceinline__ void keep(const float* v, const Place& at, uint32_t i, uint8_t* codes, float* scales)
{
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) { const uint32_t m = mag_bits(v[j]); top = m > top ? m : top; }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) { const uint32_t o = __shfl_xor(top, m); top = o > top ? o : top; }
    const RowCoder c(top);
    float q[PER_LANE];
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) q[j] = c.code(v[j], 0.f);
    uint2 w;
    w.x = pack4(q[0], q[1], q[2], q[3]);
    w.y = pack4(q[4], q[5], q[6], q[7]);
    *(uint2*)(codes + (int64_t)i * BLOCK + (threadIdx.x % LANES) * PER_LANE) = w;
    if (threadIdx.x % LANES == 0) scales[i] = c.scale;
}
__device__ __forceinline__ void kept(const uint8_t* codes, const float* scales, uint32_t i, float* v)
{
    const uint2 w = *(const uint2*)(codes + (int64_t)i * BLOCK + (threadIdx.x % LANES) * PER_LANE);
    const float s = scales[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = (float)(int8_t)(w.x >> (8 * j)) * s;
        v[4 + j] = (float)(int8_t)(w.y >> (8 * j)) * s;
    }
}

template <typename T, bool VEC, bool KEEP>
__global__ void __launch_bounds__(THREADS) swiglu8_fwd_kernel(const MoeSwiglu8 p)
{
    Place at;
    if (!place<VEC>(p, &at)) return;   // (whole blocks of lanes leave)
    float g[PER_LANE], u[PER_LANE], h[PER_LANE];
    load8<T, VEC>((const T*)p.gate + (int64_t)at.row * p.ldg, at, g);
    load8<T, VEC>((const T*)p.up + (int64_t)at.row * p.ldu, at, u);
    if (KEEP) {
        const uint32_t i = at.row * p.row_blocks + at.block;
        keep(g, at, i, p.codes[0], p.scales[0]);
        keep(u, at, i, p.codes[1], p.scales[1]);
    }
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) h[j] = g[j] * Values<T>::sigmoid(g[j]) * u[j];
    store8<T, VEC>((T*)p.h + (int64_t)at.row * p.ldh, at, h);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) swiglu8_bwd_kernel(const MoeSwiglu8 p)
{
    Place at;
    if (!place<VEC>(p, &at)) return;
    const uint32_t i = at.row * p.row_blocks + at.block;
    float g[PER_LANE], u[PER_LANE], d[PER_LANE], dg[PER_LANE], du[PER_LANE];
    kept(p.codes[0], p.scales[0], i, g);
    kept(p.codes[1], p.scales[1], i, u);
    load8<T, VEC>((const T*)p.dh + (int64_t)at.row * p.ldh, at, d);
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
        const float s = Values<T>::sigmoid(g[j]), ds = d[j] * s;
        dg[j] = ds * u[j] * (1.f + g[j] * (1.f - s));
        du[j] = ds * g[j];
    }
    store8<T, VEC>((T*)p.dgate + (int64_t)at.row * p.ldg, at, dg);
    store8<T, VEC>((T*)p.dup + (int64_t)at.row * p.ldu, at, du);
}

}  // namespace

int moe_launch_swiglu8(const MoeSwiglu8& p, int dtype, bool vec, bool backward, hipStream_t stream)
{
    const int64_t grid = ((int64_t)p.nblocks * LANES + THREADS - 1) / THREADS;
    if (!moe_grid_fits(grid, THREADS)) return MOE_ERR_UNSUPPORTED;
    const dim3 g((unsigned)grid), t(THREADS);
    MOE_DISPATCH_DTYPE(dtype, {
        if (backward) {
            if (vec) hipLaunchKernelGGL((swiglu8_bwd_kernel<T, true>), g, t, 0, stream, p);
            else hipLaunchKernelGGL((swiglu8_bwd_kernel<T, false>), g, t, 0, stream, p);
        } else if (p.codes[0]) {
            if (vec) hipLaunchKernelGGL((swiglu8_fwd_kernel<T, true, true>), g, t, 0, stream, p);
            else hipLaunchKernelGGL((swiglu8_fwd_kernel<T, false, true>), g, t, 0, stream, p);
        } else {
            if (vec) hipLaunchKernelGGL((swiglu8_fwd_kernel<T, true, false>), g, t, 0, stream, p);
            else hipLaunchKernelGGL((swiglu8_fwd_kernel<T, false, false>), g, t, 0, stream, p);
        }
    });
    return moe_launch_status();
}

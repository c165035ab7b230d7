// Rows of the 8-bit expert products: activations and gradients into codes with a scale per row, the interims between two products, and
// weights in an order that the product kernel can read.
//
// A row v becomes codes q[c] = rne(127 v[c] / a) with a = max |v| and the scale a / 127: the quotient is rounded as it is, not as some fp32 value of
// it comes out (ties are common: half the maximum is 63.5 for every row of a 2-byte type).  q is guessed with one multiplication by 127 / a and, next to a border, put right
// from its remainder 127 v - q a: 127 v is held as an fp32 number and its rounding error, and the difference with q a is exact (it is a multiple of half a unit of a's last
// place and at most a / 2; below a / 254 q is 0).  Rows of inputs and weights are what they are; rows of gradients, products of two or three numbers, are held as an fp32
// number and its error (together off by 2^-46 of it) from the start, their maximum too.  (16384 x 2048 bf16 gradient rows: 39.5 us, against 32 from fp32 products and a rounded 127 / a,
// which puts 1 code in 10^5, and ties of most maxima, on the other side.)  The MLP's own interims, h and the joint row of dgate and dup, are computed in fp32 and carry its
// rounding: their codes are of the fp32 values, by one multiplication, and a value that lies on a border to within that rounding may go to either side (1 to 2 in 10^6 codes of h;
// half as many where gate, up and h are kept in fp32).
// A row that holds an infinity or a NaN gets the scale NaN and codes 0, so that every product of it is NaN and no other row changes; a row of zeros the scale 0.
//
// Interims (h, the saved gate and up, dh) travel as 24-bit integers with a scale for each 32 columns of a row: 3 bytes per value, at most 2^-24 of the segment's
// maximum off.  Every value that a rounding on the way carries over a border of the 8-bit codes costs a whole step, so this noise falls with the root of
// the rounding only: with 16 bits 1 code in 700 changed and the MLP's error against 64 bits was 1.5e-3 of its result's norm (bf16 rows would be off by four
// times that), with 24 it is about twice that of fp32 arithmetic, at three quarters of an fp32 tensor's bytes.
#include "common.h"
#include "kernels.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Magnitudes are compared as bits: those of an infinity lie above every number's, and NaN's above those.
constexpr uint32_t NOT_FINITE = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// (at most one maximum of each type in a kernel: its place is not used twice)
template <typename U> __device__ __forceinline__ U block_max(U v)
{
    __shared__ U s_max[16];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) { const U o = __shfl_xor(v, m); v = v > o ? v : o; }
    if (blockDim.x == 64) return v;
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_max[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = v > s_max[w] ? v : s_max[w];
    return v;
}
// (g + ge) s as the nearest fp32 number and its error.  (Contracted, the sum of the product and its error would hold the error twice.)
__device__ __forceinline__ void times_with_error(float g, float ge, float s, float* v, float* lo)
{
#pragma clang fp contract(off)
    const float h = g * s, he = fmaf(g, s, -h) + ge * s;
    *v = h + he;
    *lo = he - (*v - h);
}
// Errors lo of nearest fp32 numbers v as those of their magnitudes, in an order that unsigned numbers have, and back.
__device__ __forceinline__ uint32_t error_key(float v, float lo)
{
    const uint32_t b = __float_as_uint(v < 0.f ? -lo : lo);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_error(uint32_t b) { return __uint_as_float(b >> 31 ? b & 0x7fffffffu : ~b); }

// What turns values of a row into its codes.  f: what the values are multiplied by first, so that 127 v and 127 / a stay inside fp32's range (a value that the
// factor makes subnormal is far below half a step).
struct RowCoder {
    float f, a, a_lo, inv, scale;
    __device__ __forceinline__ RowCoder(uint32_t top, float top_lo = 0.f)
    {
        const float amax = __uint_as_float(top);
        const bool fine = top < NOT_FINITE;
        f = amax > 0x1p64f ? 0x1p-64f : amax < 0x1p-64f ? 0x1p64f : 1.f;
        a = fine ? amax * f : 0.f;
        a_lo = fine ? top_lo * f : 0.f;
        inv = a > 0.f ? 127.f / a : 0.f;
        if (inv == 0.f) f = 0.f;   // every code 0
        scale = fine ? amax / 127.f : __uint_as_float(0x7fc00000u);
    }
    // The code of v + lo, lo the rounding error of v.  v times 127 / a is off by five roundings, 127 * 5 * 2^-24 < 4e-5 of a step: only beside a border does more matter.
    __device__ __forceinline__ float code(float v, float lo) const
    {
        const float t = f == 0.f ? 0.f : v * f * inv, q = rintf(t);
        return fabsf(t - q) > 0.49995f ? exact(v, lo) : q;
    }
    __device__ __forceinline__ float exact(float v, float lo) const
    {
        v = f == 0.f ? 0.f : v * f;
        lo = f == 0.f ? 0.f : lo * f;
        float q = rintf(v * inv);
        const float t = 127.f * v, te = fmaf(127.f, v, -t) + 127.f * lo - q * a_lo, r = fmaf(-q, a, t);
        const float side = copysignf(1.f, r), d = fmaf(2.f, fabsf(r), -a) + (2.f * side * te - a_lo);   // twice the distance to q, minus a step
        if (d > 0.f || (d == 0.f && a > 0.f && ((int)q & 1))) q += side;
        return q;
    }
    // ... of a value that carries fp32 rounding anyway
    __device__ __forceinline__ float nearest(float v) const { return f == 0.f ? 0.f : rintf(v * f * inv); }
};

// four whole numbers of magnitude 127 at most as bytes: 1.5 * 2^23 more, and they stand in the lowest bits
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d)
{
    constexpr float M = 12582912.f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + M), __float_as_uint(a + M), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + M), __float_as_uint(c + M), 0x04000c0cu);
    return ab | cd;
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
constexpr int64_t ZERO_PIECE = 4096;   // ints that a workgroup clears
template <typename T, bool SCALED, int KEEP>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const MoeQuantizeRows p)
{
    const int64_t m = blockIdx.x;
    if (m >= p.rows) {   // side job: the counters and sums of the products behind this launch
        const int64_t i0 = (m - p.rows) * ZERO_PIECE;
        for (int64_t i = i0 + threadIdx.x; i < i0 + ZERO_PIECE && i < p.zero_n; i += blockDim.x) p.zero[i] = 0;
        return;
    }
    int64_t src_row = m;
    float coeff = 1.f;
    const float* cs = nullptr;
    if (SCALED) {
        int64_t at = m;
        if (p.pos) {
            at = load_idx(p.pos, m, p.pos64);
            src_row = at / p.fan_out;
        }
        if (p.coeff) coeff = load_gate(p.coeff, at, p.coeff_dtype);
        if (p.col_scale) {
            const int e = expert_of_row(p.offsets, p.off64, p.E, m);
            if (e >= p.E) return;   // behind the last group: no product reads the row
            cs = p.col_scale + (int64_t)e * p.cols;
        }
    }
    const T* row = (const T*)p.src + src_row * p.lds;
    const int nt = blockDim.x;
    // eight values and, of products, their errors
    auto load = [&](int64_t c0, float* v, float* lo) {
        const bool whole = c0 + 8 <= p.cols;
        float s[8];
        if (p.vec && whole) Loader<T>::ld8(row + c0, v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c0 + i < p.cols ? Elem<T>::ld(row + c0 + i) : 0.f;
        if (!SCALED) return;
        if (cs) {
            if (p.vec_scale && whole) Loader<float>::ld8(cs + c0, s);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = c0 + i < p.cols ? cs[c0 + i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = v[i], g = coeff * x, ge = fmaf(coeff, x, -g);
            v[i] = g;
            lo[i] = ge;
            if (cs) times_with_error(g, ge, s[i], v + i, lo + i);
        }
    };
    float keep[KEEP ? KEEP : 1][8], low[KEEP ? KEEP : 1][8];
    auto each = [&](auto fn) {
        if constexpr (KEEP > 0) {
#pragma unroll
            for (int j = 0; j < KEEP; ++j) {
                const int64_t c0 = ((int64_t)j * nt + threadIdx.x) * 8;
                if (c0 < p.ldc) fn(keep[j], low[j], c0);
            }
        } else
            for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < p.ldc; c0 += (int64_t)nt * 8) { load(c0, keep[0], low[0]); fn(keep[0], low[0], c0); }
    };
    if constexpr (KEEP > 0) each([&](float* v, float* lo, int64_t c0) { load(c0, v, lo); });
    std::conditional_t<SCALED, unsigned long long, uint32_t> top = 0;
    each([&](const float* v, const float* lo, int64_t) {
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine = max(mine, mag_bits(v[i]));
        if constexpr (SCALED) {   // (errors count among equal magnitudes only)
            uint32_t error = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) error = mag_bits(v[i]) == mine ? max(error, error_key(v[i], lo[i])) : error;
            const unsigned long long key = (unsigned long long)mine << 32 | error;
            top = key > top ? key : top;
        } else top = max(top, mine);
    });
    top = block_max(top);
    RowCoder rc(0u);
    if constexpr (SCALED) rc = RowCoder((uint32_t)(top >> 32), key_error((uint32_t)top));
    else rc = RowCoder(top);
    int8_t* out = p.codes + m * p.ldc;
    each([&](const float* v, const float* lo, int64_t c0) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = rc.code(v[i], SCALED ? lo[i] : 0.f);
        uint2 w;
        w.x = pack4(q[0], q[1], q[2], q[3]);
        w.y = pack4(q[4], q[5], q[6], q[7]);
        *(uint2*)(out + c0) = w;
    });
    if (threadIdx.x == 0) p.scale[m] = rc.scale;
}

// Columns c0 .. c0 + 7 of a row of segments, of a segment whose maximum is s.  A value's three bytes go to the upper three of a word, so that one conversion makes it a float
// (256 times what it is).  ANY: also where the step of the segment would be subnormal (s below 2^-95): one product more per value.  (As a branch around those, which keeps
// the loads of a thread's later pieces behind it, 8192 rows of 14336 columns of gate, up and dh took 303 us instead of 262.)
template <bool ANY = false> __device__ __forceinline__ void ld8_seg(const uint8_t* row, int64_t c0, float s, float* v)
{
    constexpr float STEP = 1.f / (256.f * MOE_SEG_LEVELS);
    const uint8_t* seg = row + c0 / MOE_SEG_COLS * MOE_SEG_BYTES;
    const int c = (int)(c0 % MOE_SEG_COLS);
    const u32x4_t hi = *(const u32x4_t*)(seg + c * 2);
    const uint2 lo = *(const uint2*)(seg + 64 + c);
    auto value = [&](uint32_t word) { return ANY ? (float)(int)word * STEP * s : (float)(int)word * (STEP * s); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t l = i < 2 ? lo.x : lo.y;
        v[2 * i] = value(__builtin_amdgcn_perm(hi[i], l, i & 1 ? 0x0504020cu : 0x0504000cu));
        v[2 * i + 1] = value(__builtin_amdgcn_perm(hi[i], l, i & 1 ? 0x0706030cu : 0x0706010cu));
    }
}

// Rows of segments -> codes: the maximum of a row is that of its segments.
__global__ void __launch_bounds__(1024) requantize_rows_kernel(const uint8_t* src, const float* seg, int64_t cols, int8_t* codes, int64_t ldc, float* scale)
{
    const int64_t m = blockIdx.x;
    const int64_t nseg = cols / MOE_SEG_COLS;
    uint32_t top = 0;
    for (int64_t i = threadIdx.x; i < nseg; i += blockDim.x) top = max(top, mag_bits(seg[m * nseg + i]));
    const RowCoder rc(block_max(top));
    for (int64_t c0 = (int64_t)threadIdx.x * 8; c0 < ldc; c0 += (int64_t)blockDim.x * 8) {
        uint2 w = {0u, 0u};
        if (c0 < cols && rc.f != 0.f) {
            float v[8];
            ld8_seg(src + m * nseg * MOE_SEG_BYTES, c0, seg[m * nseg + c0 / MOE_SEG_COLS] * rc.f * rc.inv, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = rintf(fminf(fmaxf(v[i], -127.f), 127.f));
            w.x = pack4(v[0], v[1], v[2], v[3]);
            w.y = pack4(v[4], v[5], v[6], v[7]);
        }
        *(uint2*)(codes + m * ldc + c0) = w;
    }
    if (threadIdx.x == 0) scale[m] = rc.scale;
}

// SwiGLU's backward pass and the codes of the joint row [dgate * s1 | dup * s3] in one pass over dh, gate and up:
//   dgate = dh up sig(g) (1 + g (1 - sig(g))),  dup = dh g sig(g).
// One scale for both halves, so that the product behind it is one sum over 2 f codes.
template <int KEEP>
__global__ void __launch_bounds__(KEEP == 1 ? 256 : 512) swiglu_bwd_codes_kernel(const MoeSwigluBwdCodes p)
{
    const int64_t m = blockIdx.x;
    const int e = expert_of_row(p.offsets, p.off64, p.E, m);
    if (e >= p.E) return;
    const float *c1 = p.s1 + (int64_t)e * p.f, *c3 = p.s3 + (int64_t)e * p.f;
    const int64_t nseg = p.f / MOE_SEG_COLS;
    const uint8_t *dh_row = p.dh + m * nseg * MOE_SEG_BYTES, *gate_row = p.gate + m * nseg * MOE_SEG_BYTES, *up_row = p.up + m * nseg * MOE_SEG_BYTES;
    auto load = [&](int64_t c0, float* a, float* b) {
        float dh[8], g[8], u[8], x1[8], x3[8];
        const int64_t s = m * nseg + c0 / MOE_SEG_COLS;
        ld8_seg<true>(dh_row, c0, p.dh_seg[s], dh);
        ld8_seg<true>(gate_row, c0, p.gate_seg[s], g);
        ld8_seg<true>(up_row, c0, p.up_seg[s], u);
        Loader<float>::ld8(c1 + c0, x1);
        Loader<float>::ld8(c3 + c0, x3);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sg = __builtin_amdgcn_rcpf(1.f + __expf(-g[i])), t = dh[i] * sg;
            a[i] = t * u[i] * fmaf(g[i], 1.f - sg, 1.f) * x1[i];
            b[i] = t * g[i] * x3[i];
        }
    };
    float a[KEEP ? KEEP : 1][8], b[KEEP ? KEEP : 1][8];
    uint32_t top = 0;
    auto look = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, mag_bits(v[i]));
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
    const RowCoder rc(block_max(top));
    int8_t* out = p.codes + m * 2 * p.ldc;
    auto store = [&](int8_t* at, const float* v) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = rc.nearest(v[i]);
        uint2 w;
        w.x = pack4(q[0], q[1], q[2], q[3]);
        w.y = pack4(q[4], q[5], q[6], q[7]);
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

// Weighted sums of fp32 rows, out[t] = sum_j gates[t*k+j] y[t*k+j] (no gates: 1), in the output's type: the rows of a token's experts, or of its gradient, meet before
// they are rounded.  (Rounded to bf16 first, a result is off by 1.4 times its own rounding; the fp32 rows cost 1 % of a step of 4096 tokens.)  Four columns a thread.
template <typename T> __device__ __forceinline__ void store4(T* p, const float* v);
template <> __device__ __forceinline__ void store4(float* p, const float* v) { *(float4*)p = make_float4(v[0], v[1], v[2], v[3]); }
template <> __device__ __forceinline__ void store4(__hip_bfloat16* p, const float* v) { *(uint2*)p = make_uint2(NumBf16::pack2(v[0], v[1]), NumBf16::pack2(v[2], v[3])); }
template <> __device__ __forceinline__ void store4(__half* p, const float* v) { *(uint2*)p = make_uint2(NumF16::pack2(v[0], v[1]), NumF16::pack2(v[2], v[3])); }

template <typename T>
__global__ void __launch_bounds__(256) combine_f32_kernel(const float* y, int64_t ldy, T* out, int64_t ldo, const void* gates, int gdtype, int k, int64_t cols, int vec)
{
    const int64_t t = blockIdx.x;
    for (int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 4; c < cols; c += (int64_t)gridDim.y * 1024) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < k; ++j) {
            const float g = gates ? load_gate(gates, t * k + j, gdtype) : 1.f;
            const float* row = y + (t * k + j) * ldy + c;
            float4 x;
            if (vec) x = *(const float4*)row;
            else x = make_float4(row[0], c + 1 < cols ? row[1] : 0.f, c + 2 < cols ? row[2] : 0.f, c + 3 < cols ? row[3] : 0.f);
            v[0] = fmaf(g, x.x, v[0]); v[1] = fmaf(g, x.y, v[1]); v[2] = fmaf(g, x.z, v[2]); v[3] = fmaf(g, x.w, v[3]);
        }
        if (vec) store4(out + t * ldo + c, v);
        else
            for (int i = 0; i < 4; ++i)
                if (c + i < cols) Elem<T>::st(out + t * ldo + c + i, v[i]);
    }
}

// d_gates[p] = <y[p], dout[p / k]> of fp32 rows y; a workgroup per flat position
template <typename T>
__global__ void __launch_bounds__(256) dgates_f32_kernel(const float* y, int64_t ldy, const T* dout, int64_t ldd, void* dgates, int gdtype, int k, int64_t cols, int vec)
{
    const int64_t p = blockIdx.x;
    const float* row = y + p * ldy;
    const T* d = dout + p / k * ldd;
    float s = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * 8; c < cols; c += 2048) {
        float a[8], b[8];
        if (vec) { Loader<float>::ld8(row + c, a); Loader<T>::ld8(d + c, b); }
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) { a[i] = c + i < cols ? row[c + i] : 0.f; b[i] = c + i < cols ? Elem<T>::ld(d + c + i) : 0.f; }
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
    }
    __shared__ float part[4];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) s += __shfl_xor(s, m);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = (part[0] + part[1]) + (part[2] + part[3]);
    if (gdtype == MOE_F32) ((float*)dgates)[p] = s;
    else if (gdtype == MOE_BF16) ((uint16_t*)dgates)[p] = NumBf16::from_f32(s);
    else ((uint16_t*)dgates)[p] = NumF16::from_f32(s);
}

// Expert matrices whose rows are contiguous but not 16-byte aligned -> the same rows at a pitch of ldo, a multiple of 16.  16 bytes per lane, unaligned loads.
__global__ void __launch_bounds__(256) repitch_codes_kernel(const int8_t* W, int64_t swe, int64_t ldw, int64_t rows, int64_t cols, int8_t* out, int64_t ldo)
{
    const int64_t pieces = ldo / 16, i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / pieces, c = (i - r * pieces) * 16, e = blockIdx.y;
    if (r >= rows) return;
    const int8_t* src = W + e * swe + r * ldw + c;
    union { u32x4_t v; int8_t b[16]; } w;
    if (c + 16 <= cols) __builtin_memcpy(&w.v, src, 16);
    else
#pragma unroll
        for (int j = 0; j < 16; ++j) w.b[j] = c + j < cols ? src[j] : (int8_t)0;
    *(u32x4_t*)(out + (e * rows + r) * ldo + c) = w.v;
}

// Expert matrices contiguous along neither dimension -> [E][N][ldo], contiguous along the contraction, zeros from K on; 64 x 64 tiles through LDS.
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
            const uint32_t b = mag_bits(Elem<T>::ld(W + e * swe + k * swk + n * swn));
            best = b > best ? b : best;
        }
        atomicMax(top + e * N + n, best);
    } else {         // a wave per column
        const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (n >= N) return;
        for (int64_t k = threadIdx.x & 63; k < K; k += 64) {
            const uint32_t b = mag_bits(Elem<T>::ld(W + e * swe + k * swk + n * swn));
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
    const int64_t e = blockIdx.z;
    const bool along_n = swn <= swk;
    const int64_t inner = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t j = (int64_t)blockIdx.y * 16; j < (int64_t)blockIdx.y * 16 + 16; ++j) {
        const int64_t k = along_n ? j : inner, n = along_n ? inner : j;
        if (k >= K || n >= N) continue;
        const RowCoder rc(top[e * N + n]);
        codes[e * sce + k * sck + n * scn] = (int8_t)(int)rc.exact(Elem<T>::ld(W + e * swe + k * swk + n * swn), 0.f);
        if (k == 0) scale[e * N + n] = rc.scale;
    }
}

__global__ void zero_u32_kernel(uint32_t* p, int64_t n)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

// threads of a workgroup: pieces of 8 columns, one to four of them a thread
int quantize_threads(int64_t rows, int64_t ldc)
{
    const int64_t pieces = (ldc + 7) / 8;
    return pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 256 || (pieces <= 1024 && rows > 256) ? 256 : pieces <= 512 || (pieces <= 2048 && rows > 256) ? 512 : 1024;
}
int64_t quantize_blocks(int64_t rows, int64_t zero_n) { return rows + (zero_n + ZERO_PIECE - 1) / ZERO_PIECE; }
// (few rows: latency is all of it, and more threads have less each)
int requantize_threads(int64_t rows, int64_t ldc) { return ldc / 8 <= 64 ? 64 : ldc / 8 <= 128 ? 128 : rows > 256 || ldc / 8 <= 256 ? 256 : ldc / 8 <= 512 ? 512 : 1024; }
int swiglu_bwd_threads(int64_t f) { return f / 8 <= 64 ? 64 : f / 8 <= 128 ? 128 : f / 8 <= 256 ? 256 : 512; }

template <typename T, bool SCALED> int launch_quantize_t(const MoeQuantizeRows& p, int64_t rows, hipStream_t stream)
{
    const int64_t pieces = (p.ldc + 7) / 8, grid = quantize_blocks(rows, p.zero_n);
    const int nt = quantize_threads(rows, p.ldc);
    const int64_t keep = (pieces + nt - 1) / nt;
    if (keep <= 1) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 1>), dim3((unsigned)grid), dim3(nt), 0, stream, p);
    else if (keep <= 2) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 2>), dim3((unsigned)grid), dim3(nt), 0, stream, p);
    else if (keep <= 4) hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 4>), dim3((unsigned)grid), dim3(nt), 0, stream, p);
    else hipLaunchKernelGGL((quantize_rows_kernel<T, SCALED, 0>), dim3((unsigned)grid), dim3(nt), 0, stream, p);
    return moe_launch_status();
}

}  // namespace

bool moe_quantize_rows_supported(int64_t rows, int64_t ldc, int64_t zero_n) { return moe_grid_fits(quantize_blocks(rows, zero_n), quantize_threads(rows, ldc)); }
bool moe_requantize_rows_supported(int64_t rows, int64_t ldc) { return moe_grid_fits(rows, requantize_threads(rows, ldc)); }
bool moe_swiglu_bwd_codes_supported(int64_t rows, int64_t f) { return moe_grid_fits(rows, swiglu_bwd_threads(f)); }
bool moe_pack_codes_supported(int64_t N) { return (N + 63) / 64 <= 65535; }

int moe_launch_quantize_rows(const MoeQuantizeRows& p_, int dtype, int64_t rows, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    MoeQuantizeRows p = p_;
    p.rows = rows;
    const bool scaled = p.pos || p.coeff || p.col_scale;
    MOE_DISPATCH_DTYPE(dtype, {
        p.vec = (uintptr_t)p.src % 16 == 0 && (p.lds * sizeof(T)) % 16 == 0;
        p.vec_scale = (uintptr_t)p.col_scale % 16 == 0 && p.cols % 4 == 0;
        return scaled ? launch_quantize_t<T, true>(p, rows, stream) : launch_quantize_t<T, false>(p, rows, stream);
    });
}

int moe_launch_requantize_rows(const uint8_t* src, const float* seg, int64_t rows, int64_t cols, int8_t* codes, int64_t ldc, float* scale, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    const int nt = requantize_threads(rows, ldc);
    hipLaunchKernelGGL(requantize_rows_kernel, dim3((unsigned)rows), dim3(nt), 0, stream, src, seg, cols, codes, ldc, scale);
    return moe_launch_status();
}

int moe_launch_swiglu_bwd_codes(const MoeSwigluBwdCodes& p, int64_t rows, hipStream_t stream)
{
    if (rows == 0) return MOE_OK;
    const int64_t pieces = p.f / 8;
    const int nt = swiglu_bwd_threads(p.f);
    const int64_t keep = (pieces + nt - 1) / nt;
    if (keep <= 1 && nt <= 256) hipLaunchKernelGGL(swiglu_bwd_codes_kernel<1>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else if (keep <= 2) hipLaunchKernelGGL(swiglu_bwd_codes_kernel<2>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else if (keep <= 4) hipLaunchKernelGGL(swiglu_bwd_codes_kernel<4>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    else hipLaunchKernelGGL(swiglu_bwd_codes_kernel<0>, dim3((unsigned)rows), dim3(nt), 0, stream, p);
    return moe_launch_status();
}

int moe_launch_repitch_codes(const int8_t* W, int64_t swe, int64_t ldw, int E, int64_t rows, int64_t cols, int8_t* out, int64_t ldo, hipStream_t stream)
{
    hipLaunchKernelGGL(repitch_codes_kernel, dim3((unsigned)((rows * (ldo / 16) + 255) / 256), (unsigned)E), dim3(256), 0, stream, W, swe, ldw, rows, cols, out, ldo);
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

int moe_launch_combine_f32(const float* y, int64_t ldy, void* out, int64_t ldo, int dtype, const void* gates, int gdtype, int k, int64_t ntok, int64_t ncols, hipStream_t stream)
{
    if (ntok == 0 || ncols == 0) return MOE_OK;
    // (few tokens: the columns of one are dealt to several workgroups)
    const int64_t pieces = (ncols + 1023) / 1024;
    const int64_t parts = ntok < 1024 ? pieces : (pieces + 3) / 4;
    const dim3 grid((unsigned)ntok, (unsigned)(parts < 65535 ? parts : 65535));
    MOE_DISPATCH_DTYPE(dtype, {
        const int vec = ncols % 4 == 0 && ldy % 4 == 0 && ldo % 4 == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)out % (4 * sizeof(T)) == 0;
        hipLaunchKernelGGL(combine_f32_kernel<T>, grid, dim3(256), 0, stream, y, ldy, (T*)out, ldo, gates, gdtype, k, ncols, vec);
        return moe_launch_status();
    });
}

int moe_launch_dgates_f32(const float* y, int64_t ldy, const void* dout, int64_t ldd, int dtype, void* dgates, int gdtype, int k, int64_t ntok, int64_t ncols, hipStream_t stream)
{
    if (ntok == 0 || k == 0) return MOE_OK;
    MOE_DISPATCH_DTYPE(dtype, {
        const int vec = ncols % 8 == 0 && ldy % 4 == 0 && (uintptr_t)y % 16 == 0 && (uintptr_t)dout % 16 == 0 && ldd * sizeof(T) % 16 == 0;
        hipLaunchKernelGGL(dgates_f32_kernel<T>, dim3((unsigned)(ntok * k)), dim3(256), 0, stream, y, ldy, (const T*)dout, ldd, dgates, gdtype, k, ncols, vec);
        return moe_launch_status();
    });
}

// Products of a few rows (16 or 32 at most) with weight matrices that are streamed once: the operands of the matrix instructions come straight from memory, no LDS on the way.
//
// A wave takes blocks of 16 columns and walks the contraction in chunks of 128; chunks are requested several ahead into a ring of registers, which keeps 64 KiB and more of a
// compute unit's loads in flight.  The weight is the first operand of v_mfma_f32_16x16x32: lane (i = lane & 15, g = lane >> 4) holds 8 weights of column i, and of the result the
// columns 4 g .. 4 g + 3 of row i.  Which eight inputs a lane holds is free as long as both operands agree:
//   4-bit weights: inputs 32 g + 8 j .. + 7 of the chunk in its step j: the 16 bytes of a lane's load are one group of 32 inputs with one scale, 64 consecutive bytes of a column per load;
//   16-bit weights: inputs 32 j + 8 g .. + 7: again 64 consecutive bytes of a column per load.
// All loads are buffer loads at 32-bit offsets; what does not exist (rows, inputs behind the last) is asked for at an offset past the buffer's range, which returns zeros without
// moving a byte, so that no load stands behind a branch and the waits count exactly.
#pragma once
#include "fp4.h"

namespace few {

constexpr int CHUNK = 128;
constexpr uint32_t RANGE = 0x80000000u;      // of the buffers, and an offset that lies outside: 2 GiB (checked on the host)

typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const void* base) { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)RANGE, 0x00020000); }
constexpr int STREAMED = 2;                  // non-temporal: nobody else reads these bytes
__device__ __forceinline__ bf16x8_t load16(Buffer b, uint32_t lane_off, uint32_t off) { return __builtin_bit_cast(bf16x8_t, __builtin_amdgcn_raw_buffer_load_b128(b, lane_off, off, 0)); }
__device__ __forceinline__ fp4_u32x4_t load16_streamed(Buffer b, uint32_t lane_off, uint32_t off) { return __builtin_bit_cast(fp4_u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, lane_off, off, STREAMED)); }

// NB columns of this lane, 4-bit weights
template <class Num_, int NB_> struct Fp4Cols {
    typedef Num_ Num;
    static constexpr int NB = NB_;
    Buffer codes[2], scales[2];   // of one matrix, or of two: blocks from NB / 2 on are the second's
    bool two;
    uint32_t c[NB], s[NB];        // first byte of the column's codes plus this lane's 16 g, of its scales plus g
    int left;                     // groups of a column from this lane's first on
    struct Stage { fp4_u32x4_t c[NB]; uint32_t s[NB]; };
    static __device__ __forceinline__ int input(int j, int g) { return 32 * g + 8 * j; }
    __device__ __forceinline__ void load(Stage& t, int chunk) const
    {
        const bool in = 4 * chunk < left;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int m = two && nb >= NB / 2 ? 1 : 0;
            t.c[nb] = load16_streamed(codes[m], in ? c[nb] : RANGE, chunk * 64);
            t.s[nb] = __builtin_amdgcn_raw_buffer_load_b8(scales[m], in ? s[nb] : RANGE, chunk * 4, 0);
        }
    }
    static __device__ __forceinline__ bf16x8_t frag(const Stage& t, int nb, int j) { return fp4_expand8<Num>(t.c[nb][j], fp4_scale(t.s[nb])); }
};

// ... 16-bit weights that are contiguous along the inputs (16-byte aligned columns)
template <class Num_, int NB_> struct Cols16 {
    typedef Num_ Num;
    static constexpr int NB = NB_;
    Buffer w[2];
    uint32_t c[NB];               // first byte of the column plus this lane's 16 g
    int left;                     // inputs from this lane's first on (a multiple of 8)
    struct Stage { fp4_u32x4_t f[NB][4]; };
    static __device__ __forceinline__ int input(int j, int g) { return 32 * j + 8 * g; }
    __device__ __forceinline__ void load(Stage& t, int chunk) const
    {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                t.f[nb][j] = load16_streamed(w[nb >= NB / 2 ? 1 : 0], chunk * CHUNK + 32 * j < left ? c[nb] : RANGE, (chunk * CHUNK + 32 * j) * 2);
    }
    static __device__ __forceinline__ bf16x8_t frag(const Stage& t, int nb, int j) { return __builtin_bit_cast(bf16x8_t, t.f[nb][j]); }
};

// The rows of this lane: NA operands, each its own block of 16 rows, or parts of one whose products are added.
template <int NA> struct Rows {
    Buffer x[NA];
    uint32_t a[NA];               // the row's first byte plus that of this lane's inputs; RANGE: the row does not exist
    int K;                        // a multiple of 8
    struct Stage { bf16x8_t f[NA][4]; };
    template <class W> __device__ __forceinline__ void load(Stage& t, int chunk, int g) const
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = chunk * CHUNK + W::input(j, g) < K;
#pragma unroll
            for (int m = 0; m < NA; ++m) t.f[m][j] = load16(x[m], in ? a[m] : RANGE, (chunk * CHUNK + W::input(j, 0)) * 2);
        }
    }
};

// acc[m][nb] += rows m times columns nb over chunks [c0, c1), DEPTH of them requested ahead (SUM: all row operands into acc[0]).  c0 and c1 are the same in every lane.
template <class W, int NA, bool SUM, int DEPTH>
__device__ __forceinline__ void stream(f32x4_t (&acc)[SUM ? 1 : NA][W::NB], const W& w, const Rows<NA>& rows, int c0, int c1)
{
    const int g = (threadIdx.x & 63) >> 4;
    typename W::Stage ws[DEPTH];
    typename Rows<NA>::Stage as[DEPTH];
    auto fetch = [&](int d, int c) { w.load(ws[d], c); rows.template load<W>(as[d], c, g); };
    auto multiply = [&](int d) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int nb = 0; nb < W::NB; ++nb) {
                const bf16x8_t f = W::frag(ws[d], nb, j);
#pragma unroll
                for (int m = 0; m < NA; ++m) acc[SUM ? 0 : m][nb] = W::Num::mfma(f, as[d].f[m][j], acc[SUM ? 0 : m][nb]);
            }
    };
    int c = c0;
    if (c1 - c0 >= DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) fetch(d, c + d);
        for (; c + 2 * DEPTH <= c1; c += DEPTH)
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) { multiply(d); fetch(d, c + DEPTH + d); }
        // the ring holds chunks c .. c + DEPTH - 1, and fewer than DEPTH are left behind them
        const int more = c1 - c - DEPTH;
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) { multiply(d); if (d < more) fetch(d, c + DEPTH + d); }
#pragma unroll
        for (int d = 0; d < DEPTH - 1; ++d)
            if (d < more) multiply(d);
    } else {
#pragma unroll
        for (int d = 0; d < DEPTH - 1; ++d)
            if (c + d < c1) fetch(d, c + d);
#pragma unroll
        for (int d = 0; d < DEPTH - 1; ++d)
            if (c + d < c1) multiply(d);
    }
}

}  // namespace few

// Products of a few rows (16 or 32 at most) with weight matrices that are streamed once.
//
// A wave takes blocks of 16 columns and walks the contraction in chunks of 128; weights are requested several units (256 inputs of 4 bits, 128 of 16) ahead into a ring of registers,
// which keeps 64 KiB and more of a compute unit's loads in flight.  The weight is the first operand of v_mfma_f32_16x16x32: lane (i = lane & 15, g = lane >> 4) holds 8 weights of column i, and of the result the
// columns 4 g .. 4 g + 3 of row i.  Which eight inputs a lane holds is free as long as both operands agree:
//   4-bit weights: inputs 32 g + 8 j .. + 7 of the chunk in its step j: the 16 bytes of a lane are one group of 32 inputs with one scale;
//   16-bit weights: inputs 32 j + 8 g .. + 7.
//
// Operands do not come from memory in that order: the memory pipeline takes four neighbouring lanes at a time, and neighbours here belong to different columns, so a 1 KiB load of 16 columns
// x 64 bytes occupies it for 65 cycles, against 21 where four neighbours read one column's 64 bytes, 18 for eight columns x 128 bytes, and 17 for whole kilobytes (and for nothing at all).  And a
// 64-byte piece is half a cache line: the other half, asked for a chunk later, came from memory a second time (W2 of eight experts, 249 MB: 432 MB fetched, 106 us for 16 tokens).  So lanes load
// whole lines side by side, and an operand passes through a piece of LDS of its wave's own (no barrier) on its way into the matrix instructions.  Where a shape does not allow it (groups
// of inputs that are no multiple of eight), 4-bit weights are loaded in the operand's order.
//
// All loads are buffer loads at 32-bit offsets; what does not exist (rows, inputs behind the last) is asked for at an offset past the buffer's range, which returns zeros without
// moving a byte, so that no load stands behind a branch and the waits count exactly.
#pragma once
#include "fp4.h"
#include "kernels.h"

namespace few {

constexpr int CHUNK = 128;
constexpr uint32_t RANGE = 0x80000000u;      // of the buffers, and an offset that lies outside: 2 GiB (checked on the host)

typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const void* base) { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)RANGE, 0x00020000); }
constexpr int STREAMED = 2;                  // non-temporal: nobody else reads these bytes
__device__ __forceinline__ fp4_u32x4_t load16(Buffer b, uint32_t lane_off, uint32_t off) { return __builtin_bit_cast(fp4_u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, lane_off, off, 0)); }
__device__ __forceinline__ fp4_u32x4_t load16_streamed(Buffer b, uint32_t lane_off, uint32_t off) { return __builtin_bit_cast(fp4_u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, lane_off, off, STREAMED)); }

// The lanes of a wave pass operands to each other through LDS of the wave's own.  The hardware takes a wave's accesses to LDS in order; this tells the compiler to leave them in that order, around every
// exchange (lanes write what others read, and write again where others have read).  It costs no instruction.
__device__ __forceinline__ void in_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
}

// A block of 16 columns x 64 bytes, loaded with lane l at column l >> 2, piece quad_piece(l) of 16 bytes, as the operand's lane (i, g) holds it: through 1 KiB of LDS.  (The pieces'
// places depend on the column so that 16 columns meet all banks once.)
__device__ __forceinline__ int quad_piece(int lane) { return (lane & 3) ^ (lane >> 4); }
__device__ __forceinline__ fp4_u32x4_t from_quads(fp4_u32x4_t v, uint8_t* scratch)
{
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    in_order();
    *(fp4_u32x4_t*)(scratch + lane * 16) = v;
    in_order();
    return *(const fp4_u32x4_t*)(scratch + i * 64 + (g ^ (i >> 2)) * 16);
}

// NB columns of this lane, 4-bit weights, in the operand's order: any number of groups.  TWO: blocks from NB / 2 on are those of a second matrix.
template <class Num_, int NB_, bool TWO> struct Fp4Cols {
    typedef Num_ Num;
    static constexpr int NB = NB_, UNIT = 1, SCRATCH = 0;
    Buffer codes[2], scales[2];
    uint32_t c[NB], s[NB];        // first byte of the column's codes plus this lane's 16 g, of its scales plus g
    int left;                     // groups of a column from this lane's first on
    struct Stage { fp4_u32x4_t c[NB]; uint32_t s[NB]; };
    static __device__ __forceinline__ int piece(int j, int g) { return 4 * g + j; }
    // matrix m, of K inputs; number(nb, i): that of column i of block nb in it
    template <class F> __device__ __forceinline__ void columns(int m, const MoeFp4Weights& w, int e, int K, F number)
    {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        codes[m] = buffer(w.codes + e * w.sce);
        scales[m] = buffer(w.scales + e * w.sse);
        left = (K + FP4_GROUP - 1) / FP4_GROUP - q;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if (TWO && nb / (NB / 2) != m) continue;
            const int64_t n = number(nb, lane & 15);
            c[nb] = (uint32_t)(n * w.scn) + q * FP4_GROUP_BYTES;
            s[nb] = (uint32_t)(n * w.ssn) + q;
        }
    }
    __device__ __forceinline__ void load(Stage& t, int chunk) const
    {
        const bool in = 4 * chunk < left;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int m = TWO && nb >= NB / 2 ? 1 : 0;
            t.c[nb] = load16_streamed(codes[m], in ? c[nb] : RANGE, chunk * 64);
            t.s[nb] = __builtin_amdgcn_raw_buffer_load_b8(scales[m], in ? s[nb] : RANGE, chunk * 4, 0);
        }
    }
    __device__ __forceinline__ void ready(Stage&, uint8_t*) const {}
    static __device__ __forceinline__ bf16x8_t frag(const Stage& t, int, int nb, int j) { return fp4_expand8<Num>(t.c[nb][j], fp4_scale(t.s[nb])); }
};

// A block of 16 columns x 128 bytes (two chunks of 4-bit weights), loaded in two halves with lane l at column 8 h + (l >> 3), piece line_piece of 16 bytes, as the operand's lane (i, g)
// holds its two chunks: through 2 KiB of LDS.
__device__ __forceinline__ int line_piece(int lane, int h) { return (lane & 7) ^ (((8 * h + (lane >> 3)) >> 1) & 7); }
__device__ __forceinline__ void from_lines(fp4_u32x4_t (&v)[2], uint8_t* scratch)
{
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    in_order();
#pragma unroll
    for (int h = 0; h < 2; ++h) *(fp4_u32x4_t*)(scratch + (h * 64 + lane) * 16) = v[h];
    in_order();
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) v[cc] = *(const fp4_u32x4_t*)(scratch + i * 128 + ((cc * 4 + g) ^ ((i >> 1) & 7)) * 16);
}

// ... loaded side by side: units of 256 inputs, scales in 8-byte pieces.  NB 1, 2 or 4: lane l brings the eight scales of column l of a matrix's blocks.
template <class Num_, int NB_, bool TWO> struct Fp4Quads {
    typedef Num_ Num;
    static constexpr int NB = NB_, UNIT = 2, SCRATCH = 2048 + NB * 128, MATS = TWO ? 2 : 1, EACH = 16 * NB / MATS;
    Buffer codes[2], scales[2];
    uint32_t c[NB][2], s[MATS];
    struct Stage { fp4_u32x4_t c[NB][2]; uint32_t s[NB][2]; };
    static __device__ __forceinline__ int piece(int j, int g) { return 4 * g + j; }
    template <class F> __device__ __forceinline__ void columns(int m, const MoeFp4Weights& w, int e, int, F number)
    {
        const int lane = threadIdx.x & 63;
        codes[m] = buffer(w.codes + e * w.sce);
        scales[m] = buffer(w.scales + e * w.sse);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (!TWO || nb / (NB / 2) == m) c[nb][h] = (uint32_t)(number(nb, 8 * h + (lane >> 3)) * w.scn) + line_piece(lane, h) * 16;
        s[m] = lane < EACH ? (uint32_t)(number(m * (NB / MATS) + (lane >> 4), lane & 15) * w.ssn) : RANGE;
    }
    __device__ __forceinline__ void load(Stage& t, int unit) const
    {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) t.c[nb][h] = load16_streamed(codes[TWO && nb >= NB / 2 ? 1 : 0], c[nb][h], unit * 128);
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(scales[m], s[m], unit * 8, 0);
            t.s[m][0] = v[0];
            t.s[m][1] = v[1];
        }
    }
    __device__ __forceinline__ void ready(Stage& t, uint8_t* scratch) const
    {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) from_lines(t.c[nb], scratch);   // (the same 2 KiB for every block: a wave's accesses to LDS happen in order)
        uint2* sc = (uint2*)(scratch + 2048);
        in_order();
#pragma unroll
        for (int m = 0; m < MATS; ++m)
            if (lane < EACH) sc[m * EACH + lane] = make_uint2(t.s[m][0], t.s[m][1]);
        in_order();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const uint2 v = sc[nb * 16 + i];
            t.s[nb][0] = v.x >> (8 * g) & 0xff;
            t.s[nb][1] = v.y >> (8 * g) & 0xff;
        }
    }
    static __device__ __forceinline__ bf16x8_t frag(const Stage& t, int cc, int nb, int j) { return fp4_expand8<Num>(t.c[nb][cc][j], fp4_scale(t.s[nb][cc])); }
};

// 16-bit weights that are contiguous along the inputs (16-byte aligned columns): two matrices side by side, NB / 2 blocks of each
template <class Num_, int NB_> struct Cols16 {
    typedef Num_ Num;
    static constexpr int NB = NB_, UNIT = 1, SCRATCH = NB * 1024;
    Buffer w[2];
    uint32_t c[NB];               // first byte of the column (lane >> 2) plus this lane's piece
    int left;                     // inputs from this lane's first on (a multiple of 8)
    struct Stage { fp4_u32x4_t f[NB][4]; };
    static __device__ __forceinline__ int piece(int j, int g) { return 4 * j + g; }
    __device__ __forceinline__ void load(Stage& t, int chunk) const
    {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                t.f[nb][j] = load16_streamed(w[nb >= NB / 2 ? 1 : 0], chunk * CHUNK + 32 * j < left ? c[nb] : RANGE, (chunk * CHUNK + 32 * j) * 2);
    }
    __device__ __forceinline__ void ready(Stage& t, uint8_t* scratch) const
    {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) t.f[nb][j] = from_quads(t.f[nb][j], scratch + nb * 1024);
    }
    static __device__ __forceinline__ bf16x8_t frag(const Stage& t, int, int nb, int j) { return __builtin_bit_cast(bf16x8_t, t.f[nb][j]); }
};

// Rows, 256 bytes of each per chunk: NA operands of 16 rows, each a block of its own, or parts of one whose products are added.  Lane l loads piece l & 15 of rows 4 j + (l >> 4).
template <int NA> struct Rows {
    static constexpr int SCRATCH = NA * 4096;
    Buffer x[NA];
    uint32_t a[NA][4];            // first byte of row 4 j + (l >> 4) plus this lane's piece; RANGE: there is no such row
    int left;                     // inputs from this lane's first on
    struct Stage { fp4_u32x4_t f[NA][4]; };
    __device__ __forceinline__ void load(Stage& t, int chunk) const
    {
        const bool in = chunk * CHUNK < left;
#pragma unroll
        for (int m = 0; m < NA; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) t.f[m][j] = load16(x[m], in ? a[m][j] : RANGE, chunk * CHUNK * 2);
    }
    // ... into the operand's order: f[m][j] is row lane & 15, piece W::piece(j, g)
    template <class W> __device__ __forceinline__ void ready(Stage& t, uint8_t* scratch) const
    {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
        in_order();
#pragma unroll
        for (int m = 0; m < NA; ++m) {
            uint8_t* s = scratch + m * 4096;
#pragma unroll
            for (int j = 0; j < 4; ++j) *(fp4_u32x4_t*)(s + (4 * j + g) * 256 + (i ^ (4 * j + g)) * 16) = t.f[m][j];
            in_order();
#pragma unroll
            for (int j = 0; j < 4; ++j) t.f[m][j] = *(const fp4_u32x4_t*)(s + i * 256 + (W::piece(j, g) ^ i) * 16);
        }
    }
};

// a step's 32 products are summed by the instruction, the steps in fp32 or, where a sum decides between experts, in 64 bits
struct Wide { double v[4]; };
template <class Num> __device__ __forceinline__ void add_products(f32x4_t& a, bf16x8_t w, bf16x8_t x) { a = Num::mfma(w, x, a); }
template <class Num> __device__ __forceinline__ void add_products(Wide& a, bf16x8_t w, bf16x8_t x)
{
    const f32x4_t p = Num::mfma(w, x, (f32x4_t){0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int r = 0; r < 4; ++r) a.v[r] += (double)p[r];
}

// acc[m][nb] += rows m times columns nb over `count` units of W::UNIT chunks, `first` and every `step`th from there on, DEPTH of them requested ahead, and the rows of AHEAD chunks (SUM: all
// row operands into acc[0]).  These numbers are the same in every lane; scratch is the wave's own W::SCRATCH + Rows::SCRATCH bytes.
template <class W, int NA, bool SUM, int DEPTH, int AHEAD, class Acc>
__device__ __forceinline__ void stream(Acc (&acc)[SUM ? 1 : NA][W::NB], const W& w, const Rows<NA>& rows, int first, int count, int step, uint8_t* scratch)
{
    constexpr int UNIT = W::UNIT;
    static_assert(DEPTH * UNIT % AHEAD == 0, "a chunk's place in the ring of rows is known when the loop is compiled");
    typename W::Stage ws[DEPTH];
    typename Rows<NA>::Stage as[AHEAD];
    // (the scheduler would gather the requests of a round behind its products: each stays where it is written)
    auto fetch = [&](int d, int u) { w.load(ws[d], first + u * step); __builtin_amdgcn_sched_barrier(0); };
    auto fetch_rows = [&](int a, int c) { rows.load(as[a], (first + c / UNIT * step) * UNIT + c % UNIT); __builtin_amdgcn_sched_barrier(0); };
    auto multiply = [&](int d, int cc) {
        auto& x = as[(d * UNIT + cc) % AHEAD];
        if (cc == 0) w.ready(ws[d], scratch);
        rows.template ready<W>(x, scratch + W::SCRATCH);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int nb = 0; nb < W::NB; ++nb) {
                const bf16x8_t f = W::frag(ws[d], cc, nb, j);
#pragma unroll
                for (int m = 0; m < NA; ++m) add_products<typename W::Num>(acc[SUM ? 0 : m][nb], f, __builtin_bit_cast(bf16x8_t, x.f[m][j]));
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    const int last = count * UNIT;   // chunks from here on are not this wave's
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (d < count) fetch(d, d);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
        if (a < last) fetch_rows(a, a);
    int u = 0;
    for (; u + 2 * DEPTH <= count; u += DEPTH)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
            for (int cc = 0; cc < UNIT; ++cc) { multiply(d, cc); fetch_rows((d * UNIT + cc) % AHEAD, (u + d) * UNIT + cc + AHEAD); }
            fetch(d, u + DEPTH + d);
        }
    for (; u < count; u += DEPTH)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (u + d >= count) break;
#pragma unroll
            for (int cc = 0; cc < UNIT; ++cc) {
                multiply(d, cc);
                const int c = (u + d) * UNIT + cc + AHEAD;
                if (c < last) fetch_rows((d * UNIT + cc) % AHEAD, c);
            }
            if (u + d + DEPTH < count) fetch(d, u + d + DEPTH);
        }
}

}  // namespace few

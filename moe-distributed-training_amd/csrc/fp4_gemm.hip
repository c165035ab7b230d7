// Grouped product of 16-bit rows with 4-bit weights (fp4.h) over ragged expert groups, few rows per expert: the codes are streamed (few_rows.h).
//
//   Y[out_row(m)][n] = sum_k X[in_row(m)][k] W[e(m)][n][k]
//
// Bound by the codes (17 bytes per 32 weights) of the experts that hold a row: two rows of 4096 x 14336 15.2 us = 4.1 TB/s, of which 3 us are the launch, the look-up of the tile and its rows and the sum
// over waves; sixteen rows of eight experts 50 us = 5.0 TB/s.
#include "few_rows.h"
#include "kernels.h"

namespace {

// four consecutive values of a row
__device__ __forceinline__ void store4(void* Y, int64_t at, int dtype, f32x4_t v, int live, bool vec)
{
    if (dtype == MOE_F32) {
        float* y = (float*)Y + at;
        if (vec && live == 4) { *(float4*)y = make_float4(v[0], v[1], v[2], v[3]); return; }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < live) y[i] = v[i];
        return;
    }
    uint16_t* y = (uint16_t*)Y + at;
    uint2 o;
    if (dtype == MOE_BF16) { o.x = NumBf16::pack2(v[0], v[1]); o.y = NumBf16::pack2(v[2], v[3]); }
    else { o.x = NumF16::pack2(v[0], v[1]); o.y = NumF16::pack2(v[2], v[3]); }
    if (vec && live == 4) { *(uint2*)y = o; return; }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < live) y[i] = (uint16_t)((i < 2 ? o.x : o.y) >> (16 * (i & 1)));
}

// A workgroup: one row tile of 16 rows, 16 NB columns; its waves share the contraction and add up their sums in LDS, in wave order.
template <class Num, int NB, bool QUADS>
__global__ void __launch_bounds__(512) fp4_few_rows_kernel(const MoeFp4Gemm p)
{
    constexpr int MB = 1;
    typedef typename std::conditional<QUADS, few::Fp4Quads<Num, NB, false>, few::Fp4Cols<Num, NB, false>>::type W;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int i = lane & 15, q = lane >> 4;
    const uint32_t ncb = (uint32_t)p.col_blocks, tile = blockIdx.x / ncb, cb = blockIdx.x - tile * ncb;
    RowTile t;
    if (!find_row_tile(p.offsets, p.off64, p.E, 16 * MB, tile, &t)) return;
    const int64_t row0 = uniform_i64(t.row0);
    const int nrows = __builtin_amdgcn_readfirstlane((int)(t.row1 - t.row0)), e = __builtin_amdgcn_readfirstlane(t.expert);
    W w;
    // column i of the wave's block nb is 16 (i >> 2) + 4 nb + (i & 3) with NB = 4: a lane then holds 16 consecutive columns of its row
    const int64_t n0 = (int64_t)cb * (16 * NB);
    w.columns(0, p.w, e, p.K, [&](int nb, int c) {
        const int64_t n = n0 + (c >> 2) * (4 * NB) + 4 * nb + (c & 3);
        return n < p.N ? n : p.N - 1;
    });
    few::Rows<MB> rows;
    rows.left = p.K - 8 * i;
    const int64_t base = p.x_grouped ? row0 : 0;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        rows.x[mb] = few::buffer((const uint16_t*)p.X + base * p.ldx);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = mb * 16 + 4 * j + q;
            rows.a[mb][j] = few::RANGE;
            if (r < nrows) {
                const int64_t m = row0 + r;
                rows.a[mb][j] = (uint32_t)(((p.x_grouped ? m : load_idx(p.pos, m, p.pos64) / p.fan_out) - base) * p.ldx + 8 * i) * 2;
            }
        }
    }
    f32x4_t acc[MB][NB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) acc[mb][nb] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    constexpr int UNIT = W::UNIT * few::CHUNK, SCRATCH = W::SCRATCH + few::Rows<MB>::SCRATCH;
    const int units = (p.K + UNIT - 1) / UNIT;
    few::stream<W, MB, false, 2, 2>(acc, w, rows, wave, (units - wave + waves - 1) / waves, waves, smem + wave * SCRATCH);
    f32x4_t* red = (f32x4_t*)smem;   // [wave][MB * NB][64], in place of the operands
    static_assert(MB * NB * 1024 <= SCRATCH, "the sums fit where the operands were");
    if (waves > 1) {
        __syncthreads();
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) red[(wave * (MB * NB) + mb * NB + nb) * 64 + lane] = acc[mb][nb];
        __syncthreads();
    }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int r = mb * 16 + i;
        const int64_t m = row0 + (r < nrows ? r : 0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int unit = mb * NB + nb;
            if (unit % waves != wave) continue;
            f32x4_t v = acc[mb][nb];
            if (waves > 1) {
                v = red[unit * 64 + lane];
                for (int x = 1; x < waves; ++x) v += red[(x * (MB * NB) + unit) * 64 + lane];
            }
            const int64_t n = n0 + q * (4 * NB) + 4 * nb;
            if (r >= nrows || n >= p.N) continue;
            const int64_t out = p.y_grouped ? m : load_idx(p.pos, m, p.pos64);
            store4(p.Y, out * p.ldy + n, p.ydtype, v, p.N - n < 4 ? (int)(p.N - n) : 4, p.y_vec);
        }
    }
}

template <class Num, int NB> int launch_few_typed(MoeFp4Gemm p, int64_t tiles, int waves, hipStream_t stream)
{
    p.col_blocks = (p.N + 16 * NB - 1) / (16 * NB);
    if (!moe_grid_fits(tiles * p.col_blocks, waves * 64)) return MOE_ERR_UNSUPPORTED;
    auto go = [&](auto quads) {
        constexpr bool Q = decltype(quads)::value;
        const size_t lds = (size_t)waves * (few::Rows<1>::SCRATCH + (Q ? few::Fp4Quads<Num, NB, false>::SCRATCH : 0));
        auto kern = fp4_few_rows_kernel<Num, NB, Q>;
        static std::atomic<bool> attr_set[MOE_MAX_DEVICES];
        const int dev = moe_current_device();
        if (!attr_set[dev]) {
            if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return MOE_ERR_LAUNCH;
            attr_set[dev] = true;
        }
        hipLaunchKernelGGL(kern, dim3((unsigned)(tiles * p.col_blocks)), dim3(waves * 64), lds, stream, p);
        return moe_launch_status();
    };
    return p.quads ? go(std::true_type{}) : go(std::false_type{});
}

template <class Num> int launch_few(const MoeFp4Gemm& p, int64_t R, hipStream_t stream)
{
    const int64_t most = R / 16 + p.E, tiles = most < R ? most : R, used = p.E < R ? p.E : R;   // (a tile holds a row at least)
    const int chunks = (p.K + few::CHUNK - 1) / few::CHUNK, cus = moe_device_cus();
    const bool narrow = tiles * ((p.N + 63) / 64) < cus;   // few column blocks: blocks of 16 columns give every compute unit one
    // Waves that share a contraction: as many as the chip holds at once (by their registers, below; tiles as many as spread rows fill: evenly, or with half a tile more for each expert), two chunks each at least.  One
    // token of 4096 x 14336, 448 workgroups: 1 / 2 / 4 / 8 waves 25 / 19 / 15 / 20 us, the last in two rounds; 16 of one expert each 50 / 54 / 52 / 70; 666 rows of 1000 x 1368 12.6 / 14.9 / 16.4 / 27.
    const int64_t even = used * ((R + 16 * used - 1) / (16 * used)), uneven = R / 16 + used / 2, groups = (even > uneven ? even : uneven) * (narrow ? (p.N + 15) / 16 : (p.N + 63) / 64);
    const int64_t resident = (int64_t)cus * (narrow ? (p.quads ? 16 : 20) : p.quads ? 8 : 12);
    int waves = 1;
    while (waves < 8 && groups * waves * 2 <= resident && chunks >= 2 * waves) waves *= 2;
    return narrow ? launch_few_typed<Num, 1>(p, tiles, waves, stream) : launch_few_typed<Num, 4>(p, tiles, waves, stream);
}

}  // namespace

int moe_launch_fp4_few_rows(MoeFp4Gemm p, int64_t R, hipStream_t stream)
{
    p.quads = (p.K + FP4_GROUP - 1) / FP4_GROUP % 8 == 0;   // whole lines of codes and scales; columns of other sizes are loaded group by group (666 rows of 1000 x 1368: 17.2 us, 12.6 in lines)
    p.y_vec = p.ldy % 4 == 0 && (uintptr_t)p.Y % 16 == 0;
    return p.f16 ? launch_few<NumF16>(p, R, stream) : launch_few<NumBf16>(p, R, stream);
}

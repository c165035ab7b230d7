// The grouped product of 8-bit codes with tiles of 256 x 256, one workgroup of 8 waves per compute unit, and what both tile sizes share.
#define MOE_I8_TILE 256
#include "int8_gemm_kernel.h"

namespace {

constexpr int MAX_SPLIT = 8;   // K parts that a tile of the last, partial round of compute units may be cut into

int64_t tiles_at_most(int tile, int64_t R, int E, int64_t N, bool pair)
{
    const int64_t cols = pair ? tile / 2 : tile;
    return (R / tile + E) * ((N + cols - 1) / cols);
}

// K parts that a tile of `ktiles` K tiles can be cut into
int parts_at_most(int64_t ktiles)
{
    int s = 1;
    while (s * 2 <= MAX_SPLIT && ktiles / (s * 2) >= MIN_PART_KTILES) s *= 2;
    return s;
}

}  // namespace

// rows and columns of a launch's tiles
int moe_i8_tile(int cus, int64_t R, int E, int64_t N, bool pair)
{
    const int64_t groups = R < E ? R : E;
    const int64_t tiles = groups * (((R + groups - 1) / groups + BM - 1) / BM) * ((N + BN - 1) / BN * (pair ? 2 : 1));   // (as if the rows were dealt evenly)
    return R <= groups * 128 || 2 * tiles <= cus ? 128 : 256;
}

bool moe_i8_weights_ok(const void* W, int64_t swe, int64_t ldw) { return (uintptr_t)W % 16 == 0 && swe % 16 == 0 && ldw % 16 == 0; }

// 32-bit byte offsets: gathered rows of X from its start (grouped ones from the tile's first row), one expert's matrix (2 GiB where its last K tile is masked)
bool moe_i8_gemm_supported(const MoeI8Gemm& p, int64_t R, int64_t x_rows)
{
    (void)R;
    const int64_t rows = p.x_grouped ? BM : x_rows, limit = p.K % BK ? (int64_t)1 << 31 : (int64_t)1 << 32;
    return rows * p.ldx < ((int64_t)1 << 32) && (p.nn ? (p.K - 1) * p.ldw + p.N : (p.N - 1) * p.ldw + p.K) + 16 < limit;
}

// counters of the split tiles: two per compute unit are enough for either tile size
int moe_i8_counters() { return 2 * (moe_device_cus() / NXCD * NXCD > 0 ? moe_device_cus() / NXCD * NXCD : NXCD); }

// counters of the split tiles (one per compute unit's workgroup) and their parts' sums, of the tile size that needs more
size_t moe_i8_exchange_bytes(int64_t R, int E, int64_t K, int64_t N, bool pair)
{
    const int cus = moe_i8_counters() / 2;
    const int64_t parts = parts_at_most((K + BK - 1) / BK);
    size_t most = 0;
    for (int tile = 256; tile >= 128; tile /= 2) {
        const int64_t slots = (int64_t)(256 / tile) * cus, all = parts * tiles_at_most(tile, R, E, N, pair);
        const size_t b = parts == 1 ? 0 : (size_t)(all < slots ? all : slots) * tile * tile * sizeof(int);
        most = b > most ? b : most;
    }
    return 2 * (size_t)cus * sizeof(int) + 256 + most;
}

int moe_launch_i8_gemm(const MoeI8Gemm& p_, int64_t R, hipStream_t stream)
{
    if (R == 0 || p_.N == 0) return MOE_OK;
    MoeI8Gemm p = p_;
    const int cus = moe_i8_counters() / 2;
    p.num_cus = cus;
    p.max_split = parts_at_most((p.K + BK - 1) / BK * p.nseg);
    if (p.max_split > 1 && !p.exchange) return MOE_ERR_WORKSPACE;
    p.sk_counters = (int*)p.exchange;
    p.sk_partials = (int*)((uint8_t*)p.exchange + ((2 * (size_t)cus * sizeof(int) + 255) & ~(size_t)255));
    p.y_vec = (uintptr_t)p.Y % 16 == 0 && (p.ydtype == MOE_F32 ? p.ldy % 4 == 0 && p.N % 4 == 0 : p.ldy % 8 == 0 && p.N % 8 == 0);
    return moe_i8_tile(cus, R, p.E, p.N, p.epi == MOE_I8_SWIGLU) == 128 ? moe_launch_i8_gemm_small(p, R, stream) : launch_epilogue(p, R, stream);
}

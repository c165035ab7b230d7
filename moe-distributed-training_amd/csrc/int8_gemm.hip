// The grouped product of 8-bit codes with tiles of 256 x 256, one workgroup of 8 waves per compute unit, and what both tile sizes share.
#define MOE_I8_TILE 256
#include "int8_gemm_kernel.h"

namespace {

constexpr int MAX_SPLIT = 8;   // K parts that a tile of the last, partial round of compute units may be cut into

// compute units that the plan fills, whole rounds of the 8 XCDs
int plan_cus()
{
    const int n = moe_device_cus() / NXCD * NXCD;
    return n < NXCD ? NXCD : n;
}
int64_t counters(int cus) { return 2 * (int64_t)cus + 64; }   // ints in front of the sums or slots (whole 256 bytes)

int64_t tiles_at_most(int tile, int64_t R, int E, int64_t N, bool pair)
{
    const int64_t cols = pair ? tile / 2 : tile;
    return (R / tile + E) * ((N + cols - 1) / cols);
}

// A launch's tile size and the K parts that its tiles may be cut into, by what a launch of evenly dealt rows would take (ns):
//   - a chain of K tiles per workgroup, 550 + 1.2 per row of the tile for tiles of 128 (two workgroups per compute unit) and 750 + 1.8 for 256, times the rounds;
//   - at least the weights at 6 TB/s;
//   - where tiles are cut, the meeting of the parts: sums by atomics at 80 per ns (128), or slots written and read at 2.5 TB/s behind fences of 8 us (256).
// Measured and, in brackets, estimated (us; f=14336, d=4096), [tile, parts]; * what the rule takes:
//   h W2, 2 rows of 2 experts   *[128, 4] 24 (23)    [128, 8] 25 (23)   [128, 1] 57 (62)   [256, 8] 33 (28)
//         4 rows of 1           *[128, 8] 17 (14)    [128, 4] 22 (19)   [128, 1] 56 (62)   [256, 8] 27 (19)
//         64 rows of 1          *[256, 8] 35 (27)    [128, 4] 37 (34)   [128, 8] 40 (39)   [128, 1] 66 (70)
//         500 rows of 1         *[256, 4] 64 (68)    [256, 8] 82 (77)   [128, 1] 59 (79): 8 % slower than it could be
//         48 rows of 8          *[128, 1] 82 (78)    [256, 1] 99 (85)
//         666 rows of 8         *[128, 1] 97 (78)    [256, 4] 110 (-)   [256, 1] 132 (101)
//   gate/up, 666 rows of 8      *[128, 1] 212 (157)  [256, 1] 189 (157): both at the weights' time, and the first of equals is taken, here the slower one
//   gate/up, 16384 rows of 64, 2048 x 1024   *[256, 1] 107 (45)  [128, 1] 141 (45);   their h W2  *[256, 1] 73 (22)  [128, 1] 95 (23)
// The estimate knows neither what a tile costs before its first K tile nor how ragged the groups are: of many small tiles it says far too little, of both sizes alike.
// Where the chip is full anyway (a round of tiles or more) only tiles of 256 are cut, into parts of 16 K tiles at least: those of
// the last round (dX of 8192 rows of 2 experts 903 us uncut, 752 cut; dh, whose K is 32 tiles, 485 uncut, 510 in parts of 4).
struct Plan { int tile, split; };
Plan plan(int cus, int64_t R, int E, int64_t ktiles, int64_t N, bool pair)
{
    const int64_t groups = R < E ? R : E, rows = (R + groups - 1) / groups;
    const double weights = (double)groups * (double)ktiles * BK * (double)N * (pair ? 2 : 1) / 6000.0;
    Plan best = {128, 1};
    double best_ns = -1.0;
    for (int tile = 128; tile <= 256; tile *= 2) {
        const int64_t cols = pair ? tile / 2 : tile, tiles = groups * ((rows + tile - 1) / tile) * ((N + cols - 1) / cols), slots = tile == 128 ? 2 * (int64_t)cus : cus;
        const double ktile_ns = tile == 128 ? 550.0 + 1.2 * (double)(rows < 128 ? rows : 128) : 750.0 + 1.8 * (double)(rows < 256 ? rows : 256);
        for (int split = 1; split <= MAX_SPLIT; split *= 2) {
            if (split > 1 && (ktiles / split < MIN_PART_KTILES || tiles * split > slots)) break;
            const int64_t rounds = (tiles * split + slots - 1) / slots;
            const double chain = (double)((ktiles + split - 1) / split) * ktile_ns * (double)rounds;
            const double sums = (double)R * (double)N * (pair ? 2 : 1) * split;
            const double meet = split == 1 ? 0.0 : tile == 128 ? 3000.0 + sums / 80.0 : 8000.0 + sums * 8.0 / 2500.0;
            const double ns = (chain > weights ? chain : weights) + meet;
            if (best_ns < 0.0 || ns < best_ns) { best = {tile, split}; best_ns = ns; }
        }
        if (tile == 256 && best.tile == 256 && tiles >= cus) {
            best.split = 1;
            while (best.split * 2 <= 4 && ktiles / (best.split * 2) >= 16) best.split *= 2;
        }
    }
    return best;
}

}  // namespace

bool moe_i8_weights_ok(const void* W, int64_t swe, int64_t ldw) { return (uintptr_t)W % 16 == 0 && swe % 16 == 0 && ldw % 16 == 0; }

// 32-bit byte offsets: gathered rows of X from its start (grouped ones from the tile's first row), one expert's matrix (2 GiB where its last K tile is masked); and the
// threads of the grid
bool moe_i8_gemm_supported(const MoeI8Gemm& p, int64_t R, int64_t x_rows)
{
    const int64_t rows = p.x_grouped ? BM : x_rows, limit = p.K % BK ? (int64_t)1 << 31 : (int64_t)1 << 32;
    if (rows * p.ldx >= ((int64_t)1 << 32) || (p.nn ? (p.K - 1) * p.ldw + p.N : (p.N - 1) * p.ldw + p.K) + 16 >= limit) return false;
    const bool pair = p.epi == MOE_I8_SWIGLU;
    const int cus = plan_cus();
    auto fits = [&](int tile) { return moe_grid_fits(tiles_at_most(tile, R, p.E, p.N, pair) + (256 / tile) * cus + NXCD, 2 * tile); };   // (as plan_grid has it, or a few more)
    return fits(128) || fits(plan(cus, R, p.E, (p.K + BK - 1) / BK * p.nseg, p.N, pair).tile);
}

// Where a launch's split tiles meet: `zeros` ints, a counter per workgroup of a round (tiles of 128 have twice those of 256) and, for tiles of 128, the matrix of
// sums; and for tiles of 256 `slots` ints, a tile of them per part.
MoeI8Exchange moe_i8_exchange(int64_t R, int E, int64_t K, int64_t N, bool pair)
{
    if (R < 1) return {0, 0};
    const int cus = plan_cus();
    const Plan pl = plan(cus, R, E, (K + BK - 1) / BK, N, pair);
    if (pl.split == 1) return {0, 0};
    if (pl.tile == 128) return {counters(cus) + (pair ? 2 : 1) * R * N, 0};
    const int64_t all = pl.split * tiles_at_most(pl.tile, R, E, N, pair);
    return {counters(cus), (all < cus ? all : cus) * BM * BN};
}

int moe_i8_tile(int64_t R, int E, int64_t K, int64_t N, bool pair, int nseg, int* parts)
{
    const Plan pl = plan(plan_cus(), R, E, (K + BK - 1) / BK * nseg, N, pair);
    if (parts) *parts = pl.split;
    return pl.tile;
}

int moe_launch_i8_gemm(const MoeI8Gemm& p_, int64_t R, hipStream_t stream)
{
    if (R == 0 || p_.N == 0) return MOE_OK;
    MoeI8Gemm p = p_;
    const int cus = plan_cus();
    const Plan pl = plan(cus, R, p.E, (p.K + BK - 1) / BK * p.nseg, p.N, p.epi == MOE_I8_SWIGLU);
    p.num_cus = cus;
    p.rows = R;
    p.max_split = pl.split;
    if (p.max_split > 1 && (!p.zeros || (pl.tile == 256 && !p.slots))) return MOE_ERR_WORKSPACE;
    p.sk_counters = p.zeros;
    p.sk_partials = pl.tile == 256 ? p.slots : p.zeros + counters(cus);
    p.y_vec = (uintptr_t)p.Y % 16 == 0 && (p.ydtype == MOE_F32 ? p.ldy % 4 == 0 && p.N % 4 == 0 : p.ldy % 8 == 0 && p.N % 8 == 0);
    return pl.tile == 128 ? moe_launch_i8_gemm_small(p, R, stream) : launch_epilogue(p, R, stream);
}

// C-ABI entries of the expert products over 4-bit weights and of the SwiGLU that keeps its inputs in 8 bits: argument checks and launch sequences.  Declarations and their
// contracts: include/moe_hip.h.
#include "../../include/moe_hip.h"
#include "common.h"
#include "kernels.h"

namespace {

inline hipStream_t S(void* s) { return (hipStream_t)s; }
inline size_t al(size_t n) { return (n + 255) & ~(size_t)255; }
inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline int64_t groups_of(int64_t K) { return (K + 31) / 32; }
#define TRY(call) do { const int rc_ = (call); if (rc_ != MOE_OK) return rc_; } while (0)

// rows of codes that 16-byte loads take, and scales that lie one after the other; offsets are unsigned
bool weights_ok(const MoeFp4Weights& w)
{
    return w.codes && w.scales && aligned16(w.codes) && w.sce >= 0 && w.scn >= 0 && w.sse >= 0 && w.ssn >= 0 && w.sce % 16 == 0 && w.scn % 16 == 0;
}

// rows that 16-byte loads take as they are, within their offsets; otherwise they are packed in the order of the product
bool rows_ok(const void* x, int64_t ldx, int64_t x_rows, int64_t cols, int x_grouped)
{
    return aligned16(x) && ldx % 8 == 0 && cols % 8 == 0 && ((x_grouped ? 128 : x_rows) * ldx + cols) * 2 < MOE_FP4_RANGE;
}
int64_t packed_cols(int64_t n) { return (n + 7) / 8 * 8; }
// scales that 4-byte loads take as they are; otherwise rows of whole fours are made of them
bool scales_ok(const uint8_t* scales, int64_t sse, int64_t ssn, int64_t G) { return (uintptr_t)scales % 4 == 0 && sse % 4 == 0 && ssn % 4 == 0 && G % 4 == 0; }
int64_t packed_groups(int64_t G) { return (G + 3) / 4 * 4; }

// What a 16-bit product copies into its workspace before it starts: rows (len columns) and scales.
struct Fp4Copies {
    size_t rows, scales;
    Fp4Copies(const void* x, int64_t ldx, int64_t x_rows, int x_grouped, const uint8_t* s, int64_t sse, int64_t ssn, int64_t R, int E, int64_t K, int64_t N, int64_t len)
        : rows(rows_ok(x, ldx, x_rows, len, x_grouped) ? 0 : al((size_t)R * (size_t)packed_cols(len) * 2)),
          scales(scales_ok(s, sse, ssn, groups_of(K)) ? 0 : al((size_t)E * (size_t)N * (size_t)packed_groups(groups_of(K)))) {}
    // makes them, and has g read them; len becomes whole pieces of rows
    int make(MoeFp4Gemm& g, int64_t R, int64_t len, uint8_t* ws, hipStream_t st) const
    {
        if (rows) {
            const int64_t ld = packed_cols(len);
            TRY(moe_launch_fp4_pack_rows(g.X, g.ldx, g.x_grouped ? nullptr : g.pos, g.pos64, g.fan_out, g.offsets, g.off64, g.E, R, len, ws, ld, st));
            g.X = ws; g.ldx = ld; g.x_grouped = 1;
        }
        if (scales) {
            const int64_t G = groups_of(g.K), ld = packed_groups(G);
            TRY(moe_launch_fp4_pack_scales(g.w.scales, g.w.sse, g.w.ssn, g.E, g.N, G, ws + rows, ld, st));
            g.w.scales = ws + rows; g.w.ssn = ld; g.w.sse = g.N * ld;
        }
        return MOE_OK;
    }
};
bool fp4_sizes_ok(int64_t K, int64_t N, int E, int64_t scn, int64_t ssn)
{
    return K <= 0x3fffff && E <= 65535 && N * scn < MOE_FP4_RANGE && N * ssn < MOE_FP4_RANGE && N * packed_groups(groups_of(K)) < MOE_FP4_RANGE && packed_cols(N) * 256 < MOE_FP4_RANGE;
}

// Which of the two kernels a forward product takes, by their estimated times (us; the host knows the groups' sizes on average only).  Few rows: every 16 rows of an expert, begun ones too, stream its
// codes, at 4.6 TB/s.  Tiles: rounds of two workgroups per compute unit, 0.55 us per 64 inputs and up to as much again for the rows, and the codes once.  Measured (8 experts, rows per expert, give or
// take three: few rows / tiles):
//   4096 x 14336   8: 53 / 67    16: 82 / 67    24: 107 / 67       4096 x 4096   16: 24 / 40    32: 38 / 45    48: 48 / 47    64: 69 / 54       2048 x 2816   16: 11 / 19    64: 23 / 29
//   14336 x 4096   16: 81 / 134    32: 138 / 171    48: 172 / 174    64: 251 / 194       1000 x 1368   16: 6.8 / 11.3    64: 9.4 / 17.5    128: 13.9 / 18.9       2048 x 512   256: 20 / 31
bool fp4_few_rows(int64_t R, int E, int64_t K, int64_t N)
{
    const int64_t used = E < R ? E : R;                    // groups that hold a row, at most
    const double rows = (double)R / used, codes = (double)used * N * groups_of(K) * 17 / 4.6e6;
    const double few = 4 + codes * (rows > 8 ? rows / 16 + 0.5 : 1);
    const int64_t tiles = (R / 128 + used) * ((N + 255) / 256), slots = 2 * (int64_t)moe_device_cus();
    const double tiled = 3 + (double)((tiles + slots - 1) / slots) * ((K + 63) / 64) * (0.55 + 0.5 * (rows < 128 ? rows / 128 : 1));
    return few <= (tiled > codes + 3 ? tiled : codes + 3) || rows <= 8;
}

struct Kept { size_t codes, scales; };
Kept kept_sizes(int64_t rows, int64_t cols)
{
    const size_t blocks = (size_t)rows * (size_t)((cols + MOE_KEPT_BLOCK - 1) / MOE_KEPT_BLOCK);
    return {al(blocks * MOE_KEPT_BLOCK), al(blocks * 4)};
}
size_t kept_bytes(int64_t rows, int64_t cols) { const Kept k = kept_sizes(rows, cols); return 2 * (k.codes + k.scales); }

int swiglu8_params(MoeSwiglu8& p, uint8_t* kept, int64_t rows, int64_t cols)
{
    p.cols = cols;
    const int64_t row_blocks = (cols + MOE_KEPT_BLOCK - 1) / MOE_KEPT_BLOCK;
    // (a launch's threads, eight to a block, are counted in 32 bits)
    if (row_blocks > 0x7fffffff || rows > 0x7fffffff || rows * row_blocks >= (int64_t)1 << 28) return MOE_ERR_UNSUPPORTED;
    p.row_blocks = (uint32_t)row_blocks;
    p.nblocks = (uint32_t)(rows * row_blocks);
    if (kept) {
        const Kept k = kept_sizes(rows, cols);
        p.codes[0] = kept; p.codes[1] = kept + k.codes;
        p.scales[0] = (float*)(kept + 2 * k.codes); p.scales[1] = (float*)(kept + 2 * k.codes + k.scales);
    }
    return MOE_OK;
}

constexpr int64_t MAX_WIDTH = 1 << 20;   // hidden and ffn size of the layer for a few tokens

// what both entry points of the layer for a few tokens share
int decode_params(MoeDecode& p, const void* x, int64_t ldx, const void* wg, int64_t ldwg, int dtype, void* out, int64_t ldo, float* weights, int32_t* indices, int64_t T, int E,
                  int64_t d, int64_t f, int k, int normalize, void* workspace, size_t workspace_bytes, int bits)
{
    if (dtype < 0 || dtype > 2 || T < 0 || E < 1 || d < 64 || f < 64 || d % 64 != 0 || f % 64 != 0 || k < 1 || k > E) return MOE_ERR_BAD_ARG;
    if (dtype == MOE_F32 || T > MOE_DECODE_TOKENS || E > MOE_DECODE_EXPERTS || k > MOE_DECODE_TOPK || d > MAX_WIDTH || f > MAX_WIDTH) return MOE_ERR_UNSUPPORTED;
    if (T == 0) return MOE_OK;
    if (!x || !wg || !out || !weights || !indices || ldx < 0 || ldwg < 0 || (T > 1 && ldo < d)) return MOE_ERR_BAD_ARG;
    if (!aligned16(x) || !aligned16(wg) || ldx % 8 != 0 || ldwg % 8 != 0 || (uintptr_t)out % 8 != 0 || ldo % 4 != 0 || !aligned16(workspace)) return MOE_ERR_BAD_ARG;
    if ((T * ldx + d) * 2 >= MOE_FP4_RANGE || (E * ldwg + d) * 2 >= MOE_FP4_RANGE) return MOE_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < moe_decode_bytes((int)T, E, (int)d, (int)f, k, bits == 4)) return MOE_ERR_WORKSPACE;
    p.x = x; p.ldx = ldx; p.wg = wg; p.ldwg = ldwg; p.out = out; p.ldo = ldo; p.weights = weights; p.indices = indices;
    p.T = (int)T; p.E = E; p.d = (int)d; p.f = (int)f; p.k = k; p.normalize = normalize;
    return MOE_OK;
}

}  // namespace

extern "C" {

int moe_fp4_quantize_weights(const void* W, int64_t swe, int64_t swk, int64_t swn, int dtype, int E, int64_t K, int64_t N, uint8_t* codes, int64_t sce, int64_t scn, uint8_t* scales,
                             int64_t sse, int64_t ssn, void* stream)
{
    if (dtype < 0 || dtype > 2 || E < 1 || K < 1 || N < 1 || !W || !codes || !scales || !aligned16(codes) || sce % 16 != 0 || scn % 16 != 0 || scn < groups_of(K) * 16) return MOE_ERR_BAD_ARG;
    return moe_launch_fp4_quantize(W, swe, swk, swn, dtype, E, K, N, codes, sce, scn, scales, sse, ssn, S(stream));
}

size_t moe_linear_fp4_workspace_bytes(const void* x, int64_t ldx, int64_t x_rows, int x_grouped, int dtype, const uint8_t* scales, int64_t sse, int64_t ssn, int64_t R, int E, int64_t K,
                                      int64_t N)
{
    if (dtype < 0 || dtype > 2 || dtype == MOE_F32 || R < 1 || E < 1 || K < 1 || N < 1) return 0;
    const Fp4Copies c(x, ldx, x_rows, x_grouped, scales, sse, ssn, R, E, K, N, K);
    return c.rows + c.scales;
}

int moe_linear_fp4_fwd(const void* x, int64_t ldx, int64_t x_rows, int dtype, const uint8_t* codes, int64_t sce, int64_t scn, const uint8_t* scales, int64_t sse, int64_t ssn, void* y,
                       int64_t ldy, int y_dtype, const void* pos, int pos64, const void* offsets, int off64, int E, int64_t R, int64_t K, int64_t N, int fan_out, int x_grouped,
                       int y_grouped, void* workspace, size_t workspace_bytes, void* stream)
{
    if (dtype < 0 || dtype > 2 || y_dtype < 0 || y_dtype > 2 || E < 1 || R < 0 || x_rows < 0 || K < 1 || N < 0 || fan_out < 1) return MOE_ERR_BAD_ARG;
    if (R == 0 || N == 0) return MOE_OK;
    if (ldx < 0 || (R > 1 && ldy < N)) return MOE_ERR_BAD_ARG;   // (rows of an input may overlap)
    const MoeFp4Weights w = {codes, sce, scn, scales, sse, ssn};
    if (!x || x_rows < 1 || !weights_ok(w) || !y || !offsets || ((!x_grouped || !y_grouped) && !pos) || (x_grouped && x_rows < R) || !aligned16(workspace)) return MOE_ERR_BAD_ARG;
    const size_t need = moe_linear_fp4_workspace_bytes(x, ldx, x_rows, x_grouped, dtype, scales, sse, ssn, R, E, K, N);
    if (need && (!workspace || workspace_bytes < need)) return MOE_ERR_WORKSPACE;
    if (dtype == MOE_F32 ? y_dtype != MOE_F32 || K > 0x3fffffff : !fp4_sizes_ok(K, N, E, scn, ssn)) return MOE_ERR_UNSUPPORTED;
    MoeFp4Gemm g = {};
    g.X = x; g.ldx = ldx; g.w = w; g.Y = y; g.ldy = ldy; g.ydtype = y_dtype; g.pos = pos; g.pos64 = pos64; g.offsets = offsets; g.off64 = off64;
    g.E = E; g.K = (int)K; g.N = N; g.fan_out = fan_out; g.x_grouped = x_grouped; g.y_grouped = y_grouped; g.f16 = dtype == MOE_F16;
    if (dtype == MOE_F32) return moe_launch_fp4_f32(g, R, false, S(stream));
    const Fp4Copies c(x, ldx, x_rows, x_grouped, scales, sse, ssn, R, E, K, N, K);
    TRY(c.make(g, R, K, (uint8_t*)workspace, S(stream)));
    if (c.rows) g.K = (int)packed_cols(K);   // (the same groups of weights; the rows have zeros there)
    return fp4_few_rows(R, E, g.K, N) ? moe_launch_fp4_few_rows(g, R, S(stream)) : moe_launch_fp4_tiles(g, R, false, S(stream));
}

size_t moe_linear_fp4_bwd_workspace_bytes(const void* dy, int64_t lddy, int64_t dy_rows, int dy_grouped, int dtype, const uint8_t* scales, int64_t sse, int64_t ssn, int64_t R,
                                          int E, int64_t K, int64_t N)
{
    if (dtype < 0 || dtype > 2 || dtype == MOE_F32 || R < 1 || E < 1 || K < 1 || N < 1) return 0;
    const Fp4Copies c(dy, lddy, dy_rows, dy_grouped, scales, sse, ssn, R, E, K, N, N);
    return c.rows + c.scales;
}

int moe_linear_fp4_bwd(const void* dy, int64_t lddy, int64_t dy_rows, int dtype, int dy_grouped, int dy_fan_out, const void* gates, int gates_dtype, const uint8_t* codes, int64_t sce,
                       int64_t scn, const uint8_t* scales, int64_t sse, int64_t ssn, void* dx_rows, int64_t lddx, int dx_dtype, int dx_grouped, const void* pos, int pos64, const void* offsets,
                       int off64, int E, int64_t R, int64_t K, int64_t N, void* workspace, size_t workspace_bytes, void* stream)
{
    if (dtype < 0 || dtype > 2 || dx_dtype < 0 || dx_dtype > 2 || E < 1 || R < 0 || dy_rows < 0 || K < 1 || N < 1 || dy_fan_out < 1 || (gates && (gates_dtype < 0 || gates_dtype > 2 || dy_grouped))) return MOE_ERR_BAD_ARG;
    if (R == 0) return MOE_OK;
    const MoeFp4Weights w = {codes, sce, scn, scales, sse, ssn};
    if (lddy < 0 || (R > 1 && lddx < K) || !dy || dy_rows < 1 || !weights_ok(w) || !dx_rows || !offsets || ((!dy_grouped || !dx_grouped) && !pos) || (dy_grouped && dy_rows < R) ||
        !aligned16(workspace)) return MOE_ERR_BAD_ARG;
    const size_t need = moe_linear_fp4_bwd_workspace_bytes(dy, lddy, dy_rows, dy_grouped, dtype, scales, sse, ssn, R, E, K, N);
    if (need && (!workspace || workspace_bytes < need)) return MOE_ERR_WORKSPACE;
    if (dtype == MOE_F32 ? dx_dtype != MOE_F32 || K > 0x3fffffff : !fp4_sizes_ok(K, N, E, scn, ssn)) return MOE_ERR_UNSUPPORTED;
    MoeFp4Gemm g = {};
    g.X = dy; g.ldx = lddy; g.w = w; g.Y = dx_rows; g.ldy = lddx; g.ydtype = dx_dtype; g.pos = pos; g.pos64 = pos64; g.offsets = offsets; g.off64 = off64;
    g.E = E; g.K = (int)K; g.N = N; g.fan_out = dy_fan_out; g.x_grouped = dy_grouped; g.y_grouped = dx_grouped; g.f16 = dtype == MOE_F16;
    g.gates = gates; g.gates_dtype = gates_dtype;
    if (dtype == MOE_F32) return moe_launch_fp4_f32(g, R, true, S(stream));
    const Fp4Copies c(dy, lddy, dy_rows, dy_grouped, scales, sse, ssn, R, E, K, N, N);
    TRY(c.make(g, R, N, (uint8_t*)workspace, S(stream)));
    return moe_launch_fp4_tiles(g, R, true, S(stream));
}

size_t moe_swiglu8_kept_bytes(int64_t rows, int64_t cols) { return rows < 1 || cols < 1 ? 0 : kept_bytes(rows, cols); }

int moe_swiglu8_fwd(const void* gate, int64_t ldg, const void* up, int64_t ldu, void* h, int64_t ldh, void* kept, size_t kept_size, int64_t rows, int64_t cols, int dtype, void* stream)
{
    if (dtype < 0 || dtype > 2 || rows < 0 || cols < 0) return MOE_ERR_BAD_ARG;
    if (rows == 0 || cols == 0) return MOE_OK;
    if (!gate || !up || !h || ldg < 0 || ldu < 0 || (rows > 1 && ldh < cols) || !aligned16(kept)) return MOE_ERR_BAD_ARG;
    if (kept && kept_size < kept_bytes(rows, cols)) return MOE_ERR_WORKSPACE;
    MoeSwiglu8 p = {};
    p.gate = gate; p.up = up; p.h = h; p.ldg = ldg; p.ldu = ldu; p.ldh = ldh;
    TRY(swiglu8_params(p, (uint8_t*)kept, rows, cols));
    const bool vec = cols % 8 == 0 && ldg % 8 == 0 && ldu % 8 == 0 && ldh % 8 == 0 && aligned16(gate) && aligned16(up) && aligned16(h);
    return moe_launch_swiglu8(p, dtype, vec, false, S(stream));
}

int moe_swiglu8_bwd(const void* kept, size_t kept_size, const void* dh, int64_t lddh, void* dgate, int64_t lddg, void* dup, int64_t lddu, int64_t rows, int64_t cols, int dtype,
                    void* stream)
{
    if (dtype < 0 || dtype > 2 || rows < 0 || cols < 0) return MOE_ERR_BAD_ARG;
    if (rows == 0 || cols == 0) return MOE_OK;
    if (!kept || !dh || !dgate || !dup || lddh < 0 || (rows > 1 && (lddg < cols || lddu < cols)) || !aligned16(kept)) return MOE_ERR_BAD_ARG;
    if (kept_size < kept_bytes(rows, cols)) return MOE_ERR_WORKSPACE;
    MoeSwiglu8 p = {};
    p.dh = dh; p.dgate = dgate; p.dup = dup; p.ldg = lddg; p.ldu = lddu; p.ldh = lddh;
    TRY(swiglu8_params(p, (uint8_t*)kept, rows, cols));
    const bool vec = cols % 8 == 0 && lddh % 8 == 0 && lddg % 8 == 0 && lddu % 8 == 0 && aligned16(dh) && aligned16(dgate) && aligned16(dup);
    return moe_launch_swiglu8(p, dtype, vec, true, S(stream));
}

size_t moe_decode_layer_workspace_bytes(int64_t T, int E, int64_t d, int64_t f, int k, int bits)
{
    if (T < 1 || T > MOE_DECODE_TOKENS || E < 1 || E > MOE_DECODE_EXPERTS || d < 64 || f < 64 || d > MAX_WIDTH || f > MAX_WIDTH || k < 1 || k > E || k > MOE_DECODE_TOPK) return 0;
    return moe_decode_bytes((int)T, E, (int)d, (int)f, k, bits == 4);
}

int moe_decode_layer(const void* x, int64_t ldx, const void* wg, int64_t ldwg, int dtype, const void* w1, const void* w3, const void* w2, void* out, int64_t ldo, float* weights,
                     int32_t* indices, int64_t T, int E, int64_t d, int64_t f, int k, int normalize, void* workspace, size_t workspace_bytes, void* stream)
{
    MoeDecode p = {};
    TRY(decode_params(p, x, ldx, wg, ldwg, dtype, out, ldo, weights, indices, T, E, d, f, k, normalize, workspace, workspace_bytes, 16));
    if (T == 0) return MOE_OK;
    if (!w1 || !w3 || !w2 || !aligned16(w1) || !aligned16(w3) || !aligned16(w2)) return MOE_ERR_BAD_ARG;
    if (d * f * 2 >= MOE_FP4_RANGE) return MOE_ERR_UNSUPPORTED;
    p.w1 = w1; p.w3 = w3; p.w2 = w2;
    return moe_launch_decode(p, false, dtype == MOE_F16, workspace, S(stream));
}

int moe_decode_layer_fp4(const void* x, int64_t ldx, const void* wg, int64_t ldwg, int dtype, const uint8_t* c1, const uint8_t* s1, const uint8_t* c3, const uint8_t* s3,
                         const uint8_t* c2, const uint8_t* s2, void* out, int64_t ldo, float* weights, int32_t* indices, int64_t T, int E, int64_t d, int64_t f, int k, int normalize,
                         void* workspace, size_t workspace_bytes, void* stream)
{
    MoeDecode p = {};
    TRY(decode_params(p, x, ldx, wg, ldwg, dtype, out, ldo, weights, indices, T, E, d, f, k, normalize, workspace, workspace_bytes, 4));
    if (T == 0) return MOE_OK;
    if (d * f >= MOE_FP4_RANGE) return MOE_ERR_UNSUPPORTED;
    auto take = [](const uint8_t* c, const uint8_t* s, int64_t rows, int64_t inner) { return MoeFp4Weights{c, rows * (inner / 2), inner / 2, s, rows * (inner / 32), inner / 32}; };
    p.f1 = take(c1, s1, f, d);
    p.f3 = take(c3, s3, f, d);
    p.f2 = take(c2, s2, d, f);
    for (const MoeFp4Weights* w : {&p.f1, &p.f3, &p.f2})
        if (!weights_ok(*w) || !aligned16(w->scales)) return MOE_ERR_BAD_ARG;
    return moe_launch_decode(p, true, dtype == MOE_F16, workspace, S(stream));
}

}  // extern "C"

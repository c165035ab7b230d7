// The whole MoE layer for the few tokens of a generation step (16 at most) in two launches:
//
//   logits = x Wg^T;  s = softmax(logits);  the k largest (ties to the lower expert), w_j = s_j / sum s  (or s_j);
//   h_j = silu(x W1_j^T) * (x W3_j^T);      out = sum_j w_j (h_j W2_j^T)
//
// Launch 1 (gate_up_kernel): every workgroup computes the router for itself -- the router's weight stays in L2, and a launch of its own would cost more -- and then
// takes blocks of 16 ffn columns of the experts that some token chose: gate and up of all tokens, summed over the waves in LDS, h into the workspace.
// Launch 2 (down_kernel): a workgroup takes a block of output columns and a part of the contraction, which runs over the chosen experts one after the other; parts add up their
// sums in the workspace, the one that arrives last writes the output, in part order.  Nobody waits for anybody.
//
// Both are bound by the weights of the chosen experts, each byte read once (few_rows.h).  All tokens of the batch are rows of the matrix operand, so a weight is read once however
// many tokens chose its expert; rows of other tokens are computed in launch 1 and not stored, and are absent from launch 2.
// h travels as two numbers of the activations' type, h and what its rounding lost (16 bits more), whose products are added: the result then carries one rounding, its own.
#include "few_rows.h"
#include "kernels.h"

namespace {

constexpr int WAVES = 8, THREADS = WAVES * 64;
constexpr int TOK = MOE_DECODE_TOKENS, MAXK = MOE_DECODE_TOPK, MAXE = MOE_DECODE_EXPERTS;

// what a workgroup knows of the routing
struct Chosen {
    int idx[TOK][MAXK];
    float weight[TOK][MAXK];
    int used[MAXE];          // whether a token chose the expert
    int active[MAXE];        // those experts, in order
    int nactive;
};

// the chosen experts in order, from idx; all threads
__device__ __forceinline__ void list_active(Chosen& c, int T, int E, int k)
{
    for (int e = threadIdx.x; e < E; e += THREADS) c.used[e] = 0;
    __syncthreads();
    for (int x = threadIdx.x; x < T * k; x += THREADS) c.used[c.idx[x / k][x % k]] = 1;   // (several threads may write the same 1)
    __syncthreads();
    if (threadIdx.x < 64) {
        int n = 0;
        for (int base = 0; base < E; base += 64) {
            const int e = base + threadIdx.x;
            const bool on = e < E && c.used[e];
            const unsigned long long m = __ballot(on);
            if (on) c.active[n + __popcll(m & ((1ull << threadIdx.x) - 1))] = e;
            n += __popcll(m);
        }
        if (threadIdx.x == 0) c.nactive = n;
    }
    __syncthreads();
}

// which of token t's choices is expert e: -1 if none
__device__ __forceinline__ int choice_of(const Chosen& c, int t, int e, int k)
{
    int at = -1;
    for (int j = 0; j < k; ++j) at = c.idx[t][j] == e ? j : at;
    return at;
}

// numbers in an order that unsigned integers have (NaN, of either sign, before all others)
__device__ __forceinline__ uint32_t order_of(float v)
{
    if (v != v) return 0;
    const uint32_t b = __float_as_uint(v);
    return b >> 31 ? ~b : b | 0x80000000u;
}

// Logits, softmax and choices of all tokens, in LDS (scratch: WAVES * 1 KiB of sums and TOK * MAXE logits).
template <class Num> __device__ __forceinline__ void route(const MoeDecode& p, Chosen& c, float* red, float* logits)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    const int chunks = (p.d + few::CHUNK - 1) / few::CHUNK;
    typedef few::Cols16<Num, 1> W;
    few::Rows<1> rows;
    rows.K = p.d;
    rows.x[0] = few::buffer(p.x);
    rows.a[0] = i < p.T ? (uint32_t)(i * p.ldx + 8 * q) * 2 : few::RANGE;
    W w;
    w.w[0] = w.w[1] = few::buffer(p.wg);
    w.left = p.d - 8 * q;
    for (int eb = 0; eb < p.E; eb += 16) {
        const int e = eb + i < p.E ? eb + i : p.E - 1;
        w.c[0] = (uint32_t)(e * p.ldwg + 8 * q) * 2;
        f32x4_t acc[1][1] = {{(f32x4_t){0.f, 0.f, 0.f, 0.f}}};
        few::stream<W, 1, false, 4>(acc, w, rows, chunks * wave / WAVES, chunks * (wave + 1) / WAVES);
        *(f32x4_t*)(red + (wave * 64 + lane) * 4) = acc[0][0];
        __syncthreads();
        if (threadIdx.x < 256) {   // expert eb + x of token t
            const int t = threadIdx.x & 15, x = threadIdx.x >> 4;
            double sum = 0;   // (choices between experts are values next to a border)
            for (int v = 0; v < WAVES; ++v) sum += (double)red[(v * 64 + (x >> 2) * 16 + t) * 4 + (x & 3)];
            if (eb + x < p.E) logits[t * MAXE + eb + x] = (float)sum;
        }
        __syncthreads();
    }
    // a wave per token: softmax over its experts, then the largest one after the other
    for (int t = wave; t < p.T; t += WAVES) {
        constexpr int PER = MAXE / 64;
        float v[PER], top = -__builtin_inff();
        unsigned long long key[PER];
        bool nan = false;
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int e = r * 64 + lane;
            v[r] = e < p.E ? logits[t * MAXE + e] : -__builtin_inff();
            top = fmaxf(top, v[r]);
            nan = nan || v[r] != v[r];
            // (ties to the lower expert; an expert's key is never 0, that of a taken or absent one is)
            key[r] = e < p.E ? (unsigned long long)order_of(v[r]) << 32 | (0xffffffffu - e) : 0;
        }
        float sum = 0.f;
        for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            v[r] = r * 64 + lane < p.E ? expf(v[r] - top) : 0.f;
            sum += v[r];
        }
        for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
        if (__any(nan)) sum = __builtin_nanf("");
        float chosen[MAXK], total = 0.f;
        for (int j = 0; j < p.k; ++j) {
            unsigned long long best = 0;
#pragma unroll
            for (int r = 0; r < PER; ++r) best = key[r] > best ? key[r] : best;
            for (int m = 32; m > 0; m >>= 1) {
                const unsigned long long o = __shfl_xor(best, m);
                best = o > best ? o : best;
            }
            const int e = (int)(0xffffffffu - (uint32_t)best);
            float mine = 0.f;
#pragma unroll
            for (int r = 0; r < PER; ++r)
                if (r * 64 + lane == e) { mine = v[r]; key[r] = 0; }
            chosen[j] = __shfl(mine, e & 63) / sum;
            total += chosen[j];
            if (lane == 0) c.idx[t][j] = e;
        }
        for (int j = 0; j < p.k; ++j)
            if (lane == 0) c.weight[t][j] = p.normalize ? chosen[j] / total : chosen[j];
    }
    __syncthreads();
}

template <class W> __device__ __forceinline__ void gate_up_columns(const MoeDecode& p, W& w, int e, int n, int i, int q)
{
    if constexpr (std::is_same<W, few::Fp4Cols<typename W::Num, 2>>::value) {
        w.two = true;
        w.left = p.d / FP4_GROUP - q;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const MoeFp4Weights& f = m ? p.f3 : p.f1;
            w.codes[m] = few::buffer(f.codes + e * f.sce);
            w.scales[m] = few::buffer(f.scales + e * f.sse);
            w.c[m] = (uint32_t)((n + i) * f.scn) + q * FP4_GROUP_BYTES;
            w.s[m] = (uint32_t)((n + i) * f.ssn) + q;
        }
    } else {
        w.left = p.d - 8 * q;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            w.w[m] = few::buffer((const uint16_t*)(m ? p.w3 : p.w1) + (int64_t)e * p.f * p.d);
            w.c[m] = (uint32_t)((int64_t)(n + i) * p.d + 8 * q) * 2;
        }
    }
}

template <class Num, bool FP4>
__global__ void __launch_bounds__(THREADS) gate_up_kernel(const MoeDecode p)
{
    typedef typename std::conditional<FP4, few::Fp4Cols<Num, 2>, few::Cols16<Num, 2>>::type W;
    __shared__ Chosen c;
    __shared__ __attribute__((aligned(16))) float red[2][WAVES][2][64][4];   // sums of two jobs; before them the router's
    __shared__ float logits[TOK * MAXE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    route<Num>(p, c, &red[0][0][0][0][0], logits);
    if (blockIdx.x == 0) {
        for (int x = threadIdx.x; x < p.T * p.k; x += THREADS) {
            p.indices[x] = c.idx[x / p.k][x % p.k];
            p.weights[x] = c.weight[x / p.k][x % p.k];
        }
        for (int x = threadIdx.x; x < p.counters_n; x += THREADS) p.counters[x] = 0;   // of launch 2
    }
    list_active(c, p.T, p.E, p.k);
    const int ncb = p.f / 16, jobs = c.nactive * ncb, chunks = (p.d + few::CHUNK - 1) / few::CHUNK;
    few::Rows<1> rows;
    rows.K = p.d;
    rows.x[0] = few::buffer(p.x);
    rows.a[0] = i < p.T ? (uint32_t)(i * p.ldx + W::input(0, q)) * 2 : few::RANGE;
    int turn = 0;
    for (int job = blockIdx.x; job < jobs; job += gridDim.x, ++turn) {
        const int e = __builtin_amdgcn_readfirstlane(c.active[job / ncb]), n = __builtin_amdgcn_readfirstlane(job % ncb) * 16;
        W w;
        gate_up_columns(p, w, e, n, i, q);
        f32x4_t acc[1][2] = {{(f32x4_t){0.f, 0.f, 0.f, 0.f}, (f32x4_t){0.f, 0.f, 0.f, 0.f}}};
        few::stream<W, 1, false, FP4 ? 4 : 2>(acc, w, rows, chunks * wave / WAVES, chunks * (wave + 1) / WAVES);
        float (*r)[2][64][4] = red[turn & 1];   // (the other one may still be read)
        *(f32x4_t*)r[wave][0][lane] = acc[0][0];
        *(f32x4_t*)r[wave][1][lane] = acc[0][1];
        __syncthreads();
        if (wave == (turn & (WAVES - 1)) && i < p.T) {
            const int j = choice_of(c, i, e, p.k);
            if (j >= 0) {
                f32x4_t g = (f32x4_t){0.f, 0.f, 0.f, 0.f}, u = g;
#pragma unroll
                for (int v = 0; v < WAVES; ++v) { g += *(const f32x4_t*)r[v][0][lane]; u += *(const f32x4_t*)r[v][1][lane]; }
                float hi[4], lo[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float h = g[v] / (1.f + __expf(-g[v])) * u[v];
                    hi[v] = Num::to_f32(Num::from_f32(h));
                    lo[v] = fabsf(hi[v]) < __builtin_inff() ? h - hi[v] : 0.f;
                }
                uint16_t* h = p.h + ((int64_t)(i * p.k + j) * p.f + n + 4 * q);
                *(uint2*)h = make_uint2(Num::pack2(hi[0], hi[1]), Num::pack2(hi[2], hi[3]));
                *(uint2*)(h + p.h_lo) = make_uint2(Num::pack2(lo[0], lo[1]), Num::pack2(lo[2], lo[3]));
            }
        }
    }
}

// ---- launch 2
// 4-bit W2 (E, d, f): 64 output columns, NB = 4 blocks whose columns are dealt so that a lane holds 4 NB consecutive ones.  16-bit W2 (E, f, d), contiguous along the output:
// 128 columns; a lane loads 8 of them (16 bytes) in 8 rows and transposes the 8 x 8 block in registers, one instruction for two values; the weight is the second operand, so a lane
// ends up with 8 consecutive columns of four tokens.
constexpr int DOWN_PARTS_MAX = 64;

template <class Num, bool FP4>
__global__ void __launch_bounds__(THREADS) down_kernel(const MoeDecode p)
{
    constexpr int UNITS = 4, PER = FP4 ? 4 : 8;   // floats of a lane and unit: unit nb holds 4 columns of one token, unit r 8 columns of one
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ Chosen c;
    __shared__ int arrival;
    float* red = (float*)smem;   // [wave][unit][64][PER]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    const int tile = blockIdx.x / p.parts, part = blockIdx.x - tile * p.parts;
    for (int x = threadIdx.x; x < p.T * p.k; x += THREADS) {
        c.idx[x / p.k][x % p.k] = p.indices[x];
        c.weight[x / p.k][x % p.k] = p.weights[x];
    }
    __syncthreads();
    list_active(c, p.T, p.E, p.k);
    // this wave's share of the contraction: steps of the chosen experts one after the other
    const int steps = FP4 ? (p.f + few::CHUNK - 1) / few::CHUNK : p.f / 32;
    const int64_t total = (int64_t)c.nactive * steps;
    const int shares = p.parts * WAVES, share = part * WAVES + wave;
    int64_t at = total * share / shares;
    const int64_t end = total * (share + 1) / shares;
    float out[UNITS][PER];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int v = 0; v < PER; ++v) out[u][v] = 0.f;
    while (at < end) {
        const int a = (int)(at / steps), s0 = __builtin_amdgcn_readfirstlane((int)(at - (int64_t)a * steps));
        const int s1 = __builtin_amdgcn_readfirstlane(end - at < steps - s0 ? s0 + (int)(end - at) : steps);
        const int e = __builtin_amdgcn_readfirstlane(c.active[a]);
        at += s1 - s0;
        const int j = i < p.T ? choice_of(c, i, e, p.k) : -1;
        few::Rows<2> rows;
        rows.K = p.f;
        rows.x[0] = few::buffer(p.h);
        rows.x[1] = few::buffer(p.h + p.h_lo);
        if constexpr (FP4) {
            typedef few::Fp4Cols<Num, 4> W;
            W w;
            w.two = false;
            w.left = p.f / FP4_GROUP - q;
            w.codes[0] = few::buffer(p.f2.codes + e * p.f2.sce);
            w.scales[0] = few::buffer(p.f2.scales + e * p.f2.sse);
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) {
                const int n = tile * 64 + (i >> 2) * 16 + 4 * nb + (i & 3);   // (d is a multiple of 64)
                w.c[nb] = (uint32_t)(n * p.f2.scn) + q * FP4_GROUP_BYTES;
                w.s[nb] = (uint32_t)(n * p.f2.ssn) + q;
            }
            rows.a[0] = rows.a[1] = j >= 0 ? (uint32_t)((i * p.k + j) * p.f + W::input(0, q)) * 2 : few::RANGE;
            f32x4_t acc[1][4];
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[0][nb] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            few::stream<W, 2, true, 2>(acc, w, rows, s0, s1);
            const float g = j >= 0 ? c.weight[i][j] : 0.f;
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int v = 0; v < PER; ++v) out[u][v] = j >= 0 ? out[u][v] + g * acc[0][u][v] : out[u][v];   // (what other tokens' rows hold may not be finite)
        } else {
            const few::Buffer w = few::buffer((const uint16_t*)p.w2 + (int64_t)e * p.f * p.d);
            const int n = tile * 128 + 8 * i;
            const uint32_t col = n < p.d ? (uint32_t)(n + 8 * q * p.d) * 2 : few::RANGE;
            const uint32_t row = j >= 0 ? (uint32_t)((i * p.k + j) * p.f + 8 * q) * 2 : few::RANGE;
            f32x4_t acc[8];
#pragma unroll
            for (int b = 0; b < 8; ++b) acc[b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            constexpr int DEPTH = 2;
            fp4_u32x4_t ws[DEPTH][8];
            bf16x8_t as[DEPTH][2];
            auto fetch = [&](int dst, int s) {
#pragma unroll
                for (int r = 0; r < 8; ++r) ws[dst][r] = few::load16_streamed(w, col, (uint32_t)(s * 32 + r) * (uint32_t)p.d * 2);
#pragma unroll
                for (int m = 0; m < 2; ++m) as[dst][m] = few::load16(rows.x[m], row, (uint32_t)s * 64);
            };
            auto multiply = [&](int src) {
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    fp4_u32x4_t f;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        f[r] = __builtin_amdgcn_perm(ws[src][2 * r + 1][b / 2], ws[src][2 * r][b / 2], b & 1 ? 0x07060302u : 0x05040100u);
                    const bf16x8_t wf = __builtin_bit_cast(bf16x8_t, f);
                    acc[b] = Num::mfma(as[src][0], wf, acc[b]);
                    acc[b] = Num::mfma(as[src][1], wf, acc[b]);
                }
            };
            int s = s0;
            if (s1 - s0 >= DEPTH) {
#pragma unroll
                for (int x = 0; x < DEPTH; ++x) fetch(x, s + x);
                for (; s + 2 * DEPTH <= s1; s += DEPTH)
#pragma unroll
                    for (int x = 0; x < DEPTH; ++x) { multiply(x); fetch(x, s + DEPTH + x); }
                const int more = s1 - s - DEPTH;
#pragma unroll
                for (int x = 0; x < DEPTH; ++x) { multiply(x); if (x < more) fetch(x, s + DEPTH + x); }
#pragma unroll
                for (int x = 0; x < DEPTH - 1; ++x)
                    if (x < more) multiply(x);
            } else {
                fetch(0, s);
                multiply(0);
            }
            // acc[b][r] is column 8 i + b of token 4 q + r
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 4 * q + r, jr = t < p.T ? choice_of(c, t, e, p.k) : -1;
                const float g = jr >= 0 ? c.weight[t][jr] : 0.f;
#pragma unroll
                for (int b = 0; b < 8; ++b) out[r][b] = jr >= 0 ? out[r][b] + g * acc[b][r] : out[r][b];
            }
        }
    }
    // ---- the waves' sums, in wave order
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int v = 0; v < PER; v += 4)
            *(f32x4_t*)(red + ((wave * UNITS + u) * 64 + lane) * PER + v) = (f32x4_t){out[u][v], out[u][v + 1], out[u][v + 2], out[u][v + 3]};
    __syncthreads();
    float sum[PER];
    const bool mine = wave < UNITS;
    const int t = FP4 ? i : 4 * q + wave;                                         // the token and the first column of this lane's sums
    const int n = FP4 ? tile * 64 + q * 16 + 4 * wave : tile * 128 + 8 * i;
    const bool live = mine && t < p.T && n < p.d;
    if (live) {
#pragma unroll
        for (int v = 0; v < PER; ++v) sum[v] = 0.f;
        for (int x = 0; x < WAVES; ++x)
#pragma unroll
            for (int v = 0; v < PER; ++v) sum[v] += red[((x * UNITS + wave) * 64 + lane) * PER + v];
    }
    if (p.parts > 1) {
        // A part's sums go to a slot of their own by device-scope stores, then the tile's counter; the part that counts last adds up all slots in part order.
        constexpr int DEVICE_SCOPE = 16;
        const few::Buffer slots = few::buffer(p.slots);
        auto slot = [&](int x) { return (uint32_t)((((int64_t)tile * p.parts + x) * UNITS + wave) * 64 + lane) * (PER * 4); };
        if (live)
#pragma unroll
            for (int v = 0; v < PER; v += 4)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(fp4_u32x4_t, (f32x4_t){sum[v], sum[v + 1], sum[v + 2], sum[v + 3]}), slots, slot(part) + 4 * v, 0, DEVICE_SCOPE);
        __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's stores are acknowledged
        __syncthreads();                      // ... and every wave's
        if (threadIdx.x == 0) arrival = __hip_atomic_fetch_add(&p.counters[tile], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrival != p.parts - 1) return;
        if (live) {
#pragma unroll
            for (int v = 0; v < PER; ++v) sum[v] = 0.f;
            for (int x = 0; x < p.parts; ++x)
#pragma unroll
                for (int v = 0; v < PER; v += 4) {
                    const f32x4_t s = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(slots, slot(x) + 4 * v, 0, DEVICE_SCOPE));
#pragma unroll
                    for (int y = 0; y < 4; ++y) sum[v + y] += s[y];
                }
        }
    }
    if (!live) return;
    uint16_t* o = (uint16_t*)p.out + t * p.ldo + n;
#pragma unroll
    for (int v = 0; v < PER; v += 4) *(uint2*)(o + v) = make_uint2(Num::pack2(sum[v], sum[v + 1]), Num::pack2(sum[v + 2], sum[v + 3]));
}

struct Plan { int grid1, tiles, parts; size_t h_bytes, counter_bytes, slot_bytes; };
Plan plan(int T, int E, int d, int f, int k, bool fp4)
{
    Plan r = {};
    const int cus = moe_device_cus();
    const int64_t jobs = (int64_t)(E < T * k ? E : T * k) * (f / 16);
    r.grid1 = (int)(jobs < 2 * cus ? jobs : 2 * cus);
    r.tiles = fp4 ? d / 64 : (d + 127) / 128;
    r.parts = 1;
    while (r.parts < DOWN_PARTS_MAX && r.tiles * r.parts < cus) r.parts *= 2;
    auto al = [](size_t n) { return (n + 255) & ~(size_t)255; };
    r.h_bytes = al((size_t)T * k * f * 2);
    r.counter_bytes = al((size_t)r.tiles * 4);
    r.slot_bytes = r.parts > 1 ? al((size_t)r.tiles * r.parts * 4 * 64 * (fp4 ? 4 : 8) * 4) : 0;
    return r;
}

template <class Num, bool FP4> int launch_typed(const MoeDecode& p, const Plan& pl, hipStream_t stream)
{
    constexpr size_t lds = (size_t)WAVES * 4 * 64 * (FP4 ? 4 : 8) * 4;
    hipLaunchKernelGGL((gate_up_kernel<Num, FP4>), dim3((unsigned)pl.grid1), dim3(THREADS), 0, stream, p);
    hipLaunchKernelGGL((down_kernel<Num, FP4>), dim3((unsigned)(pl.tiles * pl.parts)), dim3(THREADS), lds, stream, p);
    return moe_launch_status();
}

}  // namespace

size_t moe_decode_bytes(int T, int E, int d, int f, int k, bool fp4)
{
    const Plan pl = plan(T, E, d, f, k, fp4);
    return 2 * pl.h_bytes + pl.counter_bytes + pl.slot_bytes;
}

int moe_launch_decode(MoeDecode p, bool fp4, bool f16, void* workspace, hipStream_t stream)
{
    const Plan pl = plan(p.T, p.E, p.d, p.f, p.k, fp4);
    uint8_t* b = (uint8_t*)workspace;
    p.h = (uint16_t*)b; p.h_lo = (int64_t)(pl.h_bytes / 2);
    p.counters = (int*)(b + 2 * pl.h_bytes); p.counters_n = pl.tiles;
    p.slots = (float*)(b + 2 * pl.h_bytes + pl.counter_bytes);
    p.parts = pl.parts;
    if (f16) return fp4 ? launch_typed<NumF16, true>(p, pl, stream) : launch_typed<NumF16, false>(p, pl, stream);
    return fp4 ? launch_typed<NumBf16, true>(p, pl, stream) : launch_typed<NumBf16, false>(p, pl, stream);
}

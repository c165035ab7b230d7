// The whole MoE layer for the few tokens of a generation step (16 at most) in two launches:
//
//   logits = x Wg^T;  s = softmax(logits), fp32;  the k largest s (ties to the lower expert), w_j = s_j / sum s  (or s_j);
//   h_j = silu(x W1_j^T) * (x W3_j^T);      out = sum_j w_j (h_j W2_j^T)
//
// Launch 1 (gate_up_kernel): every workgroup computes the router for itself -- the router's weight stays in L2, and a launch of its own would cost more -- and then
// takes blocks of 16 ffn columns of the experts that some token chose: gate and up of all tokens, summed over the waves in LDS, h into the workspace.
// Launch 2 (down_kernel): a workgroup takes a block of output columns and a part of the contraction, which runs over the chosen experts one after the other; parts add up their
// sums in the workspace, the one that arrives last writes the output, in part order.  Nobody waits for anybody.
//
// Both are bound by the weights of the chosen experts, each byte read once (few_rows.h).  All tokens of the batch are rows of the matrix operand, so a weight is read once however
// many tokens chose its expert; rows of other tokens are computed in launch 1 and not stored, and are absent from launch 2.
// Measured (launch 1 + launch 2, 4096 x 14336, 8 experts, top-2): one token in 16 bits 84 + 49 us (5.6 and 4.8 TB/s), in 4 bits 30 + 22.5; sixteen tokens in 4 bits 87 + 65 (5.7 and 3.9; their rows of h, read by
// every tile, cost 10).  Of launch 1 the router takes 6 us (11 with 64 experts), of launch 2 the meeting of the parts 4.
// h travels as two numbers of the activations' type, h and what its rounding lost, whose products are added: h to 2^-17 of itself in bf16; in fp16 to 2^-23, or to 2^-25 where that is more (half the
// subnormal step), and infinite beyond 65504.  Besides that the result carries one rounding, its own.  (A third number would be half as many products and
// bytes of rows again; for the lack of it 10 of a bf16 result's 4096 values round the other way, at the same error.)
#include "few_rows.h"
#include "gemm_tiles.h"
#include "kernels.h"

namespace {

constexpr int WAVES = 8, THREADS = WAVES * 64;
constexpr int TOK = MOE_DECODE_TOKENS, MAXK = MOE_DECODE_TOPK, MAXE = MOE_DECODE_EXPERTS;

// what a workgroup knows of the routing
struct Chosen {
    int idx[TOK][MAXK];
    float weight[TOK][MAXK];
    uint32_t used[MAXE / 32];   // bits of the experts that a token chose
    int active[MAXE];           // those experts, in order
};

// the chosen experts in order, from their bits; all threads, behind a barrier
__device__ __forceinline__ int list_active(Chosen& c)
{
    static_assert(THREADS >= MAXE, "a thread per expert");
    const int e = threadIdx.x;
    int n = 0, before = 0;
#pragma unroll
    for (int w = 0; w < MAXE / 32; ++w) {
        const uint32_t bits = c.used[w];
        before += __popc(e >> 5 > w ? bits : e >> 5 == w ? bits & ((1u << (e & 31)) - 1) : 0u);
        n += __popc(bits);
    }
    if (e < MAXE && c.used[e >> 5] >> (e & 31) & 1) c.active[before] = e;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(n);
}

// which of token t's choices is expert e: -1 if none
__device__ __forceinline__ int choice_of(const Chosen& c, int t, int e, int k)
{
    int at = -1;
    for (int j = 0; j < k; ++j) at = c.idx[t][j] == e ? j : at;
    return at;
}

// numbers in an order that positive integers have (NaN, of either sign, before all others)
__device__ __forceinline__ uint32_t order_of(float v)
{
    if (v != v) return 1;
    const uint32_t b = __float_as_uint(v);
    return b >> 31 ? ~b : b | 0x80000000u;
}

// the largest value of the wave's lanes, in every lane: within rows of 16 lanes and from row to row without LDS
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    auto with = [&](auto ctrl, auto rows) {
        const uint32_t o = __builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, true);
        v = o > v ? o : v;
    };
    with(std::integral_constant<int, DPP_ROW_SHR + 1>{}, std::integral_constant<int, 0xf>{});
    with(std::integral_constant<int, DPP_ROW_SHR + 2>{}, std::integral_constant<int, 0xf>{});
    with(std::integral_constant<int, DPP_ROW_SHR + 4>{}, std::integral_constant<int, 0xf>{});
    with(std::integral_constant<int, DPP_ROW_SHR + 8>{}, std::integral_constant<int, 0xf>{});
    with(std::integral_constant<int, DPP_ROW_BCAST15>{}, std::integral_constant<int, 0xa>{});
    with(std::integral_constant<int, DPP_ROW_BCAST31>{}, std::integral_constant<int, 0xc>{});
    return __builtin_amdgcn_readlane(v, 63);
}

// Softmax and choices of all tokens from their logits, which make room for the exponentials: a wave per token.  Experts are ranked by their fp32 scores, as the router of the other paths ranks them (softmax_topk_token of routing.hip, with
// the exponentials added in expert order there too, so that equal logits get the same bits): scores that underflow or round to the same number are ties, and NaN scores lose to every number and
// are taken in expert order.
__device__ __forceinline__ void choose(const MoeDecode& p, Chosen& c, float* logits)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int PER = MAXE / 64;
    const int per = (p.E + 63) / 64;
    for (int t = wave; t < p.T; t += WAVES) {
        float v[PER];
        uint32_t key[PER], top = 0;
        for (int r = 0; r < PER; ++r) { v[r] = 0.f; key[r] = 0; }
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (r < per && r * 64 + lane < p.E) {
                v[r] = logits[t * MAXE + r * 64 + lane];
                const uint32_t o = order_of(v[r]);
                top = o > top ? o : top;
            }
        float sum = 0.f;
        const uint32_t most = wave_max(top);
        const float shift = __uint_as_float(most >> 31 ? most & 0x7fffffffu : ~most);   // the largest logit
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (r < per) {
                v[r] = r * 64 + lane < p.E ? expf(v[r] - shift) : 0.f;
                logits[t * MAXE + r * 64 + lane] = v[r];
            }
        few::in_order();
        // (every lane adds all of them, from LDS: with moves between lanes 64 experts took 2 us more, 256 experts and 16 tokens 17)
#pragma unroll 4
        for (int e = 0; e < p.E; e += 4) {
            const f32x4_t x = *(const f32x4_t*)(logits + t * MAXE + e);
            sum += x[0]; sum += x[1]; sum += x[2]; sum += x[3];
        }
        // (the key of a taken or absent expert is 0, of a NaN score 1)
#pragma unroll
        for (int r = 0; r < PER; ++r)
            if (r < per && r * 64 + lane < p.E) {
                v[r] /= sum;
                key[r] = v[r] >= 0.f ? __float_as_uint(v[r]) + 2 : 1;
            }
        float total = 0.f;
        float chosen = 0.f;   // lane j keeps the weight of choice j
        int choice = 0;
        for (int j = 0; j < p.k; ++j) {
            uint32_t best = 0;
#pragma unroll
            for (int r = 0; r < PER; ++r) best = key[r] > best ? key[r] : best;
            best = wave_max(best);
            int e = 0;
            float s = 0.f;
            bool found = false;
#pragma unroll
            for (int r = 0; r < PER; ++r)
                if (r < per && !found) {   // ties: the lower expert
                    const unsigned long long hit = __ballot(key[r] == best);
                    if (hit != 0) {
                        const int l = __ffsll(hit) - 1;
                        e = r * 64 + l;
                        s = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v[r]), l));
                        if (lane == l) key[r] = 0;
                        found = true;
                    }
                }
            total += s;
            if (lane == j) { chosen = s; choice = e; }
        }
        if (lane < p.k) {
            c.idx[t][lane] = choice;
            c.weight[t][lane] = p.normalize ? chosen / total : chosen;
            atomicOr(&c.used[choice >> 5], 1u << (choice & 31));
        }
    }
    __syncthreads();
}

// (Steps of 32 products and waves are summed in 64 bits, as in the wide router of routing.hip: choices between experts are values next to a border.  Against fp32 chains of a wave's share: 64 experts 0.7 us more, 8 experts 0.3, 8 of hidden size 4224 1.0.)
__device__ __forceinline__ f32x4_t rounded(const few::Wide& a) { return (f32x4_t){(float)a.v[0], (float)a.v[1], (float)a.v[2], (float)a.v[3]}; }
// Logits of all tokens for experts of a block of 16 each, from the waves' sums [64][4], `stride` apart: each of `blocks` blocks from eb on is shared by `split` waves.
__device__ __forceinline__ void sum_logits(const MoeDecode& p, const float* red, int stride, float* logits, int eb, int blocks, int split)
{
    for (int x = threadIdx.x; x < blocks * 256; x += THREADS) {
        const int t = x & 15, y = x >> 4 & 15, b = x >> 8, e = (eb + b) * 16 + y;
        double sum = 0;
        for (int v = 0; v < split; ++v) sum += (double)red[(b * split + v) * stride + ((y >> 2) * 16 + t) * 4 + (y & 3)];
        if (e < p.E) logits[t * MAXE + e] = (float)sum;
    }
}

// rows of x
__device__ __forceinline__ few::Rows<1> token_rows(const MoeDecode& p, const void* x, int64_t ldx, int K)
{
    const int lane = threadIdx.x & 63;
    few::Rows<1> r;
    r.x[0] = few::buffer(x);
    r.left = K - 8 * (lane & 15);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int t = 4 * j + (lane >> 4);
        r.a[0][j] = t < p.T ? (uint32_t)(t * ldx + 8 * (lane & 15)) * 2 : few::RANGE;
    }
    return r;
}

// Logits, softmax and choices where x is not kept
template <class Num> __device__ __forceinline__ void route(const MoeDecode& p, Chosen& c, float* red, float* logits, uint8_t* scratch)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunks = (p.d + few::CHUNK - 1) / few::CHUNK;
    typedef few::Cols16<Num, 1> W;
    const few::Rows<1> rows = token_rows(p, p.x, p.ldx, p.d);
    W w;
    w.w[0] = w.w[1] = few::buffer(p.wg);
    w.left = p.d - 8 * few::quad_piece(lane);
    for (int eb = 0; eb * 16 < p.E; ++eb) {
        const int x = eb * 16 + (lane >> 2), e = x < p.E ? x : p.E - 1;
        w.c[0] = (uint32_t)(e * p.ldwg + 8 * few::quad_piece(lane)) * 2;
        few::Wide acc[1][1] = {};
        few::stream<W, 1, false, 4, 4>(acc, w, rows, wave, (chunks - wave + WAVES - 1) / WAVES, WAVES, scratch);
        *(f32x4_t*)(red + (wave * 64 + lane) * 4) = rounded(acc[0][0]);
        __syncthreads();
        sum_logits(p, red, 256, logits, eb, 1, WAVES);
        __syncthreads();
    }
    choose(p, c, logits);
}

// ... and where it is, in the order of W's pieces: the waves of a group of `split` share a block's inputs, groups take different blocks, and the router's rows of the next block are on
// their way while one is summed.  (Loaded as rows of x are: 16 experts x 256 bytes.)
// xs: this wave's chunks of x, loaded on entry and in the operand's order on return.
template <class W> __device__ __forceinline__ void route_kept(const MoeDecode& p, Chosen& c, float* red, int stride, float* logits, few::Rows<1>::Stage (&xs)[4], uint8_t* scratch)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    const int group = wave / p.split, groups = WAVES / p.split, c0 = (wave & (p.split - 1)) * 4, nblocks = (p.E + 15) / 16;
    few::Rows<1>::Stage f[2][4];
    auto fetch = [&](int to, int eb) {
        few::Rows<1> r;
        r.x[0] = few::buffer(p.wg);
        r.left = p.d - 8 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = eb * 16 + 4 * j + q;
            r.a[0][j] = e < p.E ? (uint32_t)(e * p.ldwg + 8 * i) * 2 : few::RANGE;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) r.load(f[to][d], c0 + d);
    };
    auto block = [&](int from, int eb0) {   // blocks eb0 .. eb0 + groups - 1
        few::Wide acc = {};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            few::Rows<1>().template ready<W>(f[from][d], scratch);
#pragma unroll
            for (int j = 0; j < 4; ++j) few::add_products<typename W::Num>(acc, __builtin_bit_cast(bf16x8_t, f[from][d].f[0][j]), __builtin_bit_cast(bf16x8_t, xs[d].f[0][j]));
        }
        *(f32x4_t*)(red + wave * stride + lane * 4) = rounded(acc);
        __syncthreads();
        sum_logits(p, red, stride, logits, eb0, groups, p.split);
        __syncthreads();
    };
    fetch(0, group);
    if (groups < nblocks) fetch(1, groups + group);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < 4; ++d) few::Rows<1>().template ready<W>(xs[d], scratch);
    for (int eb0 = 0; eb0 < nblocks; eb0 += 2 * groups) {
        block(0, eb0);
        if (eb0 + 2 * groups < nblocks) fetch(0, eb0 + 2 * groups + group);
        if (eb0 + groups < nblocks) block(1, eb0 + groups);
        if (eb0 + 3 * groups < nblocks) fetch(1, eb0 + 3 * groups + group);
    }
    choose(p, c, logits);
}

// One job's columns [n, n + 16) of both projections of expert e.
template <class W> __device__ __forceinline__ void gate_up_columns(const MoeDecode& p, W& w, int e, int n)
{
    const int lane = threadIdx.x & 63;
    if constexpr (!std::is_same<W, few::Cols16<typename W::Num, 2>>::value) {
        w.columns(0, p.f1, e, p.d, [&](int, int c) { return (int64_t)n + c; });
        w.columns(1, p.f3, e, p.d, [&](int, int c) { return (int64_t)n + c; });
    } else {
        w.left = p.d - 8 * few::quad_piece(lane);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            w.w[m] = few::buffer((const uint16_t*)(m ? p.w3 : p.w1) + (int64_t)e * p.f * p.d);
            w.c[m] = (uint32_t)((int64_t)(n + (lane >> 2)) * p.d + 8 * few::quad_piece(lane)) * 2;
        }
    }
}

// silu(gate) * up of four columns of a token, as two numbers of the type
template <class Num> __device__ __forceinline__ void store_h(const MoeDecode& p, int row, int n, f32x4_t g, f32x4_t u)
{
    float hi[4], lo[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float h = g[v] / (1.f + __expf(-g[v])) * u[v];
        hi[v] = Num::to_f32(Num::from_f32(h));
        lo[v] = fabsf(hi[v]) < __builtin_inff() ? h - hi[v] : 0.f;
    }
    uint16_t* h = p.h + ((int64_t)row * p.f + n);
    *(uint2*)h = make_uint2(Num::pack2(hi[0], hi[1]), Num::pack2(hi[2], hi[3]));
    *(uint2*)(h + p.h_lo) = make_uint2(Num::pack2(lo[0], lo[1]), Num::pack2(lo[2], lo[3]));
}

// A job's sums [wave][gate, up][64][4] of `split` waves, in wave order; h of the tokens that chose its expert.
template <class Num, class P> __device__ __forceinline__ void finish_job(const MoeDecode& p, const Chosen& c, const P& place, int job, const float* sums, int split)
{
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    if (i >= p.T) return;
    int e, n;
    place(job, &e, &n);
    const int j = choice_of(c, i, e, p.k);
    if (j < 0) return;
    f32x4_t g = (f32x4_t){0.f, 0.f, 0.f, 0.f}, u = g;
    for (int v = 0; v < split; ++v) { g += *(const f32x4_t*)(sums + (v * 128 + lane) * 4); u += *(const f32x4_t*)(sums + (v * 128 + 64 + lane) * 4); }
    store_h<Num>(p, i * p.k + j, n + 4 * q, g, u);
}

// what launch 1 leaves for the caller and for launch 2; all threads of the first workgroup
__device__ __forceinline__ void store_choices(const MoeDecode& p, const Chosen& c)
{
    if (blockIdx.x != 0) return;
    for (int x = threadIdx.x; x < p.T * p.k; x += THREADS) {
        p.indices[x] = c.idx[x / p.k][x % p.k];
        p.weights[x] = c.weight[x / p.k][x % p.k];
    }
    for (int x = threadIdx.x; x < p.counters_n; x += THREADS) p.counters[x] = 0;
}

// Launch 1, hidden sizes up to 4096 (KEPT): p.split waves share a job's contraction, four chunks each, so that every job meets a wave with the same chunks of x: they stay in registers,
// with 8 / p.split jobs at a time.  The ring holds exactly one job (256 KiB of a compute unit): while a chunk of a job is multiplied, that of the next one is on its way into its place.
// Otherwise all eight waves share a job, through few::stream.
// a wave's scratch: its rows of x and its weights, or the router's
template <class W, bool KEPT> constexpr int gate_up_scratch()
{
    constexpr int router = few::Cols16<typename W::Num, 1>::SCRATCH;
    return few::Rows<1>::SCRATCH + (KEPT ? 0 : W::SCRATCH > router ? W::SCRATCH : router);
}

template <class Num, int BITS, bool KEPT, bool QUADS>
__global__ void __launch_bounds__(THREADS, 2) gate_up_kernel(const MoeDecode p)
{
    constexpr bool FP4 = BITS == 4;
    typedef typename std::conditional<FP4, typename std::conditional<QUADS, few::Fp4Quads<Num, 2, true>, few::Fp4Cols<Num, 2, true>>::type, few::Cols16<Num, 2>>::type W;
    static_assert(!KEPT || !FP4, "4-bit weights: gate_up_fp4_kernel");
    constexpr int SCRATCH = gate_up_scratch<W, KEPT>();
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];   // every wave's scratch
    __shared__ Chosen c;
    __shared__ __attribute__((aligned(16))) float red[2][WAVES][2][64][4];   // sums of two jobs; before them the router's
    __shared__ __attribute__((aligned(16))) float logits[TOK * MAXE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    if (threadIdx.x < MAXE / 32) c.used[threadIdx.x] = 0;   // (the router's barriers lie in between)
    uint8_t* scratch = smem + wave * SCRATCH;
    const few::Rows<1> rows = token_rows(p, p.x, p.ldx, p.d);
    few::Rows<1>::Stage xs[4];
    const int member = KEPT ? wave & (p.split - 1) : 0, c0 = member * 4;
    if constexpr (KEPT) {
#pragma unroll
        for (int d = 0; d < 4; ++d) rows.load(xs[d], c0 + d);
        route_kept<W>(p, c, &red[0][0][0][0][0], 256, logits, xs, scratch);
    } else route<Num>(p, c, &red[0][0][0][0][0], logits, scratch);
    store_choices(p, c);
    const int ncb = p.f / 16, jobs = list_active(c) * ncb;
    auto place = [&](int job, int* e, int* n) {
        *e = __builtin_amdgcn_readfirstlane(c.active[job / ncb]);
        *n = __builtin_amdgcn_readfirstlane(job % ncb) * 16;
    };
    if constexpr (KEPT) {
        const int split = p.split, at_once = WAVES / split;
        const int step = gridDim.x * at_once, first = blockIdx.x * at_once + wave / split;
        const int rounds = (jobs - (int)blockIdx.x * at_once + step - 1) / step;   // of this workgroup, the same for all of its waves
        W w;
        typename W::Stage ring[4];
        auto turn_to = [&](int job) {   // where a job's weights lie; there may be none
            int e = 0, n = 0;
            if (job < jobs) place(job, &e, &n);
            gate_up_columns(p, w, e, n);
            if (job >= jobs) w.left = 0;
        };
        turn_to(rounds > 0 ? first : jobs);
#pragma unroll
        for (int d = 0; d < 4; ++d) w.load(ring[d], c0 + d);
        for (int r = 0; r < rounds; ++r) {
            const int job = first + r * step;
            turn_to(r + 1 < rounds ? job + step : jobs);
            f32x4_t acc[2] = {(f32x4_t){0.f, 0.f, 0.f, 0.f}, (f32x4_t){0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                w.ready(ring[d], scratch);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m) acc[m] = Num::mfma(W::frag(ring[d], 0, m, j), __builtin_bit_cast(bf16x8_t, xs[d].f[0][j]), acc[m]);
                __builtin_amdgcn_sched_barrier(0);   // (as in few::stream)
                w.load(ring[d], c0 + d);
                __builtin_amdgcn_sched_barrier(0);
            }
            float (*s)[2][64][4] = red[r & 1];   // (the other one may still be read)
            *(f32x4_t*)s[wave][0][lane] = acc[0];
            *(f32x4_t*)s[wave][1][lane] = acc[1];
            __syncthreads();
            if (member == (r & (split - 1)) && job < jobs) finish_job<Num>(p, c, place, job, &s[wave - member][0][0][0], split);
        }
    } else {
        constexpr int UNIT = W::UNIT * few::CHUNK;
        const int units = (p.d + UNIT - 1) / UNIT;
        int turn = 0;
        for (int job = blockIdx.x; job < jobs; job += gridDim.x, ++turn) {
            int e, n;
            place(job, &e, &n);
            W w;
            gate_up_columns(p, w, e, n);
            f32x4_t acc[1][2] = {{(f32x4_t){0.f, 0.f, 0.f, 0.f}, (f32x4_t){0.f, 0.f, 0.f, 0.f}}};
            few::stream<W, 1, false, 2, 2>(acc, w, rows, wave, (units - wave + WAVES - 1) / WAVES, WAVES, scratch);
            float (*s)[2][64][4] = red[turn & 1];
            *(f32x4_t*)s[wave][0][lane] = acc[0][0];
            *(f32x4_t*)s[wave][1][lane] = acc[0][1];
            __syncthreads();
            if (wave == (turn & (WAVES - 1))) finish_job<Num>(p, c, place, job, &s[0][0][0][0], WAVES);
        }
    }
}

// Launch 1 over 4-bit weights, hidden sizes up to 4096 that are multiples of 512: as KEPT above, but codes go straight into LDS, a ring of four units (256 inputs of 16 columns of both
// projections, 4 KiB) per wave, two jobs: a job is only 64 KiB of a compute unit, and with one of them in registers the loop waited for memory (4 us a job).  Requests are counted by
// hand: a job is the scales of gate and up and two units of four loads; scales and a unit are awaited with what was requested behind them still on its way.
constexpr int FP4_UNIT_LDS = 4096, FP4_SCALES_LDS = 512, FP4_WAVE_LDS = 4 * FP4_UNIT_LDS + 2 * FP4_SCALES_LDS, FP4_LDS = WAVES * FP4_WAVE_LDS + WAVES * 2 * 1024;

template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <class Num>
__global__ void __launch_bounds__(THREADS, 2) gate_up_fp4_kernel(const MoeDecode p)
{
    typedef few::Fp4Quads<Num, 2, true> W;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];   // every wave's ring and scales, and the sums of a job [wave][gate, up][64][4]
    __shared__ Chosen c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    float* red = (float*)(smem + WAVES * FP4_WAVE_LDS);
    uint8_t* area = smem + wave * FP4_WAVE_LDS;
    if (threadIdx.x < MAXE / 32) c.used[threadIdx.x] = 0;   // (the router's barriers lie in between)
    const int split = p.split, member = wave & (split - 1), c0 = member * 4;
    const few::Rows<1> rows = token_rows(p, p.x, p.ldx, p.d);
    few::Rows<1>::Stage xs[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) rows.load(xs[d], c0 + d);
    // (the router's sums lie behind every wave's scratch, its logits where a job's sums will be)
    static_assert(TOK * MAXE * 4 <= WAVES * 2 * 1024 && few::Rows<1>::SCRATCH + 1024 <= FP4_WAVE_LDS, "");
    route_kept<W>(p, c, (float*)(smem + few::Rows<1>::SCRATCH), FP4_WAVE_LDS / 4, red, xs, area);
    store_choices(p, c);
    const int ncb = p.f / 16, jobs = list_active(c) * ncb;
    auto place = [&](int job, int* e, int* n) {
        *e = __builtin_amdgcn_readfirstlane(c.active[job / ncb]);
        *n = __builtin_amdgcn_readfirstlane(job % ncb) * 16;
    };
    const int at_once = WAVES / split, step = gridDim.x * at_once, first = blockIdx.x * at_once + wave / split;
    const int rounds = (jobs - (int)blockIdx.x * at_once + step - 1) / step;   // of this workgroup, the same for all of its waves
    // where a job's weights lie (there may be none: requests outside the buffer's range)
    i32x4_t codes[2], scales[2];
    uint32_t col[2], scale_at = few::RANGE;   // of the two halves of a block's columns, from the job's first one
    const uint32_t area_u = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(area));
    auto turn_to = [&](int job) {
        const bool some = job < jobs && c0 * few::CHUNK < p.d;
        int e = 0, n = 0;
        if (job < jobs) place(job, &e, &n);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const MoeFp4Weights& f = m ? p.f3 : p.f1;
            codes[m] = make_buffer(f.codes + e * f.sce + n * f.scn, few::RANGE);
            scales[m] = make_buffer(f.scales + e * f.sse + n * f.ssn, few::RANGE);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) col[h] = some ? (uint32_t)((8 * h + (lane >> 3)) * p.f1.scn) + few::line_piece(lane, h) * 16 : few::RANGE;   // (w1 and w3 have the same pitch)
        scale_at = some ? (uint32_t)(lane * p.f1.ssn) : few::RANGE;
    };
    auto fetch_scales = [&](int slot) {
        if (lane < 16)
#pragma unroll
            for (int m = 0; m < 2; ++m) load_to_lds_16(scales[m], scale_at, c0 * 4, area_u + 4 * FP4_UNIT_LDS + slot * FP4_SCALES_LDS + m * 256);
    };
    auto fetch = [&](int slot, int u) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) load_to_lds_16<true>(codes[m], col[h], (c0 / 2 + u) * 128, area_u + (slot * 2 + u) * FP4_UNIT_LDS + m * 2048 + h * 1024);
    };
    constexpr int UNIT_LOADS = 4, JOB_LOADS = 2 + 2 * UNIT_LOADS;
#pragma unroll 1
    for (int r = 0; r < 2; ++r) {
        turn_to(r < rounds ? first + r * step : jobs);
        fetch_scales(r);
        fetch(r, 0);
        fetch(r, 1);
    }
#pragma unroll 1
    for (int r = 0; r < rounds; ++r) {
        const int job = first + r * step, slot = r & 1;
        turn_to(r + 2 < rounds ? job + 2 * step : jobs);
        f32x4_t acc[2] = {(f32x4_t){0.f, 0.f, 0.f, 0.f}, (f32x4_t){0.f, 0.f, 0.f, 0.f}};
        fp4_u32x4_t now[2];   // scales of column i: byte q of word d
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (u == 0) {
                wait_loads<UNIT_LOADS + JOB_LOADS>();
#pragma unroll
                for (int m = 0; m < 2; ++m) now[m] = *(const fp4_u32x4_t*)(area + 4 * FP4_UNIT_LDS + slot * FP4_SCALES_LDS + m * 256 + i * 16);
            } else wait_loads<JOB_LOADS + 2 + UNIT_LOADS>();
            fp4_u32x4_t f[2][2];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) f[m][cc] = *(const fp4_u32x4_t*)(area + (slot * 2 + u) * FP4_UNIT_LDS + m * 2048 + i * 128 + ((cc * 4 + q) ^ ((i >> 1) & 7)) * 16);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        acc[m] = Num::mfma(fp4_expand8<Num>(f[m][cc][j], fp4_scale(now[m][2 * u + cc] >> (8 * q) & 0xff)), __builtin_bit_cast(bf16x8_t, xs[2 * u + cc].f[0][j]), acc[m]);
            // every read of this unit's place has come back: the job after the next goes there
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            if (u == 0) fetch_scales(slot);
            fetch(slot, u);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();   // the sums of the job before have been read
        *(f32x4_t*)(red + (wave * 128 + lane) * 4) = acc[0];
        *(f32x4_t*)(red + (wave * 128 + 64 + lane) * 4) = acc[1];
        __syncthreads();
        if (member == (r & (split - 1)) && job < jobs) finish_job<Num>(p, c, place, job, red + (wave - member) * 512, split);
    }
    wait_loads<0>();   // (nothing lands in LDS that is no longer this workgroup's)
}

// ---- launch 2
// 4-bit W2 (E, d, f): 64 output columns, NB = 4 blocks whose columns are dealt so that a lane holds 4 NB consecutive ones.  16-bit W2 (E, f, d), contiguous along the output:
// 128 columns; a lane loads 8 of them (16 bytes) in 8 rows and transposes the 8 x 8 block in registers, one instruction for two values; the weight is the second operand, so a lane
// ends up with 8 consecutive columns of four tokens.
constexpr int DOWN_PARTS_MAX = 64;

// HALVES (up to 8 tokens): rows 8 on of the operand are what the rounding of h lost, so that one product takes both numbers; otherwise two products.
template <class Num, int BITS, bool QUADS, bool HALVES>
__global__ void __launch_bounds__(THREADS) down_kernel(const MoeDecode p)
{
    constexpr bool FP4 = BITS == 4;
    typedef typename std::conditional<QUADS, few::Fp4Quads<Num, 4, false>, few::Fp4Cols<Num, 4, false>>::type W;
    constexpr int NA = HALVES ? 1 : 2, SCRATCH = W::SCRATCH + few::Rows<NA>::SCRATCH;   // of a wave, with 4-bit weights
    constexpr int UNITS = 4, PER = FP4 ? 4 : 8;   // floats of a lane and unit: unit nb holds 4 columns of one token, unit r 8 columns of one
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ Chosen c;
    __shared__ int arrival;
    float* red = (float*)smem;   // [wave][unit][64][PER]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, q = lane >> 4;
    // (tiles side by side, so that an XCD has every row of a few tiles: with a few rows of every tile each, columns 256 bytes apart in rows of 8 KiB came out of its L2 at two speeds, 34 and 49 us of
    // one token's 53 of 4096 x 14336 in 16 bits; now 34 to 41)
    const int tiles = gridDim.x / p.parts, part = blockIdx.x / tiles, tile = blockIdx.x - part * tiles;
    static_assert(THREADS >= TOK * MAXK, "a thread per choice");
    const int x = threadIdx.x;
    const int choice = x < p.T * p.k ? p.indices[x] : 0;
    if (x < MAXE / 32) c.used[x] = 0;
    __syncthreads();
    if (x < p.T * p.k) {
        c.idx[x / p.k][x % p.k] = choice;
        c.weight[x / p.k][x % p.k] = p.weights[x];
        atomicOr(&c.used[choice >> 5], 1u << (choice & 31));
    }
    __syncthreads();
    const int nactive = list_active(c);
    // this wave's share of the contraction: steps of the chosen experts one after the other
    constexpr int STEP = FP4 ? W::UNIT * few::CHUNK : 32;
    const int steps = (p.f + STEP - 1) / STEP;
    const int64_t total = (int64_t)nactive * steps;
    // (the waves of a part take every eighth step, side by side in memory; where an expert has few, ranges of their own)
    const bool side_by_side = FP4 && steps >= 2 * WAVES;
    const int shares = side_by_side ? p.parts : p.parts * WAVES, share = side_by_side ? part : part * WAVES + wave;
    int64_t at = total * share / shares;
    const int64_t end = total * (share + 1) / shares;
    // the token that row r of the operand belongs to, and where its numbers lie
    auto token = [&](int r) { return HALVES ? r & 7 : r; };
    auto row_of = [&](int r, int j) { return (uint32_t)((token(r) * p.k + j) * p.f + (HALVES && r >= 8 ? (int)p.h_lo : 0)) * 2; };
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
        const int j = token(i) < p.T ? choice_of(c, token(i), e, p.k) : -1;
        if constexpr (FP4) {
            W w;
            w.columns(0, p.f2, e, p.f, [&](int nb, int c) { return (int64_t)tile * 64 + (c >> 2) * 16 + 4 * nb + (c & 3); });   // (d is a multiple of 64)
            few::Rows<NA> rows;
#pragma unroll
            for (int m = 0; m < NA; ++m) rows.x[m] = few::buffer(p.h + m * p.h_lo);
            rows.left = p.f - 8 * i;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int r = 4 * y + q, jt = token(r) < p.T ? choice_of(c, token(r), e, p.k) : -1;
#pragma unroll
                for (int m = 0; m < NA; ++m) rows.a[m][y] = jt >= 0 ? row_of(r, jt) + 16 * i : few::RANGE;
            }
            f32x4_t acc[1][4];
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[0][nb] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            const int step = side_by_side ? WAVES : 1, first = side_by_side ? s0 + wave : s0;
            few::stream<W, NA, true, HALVES ? 3 : 2, HALVES && W::UNIT == 1 ? 3 : 2>(acc, w, rows, first, (s1 - first + step - 1) / step, step, smem + wave * SCRATCH);
            const float g = j >= 0 ? c.weight[token(i)][j] : 0.f;
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int v = 0; v < PER; ++v) out[u][v] = j >= 0 ? out[u][v] + g * acc[0][u][v] : out[u][v];   // (what other tokens' rows hold may not be finite)
        } else {
            const few::Buffer w = few::buffer((const uint16_t*)p.w2 + (int64_t)e * p.f * p.d);
            const int n = tile * 128 + 8 * i;
            const uint32_t col = n < p.d ? (uint32_t)(n + 8 * q * p.d) * 2 : few::RANGE;
            const uint32_t row = j >= 0 ? row_of(i, j) + 16 * q : few::RANGE;
            const few::Buffer hb[2] = {few::buffer(p.h), few::buffer(p.h + p.h_lo)};
            f32x4_t acc[8];
#pragma unroll
            for (int b = 0; b < 8; ++b) acc[b] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            constexpr int DEPTH = HALVES ? 3 : 2;
            fp4_u32x4_t ws[DEPTH][8];
            bf16x8_t as[DEPTH][NA];
            auto fetch = [&](int dst, int s) {
#pragma unroll
                for (int r = 0; r < 8; ++r) ws[dst][r] = few::load16_streamed(w, col, (uint32_t)(s * 32 + r) * (uint32_t)p.d * 2);
#pragma unroll
                for (int m = 0; m < NA; ++m) as[dst][m] = __builtin_bit_cast(bf16x8_t, few::load16(hb[m], row, (uint32_t)s * 64));
                __builtin_amdgcn_sched_barrier(0);
            };
            auto multiply = [&](int src) {
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    fp4_u32x4_t f;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        f[r] = __builtin_amdgcn_perm(ws[src][2 * r + 1][b / 2], ws[src][2 * r][b / 2], b & 1 ? 0x07060302u : 0x05040100u);
                    const bf16x8_t wf = __builtin_bit_cast(bf16x8_t, f);
#pragma unroll
                    for (int m = 0; m < NA; ++m) acc[b] = Num::mfma(as[src][m], wf, acc[b]);
                }
                __builtin_amdgcn_sched_barrier(0);   // (as in few::stream)
            };
#pragma unroll
            for (int x = 0; x < DEPTH; ++x)
                if (s0 + x < s1) fetch(x, s0 + x);
            int s = s0;
            for (; s + 2 * DEPTH <= s1; s += DEPTH)
#pragma unroll
                for (int x = 0; x < DEPTH; ++x) { multiply(x); fetch(x, s + DEPTH + x); }
            for (; s < s1; s += DEPTH)
#pragma unroll
                for (int x = 0; x < DEPTH; ++x) {
                    if (s + x >= s1) break;
                    multiply(x);
                    if (s + x + DEPTH < s1) fetch(x, s + x + DEPTH);
                }
            // acc[b][r] is column 8 i + b of row 4 q + r
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = token(4 * q + r), jr = t < p.T ? choice_of(c, t, e, p.k) : -1;
                const float g = jr >= 0 ? c.weight[t][jr] : 0.f;
#pragma unroll
                for (int b = 0; b < 8; ++b) out[r][b] = jr >= 0 ? out[r][b] + g * acc[b][r] : out[r][b];
            }
        }
    }
    if constexpr (HALVES)   // both numbers' products
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int v = 0; v < PER; ++v) out[u][v] += __shfl_xor(out[u][v], FP4 ? 8 : 32);
    // ---- the waves' sums, in wave order
    __syncthreads();   // (they take the place of the operands)
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
            // (eight parts' sums are requested together: one after the other they cost a trip to memory each, 3 us with four parts)
            constexpr int BATCH = 8;
            for (int x0 = 0; x0 < p.parts; x0 += BATCH) {
                f32x4_t s[BATCH][PER / 4];
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
#pragma unroll
                    for (int v = 0; v < PER / 4; ++v)
                        s[b][v] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(slots, x0 + b < p.parts ? slot(x0 + b) + 16 * v : few::RANGE, 0, DEVICE_SCOPE));
#pragma unroll
                for (int b = 0; b < BATCH; ++b)
#pragma unroll
                    for (int v = 0; v < PER; ++v) sum[v] += s[b][v / 4][v % 4];
            }
        }
    }
    if (!live) return;
    uint16_t* o = (uint16_t*)p.out + t * p.ldo + n;
#pragma unroll
    for (int v = 0; v < PER; v += 4) *(uint2*)(o + v) = make_uint2(Num::pack2(sum[v], sum[v + 1]), Num::pack2(sum[v + 2], sum[v + 3]));
}

inline int64_t chunks_of(int64_t n) { return (n + few::CHUNK - 1) / few::CHUNK; }

struct Plan { int grid1, split, tiles, parts; size_t h_bytes, counter_bytes, slot_bytes; };
Plan plan(int T, int E, int d, int f, int k, bool fp4)
{
    Plan r = {};
    const int cus = moe_device_cus();
    const int64_t jobs = (int64_t)(E < T * k ? E : T * k) * (f / 16);
    // split: 0 where a wave cannot keep its part of x (gate_up_kernel)
    const int chunks = (d + few::CHUNK - 1) / few::CHUNK;
    r.split = 0;
    // (nor where there is at most one job per compute unit: nothing to keep x for, and a ring of whole jobs costs more than it hides: d = 256, f = 512, 3 tokens 13.3 us)
    if (jobs > cus && chunks <= 4 * WAVES && (!fp4 || d % (4 * few::CHUNK) == 0))
        for (r.split = 1; r.split * 4 < chunks;) r.split *= 2;
    const int64_t at_once = r.split ? WAVES / r.split : 1, groups = (jobs + at_once - 1) / at_once;
    r.grid1 = (int)(groups < cus ? groups : cus);
    r.tiles = fp4 ? d / 64 : (d + 127) / 128;
    // parts of launch 2, one workgroup per compute unit at a time: as few as come near the least time in rounds, as long as their waves have two steps each
    const int64_t steps = (int64_t)(E < T * k ? E : T * k) * (fp4 ? chunks_of(f) : f / 32);
    auto time = [&](int parts) { return (double)((r.tiles * (int64_t)parts + cus - 1) / cus) / parts; };
    r.parts = 1;
    for (int parts = 2; parts <= DOWN_PARTS_MAX && steps >= (int64_t)parts * 2 * WAVES; ++parts)
        if (time(parts) < 0.9 * time(r.parts)) r.parts = parts;
    auto al = [](size_t n) { return (n + 255) & ~(size_t)255; };
    r.h_bytes = al((size_t)T * k * f * 2);
    r.counter_bytes = al((size_t)r.tiles * 4);
    r.slot_bytes = r.parts > 1 ? al((size_t)r.tiles * r.parts * 4 * 64 * (fp4 ? 4 : 8) * 4) : 0;
    return r;
}

template <class Num, int BITS> int launch_typed(const MoeDecode& p, const Plan& pl, hipStream_t stream)
{
    constexpr bool FP4 = BITS == 4;
    auto go = [&](auto kern, int grid, size_t lds, std::atomic<bool>* attr_set) {
        const int dev = moe_current_device();
        if (!attr_set[dev]) {
            if (hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return MOE_ERR_LAUNCH;
            attr_set[dev] = true;
        }
        hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(THREADS), lds, stream, p);
        return moe_launch_status();
    };
    static std::atomic<bool> set1[3][MOE_MAX_DEVICES], set2[4][MOE_MAX_DEVICES];
    typedef few::Fp4Quads<Num, 2, true> Q2;
    typedef few::Fp4Quads<Num, 4, false> Q4;
    constexpr size_t rows2 = few::Rows<2>::SCRATCH, sums = (size_t)4 * 64 * (FP4 ? 4 : 8) * 4;
    int rc;
    if constexpr (FP4) {
        if (p.split) rc = go(gate_up_fp4_kernel<Num>, pl.grid1, FP4_LDS, set1[0]);
        else if (p.d % (2 * few::CHUNK)) rc = go(gate_up_kernel<Num, 4, false, false>, pl.grid1, WAVES * gate_up_scratch<few::Fp4Cols<Num, 2, true>, false>(), set1[1]);
        else rc = go(gate_up_kernel<Num, 4, false, true>, pl.grid1, WAVES * gate_up_scratch<Q2, false>(), set1[2]);
    } else {
        if (p.split) rc = go(gate_up_kernel<Num, 16, true, true>, pl.grid1, WAVES * gate_up_scratch<few::Cols16<Num, 2>, true>(), set1[0]);
        else rc = go(gate_up_kernel<Num, 16, false, true>, pl.grid1, WAVES * gate_up_scratch<few::Cols16<Num, 2>, false>(), set1[1]);
    }
    if (rc != MOE_OK) return rc;
    constexpr size_t operands = FP4 ? Q4::SCRATCH + rows2 : 0;
    const bool halves = p.T <= 8, odd = FP4 && p.f % (2 * few::CHUNK);
    const size_t lds = WAVES * (odd ? (rows2 > sums ? rows2 : sums) : operands > sums ? operands : sums);
    if constexpr (FP4)
        if (odd) return halves ? go(down_kernel<Num, BITS, false, true>, pl.tiles * pl.parts, lds, set2[0]) : go(down_kernel<Num, BITS, false, false>, pl.tiles * pl.parts, lds, set2[1]);
    return halves ? go(down_kernel<Num, BITS, true, true>, pl.tiles * pl.parts, lds, set2[2]) : go(down_kernel<Num, BITS, true, false>, pl.tiles * pl.parts, lds, set2[3]);
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
    p.split = pl.split;
    if (f16) return fp4 ? launch_typed<NumF16, 4>(p, pl, stream) : launch_typed<NumF16, 16>(p, pl, stream);
    return fp4 ? launch_typed<NumBf16, 4>(p, pl, stream) : launch_typed<NumBf16, 16>(p, pl, stream);
}

// f4_moe.cuh — a whole mixture-of-experts layer for few tokens, in two kernels: 16-bit activations x 4-bit weights.
//
//   logits[t][e] = x[t] . router[e];  the `top` largest of a token, their softmax p (or their share of the softmax over all)
//   y[t] = sum over the chosen experts of p * W2_e ( silu(G_e x[t]) * (U_e x[t]) )
//
// What bounds it: every chosen expert's weights are read once, 9/16 (17/32) of a byte a weight; the products are few.
//
// The products run on tcgen05.mma.kind::mxf4nvf4, which takes the weights as they are stored; nothing is done per weight outside
// the tensor core.  (Converting them to fp16 in registers for mma.sync took 2.2 instructions a weight and reached
// 1.9 TB/s; the conversion instruction alone runs at 16 weights a clock and SM, a third of what HBM delivers.)  It wants
// the activations in 4 bits too, so each is written with eight digits of base 8 under its block's scale,
//     x = s * sum over i < 8 of 8^-i * d_i / 2,   d_i from -4 to 3: all of them E2M1 numbers when halved.
// s is a power of two, so multiples of 2^-22 s (fp16 numbers down to 2^-10 of their block's largest, bf16 down to 2^-13) are exact,
// others off by at most 2^-23 s < 2^-22.7 of the block's largest.  (Six digits, 2^-16.7, were not
// enough beside a channel a thousand times larger: 2^-7 of the others.)  The eight digits are eight columns of the MMA, the
// least it takes, and cost nothing: an MMA takes as long with 8 columns as with 100.  All have the block's scale; the powers of 8
// are applied to the columns' fp32 sums when they are added.
//
// Kernel 1, moe_router_kernel: clusters of 8 CTAs per group of at most 8 tokens.  One set of clusters makes the logits: the warps share the
// experts and 16 pieces of K (mma.sync, 16 experts x 8 tokens), the pieces meet in the shared memory of one CTA per token, whose first
// warp selects.  Another set of clusters cuts the same tokens into their digits meanwhile, a CTA per token.
// Logits are products and sums in 64 bits (mma.sync on fp64), in an order that is the same for every token of every batch.  With sums
// of 16 products in fp32 the kernel was 1.6 us shorter, but logits that large channels cancel in were ordered wrongly, equal ones
// told apart, and products of bf16 beyond 2^128 made infinities of finite logits.
//
// Kernel 2, moe_experts_kernel: one CTA per SM, all resident (cooperative launch).  The unit of work is 128 weight rows (gate / up: 64
// channels of each) times the tokens of one expert; where units are few they are cut along K, and the parts' sums are
// added by whoever reads them.  Units are dealt out in contiguous ranges, expert by expert, so a CTA keeps its expert's
// activations in shared memory.  Weights and scales come through a ring of TMA stages; the scales, stored in rows, are put into
// tensor memory by four warps (tcgen05.st) on the way.  The ring runs ahead into the next expert and, over the wait
// for the other CTAs' gate / up sums, into the down projection's weights.
//   The gate / up sums go to the workspace in fp32; whoever needs an expert's hidden activations waits for its sums, applies
// SiLU and cuts them into digits.  The experts' outputs go to the workspace in fp32 and are added per token after a last wait, every fourth
// choice by one lane and the four sums in a fixed tree: no atomics on sums, the same bits on every call.
//   Measured (device, both kernels): 64 tokens on 64 experts of 4096 x 1408, top 6, E8M0, 589 MB: 133 us, 4.4 TB/s; 16 tokens on 128 experts
// of 2048 x 768, top 8, E4M3, 221 MB: 62.6 us, 3.5 TB/s; 1 token, 59 MB: 34.2 us.  About 17 us of each is not streaming: the router kernel and
// the hand-over 8, the wait between the phases for the last sums and the first activations 4, the last wait and the sum over the
// experts 5.  Beyond that it is the chain of a stage (TMA, scales to tensor memory, MMA, release) more than the bytes: with the
// loads taken out 64 tokens take 98 us, 16 tokens 51 and 1 token 29.
#pragma once
#include "f4_format.cuh"
#include "f4_gemm.cuh"
#include "sm100_ptx.cuh"

namespace bm {

constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxExperts = 256;
constexpr int kMoeMaxTop = 16;
constexpr int kMoeMaxDim = 16384;
constexpr int kMoeParts = 8;                                    // digits of an activation
constexpr int kMoeMaxSplit = 4;                                 // pieces of K of a unit at most
constexpr int kMoeMaxRuns = 80;

// Activations cut up: per token and 256 of K 1 KiB, 8 rows (the digits) of 128 bytes in the 128-byte swizzle of an MMA operand, and the
// scales, a byte per block (the digits share it), rows of whole 16 bytes.
__host__ __device__ constexpr int moe_k_blocks(int k) { return (k + kF4BK - 1) / kF4BK; }
__host__ __device__ constexpr int moe_value_bytes(int k) { return moe_k_blocks(k) * 1024; }
__host__ __device__ constexpr int moe_scale_bytes(int k, int fmt) { return (moe_k_blocks(k) * f4_stage_tiles(fmt) * 4 + 15) / 16 * 16; }

struct MoeWorkspace {            // byte offsets
    size_t counters, x_scale, ids, weights, x_values, x_scales, gu, y, bytes;
    int counter_words;           // done[E], arrived
    int gu_pitch, y_pitch;       // elements: gate sums and up sums of an assignment (half each); outputs
    int split;                   // pieces of K that the sums have room for
};

struct MoeParams {
    const uint16_t* x;
    const uint16_t* router;
    long long ldx, ldy;
    uint16_t* y;
    int* ids_out;                // may be NULL
    float* weights_out;          // may be NULL
    const float* r13;            // row factors or NULL
    const float* r2;
    int tokens, hidden, inter, experts, top;
    int normalize;
    int x_vec_ok, router_vec_ok;
    unsigned* counters;
    int counter_words;
    float* x_scale;
    int* ids;
    float* weights;
    uint8_t* x_values;
    uint8_t* x_scales;
    float* gu;
    float* yp;
    int gu_pitch, y_pitch;
    int split;
    int* status;
};

template <bool BF16>
__device__ __forceinline__ uint4 moe_piece(const uint16_t* row, int v, int k, bool vec_ok) {
    const int k0 = v * 8;
    if (vec_ok && k0 + 8 <= k) return __ldg(reinterpret_cast<const uint4*>(row + k0));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k0 + j < k) w[j >> 1] |= static_cast<uint32_t>(__ldg(row + k0 + j)) << (16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// FMT_E4M3: the power of two 2^e that puts a row's largest |v| (fp32 bits) in [2^7, 2^8), where its scale is at most 2^8, as v / 2^e
template <int FMT>
__device__ __forceinline__ void moe_row_factor(uint32_t top_bits, float& factor, float& inv) {
    factor = inv = 1.f;
    if (FMT == FMT_E8M0 || top_bits == 0 || top_bits >= 0x7F800000u) return;
    const int lg = static_cast<int>(top_bits >> 23), e = lg > 8 ? lg - 7 : 1;
    factor = __uint_as_float(static_cast<uint32_t>(e) << 23);
    inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

// Eight activations (piece v of a row, two or four neighbouring lanes share a block) as digits and scales.  `values`, `scales`: the
// token's own places, in shared or global memory.  Whole warps.
//   The scale is the smallest power of two of at least |largest| / 1.7 (eight digits reach 1.714) that the format has: 2^-126
// (E8M0), or 2^-9 under the row's factor (E4M3: 2^-16 of the row's largest or less).  A number times 2^22 / s, rounded to an integer, plus 4 in every
// digit, is 24 bits, three of them a digit + 4.
template <int FMT>
__device__ __forceinline__ void moe_cut(float (&x)[8], int v, uint8_t* values, uint8_t* scales) {
    constexpr int SHARE = f4_block(FMT) / 8;
    float odd = 0.f;                                              // a NaN where one of the block's numbers is none
#pragma unroll
    for (int j = 0; j < 8; ++j) odd = fmaf(x[j], 0.f, odd);
    float top = fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))),
                      fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7]))));
#pragma unroll
    for (int o = 1; o < SHARE; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        odd += __shfl_xor_sync(0xFFFFFFFFu, odd, o);
    }
    // the scale's exponent + 127; 255 for an infinity and for a number above 1.7 * 2^127, which no E8M0 scale holds
    uint32_t e = (__float_as_uint(top * 0.58823530f) + 0x007FFFFFu) >> 23;
    uint32_t byte = e;
    if constexpr (FMT == FMT_E4M3) {
        e = min(max(e, 127u - 9u), 127u + 8u);
        byte = e >= 121u ? (e - 120u) << 3 : 1u << (e - 118u);   // a normal E4M3 number from 2^-6 on
    } else if (e < 22u) {                                         // 2^22 / s would leave fp32's range
        e += 64u;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= 0x1p64f;
    }
    const float inv = __uint_as_float((254u + 22u - e) << 23);   // 2^22 / s
    uint32_t t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = static_cast<uint32_t>(__float2int_rn(x[j] * inv)) + 9586980u;
    const int block = v / SHARE, chunk = (v & 31) >> 2;
    uint8_t* row = values + (v >> 5) * 1024 + (v & 3) * 4;
    if (odd != 0.f) byte = FMT == FMT_E4M3 ? 127u : 255u;
#pragma unroll
    for (int i = 0; i < kMoeParts; ++i) {
        constexpr int kTopDigit = 3 * (kMoeParts - 1);
        uint32_t u = 0;                                           // digits + 4, a nibble each
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int shift = 4 * j - (kTopDigit - 3 * i);
            u |= (shift >= 0 ? t[j] << (shift & 31) : t[j] >> (-shift & 31)) & (7u << (4 * j));
        }
        // 4 + d -> the code of d / 2: d itself, or 8 | -d
        const uint32_t neg = (~u >> 2) & 0x11111111u;
        const uint32_t codes = (((u & 0x33333333u) ^ (neg * 3u)) + neg) | (neg << 3);
        *reinterpret_cast<uint32_t*>(row + i * 128 + ((chunk ^ i) << 4)) = codes;
    }
    if (v % SHARE == 0) scales[block] = static_cast<uint8_t>(byte);
}

// Clusters of 8 CTAs: the first ones choose the experts of up to 8 tokens each, the others cut these tokens up (a CTA per token).
constexpr int kMoeRouterCtas = 8, kMoeRouterThreads = 256, kMoeRouterTokens = 8;
constexpr int kMoeRouterChunks = 16;                             // pieces of K that the logits are added up from

// D = A B + C in 64 bits: A 16 x 16, B 16 x 8.  Lane (g, q) of the warp holds a[2 i], a[2 i + 1]: rows g, g + 8 of column 4 i + q; b[i]: row 4 i + q of
// column g; c: rows g, g, g + 8, g + 8 of columns 2 q, 2 q + 1.
__device__ __forceinline__ void mma_f64_16x8x16(double (&c)[4], const double (&a)[8], const double (&b)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f64.f64.f64.f64 {%0, %1, %2, %3}, {%4, %5, %6, %7, %8, %9, %10, %11}, {%12, %13, %14, %15}, {%0, %1, %2, %3};"
        : "+d"(c[0]), "+d"(c[1]), "+d"(c[2]), "+d"(c[3])
        : "d"(a[0]), "d"(a[1]), "d"(a[2]), "d"(a[3]), "d"(a[4]), "d"(a[5]), "d"(a[6]), "d"(a[7]), "d"(b[0]), "d"(b[1]), "d"(b[2]), "d"(b[3]));
}
template <bool BF16>
__device__ __forceinline__ void pair_to_double(uint32_t w, double& lo, double& hi) {
    const float2 f = pair_to_float<BF16>(w);
    lo = static_cast<double>(f.x);
    hi = static_cast<double>(f.y);
}

// Logits of 16 experts (rows a0 and a1 of lane group g: experts g and g + 8) and 8 tokens over pieces [v0, v1) of 8 of K.  Lane (g, q) holds
// the 8 numbers of piece 4 i + q of its rows and of token g: any order of K serves an MMA if both operands keep it.
// All in 64 bits, where the products are exact: which expert a token gets must not depend on a sum's rounding.
template <bool BF16, bool VEC>
__device__ __forceinline__ void moe_logits(const uint16_t* a0, const uint16_t* a1, const uint16_t* x, int k, int v0, int v1, int q, double (&sum)[4]) {
    constexpr int AHEAD = 4;                                      // MMA pairs (32 of K) whose loads are in flight together
#pragma unroll 1
    for (int v = v0; v < v1; v += 4 * AHEAD) {
        uint4 a[AHEAD], c[AHEAD], b[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int at = v + 4 * i + q;
            a[i] = c[i] = b[i] = make_uint4(0, 0, 0, 0);
            if (at < v1) {
                if constexpr (VEC) {
                    a[i] = __ldg(reinterpret_cast<const uint4*>(a0) + at);
                    c[i] = __ldg(reinterpret_cast<const uint4*>(a1) + at);
                    b[i] = __ldg(reinterpret_cast<const uint4*>(x) + at);
                } else {
                    a[i] = moe_piece<BF16>(a0, at, k, false);
                    c[i] = moe_piece<BF16>(a1, at, k, false);
                    b[i] = moe_piece<BF16>(x, at, k, false);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t wa[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, wc[4] = {c[i].x, c[i].y, c[i].z, c[i].w}, wb[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                double da[8], db[4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pair_to_double<BF16>(wa[half * 2 + j], da[4 * j], da[4 * j + 2]);
                    pair_to_double<BF16>(wc[half * 2 + j], da[4 * j + 1], da[4 * j + 3]);
                    pair_to_double<BF16>(wb[half * 2 + j], db[2 * j], db[2 * j + 1]);
                }
                mma_f64_16x8x16(sum, da, db);
            }
        }
    }
}

// order of doubles as unsigned integers, NaN below every number; 0 is left for "no candidate"
__device__ __forceinline__ unsigned long long logit_key(double v) {
    if (v != v) return 1ull;
    const long long b = __double_as_longlong(v + 0.0);           // -0 counts as +0
    return (b < 0 ? ~static_cast<unsigned long long>(b) : static_cast<unsigned long long>(b) | (1ull << 63)) + 2ull;
}

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kMoeRouterThreads)
moe_router_kernel(const MoeParams p) {
    constexpr int kWarps = kMoeRouterThreads / 32;
    extern __shared__ double parts[];                             // [chunk][expert] of this CTA's token
    __shared__ double logits[kMoeMaxExperts];
    __shared__ uint32_t warp_max[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_ctarank());
    const int groups = (p.tokens + kMoeRouterTokens - 1) / kMoeRouterTokens;
    const int cluster = blockIdx.x / kMoeRouterCtas, group = cluster < groups ? cluster : cluster - groups;
    const int t0 = group * kMoeRouterTokens, n = min(p.tokens - t0, kMoeRouterTokens);
    const int t = t0 + rank;                                      // the token this CTA selects for, or cuts up
    const int pieces = (p.hidden + 7) / 8;
    pdl_launch_dependents();
    pdl_wait_prior_grid();        // the call before may still be using the workspace
    if (cluster >= groups) {
        // ------------------------------------------------------------------ a token's activations cut up
        if (rank >= n) return;
        const uint16_t* row = p.x + t * p.ldx;
        float factor = 1.f, inv = 1.f;
        if (FMT == FMT_E4M3) {
            uint32_t m = 0;
#pragma unroll 2
            for (int v = threadIdx.x; v < pieces; v += kMoeRouterThreads) {
                const uint4 d = moe_piece<BF16>(row, v, p.hidden, p.x_vec_ok);
                const uint32_t b = __vmaxu2(__vmaxu2(d.x & 0x7FFF7FFFu, d.y & 0x7FFF7FFFu), __vmaxu2(d.z & 0x7FFF7FFFu, d.w & 0x7FFF7FFFu));
                m = max(m, max(b & 0xFFFFu, b >> 16));
            }
            m = __reduce_max_sync(0xFFFFFFFFu, m);
            if (lane == 0) warp_max[warp] = m;
            __syncthreads();
            for (int w = 0; w < kWarps; ++w) m = max(m, warp_max[w]);
            const float top = BF16 ? __uint_as_float(m << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
            moe_row_factor<FMT>(__float_as_uint(top), factor, inv);
        }
        if (threadIdx.x == 0) p.x_scale[t] = factor;
        uint8_t* values = p.x_values + static_cast<size_t>(t) * moe_value_bytes(p.hidden);
        uint8_t* scales = p.x_scales + static_cast<size_t>(t) * moe_scale_bytes(p.hidden, FMT);
        for (int v = threadIdx.x; v < moe_k_blocks(p.hidden) * (kF4BK / 8); v += kMoeRouterThreads) {      // whole warps
            const uint4 d = moe_piece<BF16>(row, v, p.hidden, p.x_vec_ok);
            const uint32_t w[4] = {d.x, d.y, d.z, d.w};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 two = pair_to_float<BF16>(w[j]);
                f[2 * j] = two.x * inv;
                f[2 * j + 1] = two.y * inv;
            }
            moe_cut<FMT>(f, v, values, scales);
        }
        return;
    }
    // ---------------------------------------------------------------------- the choice of experts
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.counter_words; i += kMoeRouterThreads) p.counters[i] = 0u;
    cluster_arrive();             // every CTA of the cluster runs: its shared memory may be written
    cluster_wait();
    {
        const bool vec_ok = p.x_vec_ok && p.router_vec_ok;        // (the router's rows are whole pieces then)
        const int g = lane >> 2, q = lane & 3, tiles = (p.experts + 15) / 16, chunk = (pieces + 4 * kMoeRouterChunks - 1) / (4 * kMoeRouterChunks) * 4;
        const uint16_t* x = p.x + (t0 + min(g, n - 1)) * p.ldx;
        for (int task = rank * kWarps + warp; task < tiles * kMoeRouterChunks; task += kMoeRouterCtas * kWarps) {
            const int tile = task / kMoeRouterChunks, c = task % kMoeRouterChunks;
            const uint16_t* a0 = p.router + static_cast<size_t>(min(tile * 16 + g, p.experts - 1)) * p.hidden;
            const uint16_t* a1 = p.router + static_cast<size_t>(min(tile * 16 + g + 8, p.experts - 1)) * p.hidden;
            double sum[4] = {0.0, 0.0, 0.0, 0.0};
            const int v0 = min(c * chunk, pieces), v1 = min(v0 + chunk, pieces);
            if (vec_ok) moe_logits<BF16, true>(a0, a1, x, p.hidden, v0, v1, q, sum);
            else moe_logits<BF16, false>(a0, a1, x, p.hidden, v0, v1, q, sum);
#pragma unroll
            for (int j = 0; j < 4; ++j) {                         // (expert g, tokens 2q, 2q + 1), (expert g + 8, the same)
                const int token = q * 2 + (j & 1), e = tile * 16 + g + (j >> 1) * 8;
                if (token < n && e < p.experts)
                    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(parts + c * p.experts + e), token)), "d"(sum[j]) : "memory");
            }
        }
    }
    cluster_arrive();
    cluster_wait();
    if (rank >= n) return;
    for (int e = threadIdx.x; e < p.experts; e += kMoeRouterThreads) {
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < kMoeRouterChunks; ++c) sum += parts[c * p.experts + e];
        logits[e] = sum;
    }
    __syncthreads();
    if (warp != 0) return;
    constexpr int PER = kMoeMaxExperts / 32;
    unsigned long long key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = lane + 32 * i < p.experts ? logit_key(logits[lane + 32 * i]) : 0ull;
    double first = 0.0;
    double mine_logit = 0.0;                                      // lane r: the r-th choice
    int mine_id = 0;
    for (int r = 0; r < p.top; ++r) {
        unsigned long long best = 0ull;
        int at = kMoeMaxExperts;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (32 * i >= p.experts) break;
            if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
        }
        const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(best >> 32));
        const bool top_hi = static_cast<uint32_t>(best >> 32) == hi;
        const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, top_hi ? static_cast<uint32_t>(best) : 0u);
        const int id = __reduce_min_sync(0xFFFFFFFFu, top_hi && static_cast<uint32_t>(best) == lo ? at : kMoeMaxExperts);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i == id) key[i] = 0ull;
        const double v = logits[id];
        if (r == 0) first = v;
        if (lane == r) { mine_logit = v; mine_id = id; }
    }
    const float mine = expf(static_cast<float>(mine_logit - first));
    float z = lane < p.top ? mine : 0.f;
    if (!p.normalize) {
        z = 0.f;
        for (int e = lane; e < p.experts; e += 32) z += expf(static_cast<float>(logits[e] - first));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, o);
    if (lane < p.top) {
        const float weight = __fdiv_rn(mine, z);
        const int at = t * p.top + lane;
        p.ids[at] = mine_id;
        p.weights[at] = weight;
        if (p.ids_out) p.ids_out[at] = mine_id;
        if (p.weights_out) p.weights_out[at] = weight;
    }
}

constexpr int kMoeBuilderWarps = 12;
constexpr int kMoeBuilders = 32 * kMoeBuilderWarps;             // the last warps
constexpr int kMoeFirstBuilder = 11;
constexpr int kMoeThreads = kMoeFirstBuilder * 32 + kMoeBuilders;   // values producer, MMA issuer, 4 scale warps, 4 epilogue warps, scales producer, builders
constexpr int kMoeStages = 5;                                   // weight values, 256 of K, and as many sets of scales in tensor memory
constexpr int kMoeScaleStages = 4;                              // scales on their way there
constexpr int kMoeTileTokens = 16;                              // tokens of a pass at most: 128 MMA columns
constexpr int kMoeTileBytes = 128 * 1024;                       // activations of a pass: 8 tokens of 4096, 16 of 2048
constexpr int kMoeTileScales = 2560;                            // 2 KB and 16 bytes for each of 16 tokens, or two halves of half as much
constexpr int kMoeStageValues = 128 * 128, kMoeStageScales = 128 * 16;
constexpr int kMoeAccStride = 128, kMoeSfBase = 256;            // tensor memory: two accumulators, a set of scales (32 columns) per stage

// Tiles of activations: one, or two halves where a half holds 8 tokens, so that the next is made while one is multiplied.
__host__ __device__ constexpr int moe_tiles(int k) { return 8 * moe_value_bytes(k) <= kMoeTileBytes / 2 ? 2 : 1; }
__host__ __device__ constexpr int moe_pass_tokens(int k) {       // an even number
    const int n = kMoeTileBytes / moe_tiles(k) / moe_value_bytes(k);
    return n < kMoeTileTokens ? n / 2 * 2 : kMoeTileTokens;
}
__host__ __device__ constexpr int moe_tile_scale_pitch(int k, int fmt) { return moe_scale_bytes(k, fmt) + 16; }   // tokens 4 banks apart

// Part of a phase's work that one CTA does with one tile of activations: elements [first, last) of an expert (element = unit *
// pieces of K + piece), tokens of one pass.
struct MoeRun {
    uint16_t expert, pass, first, last;
};

struct MoeShared {
    unsigned long long token_mask[kMoeMaxExperts];
    int start[2][kMoeMaxExperts + 1];            // units x passes before each expert, per phase
    MoeRun runs[2][kMoeMaxRuns];
    int run_count[2], split[2];
    uint8_t ids[kMoeMaxTokens * kMoeMaxTop];     // the router's choices
    float x_scale[kMoeMaxTokens];
    uint16_t slot_row[4][kMoeTileTokens];        // per run (mod 4): assignment (token * top + choice) of each token of the pass
    float slot_scale[4][kMoeTileTokens];         // what its sums are multiplied with
    uint32_t slot_top[2][kMoeTileTokens];        // per run (mod 2): largest hidden activation, fp32 bits
    int abort_flag;
    uint32_t tmem_slot;
    unsigned long long full[kMoeStages], empty[kMoeStages], scale_full[kMoeScaleStages], scale_empty[kMoeScaleStages];
    unsigned long long acc_full[2], acc_empty[2], tile_full[2][2], tile_empty[2][2], slot_full[4], drain;
};
constexpr int kMoeStageScaleOffset = kMoeStages * kMoeStageValues;
constexpr int kMoeTileOffset = (kMoeStageScaleOffset + kMoeScaleStages * kMoeStageScales + 1023) / 1024 * 1024;
constexpr int kMoeTileScaleOffset = kMoeTileOffset + kMoeTileBytes;
constexpr int kMoeSharedOffset = kMoeTileScaleOffset + kMoeTileScales;
constexpr int kMoeSmemBytes = kMoeSharedOffset + static_cast<int>(sizeof(MoeShared)) + 1024;
static_assert(kMoeSmemBytes <= 227 * 1024, "shared memory over-subscribed");

__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
          "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
          "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void builders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kMoeBuilders) : "memory"); }

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kMoeThreads, 1)
moe_experts_kernel(const __grid_constant__ CUtensorMap map_w13, const __grid_constant__ CUtensorMap map_s13,
                   const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_s2, const MoeParams p) {
    constexpr int KT = f4_stage_tiles(FMT);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    MoeShared& sh = *reinterpret_cast<MoeShared*>(smem_gen + kMoeSharedOffset);
    uint8_t* tiles0 = smem_gen + kMoeTileOffset;
    uint8_t* tile_scales0 = smem_gen + kMoeTileScaleOffset;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int* abort_flag = &sh.abort_flag;
    unsigned* done = p.counters;
    unsigned* arrived = p.counters + p.experts;
    auto bar_of = [&](const unsigned long long& b) { return smem_u32(&b); };

    if (warp == 0 && elect_one()) {
        prefetch_tensormap(&map_w13);
        prefetch_tensormap(&map_s13);
        prefetch_tensormap(&map_w2);
        prefetch_tensormap(&map_s2);
    }
    const int units[2] = {(p.inter + 63) / 64, (p.hidden + 127) / 128};
    const int pass_tokens[2] = {moe_pass_tokens(p.hidden), moe_pass_tokens(p.inter)};
    const int items[2] = {moe_k_blocks(p.hidden), moe_k_blocks(p.inter)};
    const int tiles[2] = {moe_tiles(p.hidden), moe_tiles(p.inter)};

    // ---- who does what: token sets of the experts, work before each expert, this CTA's runs
    for (int e = threadIdx.x; e < p.experts; e += kMoeThreads) sh.token_mask[e] = 0ull;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMoeStages; ++i) {
            mbar_init(bar_of(sh.full[i]), 5);                            // the values, and each scale warp
            mbar_init(bar_of(sh.empty[i]), 1);
        }
        for (int i = 0; i < kMoeScaleStages; ++i) {
            mbar_init(bar_of(sh.scale_full[i]), 1);
            mbar_init(bar_of(sh.scale_empty[i]), 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_of(sh.acc_full[i]), 1);
            mbar_init(bar_of(sh.acc_empty[i]), 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_of(sh.tile_full[0][i]), 1);                   // gate / up: copies of what the router kernel cut
            mbar_init(bar_of(sh.tile_full[1][i]), kMoeBuilderWarps);    // down: cut here
            mbar_init(bar_of(sh.tile_empty[0][i]), 1);
            mbar_init(bar_of(sh.tile_empty[1][i]), 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(bar_of(sh.slot_full[i]), 1);
        mbar_init(bar_of(sh.drain), 1);
        sh.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&sh.tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_slot);
    pdl_launch_dependents();
    pdl_wait_prior_grid();        // what the router kernel wrote
    for (int a = threadIdx.x; a < p.tokens * p.top; a += kMoeThreads) {
        const int e = p.ids[a];
        sh.ids[a] = static_cast<uint8_t>(e);
        atomicOr(&sh.token_mask[e], 1ull << (a / p.top));
    }
    if (static_cast<int>(threadIdx.x) < p.tokens) sh.x_scale[threadIdx.x] = p.x_scale[threadIdx.x];
    __syncthreads();
    if (warp < 2) {
        const int ph = warp;
        int carry = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            const int mine = e < p.experts ? (__popcll(sh.token_mask[e]) + pass_tokens[ph] - 1) / pass_tokens[ph] * units[ph] : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
                if (lane >= o) sum += up;
            }
            if (e < p.experts) sh.start[ph][e] = carry + sum - mine;
            carry += __shfl_sync(0xFFFFFFFFu, sum, 31);
        }
        // pieces of K: as few as leave no CTA with much more than its share (one piece more costs about a twentieth of a unit)
        int split = 1;
        float best = 1e30f;
        for (int s = 1; s <= min(p.split, items[ph]); ++s) {
            const float cost = static_cast<float>((carry * s + gridDim.x - 1) / gridDim.x) / s + 0.05f * s;
            if (cost < best) { best = cost; split = s; }
        }
        if (lane == 0) {
            sh.start[ph][p.experts] = carry;
            sh.split[ph] = split;
        }
        __syncwarp();
        const unsigned total = static_cast<unsigned>(carry) * split, share = total / gridDim.x, rest = total - share * gridDim.x;
        const int from = static_cast<int>(share * blockIdx.x + min(blockIdx.x, rest)), to = from + static_cast<int>(share + (blockIdx.x < rest ? 1u : 0u));
        int count = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            const int lo = e < p.experts ? sh.start[ph][e] * split : 0, hi = e < p.experts ? sh.start[ph][e + 1] * split : 0;
            unsigned todo = __ballot_sync(0xFFFFFFFFu, lo < hi && lo < to && hi > from);
            while (todo) {
                const int ex = e0 + __ffs(todo) - 1;
                todo &= todo - 1;
                const int base = sh.start[ph][ex] * split, end = sh.start[ph][ex + 1] * split;
                const int passes = (end - base) / (units[ph] * split);
                const int a = max(from, base) - base, b = min(to, end) - base;
                // position = element * passes + pass: the passes over the same rows follow one another
                for (int p0 = 0; p0 < passes; p0 += 32) {
                    const int pass = p0 + lane;
                    const int first = a > pass ? (a - pass + passes - 1) / passes : 0, last = b > pass ? (b - pass + passes - 1) / passes : 0;
                    const unsigned some = __ballot_sync(0xFFFFFFFFu, pass < passes && first < last);
                    const int at = count + __popc(some & ((1u << lane) - 1u));
                    if (((some >> lane) & 1u) && at < kMoeMaxRuns)
                        sh.runs[ph][at] = MoeRun{static_cast<uint16_t>(ex), static_cast<uint16_t>(pass), static_cast<uint16_t>(first),
                                                 static_cast<uint16_t>(last)};
                    count += __popc(some);
                }
            }
        }
        if (lane == 0) sh.run_count[ph] = count < kMoeMaxRuns ? count : kMoeMaxRuns;
    }
    __syncthreads();
    const int count0 = sh.run_count[0], runs = count0 + sh.run_count[1];
    auto run_tokens = [&](const MoeRun& r, int ph) { return min(pass_tokens[ph], __popcll(sh.token_mask[r.expert]) - r.pass * pass_tokens[ph]); };
    // the assignment that token number j of a run's pass is
    auto slot_of = [&](const MoeRun& r, int ph, int j) {
        unsigned long long m = sh.token_mask[r.expert];
        for (int i = 0; i < r.pass * pass_tokens[ph] + j; ++i) m &= m - 1;
        const int t = __ffsll(static_cast<long long>(m)) - 1;
        int choice = 0;
        while (choice < p.top - 1 && sh.ids[t * p.top + choice] != r.expert) ++choice;
        return t * p.top + choice;
    };

    // pieces of K: unit and range of an element
    auto part_of = [&](int el, int ph, int split, int& unit, int& piece, int& kb0, int& kb1) {
        unit = el;
        piece = kb0 = 0;
        kb1 = items[ph];
        if (split == 1) return;                                   // (divisions are long for one thread)
        unit = el / split;
        piece = el - unit * split;
        kb0 = items[ph] * piece / split;
        kb1 = items[ph] * (piece + 1) / split;
    };

    // Every role goes through the CTA's runs, their elements and these elements' stages in the same order.
    if (warp == 0 || warp == 10) {
        // ------------------------------------------------------------------ producers: the weights' values, and their scales.  The scales run
        // further ahead: they are in tensor memory when the values arrive, and a stage of these is held for its MMAs only.
        const bool is_scales = warp == 10;
        const uint32_t stages = is_scales ? kMoeScaleStages : kMoeStages;
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        if (elect_one())
        for (int it = 0; it < runs && ok; ++it) {
            const int ph = it >= count0, split = sh.split[ph];
            const MoeRun r = sh.runs[ph][ph ? it - count0 : it];
            const CUtensorMap* map = is_scales ? (ph ? &map_s2 : &map_s13) : (ph ? &map_w2 : &map_w13);
            for (int el = r.first; el < r.last && ok; ++el) {
                int unit, piece, kb0, kb1;
                part_of(el, ph, split, unit, piece, kb0, kb1);
                const int row = unit * (ph ? 128 : 64), outer = ph ? r.expert : 2 * r.expert;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!bounded_wait(is_scales ? bar_of(sh.scale_empty[stage]) : bar_of(sh.empty[stage]), phase ^ 1u, abort_flag, p.status,
                                      DEV_TIMEOUT_PRODUCER_EMPTY)) { ok = false; break; }
                    if (is_scales) {
                        const uint32_t bar = bar_of(sh.scale_full[stage]);
                        mbar_expect_tx(bar, kMoeStageScales);
                        tma_load_3d(smem_base + kMoeStageScaleOffset + stage * kMoeStageScales, map, bar, (FMT == FMT_E4M3 ? kb : kb >> 1) * 16, row, outer);
                    } else {
                        const uint32_t bar = bar_of(sh.full[stage]);
                        mbar_expect_tx(bar, kMoeStageValues);
                        tma_load_3d(smem_base + stage * kMoeStageValues, map, bar, kb * 128, row, outer);
                    }
                    if (++stage == stages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        // One thread does it all, and a stage's barrier counts its values and the four scale warps: as a warp with two barriers and two
        // commits a stage it took 850 clocks each, of which the tensor core works 170 (64 tokens 139 us, now 130).
        const uint64_t stage_desc = make_smem_desc(smem_base, 0, 1024, SWIZZLE_128B_DESC);
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (int it = 0; it < runs && ok; ++it) {
                const int ph = it >= count0, run = ph ? it - count0 : it, split = sh.split[ph];
                const MoeRun r = sh.runs[ph][run];
                const int columns = (run_tokens(r, ph) + 1) / 2 * 16;
                const uint32_t idesc0 = make_idesc_f4<FMT>(128, columns, 0), idesc2 = make_idesc_f4<FMT>(128, columns, 2);
                const int tile_at = run & (tiles[ph] - 1), tile_use = run >> (tiles[ph] - 1);      // (one or two tiles)
                // the 8 columns of a token are one row group; the groups lie a token's activations apart
                const uint64_t tile_desc = make_smem_desc(smem_base + kMoeTileOffset + tile_at * (kMoeTileBytes / 2), 0, items[ph] * 1024, SWIZZLE_128B_DESC);
                if (!bounded_wait(bar_of(sh.tile_full[ph][tile_at]), tile_use & 1, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
                for (int el = r.first; el < r.last && ok; ++el) {
                    int unit, piece, kb0, kb1;
                    part_of(el, ph, split, unit, piece, kb0, kb1);
                    if (!bounded_wait(bar_of(sh.acc_empty[acc]), acc_phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_MMA_ACC_EMPTY)) { ok = false; break; }
                    const uint32_t d = tmem_base + acc * kMoeAccStride;
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!bounded_wait(bar_of(sh.full[stage]), phase, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
                        tc_fence_after_sync();
                        const uint32_t sfa = tmem_base + kMoeSfBase + stage * 32, sfb = sfa + 4 * KT;
                        const uint64_t a_desc = stage_desc + stage * (kMoeStageValues >> 4), b_desc = tile_desc + kb * (1024 >> 4);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const int t = ks * KT / 4;
                            mma_f4<false, FMT>(d, a_desc + ks * 2, b_desc + ks * 2, FMT == FMT_E8M0 && (ks & 1) ? idesc2 : idesc0, sfa + t * 4, sfb + t * 4,
                                               (kb != kb0 || ks != 0) ? 1u : 0u);
                        }
                        tc_commit(bar_of(sh.empty[stage]));       // for the next values, and for the next scales
                        if (++stage == kMoeStages) { stage = 0; phase ^= 1u; }
                    }
                    if (!ok) break;
                    tc_commit(bar_of(sh.acc_full[acc]));
                    acc ^= 1u;
                    if (acc == 0) acc_phase ^= 1u;
                }
                if (!ok) break;
                tc_commit(bar_of(sh.tile_empty[ph][tile_at]));
            }
            if (!ok) {
                tc_commit(bar_of(sh.drain));
                const uint64_t t0 = global_timer_ns();
                while (!mbar_try_wait(bar_of(sh.drain), 0) && global_timer_ns() - t0 < 20000000ull) {}
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------------ scale warps, epilogue warps and builders
        const int quarter = warp & 3, tid = static_cast<int>(threadIdx.x) - 32 * kMoeFirstBuilder;
        const bool scales_role = warp < 6, epilogue_role = warp >= 6 && warp < 10;
        uint32_t stage = 0, phase = 0, buf = 0, buf_phase = 0, acc = 0, acc_phase = 0;
        bool ok = true;                                           // a builder that gave up still meets the others at their barriers
        for (int it = 0; it < runs; ++it) {
            const int ph = it >= count0, run = ph ? it - count0 : it, split = sh.split[ph], k = ph ? p.inter : p.hidden;
            const int tile_at = run & (tiles[ph] - 1), tile_use = run >> (tiles[ph] - 1);      // (one or two tiles)
            const MoeRun r = sh.runs[ph][run];
            const int n = run_tokens(r, ph), value_bytes = moe_value_bytes(k), scale_pitch = moe_tile_scale_pitch(k, FMT);
            uint8_t* tile = tiles0 + tile_at * (kMoeTileBytes / 2);
            uint8_t* tile_scales = tile_scales0 + tile_at * (kMoeTileScales / 2);
            uint16_t* slot_row = sh.slot_row[it & 3];
            float* slot_scale = sh.slot_scale[it & 3];
            if (!scales_role && !epilogue_role) {
                // The tile's last use is over.  Only the first builder warp waits for that, and for every use in turn, so the barrier is never two
                // phases ahead of it: no tile is filled without it.  The others, who have nothing to do for gate / up, could be any number
                // of phases behind; they touch a tile only behind the builders' own barrier.
                auto wait_empty = [&](int phs, int at, int parity) {
                    ok = ok && warp_bounded_wait(bar_of(sh.tile_empty[phs][at]), parity, abort_flag, p.status, DEV_TIMEOUT_PRODUCER_EMPTY);
                };
                if (ph == 0 && warp != kMoeFirstBuilder) continue;
                if (warp == kMoeFirstBuilder) wait_empty(ph, tile_at, (tile_use & 1) ^ 1);
                if (ph == 0) {
                    if (ok) {                                     // copies what the router kernel has cut
                        const uint32_t bar = bar_of(sh.tile_full[0][tile_at]);
                        const int scale_bytes = moe_scale_bytes(k, FMT);
                        int t = 0;
                        if (lane < n) {
                            const int row = slot_of(r, 0, lane);
                            t = row / p.top;
                            slot_row[lane] = static_cast<uint16_t>(row);
                            slot_scale[lane] = sh.x_scale[t];
                        }
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(bar_of(sh.slot_full[it & 3]));
                            mbar_expect_tx(bar, n * (value_bytes + scale_bytes));
                        }
                        __syncwarp();
                        if (lane < n) {
                            bulk_load(smem_u32(tile) + lane * value_bytes, p.x_values + static_cast<size_t>(t) * value_bytes, value_bytes, bar);
                            bulk_load(smem_u32(tile_scales) + lane * scale_pitch, p.x_scales + static_cast<size_t>(t) * scale_bytes, scale_bytes, bar);
                        }
                    }
                    continue;
                }
                // ---- hidden activations of the pass: silu(gate) * up from the sums of all CTAs, cut into their parts
                if (run == 0 && warp == kMoeFirstBuilder)         // (the tiles of both phases share their memory)
                    for (int i = 0; i < tiles[0] && i < count0; ++i) {
                        const int last = (count0 - 1 - i) / tiles[0];     // use of the tile that run count0 - 1 - i had
                        wait_empty(0, (count0 - 1 - i) % tiles[0], last & 1);
                    }
                if (tid < n) {
                    slot_row[tid] = static_cast<uint16_t>(slot_of(r, 1, tid));
                    sh.slot_top[run & 1][tid] = 0u;
                }
                if (tid == 32) {
                    const unsigned want = static_cast<unsigned>(sh.start[0][r.expert + 1] - sh.start[0][r.expert]) * sh.split[0] * 4u;
                    const uint64_t t0 = global_timer_ns();
                    while (!*abort_flag) {
                        unsigned v;
                        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(done + r.expert) : "memory");
                        if (v >= want) break;
                        if (global_timer_ns() - t0 > BM_WAIT_LIMIT_NS) {
                            *abort_flag = 1;
                            if (p.status) atomicCAS(p.status, 0, DEV_TIMEOUT_EXPERTS);
                        }
                    }
                }
                builders_sync();
                // a warp takes 256 activations of a token at a time: 1 KiB of the tile, in fp32 as well as cut up
                const int split0 = sh.split[0];
                const int tasks = n * items[1];
                struct Sums { float4 g0, g1, u0, u1; };
                auto source = [&](int at) {
                    const int j = at / items[1], v = (at - j * items[1]) * 32 + lane;
                    return p.gu + static_cast<size_t>(slot_row[j]) * p.split * p.gu_pitch + v * 8;
                };
                auto load = [&](const float* src) {
                    const float4* gp = reinterpret_cast<const float4*>(src);
                    const float4* upp = reinterpret_cast<const float4*>(src + p.gu_pitch / 2);
                    return Sums{__ldcg(gp), __ldcg(gp + 1), __ldcg(upp), __ldcg(upp + 1)};
                };
                Sums next{};                                      // the task after the one at hand is on its way
                if (warp - kMoeFirstBuilder < tasks) next = load(source(warp - kMoeFirstBuilder));
                auto hidden = [&](int at, float (&h)[8]) {
                    const Sums c = next;
                    if (at + kMoeBuilderWarps < tasks) next = load(source(at + kMoeBuilderWarps));
                    float g[8] = {c.g0.x, c.g0.y, c.g0.z, c.g0.w, c.g1.x, c.g1.y, c.g1.z, c.g1.w};
                    float up[8] = {c.u0.x, c.u0.y, c.u0.z, c.u0.w, c.u1.x, c.u1.y, c.u1.z, c.u1.w};
#pragma unroll 1
                    for (int s = 1; s < split0; ++s) {
                        const Sums m = load(source(at) + static_cast<size_t>(s) * p.gu_pitch);
                        g[0] += m.g0.x; g[1] += m.g0.y; g[2] += m.g0.z; g[3] += m.g0.w; g[4] += m.g1.x; g[5] += m.g1.y; g[6] += m.g1.z; g[7] += m.g1.w;
                        up[0] += m.u0.x; up[1] += m.u0.y; up[2] += m.u0.z; up[3] += m.u0.w; up[4] += m.u1.x; up[5] += m.u1.y; up[6] += m.u1.z; up[7] += m.u1.w;
                    }
                    const int k0 = ((at % items[1]) * 32 + lane) * 8;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float e = __expf(-fabsf(g[i]));       // not exp(-g): beyond 2^126 the quotient would be zero
                        h[i] = k0 + i < k ? __fdividef(g[i] < 0.f ? g[i] * e : g[i], 1.f + e) * up[i] : 0.f;      // (nobody wrote what is behind)
                    }
                };
                if constexpr (FMT == FMT_E4M3) {                  // the rows' factors first; the numbers wait in the tile
#pragma unroll 1
                    for (int at = warp - kMoeFirstBuilder; at < tasks; at += kMoeBuilderWarps) {
                        const int j = at / items[1], kb = at - j * items[1];
                        float h[8];
                        hidden(at, h);
                        uint32_t top = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t b = __float_as_uint(h[i]) & 0x7FFFFFFFu;
                            if (b < 0x7F800000u) top = max(top, b);
                        }
                        float4* keep = reinterpret_cast<float4*>(tile + j * value_bytes + kb * 1024) + lane;
                        keep[0] = make_float4(h[0], h[1], h[2], h[3]);
                        keep[32] = make_float4(h[4], h[5], h[6], h[7]);
                        top = __reduce_max_sync(0xFFFFFFFFu, top);
                        if (lane == 0) atomicMax(&sh.slot_top[run & 1][j], top);
                    }
                    builders_sync();
                }
                if (tid < n) {
                    float factor, inv;
                    moe_row_factor<FMT>(sh.slot_top[run & 1][tid], factor, inv);
                    slot_scale[tid] = factor;
                }
                if (warp == kMoeFirstBuilder) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_of(sh.slot_full[it & 3]));
                }
#pragma unroll 1
                for (int at = warp - kMoeFirstBuilder; at < tasks; at += kMoeBuilderWarps) {
                    const int j = at / items[1], kb = at - j * items[1];
                    float h[8];
                    if constexpr (FMT == FMT_E4M3) {
                        float factor, inv;
                        moe_row_factor<FMT>(sh.slot_top[run & 1][j], factor, inv);
                        const float4* keep = reinterpret_cast<const float4*>(tile + j * value_bytes + kb * 1024) + lane;
                        const float4 lo = keep[0], hi = keep[32];
                        h[0] = lo.x * inv; h[1] = lo.y * inv; h[2] = lo.z * inv; h[3] = lo.w * inv;
                        h[4] = hi.x * inv; h[5] = hi.y * inv; h[6] = hi.z * inv; h[7] = hi.w * inv;
                        __syncwarp();                             // all lanes have theirs: the cut numbers take the place
                    } else {
                        hidden(at, h);
                    }
                    moe_cut<FMT>(h, kb * 32 + lane, tile + j * value_bytes, tile_scales + j * scale_pitch);
                }
                fence_proxy_async_smem();                         // visible to the tensor core
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_of(sh.tile_full[1][tile_at]));
                ok = __all_sync(0xFFFFFFFFu, ok && *abort_flag == 0);
                continue;
            }
            // The epilogue may be three runs behind the builders (two sums wait for it), so it has a barrier per slot of the four: a tile's
            // barrier could have moved on by two uses.  The scale warps are never behind: an element's MMAs need their part of it.
            ok = ok && (scales_role ? warp_bounded_wait(bar_of(sh.tile_full[ph][tile_at]), tile_use & 1, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)
                                    : warp_bounded_wait(bar_of(sh.slot_full[it & 3]), (it >> 2) & 1, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL));
            if (!ok) continue;
            const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
            if (scales_role) {
                // rows of scales -> tensor memory: row r of an operand in lane r % 32 of column r / 32, the same in each quarter
                const int groups = (n * 8 + 31) / 32;             // columns of 32 activations
                const int token = lane >> 3;
                const uint8_t* token_scales = tile_scales + token * scale_pitch;
                for (int el = r.first; el < r.last && ok; ++el) {
                    int unit, piece, kb0, kb1;
                    part_of(el, ph, split, unit, piece, kb0, kb1);
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!warp_bounded_wait(bar_of(sh.scale_full[stage]), phase, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
                        const uint4* rows = reinterpret_cast<const uint4*>(smem_gen + kMoeStageScaleOffset + stage * kMoeStageScales);
                        uint32_t set[8 * KT];                     // KT tiles of 4 columns of W's scales, then of the activations'
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint4 s = rows[c * 32 + lane];
                            // all columns of a token have its scales
                            const uint8_t* from = token_scales + c * 4 * scale_pitch + kb * KT * 4;
                            const bool some = c < groups && c * 4 + token < n;
                            if constexpr (FMT == FMT_E4M3) {
                                const uint4 x = some ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
                                set[c] = s.x; set[4 + c] = s.y; set[8 + c] = s.z; set[12 + c] = s.w;
                                set[16 + c] = x.x; set[20 + c] = x.y; set[24 + c] = x.z; set[28 + c] = x.w;
                            } else {                              // 16 bytes are 512 of K: this stage's half of them
                                const uint2 x = some ? *reinterpret_cast<const uint2*>(from) : make_uint2(0, 0);
                                set[c] = kb & 1 ? s.z : s.x; set[4 + c] = kb & 1 ? s.w : s.y;
                                set[8 + c] = x.x; set[12 + c] = x.y;
                            }
                        }
                        if (!warp_bounded_wait(bar_of(sh.empty[buf]), buf_phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_MMA_ACC_EMPTY)) { ok = false; break; }
                        tc_fence_after_sync();
                        tmem_st_32(tmem_base + lanes + kMoeSfBase + buf * 32, set);
                        tmem_st_wait();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(bar_of(sh.full[buf]));
                            mbar_arrive(bar_of(sh.scale_empty[stage]));       // what was read has been used
                        }
                        if (++stage == kMoeScaleStages) { stage = 0; phase ^= 1u; }
                        if (++buf == kMoeStages) { buf = 0; buf_phase ^= 1u; }
                    }
                }
            } else {
                const int row = quarter * 32 + lane;              // gate / up: rows 0-63 gate, 64-127 up of 64 channels
                for (int el = r.first; el < r.last && ok; ++el) {
                    int unit, piece, kb0, kb1;
                    part_of(el, ph, split, unit, piece, kb0, kb1);
                    const int channel = ph ? unit * 128 + row : unit * 64 + (row & 63), limit = ph ? p.hidden : p.inter;
                    const bool in = channel < limit;
                    float factor = 1.f;
                    float* out;
                    size_t step;
                    if (ph == 0) {
                        if (in && p.r13) factor = __ldg(p.r13 + (static_cast<size_t>(r.expert) * 2 + (row >> 6)) * p.inter + channel);
                        out = p.gu + static_cast<size_t>(piece) * p.gu_pitch + (row >> 6) * (p.gu_pitch / 2) + channel;
                        step = static_cast<size_t>(p.split) * p.gu_pitch;
                    } else {
                        if (in && p.r2) factor = __ldg(p.r2 + static_cast<size_t>(r.expert) * p.hidden + channel);
                        out = p.yp + static_cast<size_t>(piece) * p.y_pitch + channel;
                        step = static_cast<size_t>(p.split) * p.y_pitch;
                    }
                    if (!warp_bounded_wait(bar_of(sh.acc_full[acc]), acc_phase, abort_flag, p.status, DEV_TIMEOUT_EPI_ACC_FULL)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t taddr = tmem_base + lanes + acc * kMoeAccStride;
                    for (int j = 0; j < n; ++j) {
                        uint32_t v[8];
                        tmem_ld_32x8(taddr + j * 8, v);
                        tmem_ld_wait();
                        float sum = __uint_as_float(v[kMoeParts - 1]);        // the smallest first
#pragma unroll
                        for (int i = kMoeParts - 2; i >= 0; --i) sum = fmaf(sum, 0.125f, __uint_as_float(v[i]));
                        // factors on different sides of one are multiplied first, others one by one: nothing leaves fp32's range that the result is in
                        const float scale = slot_scale[j];
                        if (in) __stcg(out + slot_row[j] * step, (factor < 1.f) != (scale < 1.f) ? sum * (factor * scale) : sum * factor * scale);
                    }
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar_of(sh.acc_empty[acc]));
                        if (ph == 0) {
                            __threadfence();
                            atomicAdd(done + r.expert, 1u);
                        }
                    }
                    acc ^= 1u;
                    if (acc == 0) acc_phase ^= 1u;
                }
            }
        }
    }

    // ---- all experts' outputs exist: add them up
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();                    // copies still in flight land before the CTA leaves
        while (global_timer_ns() - t0 < 200000ull) {}
    } else if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(arrived, 1u);
        const uint64_t t0 = global_timer_ns();
        for (;;) {
            unsigned v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(arrived) : "memory");
            if (v >= gridDim.x) break;
            if (global_timer_ns() - t0 > BM_WAIT_LIMIT_NS) {
                *abort_flag = 1;
                if (p.status) atomicCAS(p.status, 0, DEV_TIMEOUT_EXPERTS);
                break;
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
    if (*abort_flag) return;
    // a warp takes 32 channels of a token: 8 lanes 4 each, of every fourth addend; neighbouring lines are in different CTAs
    const int split1 = sh.split[1], lines = (p.hidden + 31) / 32, addends = p.top * split1;
    for (int line = warp * gridDim.x + blockIdx.x; line < p.tokens * lines; line += (kMoeThreads / 32) * gridDim.x) {
        const int t = line / lines, c = (line - t * lines) * 32 + (lane & 7) * 4;      // (the rows of the sums are whole 32s long)
        const float* rows = p.yp + static_cast<size_t>(t) * p.top * p.split * p.y_pitch + c;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int a0 = lane >> 3; a0 < addends; a0 += 16) {        // four addends' loads in flight
            float4 y[4];
            float weight[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int a = min(a0 + 4 * i, addends - 1), choice = a / split1, s = a - choice * split1;
                y[i] = __ldcg(reinterpret_cast<const float4*>(rows + static_cast<size_t>(choice * p.split + s) * p.y_pitch));
                weight[i] = __ldcg(p.weights + t * p.top + choice);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (a0 + 4 * i >= addends) break;
                sum.x = fmaf(weight[i], y[i].x, sum.x);
                sum.y = fmaf(weight[i], y[i].y, sum.y);
                sum.z = fmaf(weight[i], y[i].z, sum.z);
                sum.w = fmaf(weight[i], y[i].w, sum.w);
            }
        }
#pragma unroll
        for (int o = 8; o < 32; o <<= 1) {
            sum.x += __shfl_xor_sync(0xFFFFFFFFu, sum.x, o);
            sum.y += __shfl_xor_sync(0xFFFFFFFFu, sum.y, o);
            sum.z += __shfl_xor_sync(0xFFFFFFFFu, sum.z, o);
            sum.w += __shfl_xor_sync(0xFFFFFFFFu, sum.w, o);
        }
        if (lane >= 8) continue;
        const uint32_t lo = float_to_pair<BF16>(sum.x, sum.y), hi = float_to_pair<BF16>(sum.z, sum.w);
        uint16_t* dst = p.y + t * p.ldy + c;
        if (c < p.hidden) dst[0] = static_cast<uint16_t>(lo);
        if (c + 1 < p.hidden) dst[1] = static_cast<uint16_t>(lo >> 16);
        if (c + 2 < p.hidden) dst[2] = static_cast<uint16_t>(hi);
        if (c + 3 < p.hidden) dst[3] = static_cast<uint16_t>(hi >> 16);
    }
}

}  // namespace bm

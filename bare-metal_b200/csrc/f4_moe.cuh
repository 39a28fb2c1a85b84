// f4_moe.cuh — a whole mixture-of-experts layer for few tokens, in two kernels: 16-bit activations x 4-bit weights.
//
//   logits[t][e] = x[t] . router[e];  the `top` largest of a token, their softmax p (or their share of the softmax over all)
//   y[t] = sum over the chosen experts of p * W2_e ( silu(G_e x[t]) * (U_e x[t]) )
//
// What bounds it: every chosen expert's weights are read once, 9/16 (17/32) of a byte a weight; the products are few.
//
// Kernel 1, moe_router_kernel: a cluster of 8 CTAs per group of at most 4 tokens.  64 warps share the experts, each
// token's logits meet in the shared memory of one CTA, whose first warp selects.  Logits are added in fp32 over 8 products and
// in 64 bits beyond: which expert a token gets must not depend on a sum's rounding or on the batch the token is in.
//
// Kernel 2, moe_experts_kernel: one CTA per SM, all resident (cooperative launch).  The unit of work is 16 weight rows (gate / up:
// 8 channels of each) times the tokens of one expert, taken by ONE warp over all of K, so sums never leave registers.  Units are
// dealt out in contiguous ranges, expert by expert: a CTA keeps its expert's activations in shared memory and
// meets a new expert once or twice.  A warp streams its rows through a ring of its own (TMA boxes of 16 rows x 256 of K and
// their scales), refilled by the warp itself as it empties; the refill runs ahead into the next expert and, over
// the wait for the other CTAs' gate / up results, into the down projection's weights.
//   The weights become fp16 in registers (cvt e2m1 -> f16, exact) and go through mma.m16n8k16 with fp32 sums: 8 or 16 tokens
// are the columns, so a weight is converted once for all of them.  tcgen05 would want the activations in 4 or 8 bits too.
//   E4M3: the scale is multiplied in before the MMA (2 + 4 significant bits, exact in fp16).  E8M0: its range does not fit
// fp16, so the sums of each block of 32 are scaled in fp32.  Activations are held as fp16 times a power of two per token:
// fp16 inputs as they are, bf16 inputs moved so that the row's largest is in [2^14, 2^15) (bits below 2^-24 of that, 2^-38 of the
// largest, are lost), the hidden activations rounded once from fp32 to fp16's 11 bits in the same way.
//   The experts' outputs go to the workspace in fp32 and are added per token, in the order of the selection, after a last wait:
// no atomics on sums, the same bits on every call.
#pragma once
#include "f4_format.cuh"
#include "f4_gemm.cuh"
#include "sm100_ptx.cuh"

namespace bm {

constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxExperts = 256;
constexpr int kMoeMaxTop = 16;
constexpr int kMoeMaxDim = 16384;
constexpr int kMoeWarps = 8;
constexpr int kMoeThreads = 32 * kMoeWarps;
constexpr int kMoeRing = 5;                                     // ring slots per warp
constexpr int kMoeItemK = 256;                                  // K of an item: 128 bytes a row
constexpr int kMoeItemBytes = 16 * 128, kMoeItemScales = 16 * 16;
constexpr int kMoeMaxRuns = 112;
constexpr int kMoeTileTokens = 16;                              // tokens of a pass at most (two MMA column tiles)
constexpr int kMoeTileBytes = 16 * (8192 + 64);                 // activations of a pass

struct MoeWorkspace {            // byte offsets
    size_t counters, x_scale, ids, weights, h, y, bytes;
    int counter_words;           // done[E], arrived, pad[3], h_max[T * top]
    int h_pitch, y_pitch;        // elements
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
    int tokens_per_cluster;
    int x_vec_ok, router_vec_ok;
    unsigned* counters;
    int counter_words;
    float* x_scale;
    int* ids;
    float* weights;
    float* h;
    float* yp;
    int h_pitch, y_pitch;
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

template <bool BF16>
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = pair_to_float<BF16>(x[j]), q = pair_to_float<BF16>(y[j]);
        s = fmaf(p.x, q.x, s);
        s = fmaf(p.y, q.y, s);
    }
    return s;
}

// 2^(14 - floor(log2 m)) and its inverse for a finite m > 0 given as fp32 bits; 1 otherwise (a NaN or infinity shows by itself)
__device__ __forceinline__ void moe_power(uint32_t bits, float& up, float& down) {
    const int e = static_cast<int>(bits >> 23);                  // floor(log2 m) + 127
    up = down = 1.f;
    if (bits == 0 || e == 255) return;
    const int n = e < 15 ? 126 : 14 + 127 - e;                   // exponent of `up`, at most 126
    up = __uint_as_float(static_cast<uint32_t>(n + 127) << 23);
    down = __uint_as_float(static_cast<uint32_t>(127 - n) << 23);
}

constexpr int kMoeRouterCtas = 8, kMoeRouterThreads = 256, kMoeRouterTokens = 4;

// order of doubles as unsigned integers, NaN below every number; 0 is left for "no candidate"
__device__ __forceinline__ unsigned long long logit_key(double v) {
    if (v != v) return 1ull;
    const long long b = __double_as_longlong(v + 0.0);           // -0 counts as +0
    return (b < 0 ? ~static_cast<unsigned long long>(b) : static_cast<unsigned long long>(b) | (1ull << 63)) + 2ull;
}

template <bool BF16>
__global__ void __launch_bounds__(kMoeRouterThreads)
moe_router_kernel(const MoeParams p) {
    __shared__ double logits[kMoeMaxExperts];
    __shared__ uint32_t warp_max[kMoeRouterThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_ctarank());
    const int t0 = blockIdx.x / kMoeRouterCtas * p.tokens_per_cluster;
    const int left = p.tokens - t0, n = left < p.tokens_per_cluster ? left : p.tokens_per_cluster;
    pdl_launch_dependents();
    pdl_wait_prior_grid();        // the call before may still be using the workspace
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.counter_words; i += kMoeRouterThreads) p.counters[i] = 0u;
    const int pieces = (p.hidden + 7) / 8;
    cluster_arrive();             // every CTA of the cluster runs: its shared memory may be written
    cluster_wait();
    for (int e = rank * (kMoeRouterThreads / 32) + warp; e < p.experts; e += kMoeRouterCtas * (kMoeRouterThreads / 32)) {
        const uint16_t* row = p.router + static_cast<size_t>(e) * p.hidden;
        double sum[kMoeRouterTokens] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
        for (int v = lane; v < pieces; v += 32) {
            const uint4 w = moe_piece<BF16>(row, v, p.hidden, p.router_vec_ok);
#pragma unroll
            for (int j = 0; j < kMoeRouterTokens; ++j)
                if (j < n) sum[j] += static_cast<double>(dot8<BF16>(moe_piece<BF16>(p.x + (t0 + j) * p.ldx, v, p.hidden, p.x_vec_ok), w));
        }
#pragma unroll
        for (int j = 0; j < kMoeRouterTokens; ++j) {
            if (j >= n) break;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum[j] += __shfl_xor_sync(0xFFFFFFFFu, sum[j], o);
            if (lane == 0)
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(logits + e), j)), "d"(sum[j]) : "memory");
        }
    }
    const bool owner = rank < n;                                  // this CTA selects for token t0 + rank
    if (BF16 && owner) {
        const uint16_t* row = p.x + (t0 + rank) * p.ldx;
        uint32_t m = 0;
        for (int v = threadIdx.x; v < pieces; v += kMoeRouterThreads) {
            const uint4 d = moe_piece<BF16>(row, v, p.hidden, p.x_vec_ok);
            const uint32_t b = __vmaxu2(__vmaxu2(d.x & 0x7FFF7FFFu, d.y & 0x7FFF7FFFu), __vmaxu2(d.z & 0x7FFF7FFFu, d.w & 0x7FFF7FFFu));
            m = max(m, max(b & 0xFFFFu, b >> 16));
        }
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        if (lane == 0) warp_max[warp] = m;
    }
    cluster_arrive();
    cluster_wait();
    if (!owner || warp != 0) return;
    const int t = t0 + rank;
    float up = 1.f, down = 1.f;
    if (BF16) {
        uint32_t m = lane < kMoeRouterThreads / 32 ? warp_max[lane] : 0u;
        m = __reduce_max_sync(0xFFFFFFFFu, m);
        moe_power(m << 16, up, down);
    }
    if (lane == 0) p.x_scale[t] = up;
    constexpr int PER = kMoeMaxExperts / 32;
    unsigned long long key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = lane + 32 * i < p.experts ? logit_key(logits[lane + 32 * i]) : 0ull;
    double first = 0.0;
    float mine = 0.f;                                             // lane r: weight of the r-th choice
    int mine_id = 0;
    for (int r = 0; r < p.top; ++r) {
        unsigned long long best = 0ull;
        int at = kMoeMaxExperts;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
        const uint32_t hi = __reduce_max_sync(0xFFFFFFFFu, static_cast<uint32_t>(best >> 32));
        const bool top_hi = static_cast<uint32_t>(best >> 32) == hi;
        const uint32_t lo = __reduce_max_sync(0xFFFFFFFFu, top_hi ? static_cast<uint32_t>(best) : 0u);
        const int id = __reduce_min_sync(0xFFFFFFFFu, top_hi && static_cast<uint32_t>(best) == lo ? at : kMoeMaxExperts);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i == id) key[i] = 0ull;
        const double v = logits[id];
        if (r == 0) first = v;
        if (lane == r) { mine = expf(static_cast<float>(v - first)); mine_id = id; }
    }
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

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// scales 2i and 2i + 1 (bytes `sel`) of one word as fp16, each in both halves
__device__ __forceinline__ void e4m3_pair(uint32_t word, uint32_t sel, uint32_t& s0, uint32_t& s1) {
    const uint32_t two = __byte_perm(word, 0, sel);
    uint32_t h;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n" : "=r"(h) : "r"(two));
    s0 = __byte_perm(h, 0, 0x1010);
    s1 = __byte_perm(h, 0, 0x3232);
}

// One item: 16 rows x (32 * chunks) of K against NT tiles of 8 tokens.  Lane (g, q) of a warp (g = lane / 4, q = lane % 4) holds rows
// g and g + 8 and, of every 32 of K, the 8 from 8 q on; the same 8 of its token's activations: any order of K
// serves an MMA if both operands keep it.
template <int FMT, int NT>
__device__ __forceinline__ void moe_item(uint32_t w, uint32_t scales, uint32_t b_addr, uint32_t b_next, int live, int chunks, int kb, int lane,
                                         float (&acc)[NT][4]) {
    const int g = lane >> 2, q = lane & 3;
    const uint4 sa = lds128(scales + g * 16), sb = lds128(scales + 128 + g * 16);
    uint32_t s_lo[4], s_hi[4];
    if constexpr (FMT == FMT_E4M3) {
        s_lo[0] = sa.x; s_lo[1] = sa.y; s_lo[2] = sa.z; s_lo[3] = sa.w;
        s_hi[0] = sb.x; s_hi[1] = sb.y; s_hi[2] = sb.z; s_hi[3] = sb.w;
    } else {                                                      // 16 bytes are 512 of K: this item's half of them
        s_lo[0] = kb & 1 ? sa.z : sa.x; s_lo[1] = kb & 1 ? sa.w : sa.y;
        s_hi[0] = kb & 1 ? sb.z : sb.x; s_hi[1] = kb & 1 ? sb.w : sb.y;
        if (__vcmpeq4(s_lo[0], 0xFFFFFFFFu) | __vcmpeq4(s_lo[1], 0xFFFFFFFFu)) {       // byte 255 is a NaN (the shift below makes it infinity)
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = __uint_as_float(0x7FC00000u);
        }
        if (__vcmpeq4(s_hi[0], 0xFFFFFFFFu) | __vcmpeq4(s_hi[1], 0xFFFFFFFFu)) {
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i][2] = acc[i][3] = __uint_as_float(0x7FC00000u);
        }
    }
    const uint32_t row = w + g * 128 + q * 4;
    const uint32_t sel = q < 2 ? 0x4420u : 0x4431u;               // blocks of 16: lanes 0, 1 the first, lanes 2, 3 the second of a chunk
    uint32_t m0[2], m1[2];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        if (c >= chunks) break;
        uint32_t h0[4], h1[4];
        const uint32_t at = row + ((c ^ g) << 4);                 // 128-byte swizzle
        e2m1x8_to_half(lds32(at), h0);
        e2m1x8_to_half(lds32(at + 1024), h1);
        if constexpr (FMT == FMT_E4M3) {
            if ((c & 1) == 0) {
                e4m3_pair(s_lo[c >> 1], sel, m0[0], m0[1]);
                e4m3_pair(s_hi[c >> 1], sel, m1[0], m1[1]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h0[j] = hmul2(h0[j], m0[c & 1]);
                h1[j] = hmul2(h1[j], m1[c & 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            uint4 b = make_uint4(0, 0, 0, 0);
            if (g + 8 * i < live) b = lds128(b_addr + i * b_next + c * 64);
            if constexpr (FMT == FMT_E4M3) {
                mma_16x8x16(acc[i], h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                mma_16x8x16(acc[i], h0[2], h1[2], h0[3], h1[3], b.z, b.w);
            } else {
                float part[4] = {0.f, 0.f, 0.f, 0.f};
                mma_16x8x16(part, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                mma_16x8x16(part, h0[2], h1[2], h0[3], h1[3], b.z, b.w);
                // byte c of the row's scales << 23 (byte 0 stands for 2^-127, here for 0: nothing in fp32)
                const float f0 = __uint_as_float(__byte_perm(s_lo[c >> 2], 0, 0x0444 | ((c & 3) << 12)) >> 1);
                const float f1 = __uint_as_float(__byte_perm(s_hi[c >> 2], 0, 0x0444 | ((c & 3) << 12)) >> 1);
                acc[i][0] = fmaf(part[0], f0, acc[i][0]);
                acc[i][1] = fmaf(part[1], f0, acc[i][1]);
                acc[i][2] = fmaf(part[2], f1, acc[i][2]);
                acc[i][3] = fmaf(part[3], f1, acc[i][3]);
            }
        }
    }
}

// Part of a phase's work that one CTA does with one tile of activations: units [first, last) of an expert, tokens of one pass.
struct MoeRun {
    uint16_t expert, pass, first, last;
};

struct MoeShared {
    unsigned long long token_mask[kMoeMaxExperts];
    int start[2][kMoeMaxExperts + 1];            // work before each expert, per phase
    MoeRun runs[2][kMoeMaxRuns];
    int run_count[2];
    int slot_row[kMoeTileTokens];                // assignment (token * top + choice) of each token of the pass
    float slot_scale[kMoeTileTokens];            // what a sum of the pass is multiplied with
    int abort_flag;
    unsigned long long full[kMoeWarps * kMoeRing];
};
constexpr int kMoeRingOffset = 0;
constexpr int kMoeScaleOffset = kMoeWarps * kMoeRing * kMoeItemBytes;
constexpr int kMoeTileOffset = kMoeScaleOffset + kMoeWarps * kMoeRing * kMoeItemScales;
constexpr int kMoeSharedOffset = kMoeTileOffset + kMoeTileBytes;
constexpr int kMoeSmemBytes = kMoeSharedOffset + static_cast<int>(sizeof(MoeShared)) + 1024;
static_assert(kMoeSmemBytes <= 227 * 1024, "shared memory over-subscribed");

__host__ __device__ constexpr int moe_tile_pitch(int k_padded) { return (2 * k_padded + 63) / 128 * 128 + 64; }   // 64 mod 128: no bank conflicts
__host__ __device__ constexpr int moe_pass_tokens(int k_padded) {
    const int n = kMoeTileBytes / moe_tile_pitch(k_padded);
    return n < kMoeTileTokens ? n : kMoeTileTokens;
}

// A warp's own sequence of items: phase, run, unit, K.
struct MoeCursor {
    int phase, run, unit, kb;
    bool done;
};

template <int FMT, bool BF16>
__global__ void __launch_bounds__(kMoeThreads, 1)
moe_experts_kernel(const __grid_constant__ CUtensorMap map_w13, const __grid_constant__ CUtensorMap map_s13,
                   const __grid_constant__ CUtensorMap map_w2, const __grid_constant__ CUtensorMap map_s2, const MoeParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    MoeShared& sh = *reinterpret_cast<MoeShared*>(smem_gen + kMoeSharedOffset);
    uint8_t* tile = smem_gen + kMoeTileOffset;
    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;
    const uint32_t ring = smem_base + warp * kMoeRing * kMoeItemBytes, ring_scales = smem_base + kMoeScaleOffset + warp * kMoeRing * kMoeItemScales;
    const uint32_t full0 = smem_u32(sh.full + warp * kMoeRing);
    volatile int* abort_flag = &sh.abort_flag;
    unsigned* done = p.counters;
    unsigned* arrived = p.counters + p.experts;
    unsigned* h_max = p.counters + p.experts + 4;

    const int k_padded[2] = {(p.hidden + 31) / 32 * 32, (p.inter + 31) / 32 * 32};
    const int units[2] = {(p.inter + 7) / 8, (p.hidden + 15) / 16};
    const int pass_tokens[2] = {moe_pass_tokens(k_padded[0]), moe_pass_tokens(k_padded[1])};

    // ---- who does what: token sets of the experts, work before each expert, this CTA's runs
    for (int e = threadIdx.x; e < p.experts; e += kMoeThreads) sh.token_mask[e] = 0ull;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMoeWarps * kMoeRing; ++i) mbar_init(smem_u32(sh.full + i), 1);
        sh.abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    for (int a = threadIdx.x; a < p.tokens * p.top; a += kMoeThreads) atomicOr(&sh.token_mask[p.ids[a]], 1ull << (a / p.top));
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
        if (lane == 0) sh.start[ph][p.experts] = carry;
        __syncwarp();
        const long long total = carry;
        const int from = static_cast<int>(total * blockIdx.x / gridDim.x), to = static_cast<int>(total * (blockIdx.x + 1) / gridDim.x);
        int count = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            const bool hit = e < p.experts && sh.start[ph][e] < to && sh.start[ph][e + 1] > from && sh.start[ph][e] < sh.start[ph][e + 1];
            unsigned todo = __ballot_sync(0xFFFFFFFFu, hit);
            while (todo) {
                const int ex = e0 + __ffs(todo) - 1;
                todo &= todo - 1;
                const int base = sh.start[ph][ex], passes = (sh.start[ph][ex + 1] - base) / units[ph];
                const int a = max(from, base) - base, b = min(to, sh.start[ph][ex + 1]) - base;
                // position = unit * passes + pass: the passes over the same rows follow one another
                for (int pass = lane; pass < passes; pass += 32) {
                    const int first = a > pass ? (a - pass + passes - 1) / passes : 0, last = b > pass ? (b - pass + passes - 1) / passes : 0;
                    if (count + pass < kMoeMaxRuns)
                        sh.runs[ph][count + pass] = MoeRun{static_cast<uint16_t>(ex), static_cast<uint16_t>(pass), static_cast<uint16_t>(first),
                                                           static_cast<uint16_t>(last)};
                }
                count += passes;
            }
        }
        if (lane == 0) sh.run_count[ph] = count < kMoeMaxRuns ? count : kMoeMaxRuns;
    }
    __syncthreads();

    // ---- a warp's items and its ring
    auto settle = [&](MoeCursor& c) {                             // on to the next unit of this warp, if (c.unit) is past its run
        for (;;) {
            if (c.run >= sh.run_count[c.phase]) {
                if (c.phase == 1) { c.done = true; return; }
                c.phase = 1;
                c.run = 0;
                if (sh.run_count[1] > 0) c.unit = sh.runs[1][0].first + warp;
                continue;
            }
            if (c.unit < sh.runs[c.phase][c.run].last) return;
            if (++c.run < sh.run_count[c.phase]) c.unit = sh.runs[c.phase][c.run].first + warp;
        }
    };
    MoeCursor ahead{0, 0, sh.run_count[0] > 0 ? sh.runs[0][0].first + warp : 0, 0, false};
    settle(ahead);
    uint32_t issued = 0, taken = 0;
    auto refill = [&] {                                           // the next item into the slot that `issued` names
        if (ahead.done) return;
        const int slot = issued % kMoeRing;
        const uint32_t bar = full0 + 8u * slot;
        const int expert = sh.runs[ahead.phase][ahead.run].expert;
        if (elect_one()) {
            mbar_expect_tx(bar, kMoeItemBytes + kMoeItemScales);
            const int sx = (FMT == FMT_E4M3 ? ahead.kb : ahead.kb >> 1) * 16;
            if (ahead.phase == 0) {
                tma_load_3d(ring + slot * kMoeItemBytes, &map_w13, bar, ahead.kb * 128, ahead.unit * 8, expert * 2);
                tma_load_3d(ring_scales + slot * kMoeItemScales, &map_s13, bar, sx, ahead.unit * 8, expert * 2);
            } else {
                tma_load_3d(ring + slot * kMoeItemBytes, &map_w2, bar, ahead.kb * 128, ahead.unit * 16, expert);
                tma_load_3d(ring_scales + slot * kMoeItemScales, &map_s2, bar, sx, ahead.unit * 16, expert);
            }
        }
        __syncwarp();
        ++issued;
        if (++ahead.kb * kMoeItemK >= k_padded[ahead.phase]) {
            ahead.kb = 0;
            ahead.unit += kMoeWarps;
            settle(ahead);
        }
    };
    for (int i = 0; i < kMoeRing; ++i) refill();

    bool ok = true;
    for (int ph = 0; ph < 2 && ok; ++ph) {
        const int kp = k_padded[ph], pitch = moe_tile_pitch(kp), items = (kp + kMoeItemK - 1) / kMoeItemK;
        for (int run = 0; run < sh.run_count[ph] && ok; ++run) {
            const MoeRun r = sh.runs[ph][run];
            const unsigned long long mask = sh.token_mask[r.expert];
            const int of_expert = __popcll(mask);
            const int n = r.first < r.last ? min(pass_tokens[ph], of_expert - r.pass * pass_tokens[ph]) : 0;   // (a run may be empty)
            __syncthreads();                                      // the tile before has been read, the run before is complete
            if (ph == 0 && run > 0 && threadIdx.x == 0) {
                const MoeRun b = sh.runs[0][run - 1];
                __threadfence();
                atomicAdd(done + b.expert, static_cast<unsigned>(b.last - b.first));
            }
            if (static_cast<int>(threadIdx.x) < n) {
                unsigned long long m = mask;
                for (int i = 0; i < r.pass * pass_tokens[ph] + static_cast<int>(threadIdx.x); ++i) m &= m - 1;
                const int t = __ffsll(static_cast<long long>(m)) - 1;
                int choice = 0;
                while (choice < p.top - 1 && p.ids[t * p.top + choice] != r.expert) ++choice;
                sh.slot_row[threadIdx.x] = t * p.top + choice;
            }
            if (ph == 1 && n > 0 && threadIdx.x == 0) {
                // the expert's hidden activations come from several CTAs
                const unsigned want = static_cast<unsigned>(sh.start[0][r.expert + 1] - sh.start[0][r.expert]);
                const uint64_t t0 = global_timer_ns();
                for (;;) {
                    unsigned v;
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(done + r.expert) : "memory");
                    if (v >= want) break;
                    if (global_timer_ns() - t0 > BM_WAIT_LIMIT_NS) {
                        *abort_flag = 1;
                        if (p.status) atomicCAS(p.status, 0, DEV_TIMEOUT_EXPERTS);
                        break;
                    }
                }
            }
            __syncthreads();
            if (*abort_flag) { ok = false; break; }
            // ---- activations of the pass: fp16 rows, zeros up to whole 32s
            for (int j = 0; j < n; ++j) {
                const int row = sh.slot_row[j];
                uint4* dst = reinterpret_cast<uint4*>(tile + j * pitch);
                if (ph == 0) {
                    const int t = row / p.top;
                    const float up = BF16 ? __ldcg(p.x_scale + t) : 1.f;
                    if (threadIdx.x == 0) sh.slot_scale[j] = __frcp_rn(up);                 // a power of two
                    const uint16_t* src = p.x + t * p.ldx;
                    for (int v = threadIdx.x; v < kp / 8; v += kMoeThreads) {
                        uint4 d = moe_piece<BF16>(src, v, p.hidden, p.x_vec_ok);
                        if constexpr (BF16) {
                            uint32_t* w = reinterpret_cast<uint32_t*>(&d);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 f = pair_to_float<true>(w[i]);
                                w[i] = float_to_pair<false>(__fmul_rn(f.x, up), __fmul_rn(f.y, up));
                            }
                        }
                        dst[v] = d;
                    }
                } else {
                    float up, down;
                    moe_power(__ldcg(h_max + row), up, down);
                    if (threadIdx.x == 0) sh.slot_scale[j] = down;
                    const float* src = p.h + static_cast<size_t>(row) * p.h_pitch;
                    for (int v = threadIdx.x; v < kp / 8; v += kMoeThreads) {
                        const float4 lo = __ldcg(reinterpret_cast<const float4*>(src) + 2 * v), hi = __ldcg(reinterpret_cast<const float4*>(src) + 2 * v + 1);
                        float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i] = v * 8 + i < p.inter ? __fmul_rn(f[i], up) : 0.f;     // nobody wrote what is behind
                        dst[v] = make_uint4(float_to_pair<false>(f[0], f[1]), float_to_pair<false>(f[2], f[3]), float_to_pair<false>(f[4], f[5]),
                                            float_to_pair<false>(f[6], f[7]));
                    }
                }
            }
            __syncthreads();
            const uint32_t b_lane = smem_u32(tile) + g * pitch + q * 16, b_next = 8u * pitch;
            for (int unit = r.first + warp; unit < r.last && ok; unit += kMoeWarps) {
                float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
                for (int kb = 0; kb < items; ++kb) {
                    const int slot = taken % kMoeRing;
                    if (!warp_bounded_wait(full0 + 8u * slot, (taken / kMoeRing) & 1u, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
                    ++taken;
                    const int left = kp / 32 - kb * 8, chunks = left < 8 ? left : 8;
                    const uint32_t w = ring + slot * kMoeItemBytes, s = ring_scales + slot * kMoeItemScales;
                    if (n <= 8) moe_item<FMT, 1>(w, s, b_lane + kb * 512, b_next, n, chunks, kb, lane, reinterpret_cast<float(&)[1][4]>(acc));
                    else moe_item<FMT, 2>(w, s, b_lane + kb * 512, b_next, n, chunks, kb, lane, acc);
                    __syncwarp();                                 // all lanes have read the slot
                    refill();
                }
                if (!ok) break;
                if (ph == 0) {
                    // rows g: gate, rows g + 8: up of channel unit * 8 + g
                    const int channel = unit * 8 + g;
                    const bool in = channel < p.inter;
                    const size_t base = static_cast<size_t>(r.expert) * 2 * p.inter;
                    const float fg = in && p.r13 ? __ldg(p.r13 + base + channel) : 1.f;
                    const float fu = in && p.r13 ? __ldg(p.r13 + base + p.inter + channel) : 1.f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = (i >> 1) * 8 + q * 2 + (i & 1);
                        if ((i >> 1) * 8 >= n) break;
                        float hv = 0.f;
                        if (j < n) {
                            const float s = sh.slot_scale[j];
                            const float gate = acc[i >> 1][i & 1] * fg * s, up = acc[i >> 1][2 + (i & 1)] * fu * s;
                            hv = gate / (1.f + expf(-gate)) * up;
                            if (in) __stcg(p.h + static_cast<size_t>(sh.slot_row[j]) * p.h_pitch + channel, hv);
                            else hv = 0.f;
                        }
                        uint32_t m = __float_as_uint(fabsf(hv));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
                        if (g == 0 && j < n && m != 0u) atomicMax(h_max + sh.slot_row[j], m);
                    }
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int channel = unit * 16 + half * 8 + g;
                        if (channel >= p.hidden) continue;
                        const float f = p.r2 ? __ldg(p.r2 + static_cast<size_t>(r.expert) * p.hidden + channel) : 1.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = (i >> 1) * 8 + q * 2 + (i & 1);
                            if (j < n) __stcg(p.yp + static_cast<size_t>(sh.slot_row[j]) * p.y_pitch + channel,
                                              acc[i >> 1][half * 2 + (i & 1)] * f * sh.slot_scale[j]);
                        }
                    }
                }
            }
            if (*abort_flag) ok = false;
        }
        if (ph == 0) {
            __syncthreads();
            if (threadIdx.x == 0 && sh.run_count[0] > 0 && !*abort_flag) {
                const MoeRun b = sh.runs[0][sh.run_count[0] - 1];
                __threadfence();
                atomicAdd(done + b.expert, static_cast<unsigned>(b.last - b.first));
            }
        }
    }

    // ---- all experts' outputs exist: add them up
    __syncthreads();
    if (threadIdx.x == 0 && !*abort_flag) {
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
    if (*abort_flag) {
        // copies still in flight land before the CTA leaves
        for (; taken < issued; ++taken) {
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(full0 + 8u * (taken % kMoeRing), (taken / kMoeRing) & 1u) && global_timer_ns() - t0 < 20000000ull) {}
        }
        return;
    }
    for (int at = blockIdx.x * kMoeThreads + threadIdx.x; at < p.tokens * p.hidden; at += gridDim.x * kMoeThreads) {
        const int t = at / p.hidden, c = at - t * p.hidden;
        float sum = 0.f;
        for (int k = 0; k < p.top; ++k)
            sum = fmaf(__ldcg(p.weights + t * p.top + k), __ldcg(p.yp + static_cast<size_t>(t * p.top + k) * p.y_pitch + c), sum);
        p.y[t * p.ldy + c] = BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(sum)) : __half_as_ushort(__float2half_rn(sum));
    }
}

}  // namespace bm

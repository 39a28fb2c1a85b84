// f4_gemm_few.cuh — block-scaled 4-bit GEMM for few tokens: D^T = W * X^T, weights in the MMA's A slot.
//
// With few tokens the time is that of streaming W from HBM, if all SMs stream.  A tile is 128 output channels (the accumulator
// lanes; whole 128-row tiles because that is how the scales lie) and all tokens (the columns, rounded up to 16); the K
// range of a tile is cut into `split` parts, one for each CTA of a cluster, so that N = 4096 is 128 CTAs and not 32.  The parts
// meet in shared memory: each CTA puts its fp32 sums into its own, and after a cluster barrier every CTA adds those of
// all ranks, in rank order, for its share of the tokens, applies the factors and stores; the order of the additions never changes.
// A CTA has one tile and takes half of an SM: more tiles than SMs share the memory system without a second wave,
// and the set-up of one CTA hides behind the stream of the other.
//   Measured (E4M3, fp16 out, with the call's launch): 1 token on 28672 x 8192 21.4 us, 6.2 TB/s of values and scales; 16 tokens on
// 4096 x 4096 4.7 us, of which 9.4 MB take 1.4: set-up, the first loads' latency, the cluster's sum and the stores are the rest.
#pragma once
#include "f4_gemm.cuh"

namespace bm {

constexpr int kF4FewMaxTokens = 128;
constexpr int kF4FewThreads = 192;                        // producer, MMA issuer, 4 epilogue warps
constexpr int kF4FewMaxStages = 8;
constexpr int kF4FewMaxSplit = 8;
constexpr int kF4FewRingBytes = 104 * 1024;
constexpr int kF4FewBarOffset = kF4FewRingBytes;
constexpr int kF4FewSmemBytes = kF4FewBarOffset + (2 * kF4FewMaxStages + 2) * 8 + 16 + 1024;
static_assert(2 * (kF4FewSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");

struct F4FewParams {
    void* out;                   // D [tokens x channels]
    long long ld;
    int tokens, channels;
    const float* token_scale;    // ra, or NULL
    const float* channel_scale;  // rb, or NULL
    int tokens_padded;           // MMA N
    int k_blocks, stages, split;
    int tmem_cols;
    int* status;
};

template <int TYPE>
__device__ __forceinline__ void f4_store_one(void* out, long long at, float v) {
    using T = typename F4Out<TYPE>::type;
    if constexpr (TYPE == TYPE_F32) static_cast<T*>(out)[at] = v;
    else if constexpr (TYPE == TYPE_F16) static_cast<T*>(out)[at] = __float2half_rn(v);
    else static_cast<T*>(out)[at] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

template <int FMT, int TYPE>
__global__ void __launch_bounds__(kF4FewThreads, 2)
f4_gemm_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sw,
                   const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_sx, const F4FewParams p) {
    constexpr int KT = f4_stage_tiles(FMT);
    constexpr uint32_t W_BYTES = 128 * 128, SF_BYTES = KT * kF4TileBytes;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t x_bytes = static_cast<uint32_t>(p.tokens_padded) * 128u;
    const uint32_t nstages = static_cast<uint32_t>(p.stages);
    const uint32_t w_smem0 = smem_base, x_smem0 = w_smem0 + nstages * W_BYTES;
    const uint32_t sfw_smem0 = x_smem0 + nstages * x_bytes, sfx_smem0 = sfw_smem0 + nstages * SF_BYTES;
    const uint32_t bar0 = smem_base + kF4FewBarOffset;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kF4FewMaxStages + s); };
    const uint32_t acc_bar = bar0 + 8u * (2 * kF4FewMaxStages);
    const uint32_t drain_bar = acc_bar + 8u;
    const uint32_t tmem_slot = acc_bar + 16u;
    volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + kF4FewBarOffset + 8 * (2 * kF4FewMaxStages + 2));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot_gen + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
    const int tile = blockIdx.x / p.split;
    const int kb0 = static_cast<int>(static_cast<long long>(p.k_blocks) * rank / p.split);
    const int kb1 = static_cast<int>(static_cast<long long>(p.k_blocks) * (rank + 1) / p.split);      // at least one block

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(acc_bar, 1);
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, p.tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_gen;
    pdl_launch_dependents();
    pdl_wait_prior_grid();        // nothing global is touched before the previous grid is complete

    bool ok = true;
    if (warp == 0) {
        // ------------------------------------------------------------------ producer
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_sw);
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_sx);
        uint32_t stage = 0, phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_bounded_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_PRODUCER_EMPTY)) break;
            if (elect_one()) {
                const uint32_t bar = full_bar(stage);
                mbar_expect_tx(bar, W_BYTES + x_bytes + 2 * SF_BYTES);
                tma_load_2d(w_smem0 + stage * W_BYTES, &map_w, bar, kb * 128, tile * 128);
                tma_load_3d(sfw_smem0 + stage * SF_BYTES, &map_sw, bar, 0, kb * KT * 4, tile);
                tma_load_2d(x_smem0 + stage * x_bytes, &map_x, bar, kb * 128, 0);
                tma_load_3d(sfx_smem0 + stage * SF_BYTES, &map_sx, bar, 0, kb * KT * 4, 0);
            }
            __syncwarp();
            if (++stage == nstages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        const uint32_t idesc0 = make_idesc_f4<FMT>(128, p.tokens_padded, 0), idesc2 = make_idesc_f4<FMT>(128, p.tokens_padded, 2);
        const uint32_t sfw_tmem = tmem_base + p.tokens_padded, sfx_tmem = sfw_tmem + KT * 4;
        uint32_t stage = 0, phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_bounded_wait(full_bar(stage), phase, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t sfw_desc = make_smem_desc(sfw_smem0 + stage * SF_BYTES, 0, 128, SWIZZLE_NONE_DESC);
                const uint64_t sfx_desc = make_smem_desc(sfx_smem0 + stage * SF_BYTES, 0, 128, SWIZZLE_NONE_DESC);
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    tmem_cp_scales<false>(sfw_tmem + t * 4, sfw_desc + t * (kF4TileBytes >> 4));
                    tmem_cp_scales<false>(sfx_tmem + t * 4, sfx_desc + t * (kF4TileBytes >> 4));
                }
                const uint64_t w_desc = make_smem_desc(w_smem0 + stage * W_BYTES, 0, 1024, SWIZZLE_128B_DESC);
                const uint64_t x_desc = make_smem_desc(x_smem0 + stage * x_bytes, 0, 1024, SWIZZLE_128B_DESC);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const int t = ks * KT / 4;
                    mma_f4<false, FMT>(tmem_base, w_desc + ks * 2, x_desc + ks * 2, FMT == FMT_E8M0 && (ks & 1) ? idesc2 : idesc0,
                                       sfw_tmem + t * 4, sfx_tmem + t * 4, (kb != kb0 || ks != 0) ? 1u : 0u);
                }
                tc_commit(empty_bar(stage));
            }
            __syncwarp();
            if (++stage == nstages) { stage = 0; phase ^= 1u; }
        }
        if (elect_one()) tc_commit(ok ? acc_bar : drain_bar);
        __syncwarp();
        if (!ok) {
            uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(drain_bar, 0) && global_timer_ns() - t0 < 20000000ull) {}
        }
    }
    const int quarter = warp & 3, channel = tile * 128 + quarter * 32 + lane;
    const bool drains = warp >= 2;
    float channel_s = 1.f;
    if (drains) {
        // ------------------------------------------------------------------ epilogue warps: lanes are channels
        if (channel < p.channels && p.channel_scale) channel_s = __ldg(p.channel_scale + channel);
        ok = bounded_wait(acc_bar, 0, abort_flag, p.status, DEV_TIMEOUT_EPI_ACC_FULL);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (ok) {
            tc_fence_after_sync();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
            float* part = reinterpret_cast<float*>(smem_gen) + quarter * 32 + lane;        // [token][128]; the ring has been read
            for (int t0 = 0; t0 < p.tokens; t0 += 16) {
                uint32_t r[16];
                tmem_ld_32x16(taddr + t0, r);
                const int left = p.tokens - t0;
                const float mine_s = p.split == 1 && p.token_scale && (lane & 15) < left ? __ldg(p.token_scale + t0 + (lane & 15)) : 1.f;
                tmem_ld_wait();
                if (p.split > 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(t0 + j) * 128] = __uint_as_float(r[j]);
                } else {
                    float v[16];                            // all products first, then the stores
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        v[j] = __fmul_rn(__uint_as_float(r[j]), __fmul_rn(__shfl_sync(0xFFFFFFFFu, mine_s, j), channel_s));
                    if (channel < p.channels) {
                        long long at = t0 * p.ld + channel;
#pragma unroll
                        for (int j = 0; j < 16; ++j, at += p.ld)
                            if (j < left) f4_store_one<TYPE>(p.out, at, v[j]);
                    }
                }
            }
            tc_fence_before_sync();
        }
    }
    __syncwarp();
    if (p.split > 1) {
        cluster_arrive();                                    // the sums of every rank are in place
        cluster_wait();
        if (drains && ok && channel < p.channels) {
            const uint32_t mine = smem_base + static_cast<uint32_t>(quarter * 32 + lane) * 4u;
            constexpr int kTogether = 4;                     // tokens whose sums are on their way together: a remote load takes 0.3 us
            for (int t0 = rank; t0 < p.tokens; t0 += kTogether * p.split) {
                float part[kTogether][kF4FewMaxSplit];
#pragma unroll
                for (int i = 0; i < kTogether; ++i)
#pragma unroll
                    for (int r = 0; r < kF4FewMaxSplit; ++r) {
                        const int t = t0 + i * p.split;
                        part[i][r] = r < p.split && t < p.tokens ? ld_shared_cluster_f32(mapa_shared(mine + t * 512u, r)) : 0.f;
                    }
#pragma unroll
                for (int i = 0; i < kTogether; ++i) {
                    const int t = t0 + i * p.split;
                    if (t >= p.tokens) break;
                    float sum = part[i][0];
#pragma unroll
                    for (int r = 1; r < kF4FewMaxSplit; ++r) sum += part[i][r];
                    const float token_s = p.token_scale ? __ldg(p.token_scale + t) : 1.f;
                    f4_store_one<TYPE>(p.out, t * p.ld + channel, __fmul_rn(sum, __fmul_rn(token_s, channel_s)));
                }
            }
        }
        __syncwarp();
        cluster_arrive();                                    // nobody leaves while its sums are being read
        cluster_wait();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) {
        const uint64_t t0 = global_timer_ns();               // aborting: let copies in flight land
        while (global_timer_ns() - t0 < 200000ull) {}
    }
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, p.tmem_cols);
    }
}

}  // namespace bm

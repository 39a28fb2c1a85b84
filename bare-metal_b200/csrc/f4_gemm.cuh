// f4_gemm.cuh — block-scaled 4-bit GEMM: D[m][n] = (sum_k a[m][k] sa w[n][k] sw) * ra[m] * rb[n].
//
// tcgen05.mma.kind::mxf4nvf4.block_scale multiplies E2M1 values with the scales of their blocks and adds in fp32; 64 of K
// an instruction, the scales in tensor memory.  PAIR: two CTAs compute 256 x 256 outputs as in igemm_dense_pair.cuh
// (M = 256, each CTA stages its 128 rows of A and 128 of the 256 rows of W); otherwise one CTA computes 128 x 128.
// A ring stage is 256 of K (128 bytes a row, 128-byte swizzle) and its scales: 128 rows x 4 blocks are one 512-byte tile,
// which tcgen05.cp.32x128b.warpx4 puts into 4 columns of tensor memory, row r in lane r % 32 of column r / 32, once for
// each quarter of the lanes.  Every CTA of a pair multiplies its rows with all 256 columns, so each fetches the scales
// of all 256 rows of W.
//
// Tensor memory of a pair: the accumulators are columns [0, 256) and [192, 448), the scales of a stage take 48 (24) of the
// last 64.  The 64 shared columns are drained first and the next tile's MMAs wait for them (`overlap`), as in
// igemm_sparse_pair.cuh.  Copies into tensor memory and MMAs of one thread execute in the order of their issue, so the
// scales of the next stage may follow the MMAs that read the ones before.
//
// Where at most half of the pairs would work in the last wave, its tiles are cut into two halves of 128 columns for two pairs.
//
// What bounds it: an SM needs 128 x 256 x 64 MACs = 128 clocks an MMA (512 a stage) and 38 KiB of operands a stage, 76 B/clk.
// Measured (product alone, fp16 out; in brackets without its loads, and without the epilogue): 4096^3 28.4 us (24.0, 25.4), 8192 x 22016 x 4096
// E8M0 276 us (195, 238), 8192^3 201 to 209 us (150, 179), 5.3 to 5.5 PFLOP/s (power-capped when sustained); 777 x 2260 x 1000
// 6.6 us (5.5, 4.3).
#pragma once
#include "epilogue.cuh"
#include "f4_format.cuh"
#include "igemm_dense.cuh"
#include "sm100_ptx.cuh"

namespace bm {

// Instruction descriptor of kind::mxf4nvf4 with block scales (32 bit): [4,6) scale byte of B, [7,10) A format (1 = E2M1),
// [10,12) B format, [17,23) N >> 3, [23] scale type (0 E4M3, 1 E8M0), [27,29) M >> 7, [29,31) scale byte of A.
// K is 64; both operands K-major.  With blocks of 32 an MMA takes two of a column's four scale bytes, from byte 0 or 2.
template <int FMT>
__host__ __device__ constexpr uint32_t make_idesc_f4(int m, int n, int scale_byte) {
    return (static_cast<uint32_t>(scale_byte) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (FMT == FMT_E8M0 ? 1u << 23 : 0u) | (static_cast<uint32_t>(m >> 7) << 27) | (static_cast<uint32_t>(scale_byte) << 29);
}

template <bool PAIR, int FMT>
__device__ __forceinline__ void mma_f4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
#define BM_MMA_F4(CG, VEC)                                                                                                       \
    asm volatile("{\n\t"                                                                                                         \
                 ".reg .pred p;\n\t"                                                                                             \
                 "setp.ne.b32 p, %6, 0;\n\t"                                                                                     \
                 "tcgen05.mma.cta_group::" CG ".kind::mxf4nvf4.block_scale.scale_vec::" VEC " [%0], %1, %2, %3, [%4], [%5], p;\n\t" \
                 "}\n" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                  \
                 : "memory")
    if constexpr (PAIR) {
        if constexpr (FMT == FMT_E4M3) BM_MMA_F4("2", "4X");
        else BM_MMA_F4("2", "2X");
    } else {
        if constexpr (FMT == FMT_E4M3) BM_MMA_F4("1", "4X");
        else BM_MMA_F4("1", "2X");
    }
#undef BM_MMA_F4
}

// one tile of scales: shared memory (32 rows of 16 bytes) -> 4 columns, repeated for each quarter of the lanes
template <bool PAIR>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t smem_desc) {
    if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc) : "memory");
}

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst_smem, const CUtensorMap* map, uint32_t bar_cluster, int32_t x, int32_t y,
                                                 int32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
        : "memory");
}

constexpr int kF4BK = 256;                        // K per stage
__host__ __device__ constexpr int f4_stage_tiles(int fmt) { return kF4BK / (4 * f4_block(fmt)); }     // 4 or 2 scale tiles along K

template <bool PAIR, int FMT>
struct F4Cfg {
    static constexpr int BN = PAIR ? 256 : 128;                 // tile columns
    static constexpr int ROWS = PAIR ? 256 : 128;               // tile rows
    static constexpr int KT = f4_stage_tiles(FMT);
    static constexpr int AB_BYTES = 128 * 128;                  // 128 rows of an operand
    static constexpr int SFA_BYTES = KT * kF4TileBytes;
    static constexpr int SFB_BYTES = BN / 128 * KT * kF4TileBytes;
    static constexpr int STAGE_BYTES = 2 * AB_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int STAGES = 4;
    static constexpr int ACC_STRIDE = PAIR ? 192 : 128;
    static constexpr int SF_BASE = ACC_STRIDE + BN;             // 448 or 256
    static constexpr int SF_COLS = KT * 4 * (1 + BN / 128);     // 48 / 24 or 32 / 16
    static constexpr int SF_BUFS = (512 - SF_BASE) / SF_COLS < STAGES ? (512 - SF_BASE) / SF_COLS : STAGES;
    static constexpr int NC = BN / 2;                           // columns drained per epilogue warp
    static constexpr int SFA_OFFSET = 2 * STAGES * AB_BYTES;
    static constexpr int SFB_OFFSET = SFA_OFFSET + STAGES * SFA_BYTES;
    static constexpr int STORE_OFFSET = (SFB_OFFSET + STAGES * SFB_BYTES + 1023) / 1024 * 1024;
    static constexpr int BAR_OFFSET = STORE_OFFSET + kEpiWarps * kStoreBoxBytes;
    static constexpr int STRIP_OFFSET = BAR_OFFSET + (2 * STAGES + 6) * 8 + 16;
    static constexpr int SMEM_BYTES = STRIP_OFFSET + kEpiWarps * NC * 4 + 1024;
    static_assert(SF_BUFS >= 1 && SMEM_BYTES <= 227 * 1024, "over-subscribed");
};

struct F4GemmParams {
    void* out;
    long long ld;
    int rows, cols;
    const float* row_scale;      // ra, or NULL for ones
    const float* col_scale;      // rb, or NULL for ones
    int tiles_m, tiles_n, k_blocks;
    int group_m;                 // tile order, as DenseParams::group_m
    int tail_first;              // tiles from here on are computed as two halves of 128 columns by different pairs
    int tma_ok;                  // the output is stored through TMA
    int pair_ok;                 // the output allows 4-byte stores at even columns
    int* status;
};

template <int TYPE>
struct F4Out { using type = float; };
template <>
struct F4Out<TYPE_F16> { using type = __half; };
template <>
struct F4Out<TYPE_BF16> { using type = __nv_bfloat16; };

// 16 bytes of results: accumulators r[0..] times row and column factors
template <int TYPE>
__device__ __forceinline__ uint4 f4_convert16(const uint32_t* r, const float* col, float row_s) {
    if constexpr (TYPE == TYPE_F32) {
        uint4 o;
        o.x = __float_as_uint(__fmul_rn(__uint_as_float(r[0]), __fmul_rn(row_s, col[0])));
        o.y = __float_as_uint(__fmul_rn(__uint_as_float(r[1]), __fmul_rn(row_s, col[1])));
        o.z = __float_as_uint(__fmul_rn(__uint_as_float(r[2]), __fmul_rn(row_s, col[2])));
        o.w = __float_as_uint(__fmul_rn(__uint_as_float(r[3]), __fmul_rn(row_s, col[3])));
        return o;
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = float_to_pair<TYPE == TYPE_BF16>(__fmul_rn(__uint_as_float(r[2 * j]), __fmul_rn(row_s, col[2 * j])),
                                                    __fmul_rn(__uint_as_float(r[2 * j + 1]), __fmul_rn(row_s, col[2 * j + 1])));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Drains NC columns of 32 rows (one per lane) in chunks of 32.  `reverse`: the upper half of the chunks first (NC = 128).
// `first_half` is called once, when the first 64 columns have left the accumulator.
template <int TYPE, int NC, class Hook>
__device__ __forceinline__ void f4_drain(const F4GemmParams& p, const CUtensorMap* map, uint32_t taddr, int row0, int lane, int col0,
                                         const float* strip, float row_s, uint32_t stage_smem, bool reverse, const Hook& first_half) {
    using T = typename F4Out<TYPE>::type;
    constexpr int CHUNKS = NC / 32;
    constexpr int CHUNKS_PER_BOX = TYPE == TYPE_F32 ? 1 : 2;
    constexpr int PIECES = 32 * sizeof(T) / 16;                 // 16-byte pieces per chunk
    constexpr int PER = 16 / sizeof(T);
    const int sw = lane & 7;
    auto chunk_at = [&](int i) { return reverse ? i ^ (CHUNKS / 2) : i; };
    auto live_at = [&](int i) { return col0 + chunk_at(i) * 32 < p.cols; };             // warp-uniform
    uint32_t rr[2][32];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (live_at(i)) tmem_ld_32x32(taddr + chunk_at(i) * 32, rr[i]);
    tmem_ld_wait();
    first_half();                                               // before anything is converted: the next tile's MMAs may wait for it
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int c = chunk_at(i);
        const bool live = live_at(i);
        if (i >= 2 && live) tmem_ld_wait();
        const uint32_t* r = rr[i & 1];
        const int box_c0 = col0 + (c / CHUNKS_PER_BOX) * CHUNKS_PER_BOX * 32;
        // TMA writes whole pieces of 16 bytes: a box that ends inside one, or an output that TMA cannot store, is copied by the warp
        const bool by_tma = p.tma_ok && (p.cols % PER == 0 || box_c0 + CHUNKS_PER_BOX * 32 <= p.cols);
        if (live) {
            if (i % CHUNKS_PER_BOX == 0) {
                if (lane == 0) bulk_wait_read_all();            // the box before this one has been fetched
                __syncwarp();
            }
#pragma unroll
            for (int v = 0; v < PIECES; ++v) {
                const uint4 o = f4_convert16<TYPE>(r + v * PER, strip + c * 32 + v * PER, row_s);
                const int piece = (c % CHUNKS_PER_BOX) * PIECES + v;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage_smem + lane * 128 + ((piece ^ sw) << 4)), "r"(o.x),
                             "r"(o.y), "r"(o.z), "r"(o.w)
                             : "memory");
            }
        }
        if (i + 2 < CHUNKS && live_at(i + 2)) tmem_ld_32x32(taddr + chunk_at(i + 2) * 32, rr[i & 1]);
        if (i % CHUNKS_PER_BOX == CHUNKS_PER_BOX - 1 && box_c0 < p.cols && row0 < p.rows) {
            if (by_tma) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(map, stage_smem, box_c0, row0);
                    bulk_commit_group();
                }
            } else {
                __syncwarp();
                copy_staged_box<T, 4>(p.out, p.ld, p.rows, p.cols, p.pair_ok != 0, stage_smem, row0, box_c0, lane);
                __syncwarp();
            }
        }
    }
}

// Work of one unit (a pair or a CTA): tiles unit, unit + units, ... below `tail_first`, then, on pairs, half the columns of one tile of
// the partly filled last wave.
struct F4Work {
    int tile, half;              // half < 0: the whole tile
};
struct F4WorkIter {
    int next_tile, units, tiles, tail_first, unit;
    bool tail_done;
    __device__ F4WorkIter(int unit_, int units_, const F4GemmParams& p)
        : next_tile(unit_), units(units_), tiles(p.tiles_m * p.tiles_n), tail_first(p.tail_first), unit(unit_), tail_done(false) {}
    __device__ bool next(F4Work& w) {
        w.half = -1;
        if (next_tile < tail_first) {
            w.tile = next_tile;
            next_tile += units;
            return true;
        }
        if (tail_done || unit >= (tiles - tail_first) * 2) return false;
        tail_done = true;
        w.tile = tail_first + unit / 2;
        w.half = unit % 2;
        return true;
    }
};

// map_a, map_b: packed values as byte maps, boxes of 128 bytes x 128 rows.  map_sa, map_sb: tiled scales as [128-row tile]
// [4 * tiles_k rows][128 bytes]; map_b_half, map_sb_half: the same for half a tile (PAIR).  What a box reaches beyond K or beyond the last row tile arrives as zeros.
template <bool PAIR, int FMT, int TYPE>
__global__ void __launch_bounds__(kDenseThreads, 1)
f4_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_sa,
               const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sb,
               const __grid_constant__ CUtensorMap map_b_half, const __grid_constant__ CUtensorMap map_sb_half,
               const __grid_constant__ CUtensorMap map_out, const F4GemmParams p) {
    using Cfg = F4Cfg<PAIR, FMT>;
    constexpr int STAGES = Cfg::STAGES, KT = Cfg::KT;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t a_smem0 = smem_base, b_smem0 = smem_base + STAGES * Cfg::AB_BYTES;
    const uint32_t sfa_smem0 = smem_base + Cfg::SFA_OFFSET, sfb_smem0 = smem_base + Cfg::SFB_OFFSET;
    const uint32_t bar0 = smem_base + Cfg::BAR_OFFSET;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto acc_full_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
    auto acc_empty_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 4);
    const uint32_t overlap_bar = bar0 + 8u * (2 * STAGES + 5);          // pair: in the leader
    const uint32_t tmem_slot = bar0 + 8u * (2 * STAGES + 6);
    volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + Cfg::BAR_OFFSET + 8 * (2 * STAGES + 6));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot_gen + 1);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);      // known to be the same in all lanes
    const int lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;                // 0 = leader
    const int unit = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const int units = PAIR ? gridDim.x >> 1 : gridDim.x;
    auto tile_coords = [&](int tile, int& tm, int& tn) {
        if (p.group_m <= 0) { tm = tile % p.tiles_m; tn = tile / p.tiles_m; return; }
        const int band_tiles = p.group_m * p.tiles_n;
        const int band = tile / band_tiles, r = tile - band * band_tiles;
        const int left = p.tiles_m - band * p.group_m;
        const int rows = left < p.group_m ? left : p.group_m;
        tm = band * p.group_m + r % rows;
        tn = r / rows;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full_bar(a), 1);
            mbar_init(acc_empty_bar(a), (PAIR ? 2 : 1) * kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        mbar_init(overlap_bar, kEpiWarps);               // one warp per lane quarter and CTA of a pair
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    }
    tc_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) {
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_gen;
    pdl_launch_dependents();
    pdl_wait_prior_grid();        // nothing global is touched before the previous grid is complete

    if (warp == 0) {
        // ------------------------------------------------------------------ producer (every CTA)
        prefetch_tensormap(&map_a);
        prefetch_tensormap(&map_sa);
        prefetch_tensormap(&map_b);
        prefetch_tensormap(&map_sb);
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        F4WorkIter work(unit, units, p);
        F4Work w;
        while (ok && work.next(w)) {
            int tm, tn;
            tile_coords(w.tile, tm, tn);
            const int am = tm * (Cfg::ROWS / 128) + static_cast<int>(rank);        // 128-row blocks of A and W
            const int bn = tn * (Cfg::BN / 128) + static_cast<int>(rank);
            for (int kb = 0; kb < p.k_blocks; ++kb) {
                if (!warp_bounded_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_PRODUCER_EMPTY)) { ok = false; break; }
                if (elect_one()) {
                    const uint32_t a_dst = a_smem0 + stage * Cfg::AB_BYTES, b_dst = b_smem0 + stage * Cfg::AB_BYTES;
                    const uint32_t sfa_dst = sfa_smem0 + stage * Cfg::SFA_BYTES, sfb_dst = sfb_smem0 + stage * Cfg::SFB_BYTES;
                    if constexpr (PAIR) {
                        const uint32_t bar = mapa_shared(full_bar(stage), 0);
                        const bool whole = w.half < 0;
                        if (rank == 0)
                            mbar_expect_tx(full_bar(stage), 2 * (whole ? Cfg::STAGE_BYTES : Cfg::STAGE_BYTES - (Cfg::AB_BYTES + Cfg::SFB_BYTES) / 2));
                        tma_load_2d_pair(a_dst, &map_a, bar, kb * 128, am * 128);
                        tma_load_2d_pair(b_dst, whole ? &map_b : &map_b_half, bar, kb * 128,
                                         whole ? bn * 128 : tn * 256 + w.half * 128 + static_cast<int>(rank) * 64);
                        tma_load_3d_pair(sfa_dst, &map_sa, bar, 0, kb * KT * 4, am);
                        tma_load_3d_pair(sfb_dst, whole ? &map_sb : &map_sb_half, bar, 0, kb * KT * 4, whole ? tn * 2 : tn * 2 + w.half);
                    } else {
                        const uint32_t bar = full_bar(stage);
                        mbar_expect_tx(bar, Cfg::STAGE_BYTES);
                        tma_load_2d(a_dst, &map_a, bar, kb * 128, am * 128);
                        tma_load_2d(b_dst, &map_b, bar, kb * 128, bn * 128);
                        tma_load_3d(sfa_dst, &map_sa, bar, 0, kb * KT * 4, am);
                        tma_load_3d(sfb_dst, &map_sb, bar, 0, kb * KT * 4, tn);
                    }
                }
                __syncwarp();
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (leader of a pair)
        if (rank == 0) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, sf_buf = 0;
            [[maybe_unused]] uint32_t overlap_phase = 0;
            bool ok = true, first = true;
            F4WorkIter work(unit, units, p);
            F4Work w;
            while (ok && work.next(w)) {
                if (!warp_bounded_wait(acc_empty_bar(acc), acc_phase ^ 1u, abort_flag, p.status, DEV_TIMEOUT_MMA_ACC_EMPTY)) { ok = false; break; }
                if (PAIR && !first) {
                    if (!warp_bounded_wait(overlap_bar, overlap_phase, abort_flag, p.status, DEV_TIMEOUT_MMA_ACC_EMPTY)) { ok = false; break; }
                    overlap_phase ^= 1u;
                }
                first = false;
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * Cfg::ACC_STRIDE;
                for (int kb = 0; kb < p.k_blocks; ++kb) {
                    if (!warp_bounded_wait(full_bar(stage), phase, abort_flag, p.status, DEV_TIMEOUT_MMA_FULL)) { ok = false; break; }
                    tc_fence_after_sync();
                    const uint32_t sfa_tmem = tmem_base + Cfg::SF_BASE + sf_buf * Cfg::SF_COLS, sfb_tmem = sfa_tmem + KT * 4;
                    if (elect_one()) {
                        const uint64_t sfa_desc = make_smem_desc(sfa_smem0 + stage * Cfg::SFA_BYTES, 0, 128, SWIZZLE_NONE_DESC);
                        const uint64_t sfb_desc = make_smem_desc(sfb_smem0 + stage * Cfg::SFB_BYTES, 0, 128, SWIZZLE_NONE_DESC);
#pragma unroll
                        for (int t = 0; t < KT; ++t) {
                            tmem_cp_scales<PAIR>(sfa_tmem + t * 4, sfa_desc + t * (kF4TileBytes >> 4));
#pragma unroll
                            for (int r = 0; r < Cfg::BN / 128; ++r)
                                if (r == 0 || w.half < 0) tmem_cp_scales<PAIR>(sfb_tmem + t * (Cfg::BN / 32) + r * 4, sfb_desc + (r * KT + t) * (kF4TileBytes >> 4));
                        }
                        const uint64_t a_desc = make_smem_desc(a_smem0 + stage * Cfg::AB_BYTES, 0, 1024, SWIZZLE_128B_DESC);
                        const uint64_t b_desc = make_smem_desc(b_smem0 + stage * Cfg::AB_BYTES, 0, 1024, SWIZZLE_128B_DESC);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const int t = ks * KT / 4;                                 // scale tile of these 64 of K
                            const int byte = FMT == FMT_E8M0 ? (ks & 1) * 2 : 0;
                            const uint32_t idesc = PAIR && w.half >= 0 ? make_idesc_f4<FMT>(Cfg::ROWS, Cfg::BN / 2, byte) : make_idesc_f4<FMT>(Cfg::ROWS, Cfg::BN, byte);
                            mma_f4<PAIR, FMT>(d_tmem, a_desc + ks * 2, b_desc + ks * 2, idesc,
                                              sfa_tmem + t * 4, sfb_tmem + t * (Cfg::BN / 32), (kb | ks) != 0 ? 1u : 0u);
                        }
                        if constexpr (PAIR) {
                            tc_commit_pair(empty_bar(stage));
                            tc_commit_pair(mapa_shared(empty_bar(stage), 1));
                        } else {
                            tc_commit(empty_bar(stage));
                        }
                    }
                    __syncwarp();
                    if (++sf_buf == Cfg::SF_BUFS) sf_buf = 0;
                    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                if (elect_one()) {
                    if constexpr (PAIR) {
                        tc_commit_pair(acc_full_bar(acc));
                        tc_commit_pair(mapa_shared(acc_full_bar(acc), 1));
                    } else {
                        tc_commit(acc_full_bar(acc));
                    }
                }
                __syncwarp();
                acc ^= 1u;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (!ok) {
                if (elect_one()) {
                    if constexpr (PAIR) tc_commit_pair(drain_bar);
                    else tc_commit(drain_bar);
                }
                __syncwarp();
                uint64_t t0 = global_timer_ns();
                while (!mbar_try_wait(drain_bar, 0) && global_timer_ns() - t0 < 20000000ull) {}
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue warps (every CTA)
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        float* strip = reinterpret_cast<float*>(smem_gen + Cfg::STRIP_OFFSET) + (warp - 2) * Cfg::NC;
        const uint32_t my_stage = smem_base + Cfg::STORE_OFFSET + (warp - 2) * kStoreBoxBytes;
        uint32_t acc = 0, acc_phase = 0;
        F4WorkIter work(unit, units, p);
        F4Work w;
        while (work.next(w)) {
            int tm, tn;
            tile_coords(w.tile, tm, tn);
            const int row0 = tm * Cfg::ROWS + static_cast<int>(rank) * 128 + quarter * 32;
            const int columns = w.half < 0 ? Cfg::NC : Cfg::NC / 2;          // of this warp
            const int col0 = tn * Cfg::BN + (w.half < 0 ? 0 : w.half * Cfg::NC) + half * columns;
            __syncwarp();                                        // the strip has been read
#pragma unroll
            for (int i = lane; i < Cfg::NC; i += 32) {                       // (half a tile does not use all)
                const int c = col0 + i;
                strip[i] = c < p.cols && p.col_scale ? __ldg(p.col_scale + c) : 1.f;
            }
            __syncwarp();
            const int row = row0 + lane;
            const float row_s = row < p.rows && p.row_scale ? __ldg(p.row_scale + row) : 1.f;
            if (!bounded_wait(acc_full_bar(acc), acc_phase, abort_flag, p.status, DEV_TIMEOUT_EPI_ACC_FULL)) break;
            tc_fence_after_sync();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * Cfg::ACC_STRIDE + half * columns;
            // the columns both accumulators of a pair share: the last 64 of the first, the first 64 of the second one
            const bool has_overlap = PAIR && half != static_cast<int>(acc);
            auto overlap_read = [&] {
                if (!has_overlap) return;
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(mapa_shared(overlap_bar, 0));
            };
            if (PAIR && w.half >= 0) f4_drain<TYPE, 64>(p, &map_out, taddr, row0, lane, col0, strip, row_s, my_stage, false, NoHook{});      // the last unit
            else f4_drain<TYPE, Cfg::NC>(p, &map_out, taddr, row0, lane, col0, strip, row_s, my_stage, PAIR && half == 1, overlap_read);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(mapa_shared(acc_empty_bar(acc), 0));
                else mbar_arrive(acc_empty_bar(acc));
            }
            acc ^= 1u;
            if (acc == 0) acc_phase ^= 1u;
        }
        if (lane == 0) bulk_wait_all();
    }

    // ---------------------------------------------------------------------- teardown
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) {
        const uint64_t t0 = global_timer_ns();               // aborting: let copies in flight land
        while (global_timer_ns() - t0 < 200000ull) {}
    }
    __syncthreads();
    if constexpr (PAIR) {
        cluster_arrive();
        cluster_wait();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
        else tmem_dealloc(tmem_base, 512);
    }
}

}  // namespace bm

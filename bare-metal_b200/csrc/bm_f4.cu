// bm_f4.cu — extern "C" launchers of the 4-bit floating-point operators declared in include/bm_igemm.h.
#include "host_common.cuh"
#include "f4_gemm.cuh"
#include "f4_gemm_few.cuh"
#include "f4_moe.cuh"
#include "f4_quantize.cuh"

namespace bm {

static inline int ceil_div(int a, int b) { return a / b + (a % b != 0 ? 1 : 0); }     // a + b may pass 2^31
static inline int f4_row_bytes(int k) { return ceil_div(k, 32) * 16; }
static inline int f4_tiles_k(int k, int fmt) { return ceil_div(k, 4 * f4_block(fmt)); }
static inline int f4_scale_pitch(int k, int fmt) { return ceil_div(ceil_div(k, f4_block(fmt)), 16) * 16; }

// indexes of 32 bits go as far as the end of a matrix's last tile: whole 256s of rows, a CTA's pieces of a row
constexpr int kF4MaxRows = 0x7FFFFF00, kF4MaxK = 0x7FFF0000;

static int check_format(int format, int layout) {
    if (format != BM_F4_E8M0 && format != BM_F4_E4M3) return fail_msg(BM_ERR_LAYOUT, "unknown 4-bit format tag");
    if (layout != BM_SCALE_ROWS && layout != BM_SCALE_TILED) return fail_msg(BM_ERR_LAYOUT, "unknown scale layout tag");
    return BM_OK;
}
static size_t f4_scale_bytes(int rows, int k, int fmt, int layout) {
    return layout == BM_SCALE_TILED ? static_cast<size_t>(ceil_div(rows, 128)) * f4_tiles_k(k, fmt) * kF4TileBytes
                                    : static_cast<size_t>(rows) * f4_scale_pitch(k, fmt);
}
// the widest access, up to 16 bytes, that a matrix with this base and pitch allows at every eighth column
static int access_bytes(const void* p, size_t pitch) {
    int n = 16;
    while ((reinterpret_cast<uintptr_t>(p) | pitch) % n != 0) n /= 2;
    return n;
}
static bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---- quantise ---------------------------------------------------------------------------
template <int FMT, bool BF16>
static int launch_quantize(const F4QuantParams& p, int sms, cudaStream_t stream) {
    // Threads per row: four units a thread when there are many rows, one when there are few (the chip is empty and the length of a
    // thread's own work is the latency), as far as 1024 threads reach.
    const int held = p.rows <= sms ? 1 : 4, most = held == 4 ? 512 : kF4QuantMaxThreads;
    int group = ceil_div(ceil_div(p.units, held), 32) * 32;
    if (group > most) group = most;                                // the rest of such a row is read twice
    const dim3 block(group, group == 32 ? 4 : 1);
    const dim3 grid(ceil_div(p.rows_padded, static_cast<int>(block.y)));
    if (held == 1) quantize_f4_kernel<FMT, BF16, 1><<<grid, block, 0, stream>>>(p);
    else quantize_f4_kernel<FMT, BF16, 4><<<grid, block, 0, stream>>>(p);
    BM_CUDA_TRY(cudaGetLastError());
    return BM_OK;
}

template <int FMT>
static int launch_dequantize(const F4DequantParams& p, int type, cudaStream_t stream) {
    // rows side by side in a CTA where a row is less than 256 pieces
    int x = 256;
    while (x > 32 && x / 2 >= ceil_div(p.k, 8)) x /= 2;
    const dim3 block(x, 256 / x);
    const int y = ceil_div(p.rows, static_cast<int>(block.y) * kF4DequantRows);
    const dim3 grid(ceil_div(ceil_div(p.k, 8), x), y < 65535 ? y : 65535);
    if (type == TYPE_F16) dequantize_f4_kernel<FMT, TYPE_F16><<<grid, block, 0, stream>>>(p);
    else if (type == TYPE_BF16) dequantize_f4_kernel<FMT, TYPE_BF16><<<grid, block, 0, stream>>>(p);
    else dequantize_f4_kernel<FMT, TYPE_F32><<<grid, block, 0, stream>>>(p);
    BM_CUDA_TRY(cudaGetLastError());
    return BM_OK;
}

static int sm_count(int* sms) {                    // not current_device_state(): its first use allocates
    int device = 0;
    BM_CUDA_TRY(cudaGetDevice(&device));
    BM_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    return BM_OK;
}

// ---- product ----------------------------------------------------------------------------
// tiled scales of `rows` rows as [row tile][4 * tiles_k][128 bytes], boxes of the scale tiles of one stage x `tiles` row tiles
static int scale_map(CUtensorMap* map, const void* base, int rows, int k, int fmt, int tiles) {
    const int tiles_k = f4_tiles_k(k, fmt);
    const uint64_t dims[3] = {128, 4ull * tiles_k, static_cast<uint64_t>(ceil_div(rows, 128))};
    const uint32_t box[3] = {128, 4u * f4_stage_tiles(fmt), static_cast<uint32_t>(tiles)};
    return cached_tensor_map(map, base, 3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, 128, box, CU_TENSOR_MAP_SWIZZLE_NONE, true,
                             static_cast<uint64_t>(tiles_k) * kF4TileBytes);
}

struct F4Operands {
    const uint8_t *a, *sa, *b, *sb;
    int fmt, type, M, N, K;
};

template <bool PAIR, int FMT, int TYPE>
static int launch_f4_inst(const F4Operands& o, F4GemmParams& p, DeviceState* dev, cudaStream_t stream) {
    using Cfg = F4Cfg<PAIR, FMT>;
    const size_t elem = TYPE == TYPE_F32 ? 4 : 2;
    const int pitch = f4_row_bytes(o.K);
    CUtensorMap ma, msa, mb, msb, mb_half, msb_half, mo;
    if (int rc = make_tensor_map_u8(&ma, o.a, pitch, o.M, pitch, 128, 128, true)) return rc;
    if (int rc = make_tensor_map_u8(&mb, o.b, pitch, o.N, pitch, 128, 128, true)) return rc;
    if (int rc = scale_map(&msa, o.sa, o.M, o.K, FMT, 1)) return rc;
    if (int rc = scale_map(&msb, o.sb, o.N, o.K, FMT, Cfg::BN / 128)) return rc;
    p.pair_ok = access_bytes(p.out, static_cast<size_t>(p.ld) * elem) >= 4;
    mo = ma;                                         // placeholder unless the output qualifies for TMA stores
    if (aligned16(p.out) && (static_cast<size_t>(p.ld) * elem) % 16 == 0 && opt(OPT_TMA_STORE) != 0) {
        if (int rc = make_tensor_map_out(&mo, p.out, o.N, o.M, static_cast<size_t>(p.ld) * elem, static_cast<int>(elem))) return rc;
        p.tma_ok = 1;
    }
    p.tiles_m = ceil_div(o.M, Cfg::ROWS);
    p.tiles_n = ceil_div(o.N, Cfg::BN);
    p.k_blocks = ceil_div(o.K, kF4BK);
    p.status = dev->status;
    const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
    if (tiles > 0x7FFFFFFF) return fail_msg(BM_ERR_TOO_LARGE, "more than 2^31 output tiles");
    const int slots = PAIR ? dev->sm_count / 2 : dev->sm_count;
    const int units = tiles < slots ? static_cast<int>(tiles) : slots;
    p.tail_first = static_cast<int>(tiles);
    mb_half = mb;
    msb_half = msb;
    const int rest = static_cast<int>(tiles % units);
    if (PAIR && tiles > units && rest > 0 && 2 * rest <= units && opt(OPT_TAIL_NARROW) != 0) {
        p.tail_first -= rest;
        if (int rc = make_tensor_map_u8(&mb_half, o.b, pitch, o.N, pitch, 128, 64, true)) return rc;
        if (int rc = scale_map(&msb_half, o.sb, o.N, o.K, FMT, 1)) return rc;
    }
    if (PAIR) p.group_m = p.tiles_m >= 2 * p.tiles_n && p.tiles_m >= 16 ? 8 : 0;      // as for the int8 pair kernel
    auto kern = f4_gemm_kernel<PAIR, FMT, TYPE>;
    static ConfiguredFlags flags;
    if (int rc = ensure_smem_limit(flags, kern, Cfg::SMEM_BYTES)) return rc;
    BM_CUDA_TRY(launch_pdl(kern, dim3(PAIR ? 2 * units : units), dim3(kDenseThreads), Cfg::SMEM_BYTES, stream, PAIR ? 2 : 1, ma, msa, mb,
                           msb, mb_half, msb_half, mo, p));
    return BM_OK;
}
template <bool PAIR>
static int launch_f4(const F4Operands& o, F4GemmParams& p, DeviceState* dev, cudaStream_t stream) {
#define BM_F4_CASE(F, T) if (o.fmt == F && o.type == T) return launch_f4_inst<PAIR, F, T>(o, p, dev, stream)
    BM_F4_CASE(FMT_E8M0, TYPE_F16); BM_F4_CASE(FMT_E8M0, TYPE_BF16); BM_F4_CASE(FMT_E8M0, TYPE_F32);
    BM_F4_CASE(FMT_E4M3, TYPE_F16); BM_F4_CASE(FMT_E4M3, TYPE_BF16); BM_F4_CASE(FMT_E4M3, TYPE_F32);
#undef BM_F4_CASE
    return fail_msg(BM_ERR_LAYOUT, "unknown element type tag");
}

template <int FMT, int TYPE>
static int launch_f4_few(const CUtensorMap& mw, const CUtensorMap& msw, const CUtensorMap& mx, const CUtensorMap& msx, const F4FewParams& p,
                         int tiles, cudaStream_t stream) {
    auto kern = f4_gemm_few_kernel<FMT, TYPE>;
    static ConfiguredFlags flags;
    if (int rc = ensure_smem_limit(flags, kern, kF4FewSmemBytes)) return rc;
    BM_CUDA_TRY(launch_pdl(kern, dim3(tiles * p.split), dim3(kF4FewThreads), kF4FewSmemBytes, stream, p.split, mw, msw, mx, msx, p));
    return BM_OK;
}

static int f4_few(const F4Operands& o, const F4GemmParams& g, DeviceState* dev, cudaStream_t stream) {
    F4FewParams p{};
    p.out = g.out;
    p.ld = g.ld;
    p.tokens = o.M;
    p.channels = o.N;
    p.token_scale = g.row_scale;
    p.channel_scale = g.col_scale;
    p.tokens_padded = ceil_div(o.M, 16) * 16;
    p.k_blocks = ceil_div(o.K, kF4BK);
    p.status = dev->status;
    const int stage_bytes = 128 * 128 + p.tokens_padded * 128 + 2 * f4_stage_tiles(o.fmt) * kF4TileBytes;
    p.stages = kF4FewRingBytes / stage_bytes;
    if (p.stages > kF4FewMaxStages) p.stages = kF4FewMaxStages;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.tokens_padded + 2 * f4_stage_tiles(o.fmt) * 4) p.tmem_cols *= 2;
    const int tiles = ceil_div(o.N, 128);
    p.split = 1;
    // Parts of K: as many as leave one CTA per SM (a second one per SM gained nothing: 16 tokens on 4096 x 4096 4.7 -> 5.3 us, on
    // 12288 x 4096 6.7 -> 7.9, on 4096 x 11008 6.4 -> 6.4; fewer parts: 4096 x 4096 6.7 with 2 instead of 4).
    while (p.split < kF4FewMaxSplit && 2 * p.split * tiles <= dev->sm_count && 2 * p.split <= p.k_blocks) p.split *= 2;
    CUtensorMap mw, msw, mx, msx;
    const int pitch = f4_row_bytes(o.K);
    if (int rc = make_tensor_map_u8(&mw, o.b, pitch, o.N, pitch, 128, 128, true)) return rc;
    if (int rc = make_tensor_map_u8(&mx, o.a, pitch, o.M, pitch, 128, p.tokens_padded, true)) return rc;
    if (int rc = scale_map(&msw, o.sb, o.N, o.K, o.fmt, 1)) return rc;
    if (int rc = scale_map(&msx, o.sa, o.M, o.K, o.fmt, 1)) return rc;
#define BM_F4_CASE(F, T) if (o.fmt == F && o.type == T) return launch_f4_few<F, T>(mw, msw, mx, msx, p, tiles, stream)
    BM_F4_CASE(FMT_E8M0, TYPE_F16); BM_F4_CASE(FMT_E8M0, TYPE_BF16); BM_F4_CASE(FMT_E8M0, TYPE_F32);
    BM_F4_CASE(FMT_E4M3, TYPE_F16); BM_F4_CASE(FMT_E4M3, TYPE_BF16); BM_F4_CASE(FMT_E4M3, TYPE_F32);
#undef BM_F4_CASE
    return fail_msg(BM_ERR_LAYOUT, "unknown element type tag");
}

// Which kernel (1 few tokens, 2 tiles of 128 x 128, 3 CTA pairs).  Microseconds, fitted to 1 to 2048 tokens on weights from 1024 x 1024 to
// 28672 x 8192 (E4M3, fp16 out): start-up plus waves, each a fixed part (the drain) and 256-wide blocks of K; half a wave where the pair
// kernel cuts its last one.  Used for E8M0 and fp32 results too: over 192 combinations of both formats and outputs on six weights and 1 to 2048
// tokens the choice was within 7 % of the best kernel but twice, 5.3 against 4.7 us (48 x 2260 x 1000, E8M0) and 33.0 against 30.2
// (128 x 28672 x 8192), though the model itself can be off by more (777 x 2260 x 1000 into fp32: 4.1 us, measured 5.3).
static int f4_choose(int M, int N, int K, int sms) {
    const float kb = static_cast<float>(ceil_div(K, kF4BK));
    const long long lone_tiles = static_cast<long long>(ceil_div(M, 128)) * ceil_div(N, 128);
    const long long pair_tiles = static_cast<long long>(ceil_div(M, 256)) * ceil_div(N, 256), pairs = sms / 2;
    const float lone = 2.6f + static_cast<float>((lone_tiles + sms - 1) / sms) * (0.55f + 0.23f * kb);
    float pair = 1e30f;
    if (pairs > 0) {
        const long long rest = pair_tiles % pairs;
        const float waves = static_cast<float>(pair_tiles / pairs) + (rest == 0 ? 0.f : pair_tiles > pairs && 2 * rest <= pairs ? 0.6f : 1.f);
        pair = 3.0f + waves * (2.7f + 0.28f * kb);
    }
    // Few tokens: always up to 32, beyond while the tokens' columns cost less than the wide tiles, which stream the weights at 4 TB/s.
    // Few-token kernel against 128 x 128: 4096 x 4096, 16 tokens 4.6 and 6.3 us, 64 tokens 7.4 and 6.4; 11008 x 4096, 48 tokens 8.3
    // and 10.6, 64 tokens 9.0 and 7.0; 28672 x 8192, 64 tokens 25.8 and 29.2.
    const float weight_mb = 0.5625e-6f * static_cast<float>(N) * static_cast<float>(K), stream = 2.6f + weight_mb / 4.0f;
    if (M <= 32 || (M <= kF4FewMaxTokens && 2.3f + weight_mb / 6.4f + 0.055f * M < (lone > stream ? lone : stream))) return 1;
    return pair < lone ? 3 : 2;
}

// ---- expert layer -----------------------------------------------------------------------
static MoeWorkspace moe_workspace(int T, int H, int I, int E, int top) {
    auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
    MoeWorkspace w{};
    const size_t a = static_cast<size_t>(T) * top;
    w.counter_words = E + 1;
    w.split = a <= 16 ? kMoeMaxSplit : a <= 64 ? 2 : 1;      // more assignments than that are units enough
    w.gu_pitch = 2 * moe_k_blocks(I) * kF4BK;
    w.y_pitch = ceil_div(H, 32) * 32;
    w.counters = 0;
    w.x_scale = w.counters + up(4ull * w.counter_words);
    w.ids = w.x_scale + up(4ull * T);
    w.weights = w.ids + up(4ull * a);
    w.x_values = w.weights + up(4ull * a);
    w.x_scales = w.x_values + up(static_cast<size_t>(T) * moe_value_bytes(H));
    w.gu = w.x_scales + up(static_cast<size_t>(T) * moe_scale_bytes(H, FMT_E4M3));
    w.y = w.gu + up(4ull * a * w.split * w.gu_pitch);
    w.bytes = w.y + up(4ull * a * w.split * w.y_pitch);
    return w;
}
static bool moe_in_range(int T, int H, int I, int E, int top) {
    return T > 0 && T <= kMoeMaxTokens && E > 0 && E <= kMoeMaxExperts && top > 0 && top <= kMoeMaxTop && top <= E && H > 0 && H <= kMoeMaxDim &&
           I > 0 && I <= kMoeMaxDim;
}

// expert matrices [outer][rows][K]: boxes of 128 rows, as box_outer x (128 / box_outer)
static int expert_maps(CUtensorMap* values, CUtensorMap* scales, const uint8_t* q, const uint8_t* s, int outer, int rows, int k, int fmt,
                       uint32_t box_outer) {
    const uint64_t pitch = f4_row_bytes(k), s_pitch = f4_scale_pitch(k, fmt);
    const uint64_t dims[3] = {pitch, static_cast<uint64_t>(rows), static_cast<uint64_t>(outer)};
    const uint64_t s_dims[3] = {s_pitch, static_cast<uint64_t>(rows), static_cast<uint64_t>(outer)};
    const uint32_t box[3] = {128, 128 / box_outer, box_outer}, s_box[3] = {16, 128 / box_outer, box_outer};
    if (int rc = cached_tensor_map(values, q, 3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B, true, pitch * rows))
        return rc;
    return cached_tensor_map(scales, s, 3, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, s_dims, s_pitch, s_box, CU_TENSOR_MAP_SWIZZLE_NONE, true, s_pitch * rows);
}

template <int FMT, bool BF16>
static int launch_moe(const CUtensorMap& w13, const CUtensorMap& s13, const CUtensorMap& w2, const CUtensorMap& s2, const MoeParams& p,
                      int clusters, int ctas, cudaStream_t stream) {
    auto kern = moe_experts_kernel<FMT, BF16>;
    static ConfiguredFlags flags;
    if (int rc = ensure_smem_limit(flags, kern, kMoeSmemBytes)) return rc;
    BM_CUDA_TRY(launch_pdl(moe_router_kernel<FMT, BF16>, dim3(clusters * kMoeRouterCtas), dim3(kMoeRouterThreads),
                           sizeof(double) * kMoeRouterChunks * p.experts, stream, kMoeRouterCtas, p));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = kMoeSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeCooperative;             // its CTAs wait for one another
    attr[0].val.cooperative = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = opt(OPT_PDL) != 0 ? 2 : 1;
    BM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, w13, s13, w2, s2, p));
    return BM_OK;
}

}  // namespace bm

using namespace bm;

extern "C" {

size_t bm_f4_value_bytes(int R, int K) {
    return R <= 0 || K <= 0 ? 0 : static_cast<size_t>(R) * f4_row_bytes(K);
}

size_t bm_f4_scale_bytes(int R, int K, int format, int scale_layout) {
    if (R <= 0 || K <= 0 || check_format(format, scale_layout) != BM_OK) return 0;
    return f4_scale_bytes(R, K, format, scale_layout);
}

int bm_quantize_f4(const void* X, int x_type, uint8_t* Q, uint8_t* S, float* row_scale, int R, int K, int64_t ldx, int format,
                   int scale_layout, void* stream) {
    if (!X || !Q || !S) return fail_msg(BM_ERR_NULL, "pointer is NULL");
    if (int rc = check_format(format, scale_layout)) return rc;
    if (x_type != BM_F16 && x_type != BM_BF16) return fail_msg(BM_ERR_LAYOUT, "X must be fp16 or bf16");
    if (format == BM_F4_E4M3 && !row_scale) return fail_msg(BM_ERR_NULL, "the E4M3 format needs row_scale");
    if (R <= 0 || K <= 0 || K > kF4MaxK || R > kF4MaxRows) return fail_msg(BM_ERR_SHAPE, "R and K must be positive, at most 2^31 - 256 and 2^31 - 65536");
    if (ldx < K) return fail_msg(BM_ERR_SHAPE, "row pitch is smaller than the row length");
    if (!aligned16(Q) || !aligned16(S) || !aligned_to(X, 2) || !aligned_to(row_scale, 4))
        return fail_msg(BM_ERR_ALIGN, "Q and S must be 16-byte aligned, X and row_scale to their elements");
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    F4QuantParams p{};
    p.x = static_cast<const uint16_t*>(X);
    p.ldx = ldx;
    p.q = Q;
    p.s = S;
    p.row_scale = row_scale;
    p.rows = R;
    p.k = K;
    p.k_padded = 2 * f4_row_bytes(K);
    const int share = f4_block(format) / 16;
    if (scale_layout == BM_SCALE_TILED) {
        p.tiles_k = f4_tiles_k(K, format);
        p.units = p.tiles_k * 4 * share;
        p.rows_padded = ceil_div(R, 128) * 128;
    } else {
        p.scale_pitch = f4_scale_pitch(K, format);
        p.units = p.scale_pitch * share;
        p.rows_padded = R;
    }
    p.vec_bytes = access_bytes(X, static_cast<size_t>(ldx) * 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (format == BM_F4_E8M0) return x_type == BM_BF16 ? launch_quantize<FMT_E8M0, true>(p, sms, st) : launch_quantize<FMT_E8M0, false>(p, sms, st);
    return x_type == BM_BF16 ? launch_quantize<FMT_E4M3, true>(p, sms, st) : launch_quantize<FMT_E4M3, false>(p, sms, st);
}

int bm_dequantize_f4(const uint8_t* Q, const uint8_t* S, const float* row_scale, void* out, int out_type, int R, int K, int64_t ldo,
                     int format, int scale_layout, void* stream) {
    if (!Q || !S || !out) return fail_msg(BM_ERR_NULL, "pointer is NULL");
    if (int rc = check_format(format, scale_layout)) return rc;
    if (out_type != BM_F16 && out_type != BM_BF16 && out_type != BM_F32) return fail_msg(BM_ERR_LAYOUT, "unknown element type tag");
    if (R <= 0 || K <= 0 || K > kF4MaxK || R > kF4MaxRows) return fail_msg(BM_ERR_SHAPE, "R and K must be positive, at most 2^31 - 256 and 2^31 - 65536");
    if (ldo < K) return fail_msg(BM_ERR_SHAPE, "row pitch is smaller than the row length");
    const size_t elem = out_type == BM_F32 ? 4 : 2;
    if (!aligned16(Q) || !aligned16(S) || !aligned_to(out, elem) || !aligned_to(row_scale, 4))
        return fail_msg(BM_ERR_ALIGN, "Q and S must be 16-byte aligned, the output and row_scale to their elements");
    F4DequantParams p{};
    p.q = Q;
    p.s = S;
    p.row_scale = row_scale;
    p.out = out;
    p.ldo = ldo;
    p.rows = R;
    p.k = K;
    p.k_padded = 2 * f4_row_bytes(K);
    if (scale_layout == BM_SCALE_TILED) p.tiles_k = f4_tiles_k(K, format);
    else p.scale_pitch = f4_scale_pitch(K, format);
    p.vec_bytes = access_bytes(out, static_cast<size_t>(ldo) * elem);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return format == BM_F4_E8M0 ? launch_dequantize<FMT_E8M0>(p, out_type, st) : launch_dequantize<FMT_E4M3>(p, out_type, st);
}

int bm_f4_gemm(const uint8_t* A, const uint8_t* SA, const float* ra, const uint8_t* W, const uint8_t* SW, const float* rw, void* D,
               int d_type, int M, int N, int K, int64_t ldd, int format, void* stream) {
    if (!A || !SA || !W || !SW || !D) return fail_msg(BM_ERR_NULL, "pointer is NULL");
    if (int rc = check_format(format, BM_SCALE_TILED)) return rc;
    if (d_type != BM_F16 && d_type != BM_BF16 && d_type != BM_F32) return fail_msg(BM_ERR_LAYOUT, "unknown element type tag");
    if (M <= 0 || N <= 0 || K <= 0 || K > kF4MaxK || M > kF4MaxRows || N > kF4MaxRows)
        return fail_msg(BM_ERR_SHAPE, "M, N, K must be positive, at most 2^31 - 256 (K: 2^31 - 65536)");
    if (ldd < N) return fail_msg(BM_ERR_SHAPE, "output pitch is smaller than the row length");
    if (!aligned16(A) || !aligned16(SA) || !aligned16(W) || !aligned16(SW)) return fail_msg(BM_ERR_ALIGN, "operands and scales must be 16-byte aligned");
    if (!aligned_to(D, d_type == BM_F32 ? 4 : 2) || !aligned_to(ra, 4) || !aligned_to(rw, 4))
        return fail_msg(BM_ERR_ALIGN, "output and factors must be aligned to their elements");
    DeviceState* dev = nullptr;
    if (int rc = current_device_state(&dev)) return rc;
    F4Operands o{A, SA, W, SW, format, d_type, M, N, K};
    F4GemmParams p{};
    p.out = D;
    p.ld = ldd;
    p.rows = M;
    p.cols = N;
    p.row_scale = ra;
    p.col_scale = rw;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int kernel = opt(OPT_F4_KERNEL);
    if (kernel == 1 && M > kF4FewMaxTokens) kernel = 0;
    if (kernel == 0) kernel = f4_choose(M, N, K, dev->sm_count);
    if (kernel == 1) return f4_few(o, p, dev, st);
    return kernel == 3 && dev->sm_count >= 2 ? launch_f4<true>(o, p, dev, st) : launch_f4<false>(o, p, dev, st);
}

size_t bm_moe_f4_workspace_bytes(int T, int H, int I, int E, int top) {
    return moe_in_range(T, H, I, E, top) ? moe_workspace(T, H, I, E, top).bytes : 0;
}

int bm_moe_f4(const void* X, const void* router, int x_type, const uint8_t* W13, const uint8_t* S13, const float* r13, const uint8_t* W2,
              const uint8_t* S2, const float* r2, void* Y, int32_t* ids, float* weights, int T, int H, int I, int E, int top, int64_t ldx,
              int64_t ldy, int format, int normalize, void* workspace, size_t workspace_bytes, void* stream) {
    if (!X || !router || !W13 || !S13 || !W2 || !S2 || !Y || !workspace) return fail_msg(BM_ERR_NULL, "pointer is NULL");
    if (int rc = check_format(format, BM_SCALE_ROWS)) return rc;
    if (x_type != BM_F16 && x_type != BM_BF16) return fail_msg(BM_ERR_LAYOUT, "activations must be fp16 or bf16");
    if (T <= 0 || H <= 0 || I <= 0 || E <= 0 || top <= 0 || top > E) return fail_msg(BM_ERR_SHAPE, "T, H, I, E must be positive, 1 <= top <= E");
    if (!moe_in_range(T, H, I, E, top)) return fail_msg(BM_ERR_TOO_LARGE, "at most 64 tokens, 256 experts, top 16, H and I 16384");
    if (ldx < H || ldy < H) return fail_msg(BM_ERR_SHAPE, "row pitch is smaller than the row length");
    if (!aligned16(W13) || !aligned16(S13) || !aligned16(W2) || !aligned16(S2) || !aligned_to(workspace, 256))
        return fail_msg(BM_ERR_ALIGN, "weights and scales must be 16-byte aligned, the workspace 256-byte aligned");
    if (!aligned_to(X, 2) || !aligned_to(router, 2) || !aligned_to(Y, 2) || !aligned_to(r13, 4) || !aligned_to(r2, 4) || !aligned_to(ids, 4) ||
        !aligned_to(weights, 4))
        return fail_msg(BM_ERR_ALIGN, "activations, factors and outputs must be aligned to their elements");
    const MoeWorkspace w = moe_workspace(T, H, I, E, top);
    if (workspace_bytes < w.bytes) return fail_msg(BM_ERR_TOO_LARGE, "workspace is smaller than bm_moe_f4_workspace_bytes()");
    DeviceState* dev = nullptr;
    if (int rc = current_device_state(&dev)) return rc;
    // parts of phases that one CTA can get: whole experts in its share, and all passes of the first and the last
    const int most_passes = ceil_div(T, moe_pass_tokens(H > I ? H : I));
    if (T * top / dev->sm_count + 1 + 2 * most_passes > kMoeMaxRuns) return fail_msg(BM_ERR_TOO_LARGE, "too few SMs for this many tokens and experts");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    MoeParams p{};
    p.x = static_cast<const uint16_t*>(X);
    p.router = static_cast<const uint16_t*>(router);
    p.ldx = ldx;
    p.ldy = ldy;
    p.y = static_cast<uint16_t*>(Y);
    p.ids_out = ids;
    p.weights_out = weights;
    p.r13 = r13;
    p.r2 = r2;
    p.tokens = T;
    p.hidden = H;
    p.inter = I;
    p.experts = E;
    p.top = top;
    p.normalize = normalize != 0;
    p.x_vec_ok = aligned16(X) && ldx % 8 == 0;
    p.router_vec_ok = aligned16(router) && H % 8 == 0;
    p.counters = reinterpret_cast<unsigned*>(ws + w.counters);
    p.counter_words = w.counter_words;
    p.x_scale = reinterpret_cast<float*>(ws + w.x_scale);
    p.ids = reinterpret_cast<int*>(ws + w.ids);
    p.weights = reinterpret_cast<float*>(ws + w.weights);
    p.x_values = ws + w.x_values;
    p.x_scales = ws + w.x_scales;
    p.gu = reinterpret_cast<float*>(ws + w.gu);
    p.yp = reinterpret_cast<float*>(ws + w.y);
    p.gu_pitch = w.gu_pitch;
    p.split = w.split;
    p.y_pitch = w.y_pitch;
    p.status = dev->status;
    const int clusters = 2 * ceil_div(T, kMoeRouterTokens);  // at most 128 CTAs
    CUtensorMap mw13, ms13, mw2, ms2;
    if (int rc = expert_maps(&mw13, &ms13, W13, S13, 2 * E, I, H, format, 2)) return rc;
    if (int rc = expert_maps(&mw2, &ms2, W2, S2, E, H, I, format, 1)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = x_type == BM_BF16;
    if (format == BM_F4_E8M0)
        return bf16 ? launch_moe<FMT_E8M0, true>(mw13, ms13, mw2, ms2, p, clusters, dev->sm_count, st)
                    : launch_moe<FMT_E8M0, false>(mw13, ms13, mw2, ms2, p, clusters, dev->sm_count, st);
    return bf16 ? launch_moe<FMT_E4M3, true>(mw13, ms13, mw2, ms2, p, clusters, dev->sm_count, st)
                : launch_moe<FMT_E4M3, false>(mw13, ms13, mw2, ms2, p, clusters, dev->sm_count, st);
}

}  // extern "C"

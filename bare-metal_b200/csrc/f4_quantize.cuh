// f4_quantize.cuh — rows of fp16 / bf16 to the 4-bit formats of f4_format.cuh, and back.
//
// With amax the largest |x| of a block and top that of the row (infinities and NaNs left out):
//   FMT_E8M0   s = 2^(floor(log2 amax) - 2), the rule of the OCP Microscaling specification; v = x / s
//   FMT_E4M3   t = 2^(floor(log2 top) - 10), the row's factor (1 for a row of zeros); s = E4M3(amax / (6 t)); v = x / (t s)
// and the stored code is v rounded to the nearest E2M1 number, ties to even, saturating at 6.  A power of two as the row's
// factor puts the largest block scale in [171, 342) of E4M3's 448 and costs no rounding.  A block that holds
// an infinity or a NaN gets the scale NaN and the values 0, so it shows in every product.
//
// Everything is exactly determined: x * 2^n is exact, x has at most 11 bits and s at most 4, so x / s is either a tie
// (a multiple of 1/4) or off every tie by more than 2^-13.  x * (1 / s) in fp32 is within 2^-21 of x / s; adding and
// subtracting 768 rounds it to a multiple of 2^-14, which puts ties back on the tie and moves nothing across one.
//
// 2 bytes in and 1/2 + 1/16 (1/32) out per element.  A group of threads per row holds it in registers (16-byte pieces
// of 8 numbers; two or four neighbouring threads share a block), so the row's maximum costs no second read.
#pragma once
#include "f4_format.cuh"

namespace bm {

constexpr int kF4QuantMaxThreads = 1024;

struct F4QuantParams {
    const uint16_t* x;
    long long ldx;               // elements between rows
    uint8_t* q;
    uint8_t* s;
    float* row_scale;            // FMT_E4M3
    int rows, rows_padded;       // rows of X; rows whose scales exist (whole tiles)
    int k, k_padded;             // row length; the same in whole 32s
    int pieces;                  // pieces of 8 numbers that the stored scales of a row cover
    int tiles_k;                 // tiled scales: tiles along a row; 0: scales in rows
    int scale_pitch;             // scales in rows: bytes of a row
    int vec_ok;                  // X allows 16-byte loads
};

template <bool BF16>
__device__ __forceinline__ uint4 f4_load_piece(const F4QuantParams& p, const uint16_t* row, int v) {
    const int k0 = v * 8;
    if (p.vec_ok && k0 + 8 <= p.k) return __ldg(reinterpret_cast<const uint4*>(row + k0));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k0 + j < p.k) w[j >> 1] |= static_cast<uint32_t>(__ldg(row + k0 + j)) << (16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Largest |x| of a piece as 16-bit patterns (they order like integers), numbers only; `odd`: something else was there.
template <bool BF16>
__device__ __forceinline__ uint32_t f4_piece_max(const uint4& d, bool& odd) {
    constexpr uint32_t kInf = BF16 ? 0x7F80u : 0x7C00u;
    uint32_t m = __vmaxu2(__vmaxu2(d.x & 0x7FFF7FFFu, d.y & 0x7FFF7FFFu), __vmaxu2(d.z & 0x7FFF7FFFu, d.w & 0x7FFF7FFFu));
    uint32_t one = max(m & 0xFFFFu, m >> 16);
    odd = one >= kInf;
    if (odd) {
        const uint32_t w[4] = {d.x, d.y, d.z, d.w};
        one = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = (w[j >> 1] >> (16 * (j & 1))) & 0x7FFFu;
            if (b < kInf) one = max(one, b);
        }
    }
    return one;
}
template <bool BF16>
__device__ __forceinline__ float f4_bits_value(uint32_t bits) {
    return BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// One piece: its block's scale (shared with the neighbouring threads of the block), codes and stores.
template <int FMT, bool BF16>
__device__ __forceinline__ void f4_emit(const F4QuantParams& p, const uint4& d, int row, int v, float inv_row) {
    bool odd;
    const uint32_t mine = f4_piece_max<BF16>(d, odd);
    constexpr int SHARE = f4_block(FMT) / 8;                            // threads of a block: 2 or 4
    uint32_t bits = mine | (odd ? 0x10000u : 0u);
#pragma unroll
    for (int o = 1; o < SHARE; o <<= 1) {
        const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, bits, o);
        bits = max(bits & 0xFFFFu, other & 0xFFFFu) | ((bits | other) & 0x10000u);
    }
    odd = bits > 0xFFFFu;
    const float amax = f4_bits_value<BF16>(bits & 0xFFFFu);
    uint32_t byte;
    float f[8];
    {
        const float2 a = pair_to_float<BF16>(d.x), b = pair_to_float<BF16>(d.y), c = pair_to_float<BF16>(d.z), e = pair_to_float<BF16>(d.w);
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = e.x; f[7] = e.y;
    }
    if constexpr (FMT == FMT_E8M0) {
        const int lg = static_cast<int>(__float_as_uint(amax) >> 23);   // floor(log2 amax) + 127; 0 below 2^-126
        byte = lg > 2 ? lg - 2 : 0;
        const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], inv);
        if (odd) byte = 255;
    } else {
        byte = __nv_cvt_float_to_fp8(__fdiv_rn(__fmul_rn(amax, inv_row), 6.0f), __NV_SATFINITE, __NV_E4M3);
        const float s = e4m3_value(byte);
        const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __fsub_rn(__fadd_rn(__fmul_rn(__fmul_rn(f[j], inv_row), inv), 768.f), 768.f);
        if (odd) byte = 127;
    }
    if (row < p.rows && v * 8 < p.k_padded) {
        // the sign of a zero that was a negative number is kept, as the conversion does: it is the product's sign of zero
        uint32_t codes = e2m1x8(f);
        if constexpr (FMT == FMT_E4M3) {                                // 768 - 768 has lost it
            const uint32_t w[4] = {d.x, d.y, d.z, d.w};
            uint32_t neg = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) neg |= ((w[j >> 1] >> (16 * (j & 1) + 15)) & 1u) << (4 * j + 3);
            codes |= neg;
        }
        if (odd) codes = 0;
        *reinterpret_cast<uint32_t*>(p.q + static_cast<size_t>(row) * (p.k_padded / 2) + v * 4) = codes;
    }
    // four scales to a word: lanes of 4 consecutive blocks
    const int g = v / SHARE;
    uint32_t word = byte << (8 * (g & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, SHARE);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * SHARE);
    if (v < p.pieces && (v & (4 * SHARE - 1)) == 0) {
        const size_t at = p.tiles_k ? (static_cast<size_t>(row >> 7) * p.tiles_k + (g >> 2)) * kF4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4
                                    : static_cast<size_t>(row) * p.scale_pitch + g;
        *reinterpret_cast<uint32_t*>(p.s + at) = word;
    }
}

// A group of blockDim.x threads (whole warps) per row, blockDim.y rows a CTA; a thread holds up to HELD pieces.
template <int FMT, bool BF16, int HELD>
__global__ void __launch_bounds__(HELD == 4 ? 512 : kF4QuantMaxThreads)
quantize_f4_kernel(const F4QuantParams p) {
    __shared__ uint32_t warp_bits[kF4QuantMaxThreads / 32];
    const int row = blockIdx.x * blockDim.y + threadIdx.y;
    const int tid = threadIdx.x, group = blockDim.x;
    pdl_launch_dependents();      // the GEMM behind this kernel may start its own set-up
    if (row >= p.rows_padded) return;              // whole warps: a CTA of several rows has one-warp groups
    const uint16_t* src = p.x + static_cast<long long>(row) * p.ldx;
    const int mine = row < p.rows ? p.pieces : 0;  // rows beyond X: their scales are zeros
    uint4 held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int v = tid + i * group;
        held[i] = v < mine ? f4_load_piece<BF16>(p, src, v) : make_uint4(0, 0, 0, 0);
    }
    float inv_row = 1.f;
    if constexpr (FMT == FMT_E4M3) {
        uint32_t bits = 0;
        bool odd;
#pragma unroll
        for (int i = 0; i < HELD; ++i) bits = max(bits, f4_piece_max<BF16>(held[i], odd));
        for (int v = tid + HELD * group; v < mine; v += group) bits = max(bits, f4_piece_max<BF16>(f4_load_piece<BF16>(p, src, v), odd));
        bits = __reduce_max_sync(0xFFFFFFFFu, bits);
        if (group > 32) {
            if ((tid & 31) == 0) warp_bits[tid >> 5] = bits;
            __syncthreads();
            for (int w = 0; w < group / 32; ++w) bits = max(bits, warp_bits[w]);
        }
        const float top = f4_bits_value<BF16>(bits);
        const int lg = static_cast<int>(__float_as_uint(top) >> 23);    // floor(log2 top) + 127
        const int e = top == 0.f ? 127 : lg > 11 ? lg - 10 : 1;         // the row's factor is 2^(e - 127)
        inv_row = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        if (tid == 0 && row < p.rows) p.row_scale[row] = __uint_as_float(static_cast<uint32_t>(e) << 23);
    }
    // whole warps go through every step together: neighbouring threads exchange their blocks' maxima
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int v = tid + i * group;
        if (v - (tid & 31) < p.pieces) f4_emit<FMT, BF16>(p, held[i], row, v, inv_row);
    }
    for (int v = tid + HELD * group; v - (tid & 31) < p.pieces; v += group)
        f4_emit<FMT, BF16>(p, v < mine ? f4_load_piece<BF16>(p, src, v) : make_uint4(0, 0, 0, 0), row, v, inv_row);   // second read hits L2
}

struct F4DequantParams {
    const uint8_t* q;
    const uint8_t* s;
    const float* row_scale;      // or NULL
    void* out;
    long long ldo;
    int rows, k, k_padded;
    int tiles_k, scale_pitch;
    int vec_ok;                  // the output allows 16-byte stores
};

// out = value * scale * row factor, rounded once.  A thread per 8 numbers: 4 bytes of codes, its block's scale, 16 or 32 bytes out.
template <int FMT, int TYPE>
__global__ void __launch_bounds__(256)
dequantize_f4_kernel(const F4DequantParams p) {
    const int per_row = (p.k + 7) / 8;
    const long long total = static_cast<long long>(p.rows) * per_row;
    for (long long at = blockIdx.x * 256ll + threadIdx.x; at < total; at += gridDim.x * 256ll) {
        const int row = static_cast<int>(at / per_row), v = static_cast<int>(at - static_cast<long long>(row) * per_row);
        const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>(p.q + static_cast<size_t>(row) * (p.k_padded / 2) + v * 4));
        const int g = v * 8 / f4_block(FMT);
        const size_t sat = p.tiles_k ? (static_cast<size_t>(row >> 7) * p.tiles_k + (g >> 2)) * kF4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (g & 3)
                                     : static_cast<size_t>(row) * p.scale_pitch + g;
        const float s = f4_scale_value<FMT>(__ldg(p.s + sat));
        const float t = p.row_scale ? __ldg(p.row_scale + row) : 1.f;
        uint32_t h[4];
        e2m1x8_to_half(codes, h);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 a = pair_to_float<false>(h[j]);
            f[2 * j] = __fmul_rn(__fmul_rn(a.x, s), t);
            f[2 * j + 1] = __fmul_rn(__fmul_rn(a.y, s), t);
        }
        const int k0 = v * 8;
        if constexpr (TYPE == TYPE_F32) {
            float* dst = static_cast<float*>(p.out) + static_cast<long long>(row) * p.ldo + k0;
            if (p.vec_ok && k0 + 8 <= p.k) {
                reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
                reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + j < p.k) dst[j] = f[j];
            }
        } else {
            constexpr bool BF16 = TYPE == TYPE_BF16;
            uint16_t* dst = static_cast<uint16_t*>(p.out) + static_cast<long long>(row) * p.ldo + k0;
            const uint32_t w[4] = {float_to_pair<BF16>(f[0], f[1]), float_to_pair<BF16>(f[2], f[3]), float_to_pair<BF16>(f[4], f[5]),
                                   float_to_pair<BF16>(f[6], f[7])};
            if (p.vec_ok && k0 + 8 <= p.k) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + j < p.k) dst[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
            }
        }
    }
}

}  // namespace bm

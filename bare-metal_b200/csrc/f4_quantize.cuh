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
// (a multiple of 1/4) or off every tie by more than 2^-13.  x * (1 / s) in fp32 is within 2^-20 of x / s; adding and
// subtracting 768 rounds it to a multiple of 2^-14, which puts ties back on the tie and moves nothing across one.
//
// 2 bytes in and 1/2 + 1/16 (1/32) out per element.  A group of threads per row holds it in registers, units of 16 numbers (a block,
// or half of one), so the row's maximum costs no second read.  What bounds it with many rows is instructions as much as bytes: an
// element gets one conversion, one FMA and one subtraction before the packing conversion, a unit its maximum once and its
// scale once (8 numbers a thread and two threads a block took 171 instructions per 8, this 103).  8192 x 11008 bf16 to E4M3 45.1 us, 5.1 TB/s;
// 8192 x 4096 to E8M0 15.8 us, 5.4 TB/s; 4096 x 4096 fp16 to E4M3 10.4 us.  Issue slots are 67 % busy, the rest waits for loads.
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
    int units;                   // units of 16 numbers that the stored scales of a row cover
    int tiles_k;                 // tiled scales: tiles along a row; 0: scales in rows
    int scale_pitch;             // scales in rows: bytes of a row
    int vec_bytes;               // X allows loads of 16, 8, 4 or 2 bytes
};

struct F4Unit { uint32_t w[8]; };

// unit v of a row, zeros beyond its end
__device__ __forceinline__ F4Unit f4_load_unit(const F4QuantParams& p, const uint16_t* row, int v) {
    F4Unit u;
    const int k0 = v * 16;
    const uint16_t* at = row + k0;
    if (p.vec_bytes == 16 && k0 + 16 <= p.k) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(at)), b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
        u.w[0] = a.x; u.w[1] = a.y; u.w[2] = a.z; u.w[3] = a.w; u.w[4] = b.x; u.w[5] = b.y; u.w[6] = b.z; u.w[7] = b.w;
    } else if (p.vec_bytes >= 4 && k0 + 16 <= p.k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u.w[j] = __ldg(reinterpret_cast<const uint32_t*>(at) + j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            u.w[j] = k0 + 2 * j < p.k ? __ldg(at + 2 * j) : 0u;
            if (k0 + 2 * j + 1 < p.k) u.w[j] |= static_cast<uint32_t>(__ldg(at + 2 * j + 1)) << 16;
        }
    }
    return u;
}

// Largest |x| of a unit as a 16-bit pattern (they order like integers), numbers only; bit 16: something else was there.
template <bool BF16>
__device__ __forceinline__ uint32_t f4_unit_max(const F4Unit& u) {
    constexpr uint32_t kInf = BF16 ? 0x7F80u : 0x7C00u;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = __vmaxu2(m, u.w[j] & 0x7FFF7FFFu);
    uint32_t one = max(m & 0xFFFFu, m >> 16);
    if (one >= kInf) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t lo = u.w[j] & 0x7FFFu, hi = (u.w[j] >> 16) & 0x7FFFu;
            if (lo < kInf) most = max(most, lo);
            if (hi < kInf) most = max(most, hi);
        }
        one = most | 0x10000u;
    }
    return one;
}
template <bool BF16>
__device__ __forceinline__ float f4_bits_value(uint32_t bits) {
    return BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// What a row's pieces share.
struct F4RowOut {
    uint8_t* q;                  // the row's values, NULL beyond X
    uint8_t* s;                  // byte 0 of the row's scales
    int s_step;                  // bytes from one word of four scales to the next
    float inv_row;               // FMT_E4M3: 1 / row factor ...
    float pre;                   // ... times this: the row's numbers are multiplied by it first (bf16 rows far below 1)
};

// One unit: its block's scale (FMT_E8M0: shared with the neighbouring thread), codes and stores.
template <int FMT, bool BF16>
__device__ __forceinline__ void f4_emit(const F4QuantParams& p, const F4RowOut& out, const F4Unit& u, uint32_t bits, int v) {
    constexpr int SHARE = f4_block(FMT) / 16;                           // threads of a block: 1 or 2
    if constexpr (SHARE == 2) {
        const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, bits, 1);
        bits = max(bits & 0xFFFFu, other & 0xFFFFu) | ((bits | other) & 0x10000u);
    }
    const bool odd = bits > 0xFFFFu;
    const float amax = f4_bits_value<BF16>(bits & 0xFFFFu);
    uint32_t byte;
    float f[16];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 two = pair_to_float<BF16>(u.w[j]);
        f[2 * j] = two.x;
        f[2 * j + 1] = two.y;
    }
    if constexpr (FMT == FMT_E8M0) {
        const int lg = static_cast<int>(__float_as_uint(amax) >> 23);   // floor(log2 amax) + 127; 0 below 2^-126
        byte = lg > 2 ? lg - 2 : 0;
        const float inv = __uint_as_float((254u - byte) << 23);
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = __fmul_rn(f[j], inv);
        if (odd) byte = 255;
    } else {
        float a = amax;
        if (BF16 && out.pre != 1.f) {                                   // the same for the whole row
            a *= out.pre;
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] *= out.pre;
        }
        // a / 6 rounded to the nearest: the quotient by multiplication, corrected by what it leaves
        const float t = __fmul_rn(a, out.inv_row), guess = __fmul_rn(t, 1.f / 6.f);
        byte = __nv_cvt_float_to_fp8(__fmaf_rn(__fmaf_rn(-6.f, guess, t), 1.f / 6.f, guess), __NV_SATFINITE, __NV_E4M3);
        const float s = e4m3_value(byte);
        float inv;                                                      // off by 2^-23 at most; __fdividef takes 2 % more of the kernel's time
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        inv = byte != 0 ? __fmul_rn(inv, out.inv_row) : 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = __fsub_rn(__fmaf_rn(f[j], inv, 768.f), 768.f);
        if (odd) byte = 127;
    }
    const float lo[8] = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]}, hi[8] = {f[8], f[9], f[10], f[11], f[12], f[13], f[14], f[15]};
    const uint2 codes = odd ? make_uint2(0, 0) : make_uint2(e2m1x8(lo), e2m1x8(hi));
    if (out.q != nullptr && v * 16 < p.k_padded) *reinterpret_cast<uint2*>(out.q + v * 8) = codes;
    // four scales to a word: lanes of 4 consecutive blocks
    const int g = v / SHARE;
    uint32_t word = byte << (8 * (g & 3));
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, SHARE);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * SHARE);
    if (v < p.units && (v & (4 * SHARE - 1)) == 0) *reinterpret_cast<uint32_t*>(out.s + static_cast<size_t>(g >> 2) * out.s_step) = word;
}

// A group of blockDim.x threads (whole warps) per row, blockDim.y rows a CTA; a thread holds up to HELD units.
template <int FMT, bool BF16, int HELD>
__global__ void __launch_bounds__(HELD == 4 ? 512 : kF4QuantMaxThreads)
quantize_f4_kernel(const F4QuantParams p) {
    __shared__ uint32_t warp_bits[kF4QuantMaxThreads / 32];
    const int row = blockIdx.x * blockDim.y + threadIdx.y;
    const int tid = threadIdx.x, group = blockDim.x;
    pdl_launch_dependents();      // the GEMM behind this kernel may start its own set-up
    if (row >= p.rows_padded) return;              // whole warps: a CTA of several rows has one-warp groups
    const uint16_t* src = p.x + static_cast<long long>(row) * p.ldx;
    const int mine = row < p.rows ? p.units : 0;   // rows beyond X: their scales are zeros
    F4Unit held[HELD];
    uint32_t most[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int v = tid + i * group;
        held[i] = v < mine ? f4_load_unit(p, src, v) : F4Unit{};
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) most[i] = f4_unit_max<BF16>(held[i]);
    F4RowOut out;
    out.q = row < p.rows ? p.q + static_cast<size_t>(row) * (p.k_padded / 2) : nullptr;
    out.s = p.tiles_k ? p.s + static_cast<size_t>(row >> 7) * p.tiles_k * kF4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4
                      : p.s + static_cast<size_t>(row) * p.scale_pitch;
    out.s_step = p.tiles_k ? kF4TileBytes : 4;
    out.inv_row = out.pre = 1.f;
    if constexpr (FMT == FMT_E4M3) {
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) bits = max(bits, most[i] & 0xFFFFu);
        for (int v = tid + HELD * group; v < mine; v += group) bits = max(bits, f4_unit_max<BF16>(f4_load_unit(p, src, v)) & 0xFFFFu);
        bits = __reduce_max_sync(0xFFFFFFFFu, bits);
        if (group > 32) {
            if ((tid & 31) == 0) warp_bits[tid >> 5] = bits;
            __syncthreads();
            for (int w = 0; w < group / 32; ++w) bits = max(bits, warp_bits[w]);
        }
        const float top = f4_bits_value<BF16>(bits);
        const int lg = static_cast<int>(__float_as_uint(top) >> 23);    // floor(log2 top) + 127
        int e = top == 0.f ? 127 : lg > 11 ? lg - 10 : 1;               // the row's factor is 2^(e - 127)
        if (tid == 0 && row < p.rows) p.row_scale[row] = __uint_as_float(static_cast<uint32_t>(e) << 23);
        if (BF16 && e < 64) {                                           // 1 / factor times 1 / scale would leave fp32's range
            out.pre = 0x1p64f;
            e += 64;
        }
        out.inv_row = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
    }
    // whole warps go through every step together: neighbouring threads exchange their blocks' maxima
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int v = tid + i * group;
        if (v - (tid & 31) < p.units) f4_emit<FMT, BF16>(p, out, held[i], most[i], v);
    }
    for (int v = tid + HELD * group; v - (tid & 31) < p.units; v += group) {
        const F4Unit u = v < mine ? f4_load_unit(p, src, v) : F4Unit{};                                    // second read hits L2
        f4_emit<FMT, BF16>(p, out, u, f4_unit_max<BF16>(u), v);
    }
}

struct F4DequantParams {
    const uint8_t* q;
    const uint8_t* s;
    const float* row_scale;      // or NULL
    void* out;
    long long ldo;
    int rows, k, k_padded;
    int tiles_k, scale_pitch;
    int vec_bytes;               // the output allows stores of 16, 8, 4 or 2 bytes
};

// out = value * scale * row factor in fp32, then rounded (once, if the factor is a power of two).  A thread per 8 columns and every fourth row of its CTA's: 4 bytes of codes, its block's scale,
// 16 or 32 bytes out, four rows' loads in flight.  grid: (columns, rows)
constexpr int kF4DequantRows = 4;
template <int FMT, int TYPE>
__global__ void __launch_bounds__(256)
dequantize_f4_kernel(const F4DequantParams p) {
    const int v = blockIdx.x * blockDim.x + threadIdx.x, k0 = v * 8;
    if (k0 >= p.k) return;
    const int g = k0 / f4_block(FMT);
    const unsigned rows = p.rows;                                        // (a step behind the last row may pass 2^31)
    for (unsigned row0 = (blockIdx.y * blockDim.y + threadIdx.y) * kF4DequantRows; row0 < rows; row0 += gridDim.y * blockDim.y * kF4DequantRows) {
        uint32_t codes[kF4DequantRows], byte[kF4DequantRows];
        float t[kF4DequantRows];
#pragma unroll
        for (int i = 0; i < kF4DequantRows; ++i) {
            const unsigned row = min(row0 + i, rows - 1);
            codes[i] = __ldg(reinterpret_cast<const uint32_t*>(p.q + static_cast<size_t>(row) * (p.k_padded / 2) + v * 4));
            byte[i] = __ldg(p.s + (p.tiles_k ? (static_cast<size_t>(row >> 7) * p.tiles_k + (g >> 2)) * kF4TileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (g & 3)
                                             : static_cast<size_t>(row) * p.scale_pitch + g));
            t[i] = p.row_scale ? __ldg(p.row_scale + row) : 1.f;
        }
#pragma unroll
        for (int i = 0; i < kF4DequantRows; ++i) {
            const unsigned row = row0 + i;
            if (row >= rows) break;
            const float s = f4_scale_value<FMT>(byte[i]);
            uint32_t h[4];
            e2m1x8_to_half(codes[i], h);
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 a = pair_to_float<false>(h[j]);
                f[2 * j] = __fmul_rn(__fmul_rn(a.x, s), t[i]);
                f[2 * j + 1] = __fmul_rn(__fmul_rn(a.y, s), t[i]);
            }
            constexpr int WORDS = TYPE == TYPE_F32 ? 8 : 4;
            uint32_t w[WORDS];
            if constexpr (TYPE == TYPE_F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(f[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = float_to_pair<TYPE == TYPE_BF16>(f[2 * j], f[2 * j + 1]);
            }
            constexpr int ELEM = TYPE == TYPE_F32 ? 4 : 2;
            uint8_t* dst = static_cast<uint8_t*>(p.out) + (static_cast<long long>(row) * p.ldo + k0) * ELEM;
            if (k0 + 8 <= p.k && p.vec_bytes == 16) {
#pragma unroll
                for (int j = 0; j < WORDS; j += 4) reinterpret_cast<uint4*>(dst)[j / 4] = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
            } else if (k0 + 8 <= p.k && p.vec_bytes == 8) {
#pragma unroll
                for (int j = 0; j < WORDS; j += 2) reinterpret_cast<uint2*>(dst)[j / 2] = make_uint2(w[j], w[j + 1]);
            } else if (k0 + 8 <= p.k && p.vec_bytes == 4) {
#pragma unroll
                for (int j = 0; j < WORDS; ++j) reinterpret_cast<uint32_t*>(dst)[j] = w[j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (k0 + j >= p.k) break;
                    if constexpr (TYPE == TYPE_F32) reinterpret_cast<uint32_t*>(dst)[j] = w[j];
                    else reinterpret_cast<uint16_t*>(dst)[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
    }
}

}  // namespace bm

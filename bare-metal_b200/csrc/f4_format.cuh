// f4_format.cuh — the 4-bit floating-point formats: E2M1 values in blocks along a row, one 8-bit scale per block.
//
//   FMT_E8M0  blocks of 32, scale 2^(byte - 127), byte 255 = NaN (OCP Microscaling formats, MXFP4)
//   FMT_E4M3  blocks of 16, the scale an E4M3 number, and one fp32 factor per row
//
// Values are packed two to a byte, the lower position in the low four bits, rows padded with zeros to whole 32s
// (a row is a multiple of 16 bytes, as TMA wants its pitch).  Scales lie in rows (a row padded with zeros to a multiple
// of 16 bytes) or in tiles of 128 rows x 4 blocks, the order in which the tensor core takes them:
//     byte (r, g) at ((r / 128) * tiles_k + g / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + g % 4.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "sm100_ptx.cuh"

namespace bm {

enum : int { FMT_E8M0 = 0, FMT_E4M3 = 1 };
enum : int { TYPE_F16 = 0, TYPE_BF16 = 1, TYPE_F32 = 2 };
__host__ __device__ constexpr int f4_block(int fmt) { return fmt == FMT_E8M0 ? 32 : 16; }

constexpr int kF4TileBytes = 512;                 // scales of 128 rows x 4 blocks

// the number an E8M0 byte stands for
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
}
template <int FMT>
__device__ __forceinline__ float f4_scale_value(uint32_t byte) {
    return FMT == FMT_E8M0 ? e8m0_value(byte) : e4m3_value(byte);
}

// eight fp32 numbers -> eight E2M1 codes, rounded to nearest even, saturating at 6
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// eight E2M1 codes -> four pairs of fp16 numbers, exact
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
        "}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

// two 16-bit numbers of one word as fp32
template <bool BF16>
__device__ __forceinline__ float2 pair_to_float(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <bool BF16>
__device__ __forceinline__ uint32_t float_to_pair(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

}  // namespace bm

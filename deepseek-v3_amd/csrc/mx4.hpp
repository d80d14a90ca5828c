// Microscaled 4-bit numbers: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives; bit 3 is the sign), the even one of a byte in its low
// half, and for 32 of them one power of two as an e8m0 byte, 2^(byte - 127), 255 for NaN.
#pragma once
#include "common.hpp"

namespace dsv3 {
namespace {

constexpr uint32_t kMx4Nan = 255u;
constexpr uint32_t kMx4RowSpan = 14u;                   // of a cache row: no scale lies more powers of two below the row's largest

// The smallest power of two of which no element is more than six times, from the bits of the largest |element|: largest = f 2^e with f in [1, 2)
// is at most 6 2^(e - 2) where f <= 3/2, and 6 2^(e - 1) elsewhere.  Subnormal largest elements are below 6 2^-127.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t largest) {
    if (!block_is_finite(largest)) return kMx4Nan;
    const int e = (int)(largest >> 23) - 2 + ((largest & 0x7fffffu) > 0x400000u ? 1 : 0);
    return (uint32_t)(e < 0 ? 0 : e);
}
// What elements of a block are multiplied with in front of their rounding: exact, but for products far below the smallest code (byte: up to 253).
__device__ __forceinline__ float mx4_factor(uint32_t byte) { return u32_as_f32((254u - byte) << 23); }
// 2^(byte - 127)
__device__ __forceinline__ float mx4_power(uint32_t byte) { return u32_as_f32(byte == 0u ? 0x400000u : byte == kMx4Nan ? 0x7fc00000u : byte << 23); }

// Eight binary32 -> eight codes, round to nearest even, larger ones to 6 (v_cvt_scalef32_pk_fp4_f32)
__device__ __forceinline__ uint32_t pack_fp4x8(const float (&v)[8]) {
    uint32_t r = 0u;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
}
// Codes 2 B and 2 B + 1 of a dword in binary32
template <int B> __device__ __forceinline__ v2f fp4x2_to_f32(uint32_t codes) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, B); }

}  // namespace
}  // namespace dsv3

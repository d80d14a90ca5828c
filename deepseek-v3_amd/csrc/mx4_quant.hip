// Tensors into microscaled 4-bit numbers and back (mx4.hpp).  No counterpart in the reference, whose quantiser writes e4m3 codes with binary32 scales
// per 128 (inference/kernel.py:9-57); the rule for the scale is that one's ue8m0 form (:29-31) with 6 in place of 448.
// Both pass over the data once and are bound by memory.
#include "mx4.hpp"

namespace dsv3 {
namespace {

constexpr int kThreads = 256, kUnroll = 4;
constexpr int64_t kMostItems = 0xffffffff;              // of a launch
// More 16- or 32-bit data than this (half of the last cache) pass the caches by: 18432 x 7168 of bf16 in 51.6 us in place of 59 (334 MB, 6.5 TB/s) and back in 48.6
// for 59, one after the other in 98 for 135; 9500 x 7168 in 54 for 60.  Of what the caches may hold, 4096 x 7168, such loads take 14.6 us and ordinary ones 13.3.
constexpr int64_t kPassing = 128 << 20;
template <bool PASS, class T> __device__ __forceinline__ T load_once(const T* p) {
    if constexpr (PASS) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool PASS, class T> __device__ __forceinline__ void store_once(T* p, T v) {
    if constexpr (PASS) __builtin_nontemporal_store(v, p);
    else *p = v;
}

// The largest |element| of eight, as bits of a binary32, and the eight in binary32
template <int DT> struct Eight;
template <> struct Eight<DSV3_F32> {
    v4f a, b;
    template <bool PASS> __device__ __forceinline__ void load(const void* p, int64_t i) { a = load_once<PASS>((const v4f*)p + 2 * i); b = load_once<PASS>((const v4f*)p + 2 * i + 1); }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = umax_u32(m, umax_u32(abs_bits(a[e]), abs_bits(b[e])));
        return m;
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
    }
};
struct Eight16 {
    v4u p;
    template <bool PASS> __device__ __forceinline__ void load(const void* x, int64_t i) { p = load_once<PASS>((const v4u*)x + i); }
    __device__ __forceinline__ uint32_t largest16() const {
        uint32_t m = pk_umax_u16(pk_umax_u16(p[0] & 0x7fff7fffu, p[1] & 0x7fff7fffu), pk_umax_u16(p[2] & 0x7fff7fffu, p[3] & 0x7fff7fffu));
        return umax_u32(m & 0xffffu, m >> 16);
    }
};
template <> struct Eight<DSV3_BF16> : Eight16 {
    __device__ __forceinline__ uint32_t largest() const { return largest16() << 16; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[2 * e] = bf16lo_to_f32(p[e]); f[2 * e + 1] = bf16hi_to_f32(p[e]); }
    }
};
__device__ __forceinline__ float f16_bits_to_f32(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
template <> struct Eight<DSV3_F16> : Eight16 {
    __device__ __forceinline__ uint32_t largest() const { return f32_as_u32(f16_bits_to_f32(largest16())); }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[2 * e] = f16_bits_to_f32(p[e] & 0xffffu); f[2 * e + 1] = f16_bits_to_f32(p[e] >> 16); }
    }
};

// Eight elements a lane, four lanes a block; a workgroup's loads are all on their way before the first is looked at.
template <int DT, bool PASS>
__global__ __launch_bounds__(kThreads) void mx4_quant_kernel(const void* x, uint32_t* y, uint8_t* s, int64_t eights) {
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
    Eight<DT> in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)                   // (past the end, the last eight again: a lane's three neighbours are there as well)
        in[u].template load<PASS>(x, min(first + u * kThreads, eights - 1));
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * kThreads;
        uint32_t m = in[u].largest();
        m = dpp_umax<0xb1>(m);                          // of lanes l ^ 1, then l ^ 2
        m = dpp_umax<0x4e>(m);
        const uint32_t byte = mx4_scale_byte(m);
        const float factor = mx4_factor(byte);
        float f[8];
        in[u].get(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = byte == kMx4Nan ? 0.f : f[e] * factor;
        if (i < eights) {
            y[i] = pack_fp4x8(f);
            if ((threadIdx.x & 3) == 0) s[i >> 2] = (uint8_t)byte;
        }
    }
}

// 16 bytes of results a lane: eight elements of 16 bits, four of 32, of which 18432 x 7168 take 84 us (eight a lane, with two stores that leave gaps between the
// lanes' pieces: 145, and 224 past the caches).
template <int DT, bool PASS>
__global__ __launch_bounds__(kThreads) void mx4_dequant_kernel(const void* x, const uint8_t* s, v4u* y, int64_t items) {
    constexpr bool WIDE = DT == DSV3_F32;
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
    uint32_t codes[kUnroll], byte[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = min(first + u * kThreads, items - 1);
        codes[u] = WIDE ? ((const uint16_t*)x)[i] : ((const uint32_t*)x)[i];
        byte[u] = s[i >> (WIDE ? 3 : 2)];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * kThreads;
        const float p = mx4_power(byte[u]);
        const v2f a = fp4x2_to_f32<0>(codes[u]), b = fp4x2_to_f32<1>(codes[u]), c = fp4x2_to_f32<2>(codes[u]), d = fp4x2_to_f32<3>(codes[u]);
        v4u out;
        if constexpr (WIDE) out = v4u{ f32_as_u32(a.x * p), f32_as_u32(a.y * p), f32_as_u32(b.x * p), f32_as_u32(b.y * p) };
        else if constexpr (DT == DSV3_BF16) out = v4u{ pack_bf16(a.x * p, a.y * p), pack_bf16(b.x * p, b.y * p), pack_bf16(c.x * p, c.y * p), pack_bf16(d.x * p, d.y * p) };
        else out = v4u{ pack_f16(a.x * p, a.y * p), pack_f16(b.x * p, b.y * p), pack_f16(c.x * p, c.y * p), pack_f16(d.x * p, d.y * p) };
        if (i < items) store_once<PASS>(y + i, out);
    }
}

}  // namespace

int launch_mx4_quant(const void* x, int x_dtype, void* y, void* s, int64_t numel, hipStream_t st) {
    const int64_t eights = numel / 8, grid = (eights + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    if (grid * kThreads > kMostItems) return DSV3_ERR_BAD_SHAPE;
    static void (*const kernels[3][2])(const void*, uint32_t*, uint8_t*, int64_t) = {
        { mx4_quant_kernel<DSV3_BF16, false>, mx4_quant_kernel<DSV3_BF16, true> },
        { mx4_quant_kernel<DSV3_F16, false>, mx4_quant_kernel<DSV3_F16, true> },
        { mx4_quant_kernel<DSV3_F32, false>, mx4_quant_kernel<DSV3_F32, true> },
    };
    const bool passing = numel * (x_dtype == DSV3_F32 ? 4 : 2) > kPassing;
    hipLaunchKernelGGL(kernels[x_dtype][passing], dim3((unsigned)grid), dim3(kThreads), 0, st, x, (uint32_t*)y, (uint8_t*)s, eights);
    return launch_status();
}

int launch_mx4_dequant(const void* x, const void* s, void* y, int y_dtype, int64_t numel, hipStream_t st) {
    const int64_t items = numel / (y_dtype == DSV3_F32 ? 4 : 8), grid = (items + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    if (grid * kThreads > kMostItems) return DSV3_ERR_BAD_SHAPE;
    static void (*const kernels[3][2])(const void*, const uint8_t*, v4u*, int64_t) = {
        { mx4_dequant_kernel<DSV3_BF16, false>, mx4_dequant_kernel<DSV3_BF16, true> },
        { mx4_dequant_kernel<DSV3_F16, false>, mx4_dequant_kernel<DSV3_F16, true> },
        { mx4_dequant_kernel<DSV3_F32, false>, mx4_dequant_kernel<DSV3_F32, true> },
    };
    const bool passing = numel * (y_dtype == DSV3_F32 ? 4 : 2) > kPassing;
    hipLaunchKernelGGL(kernels[y_dtype][passing], dim3((unsigned)grid), dim3(kThreads), 0, st, x, (const uint8_t*)s, (v4u*)y, items);
    return launch_status();
}

}  // namespace dsv3

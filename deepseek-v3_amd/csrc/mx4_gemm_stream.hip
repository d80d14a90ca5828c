// mx4_gemm for few rows of activations: bound by reading the weight, half a byte and 1/32 an element, once.
#include "mx4_gemm.hpp"

namespace dsv3 {
namespace {

// A workgroup: NT strips of 16 weight rows and MT tiles of 16 activation rows, W wavefronts side by side along K, sums joined in LDS in their order.
// A wavefront: v_mfma_scale_f32_16x16x128_f8f6f4 straight from memory.  Lane (r, q) = (l % 16, l / 16) holds the weight's 32 codes 32 q .. of row r in
// 128, its scale byte q, and of the activations the same or, as e4m3 codes, bytes 16 q .. + 15 and 64 + 16 q .. + 15 of 128.  The result has
// weight rows 4 q .. + 3 of activation row r in a lane.
template <bool A8, int MT, int NT, int W, int CD>
__global__ __launch_bounds__(64 * W) void mx4_stream_kernel(Mx4Args p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int steps = (int)(p.k / 128);
    const int s0 = (int)((int64_t)steps * wave / W), s1 = (int)((int64_t)steps * (wave + 1) / W);
    const uint8_t* b[NT];
    const uint32_t* bs[NT];
    const uint8_t* a[MT];
    const uint32_t* as[MT];                             // a dword per 128: four bytes, or a binary32
#pragma unroll
    for (int t = 0; t < NT; ++t) {                      // rows past the end repeat the last one; their results are dropped
        const int64_t row = min(n0 + t * 16 + r, p.n - 1);
        b[t] = p.b + row * (p.k / 2) + q * 16;
        bs[t] = (const uint32_t*)p.b_s + row * steps;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t row = min(m0 + t * 16 + r, p.m - 1);
        a[t] = p.a + row * (A8 ? p.k : p.k / 2) + q * 16;
        as[t] = (const uint32_t*)p.a_s + row * steps;
    }
    v4f acc[NT][MT] = {};
    constexpr int U = 4;
    for (int s = s0; s < s1; s += U) {
        v4u bf[U][NT], af[U][MT], ag[A8 ? U : 1][A8 ? MT : 1];
        uint32_t sb[U][NT], sa[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(s + u, s1 - 1);          // (a slice's last steps again where it is no whole U: not multiplied)
#pragma unroll
            for (int t = 0; t < NT; ++t) { bf[u][t] = *(const v4u*)(b[t] + (int64_t)at * 64); sb[u][t] = bs[t][at]; }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                af[u][t] = *(const v4u*)(a[t] + (int64_t)at * (A8 ? 128 : 64));
                if constexpr (A8) ag[u][t] = *(const v4u*)(a[t] + (int64_t)at * 128 + 64);
                sa[u][t] = as[t][at];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= s1) break;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const v8i x = __builtin_bit_cast(v8i, __builtin_shufflevector(bf[u][t], bf[u][t], 0, 1, 2, 3, 0, 1, 2, 3));
                const int xs = (int)(sb[u][t] >> (8 * q));
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    v8i y;
                    if constexpr (A8) y = __builtin_bit_cast(v8i, __builtin_shufflevector(af[u][j], ag[u][j], 0, 1, 2, 3, 4, 5, 6, 7));
                    else y = __builtin_bit_cast(v8i, __builtin_shufflevector(af[u][j], af[u][j], 0, 1, 2, 3, 0, 1, 2, 3));
                    const int ys = A8 ? (int)(sa[u][j] >> 23) : (int)(sa[u][j] >> (8 * q));
                    acc[t][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc[t][j], 4, A8 ? 0 : 4, 0, xs, 0, ys);
                }
            }
        }
    }
    __shared__ v4f part[W][NT * MT][64];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[wave][t * MT + j][lane] = acc[t][j];
    __syncthreads();
    for (int x = wave; x < NT * MT; x += W) {
        v4f sum = part[0][x][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) sum += part[w][x][lane];
        const int64_t row = m0 + (x % MT) * 16 + r, col = n0 + (x / MT) * 16 + 4 * q;
        if (row < p.m) {
            auto* c = (typename OutT<CD>::type*)p.c + row * p.n + col;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < p.n) c[e] = cvt_out<CD>(sum[e]);
        }
    }
}

template <bool A8, int MT, int NT, int W> int launch_as(const Mx4Args& p, int c_dtype, hipStream_t st) {
    const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * MT - 1) / (16 * MT);
    if (gx * (64 * W) > 0xffffffffll || gy > 65535) return DSV3_ERR_BAD_SHAPE;
    auto* kernel = c_dtype == DSV3_BF16 ? mx4_stream_kernel<A8, MT, NT, W, DSV3_BF16>
                 : c_dtype == DSV3_F16 ? mx4_stream_kernel<A8, MT, NT, W, DSV3_F16> : mx4_stream_kernel<A8, MT, NT, W, DSV3_F32>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)gx, (unsigned)gy), dim3(64 * W), 0, st, p);
    return launch_status();
}
template <bool A8> int launch_a(const Mx4Args& p, int c_dtype, hipStream_t st) {
    if (p.m <= 16) return launch_as<A8, 1, 1, 8>(p, c_dtype, st);
    if (p.m <= 32) return launch_as<A8, 2, 1, 8>(p, c_dtype, st);
    return launch_as<A8, 4, 1, 8>(p, c_dtype, st);
}

}  // namespace

int launch_mx4_stream(const Mx4Args& p, bool a8, int c_dtype, hipStream_t st) {
    return a8 ? launch_a<true>(p, c_dtype, st) : launch_a<false>(p, c_dtype, st);
}

}  // namespace dsv3

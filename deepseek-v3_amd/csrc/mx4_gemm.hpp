// The product with a weight of microscaled 4-bit numbers: what its kernels share.
//     c[i, j] = sum_k a[i, k] * b[j, k],  b = e2m1 codes * 2^(byte - 127) per 32 along k;
//     a the same, or e4m3 codes * a binary32 power of two per 128 along k (act_quant's ue8m0 form).
// All products are those of v_mfma_scale_f32_*_f8f6f4, which takes both formats and the scales as they are and sums in binary32.
#pragma once
#include "mx4.hpp"

namespace dsv3 {

struct Mx4Args {
    const uint8_t* a; const void* a_s;                  // codes [m][k / 2] and bytes [m][k / 32], or e4m3 [m][k] and binary32 [m][k / 128]
    const uint8_t* b; const uint8_t* b_s;               // codes [n][k / 2], bytes [n][k / 32]
    void* c;
    int64_t m, n, k;
};

int launch_mx4_stream(const Mx4Args& p, bool a8, int c_dtype, hipStream_t st);
size_t mx4_tile_workspace_bytes(int64_t m, int64_t n, int64_t k, bool a8);
int launch_mx4_tile(const Mx4Args& p, bool a8, int c_dtype, void* workspace, hipStream_t st);

}  // namespace dsv3

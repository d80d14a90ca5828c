// mx4_gemm: which kernel takes which sizes.
#include "mx4_gemm.hpp"

namespace dsv3 {

static bool tiles(int64_t m, int64_t n, int64_t k) { return m > 64 && mx4_tile_takes(m, n, k); }

size_t mx4_gemm_workspace_bytes(bool a8, int64_t m, int64_t n, int64_t k) { return tiles(m, n, k) ? mx4_tile_workspace_bytes(m, n, k, a8) : 0; }

int launch_mx4_gemm(const void* a, const void* a_s, bool a8, const void* b, const void* b_s, void* c, int c_dtype, int64_t m, int64_t n, int64_t k,
                    void* workspace, hipStream_t st) {
    const Mx4Args p = { (const uint8_t*)a, a_s, (const uint8_t*)b, (const uint8_t*)b_s, c, m, n, k };
    return tiles(m, n, k) ? launch_mx4_tile(p, a8, c_dtype, workspace, st) : launch_mx4_stream(p, a8, c_dtype, st);
}

}  // namespace dsv3

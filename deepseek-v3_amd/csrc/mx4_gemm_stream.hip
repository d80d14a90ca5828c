// mx4_gemm for few rows of activations, and where weights are small: bound by reading the weight, half a byte and 1/32 an element, once.
#include "mla.hpp"
#include "mx4_gemm.hpp"

namespace dsv3 {
namespace {

constexpr int kMostWaves = 8;

// A workgroup: 16 NT weight rows and 16 MT activation rows, its wavefronts side by side along k, their sums joined in LDS in their order.
//
// A wavefront takes chunks of 512 along k, which it copies into LDS for itself (no barrier), DEPTH chunks on their way: four rows of 256 bytes a copy, whole
// lines, where fragments straight from memory would ask for 16 rows of 64 bytes at a time, which the address unit takes four times as long for.  A row's piece
// of 16 bytes c stands at c ^ row % 16, so that 16 rows read at one place hit all banks.
//
// v_mfma_scale_f32_16x16x128_f8f6f4: lane (r, q) = (l % 16, l / 16) gives 32 codes of the weight's row r and their scale, of the activations' row r the same, or as
// e4m3 codes the 16-byte halves q % 2 of the blocks q / 2 and q / 2 + 2 of the four; the result has weight rows 4 q .. + 3 of activation row r in it.  Which
// 128 of the 512 a product takes is free as long as both sides take the same: product s takes blocks s, 4 + s, 8 + s and 12 + s of 32, so that a lane's scales of the
// four products are the four bytes of one dword.
//
// AR: activation rows that are copied (rows past them repeat the last one).
//
// 7168 -> 18432 (70 MB of weight, 10.8 us at the 6.5 TB/s that a read stream reaches), a weight from memory in every call: 14.4 us for one row, 18.2 for 16, 22.3 for 32
// (e4m3 15.5, 21.3 and 25.4; the first form, straight from memory into the fragments, 1 KiB of both a product, 23, 37 and 53).  One weight call after call, most of which
// the last cache keeps: 12.0, 13.9 and 17.1 (12.7, 16.4 and 19.1).  Bound by the weight's way from memory, behind it by the launch and its first line, and with 32 rows
// by the activations, which every workgroup reads (58 MB).
template <bool A8, int AR, int NT, int DEPTH> struct Geo {
    static constexpr int MT = (AR + 15) / 16, AB = A8 ? 512 : 256;      // activation tiles, bytes of an activation row in a chunk
    static constexpr int NB = 4 * NT, NA = AR * AB / 1024;              // copies of a chunk's codes
    static constexpr int PER = NB + NA + NT + MT;       // and scales: 256 bytes for each 16 rows of both
    static constexpr int STAGE = NT * 4096 + AR * AB + (NT + MT) * 256;
    static_assert(NA * 1024 == AR * AB && PER * (DEPTH - 1) < 64, "whole copies, and no more than can be counted");
};
template <int N> __device__ __forceinline__ void wait_copies() {        // all but the N youngest
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

template <bool A8, int AR, int NT, int DEPTH, int CD>
__global__ __launch_bounds__(64 * kMostWaves) void mx4_stream_kernel(Mx4Args p) {
    using G = Geo<A8, AR, NT, DEPTH>;
    constexpr int MT = G::MT, AB = G::AB;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NT), m0 = (int64_t)blockIdx.y * (16 * MT);
    const int steps = (int)(p.k / 128), chunks = (steps + 3) / 4;
    const int c0 = (int)((int64_t)chunks * wave / W), c1 = (int)((int64_t)chunks * (wave + 1) / W);
    const uint32_t mine = lds_addr_of(lds) + wave * (DEPTH * G::STAGE);
    const uint32_t b_bytes = (uint32_t)(p.k / 2), a_bytes = A8 ? (uint32_t)p.k : (uint32_t)(p.k / 2);
    const uint8_t* b0 = p.b + n0 * b_bytes;
    const uint8_t* a0 = p.a + m0 * a_bytes;
    const uint8_t* bs0 = p.b_s + n0 * (steps * 4);
    const uint8_t* as0 = (const uint8_t*)p.a_s + m0 * (steps * 4);
    const int b_last = (int)min((int64_t)16 * NT - 1, p.n - 1 - n0), a_last = (int)min((int64_t)AR - 1, p.m - 1 - m0);     // rows past the end repeat the last one

    uint32_t b_off[G::NB], a_off[G::NA], bs_off[NT], as_off[MT];
    constexpr int RPC = 1024 / AB;                      // activation rows a copy
    auto b_row = [&](int i) { return 4 * i + (lane >> 4); };
    auto a_row = [&](int i) { return RPC * i + lane / (AB / 16); };
    auto b_piece = [&](int i) { return (lane & 15) ^ (b_row(i) & 15); };
    auto a_piece = [&](int i) { return (lane & (AB / 16 - 1)) ^ (a_row(i) & 15); };
#pragma unroll
    for (int i = 0; i < G::NB; ++i) b_off[i] = min(b_row(i), b_last) * b_bytes + b_piece(i) * 16;
#pragma unroll
    for (int i = 0; i < G::NA; ++i) a_off[i] = min(a_row(i), a_last) * a_bytes + a_piece(i) * 16;
#pragma unroll
    for (int t = 0; t < NT; ++t) bs_off[t] = (min(t * 16 + (lane >> 2), b_last) * steps + (lane & 3)) * 4;
#pragma unroll
    for (int t = 0; t < MT; ++t) as_off[t] = (min(t * 16 + (lane >> 2), a_last) * steps + (lane & 3)) * 4;
    // The last chunk may be short: what is not there is the row's last piece again, with scales of zero (which multiply, below).
    auto copy = [&](int chunk, uint32_t at) {
        const int left = min(steps - chunk * 4, 4);     // of the chunk's four 128s
        auto past = [&](int piece, int have) -> uint32_t { return left == 4 ? 0u : 16u * max(piece - (left * have - 1), 0); };
#pragma unroll
        for (int i = 0; i < G::NB; ++i) copy16(b0 + (int64_t)chunk * 256, b_off[i] - past(b_piece(i), 4), at + i * 1024);
#pragma unroll
        for (int i = 0; i < G::NA; ++i) copy16(a0 + (int64_t)chunk * AB, a_off[i] - past(a_piece(i), AB / 64), at + NT * 4096 + i * 1024);
        const uint32_t back = left == 4 ? 0u : 4u * max((lane & 3) - (left - 1), 0), scales = at + NT * 4096 + AR * AB;
#pragma unroll
        for (int t = 0; t < NT; ++t) copy4(bs0 + (int64_t)chunk * 16, bs_off[t] - back, scales + t * 256);
#pragma unroll
        for (int t = 0; t < MT; ++t) copy4(as0 + (int64_t)chunk * 16, as_off[t] - back, scales + (NT + t) * 256);
    };

    v4f acc[NT][MT] = {};
    auto read16 = [](uint32_t at) -> v4u { return *(lds_v4u)(uintptr_t)at; };
    auto read4 = [](uint32_t at) -> uint32_t { return *(lds_u32)(uintptr_t)at; };
    auto multiply = [&](int chunk, uint32_t at) {
        const bool there = chunk * 4 + q < steps;
        const uint32_t a_at = at + NT * 4096, s_at = a_at + AR * AB;
        uint32_t bs[NT], as[MT], a_rd[MT];
#pragma unroll
        for (int t = 0; t < NT; ++t) { const uint32_t s = read4(s_at + t * 256 + (r * 4 + q) * 4); bs[t] = there ? s : 0u; }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int row = min(j * 16 + r, AR - 1);
            a_rd[j] = a_at + row * AB;
            const uint32_t s = read4(s_at + NT * 256 + (row * 4 + q) * 4);
            as[j] = there ? (A8 ? s >> 23 : s) : 0u;
        }
        unrolled<4>([&](auto step) {
            constexpr int s = decltype(step)::value;
            v4u b[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) b[t] = read16(at + t * 4096 + r * 256 + (((4 * q + s) ^ r) << 4));
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int swz = min(j * 16 + r, AR - 1) & 15;
                v8i y;
                if constexpr (A8) {
                    const int c = 2 * (4 * (q >> 1) + s) + (q & 1);
                    const v4u lo = read16(a_rd[j] + ((c ^ swz) << 4)), hi = read16(a_rd[j] + (((c + 16) ^ swz) << 4));
                    y = __builtin_bit_cast(v8i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                } else {
                    const v4u x = read16(a_rd[j] + (((4 * q + s) ^ swz) << 4));
                    y = __builtin_bit_cast(v8i, __builtin_shufflevector(x, x, 0, 1, 2, 3, 0, 1, 2, 3));
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const v8i w = __builtin_bit_cast(v8i, __builtin_shufflevector(b[t], b[t], 0, 1, 2, 3, 0, 1, 2, 3));
                    acc[t][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, y, acc[t][j], 4, A8 ? 0 : 4, s, (int)bs[t], A8 ? 0 : s, (int)as[j]);
                }
            }
        });
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (c0 + d < c1) copy(c0 + d, mine + d * G::STAGE);
    uint32_t at = mine;
    for (int c = c0, d = 0; c < c1; ++c) {
        // copies retire in their order: those of younger chunks may be on their way
        const int younger = c1 - 1 - c;
        if (younger >= DEPTH - 1) wait_copies<(DEPTH - 1) * G::PER>();
        else if (DEPTH > 2 && younger == 1) wait_copies<G::PER>();
        else wait_copies<0>();
        multiply(c, at);
        if (c + DEPTH < c1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the chunk has been read
            copy(c + DEPTH, at);
        }
        if (++d == DEPTH) { d = 0; at = mine; } else at += G::STAGE;
    }
    __syncthreads();
    v4f* part = (v4f*)lds;                              // [wavefront][tile][lane]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < MT; ++j) part[(wave * NT * MT + t * MT + j) * 64 + lane] = acc[t][j];
    __syncthreads();
    for (int x = wave; x < NT * MT; x += W) {
        v4f sum = part[x * 64 + lane];
        for (int w = 1; w < W; ++w) sum += part[(w * NT * MT + x) * 64 + lane];
        const int64_t row = m0 + (x % MT) * 16 + r, col = n0 + (x / MT) * 16 + 4 * q;
        if (row < p.m) {
            auto* c = (typename OutT<CD>::type*)p.c + row * p.n + col;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < p.n) c[e] = cvt_out<CD>(sum[e]);
        }
    }
}

template <bool A8, int AR, int NT, int DEPTH, int CD> int launch_cd(const Mx4Args& p, int waves, hipStream_t st) {
    using G = Geo<A8, AR, NT, DEPTH>;
    const int64_t gx = (p.n + 16 * NT - 1) / (16 * NT), gy = (p.m + 16 * G::MT - 1) / (16 * G::MT);
    if (gx * (64 * waves) > 0xffffffffll || gy > 65535) return DSV3_ERR_BAD_SHAPE;
    static LdsGrant grant;
    if (!grant.ensure((const void*)mx4_stream_kernel<A8, AR, NT, DEPTH, CD>, 160 * 1024)) return DSV3_ERR_LAUNCH;
    const int bytes = waves * (DEPTH * G::STAGE > NT * G::MT * 1024 ? DEPTH * G::STAGE : NT * G::MT * 1024);
    hipLaunchKernelGGL((mx4_stream_kernel<A8, AR, NT, DEPTH, CD>), dim3((unsigned)gx, (unsigned)gy), dim3(64 * waves), bytes, st, p);
    return launch_status();
}
template <bool A8, int AR, int NT> int launch_ar(const Mx4Args& p, int c_dtype, hipStream_t st) {
    constexpr int DEPTH = 2;
    using G = Geo<A8, AR, NT, DEPTH>;
    static_assert(DEPTH * G::STAGE <= 80 * 1024, "a wavefront's chunks");
    // Wavefronts of a workgroup: what fits a compute unit's LDS beside the workgroups that share it.  One a unit where there are no more (32 rows of e4m3,
    // 7168 -> 2112: 7.0 us, with one wavefront in half of it 11.6); three where activations take little room (one row of e4m3, 7168 -> 18432: 15.5 us, two of them
    // 16.3, one 20.5), else two (16 rows 21.3, one of them 22.6).
    const int64_t strips = (p.n + 16 * NT - 1) / (16 * NT) * ((p.m + AR - 1) / AR), chunks = (p.k + 511) / 512;
    const int room = strips <= 256 ? 160 * 1024 : AR <= 4 ? 54 * 1024 : 80 * 1024;
    int64_t w = room / (DEPTH * G::STAGE);
    w = w < 1 ? 1 : w > kMostWaves ? kMostWaves : w;
    const int64_t each = (chunks + w - 1) / w;          // chunks of the wavefronts alike
    w = chunks ? (chunks + each - 1) / each : 1;
    if (c_dtype == DSV3_BF16) return launch_cd<A8, AR, NT, DEPTH, DSV3_BF16>(p, (int)w, st);
    if (c_dtype == DSV3_F16) return launch_cd<A8, AR, NT, DEPTH, DSV3_F16>(p, (int)w, st);
    return launch_cd<A8, AR, NT, DEPTH, DSV3_F32>(p, (int)w, st);
}
// Two strips a workgroup read the activations half as often, and leave half as many workgroups: 16 x 16384 -> 7168 15.5 us with two and 17.7 with one,
// 16 x 7168 -> 4096 5.9 and 5.3.
template <bool A8, int AR> int launch_nt(const Mx4Args& p, int c_dtype, hipStream_t st) {
    return p.n >= 6144 ? launch_ar<A8, AR, 2>(p, c_dtype, st) : launch_ar<A8, AR, 1>(p, c_dtype, st);
}
template <bool A8> int launch_a(const Mx4Args& p, int c_dtype, hipStream_t st) {
    if (p.m <= 4) return launch_ar<A8, 4, 1>(p, c_dtype, st);
    if (p.m <= 16) return launch_nt<A8, 16>(p, c_dtype, st);
    return launch_nt<A8, 32>(p, c_dtype, st);
}

}  // namespace

int launch_mx4_stream(const Mx4Args& p, bool a8, int c_dtype, hipStream_t st) {
    constexpr int64_t most = 65535 * 32;                // rows of a launch, which k == 0 alone brings more of
    for (int64_t m0 = 0; m0 < p.m; m0 += most) {
        Mx4Args q = p;
        q.m = p.m - m0 < most ? p.m - m0 : most;
        q.a += m0 * (a8 ? p.k : p.k / 2);
        q.a_s = (const uint8_t*)p.a_s + m0 * (p.k / 32);
        q.c = (uint8_t*)p.c + m0 * p.n * (c_dtype == DSV3_F32 ? 4 : 2);
        const int rc = a8 ? launch_a<true>(q, c_dtype, st) : launch_a<false>(q, c_dtype, st);
        if (rc != DSV3_OK) return rc;
    }
    return DSV3_OK;
}

}  // namespace dsv3

// Behind the attention kernels of the absorbed form: the ranges' partial sums to the latent of each row, its product with the value half of
// wkv_b and, where the output projection takes it so, the quantisation of the result.
#pragma once
#include "mla.hpp"

namespace dsv3 {
namespace {

constexpr int kC = 512, kRope = 64, kNope = 128, kQd = kNope + kRope;

struct FoldArgs {
    const float* part; const v2f* ml;                   // as the attention kernel wrote them
    const v2i* plan; const int32_t* counts;             // PAGED: (first range, ranges) [sequence]; the tokens that a sequence has
    const uint8_t* w; const float* ws;                  // wkv_b fp8 [heads * 256, 512] and its block scales
    void* y; float* ys;                                 // bf16 [tokens][heads][128], or e4m3 and scales [tokens][heads]
    int tokens, per_seq, heads, rows, blocks, splits, group;    // tokens of all sequences and of one; rows of an attention workgroup and its blocks; tokens at a time, up to 16
    float scale;
};

// One workgroup: a head and up to 16 tokens at a time.  The wavefronts first form the tokens' latents from the ranges' partial sums
// (a wavefront a token and 2 KiB a range, several wavefronts a token where there are fewer than eight) and leave them in
// LDS as bf16, then multiply: wavefront (kb, dh) holds K block kb of the 64 features dh of the head's value weights and
// the four K blocks' results meet in LDS (absorb_v_ksplit_kernel's maps, wkv_b_absorb.hip).  The 128 features
// of a (token, head) are one quantisation block of the output projection's input.
// Three launches were in its place (combine 5 .. 13.7 us, the product 4.5 .. 7.5, act_quant 4.2).
// PAGED: every sequence has ranges of its own, [range][row block][row]; a row that saw no position, and one of a token that its sequence does
// not have, gives zeros (else NaN, as softmax does).  The latents go into the product as two bf16 each: rounded to one, they would be off by as
// much as the result's own rounding.  The relative error (rms) of the whole attention at 4096 positions is 0.0025 so, 0.0030 with one (0.0017: the
// rounding of the result alone); it costs 1 us of 120.
template <bool QUANT, bool PAGED>
__global__ __launch_bounds__(512, 4) void mla_fold_kernel(FoldArgs p) {
    __shared__ __attribute__((aligned(1024))) uint8_t lat[(PAGED ? 2 : 1) * 16 * 1024];         // chunk c of row r at c ^ r (low four bits); then what bf16 leaves
    __shared__ v4f sums[8][4][64];                                      // products' partial results; before, latents' partial sums
    __shared__ float norm[8];
    __shared__ uint32_t amax[8][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, kb = wave & 3, dh = wave >> 2, h = blockIdx.x;

    // The weights are loaded behind the latents, whose sums need the registers, but their lines (64 KiB, one a thread) are
    // brought into the L2 beside them.
    uint32_t touched = *(const uint32_t*)(p.w + ((int64_t)h * 256 + 128 + (threadIdx.x >> 2)) * kC + (threadIdx.x & 3) * 128);
    const float scale2 = PAGED ? 1.f : p.scale * 1.44269504088896340736f;       // (paged: maxima are exponents of two)
    for (int ms = blockIdx.z * p.group; ms < p.tokens; ms += gridDim.z * p.group) {
        const int n = min(p.group, p.tokens - ms);
        const int per = n == 1 ? 8 : n == 2 ? 4 : n <= 4 ? 2 : 1, sub = wave & (per - 1);       // wavefronts of a token
        auto put = [&](int k, int f, v4f x) {           // features f .. f + 3 of token k
            uint8_t* at = lat + k * 1024 + (((f >> 3) ^ k) << 4) + (f & 4) * 2;
            const v2u y = { pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]) };
            *(v2u*)at = y;
            if constexpr (PAGED) {                      // (beside an infinity nothing: it stays one)
                auto rest = [](float v, float r) { const float d = v - r; return d == d ? d : 0.f; };
                *(v2u*)(at + 16 * 1024) = v2u{ pack_bf16(rest(x[0], bf16lo_to_f32(y[0])), rest(x[1], bf16hi_to_f32(y[0]))),
                                               pack_bf16(rest(x[2], bf16lo_to_f32(y[1])), rest(x[3], bf16hi_to_f32(y[1]))) };
            }
        };
        for (int k = wave / per; k < n; k += 8 / per) {
            const int t = ms + k, b = t / p.per_seq, row = (t - b * p.per_seq) * p.heads + h;
            int splits = p.splits;
            int64_t bb = (int64_t)b * p.blocks + row / p.rows, part = (int64_t)p.rows * kC;
            const v2f* ml = p.ml + (bb * p.rows + row % p.rows) * p.splits;
            const float* src = p.part + bb * p.splits * part + (row % p.rows) * kC + lane * 4;
            int64_t ml_step = 1;
            if constexpr (PAGED) {
                const v2i mine = p.plan[b];
                splits = t - b * p.per_seq < p.counts[b] ? mine[1] : 0;
                bb = (int64_t)mine[0] * p.blocks + row / p.rows;
                ml = p.ml + bb * p.rows + row % p.rows;
                src = p.part + bb * part + (row % p.rows) * kC + lane * 4;
                ml_step = (int64_t)p.blocks * p.rows;
                part *= p.blocks;
            }
            // a chunk of 64 ranges, a lane each; up to six ranges' sums are requested before the first is added
            const v2f none = { -__builtin_inff(), 0.f };
            v2f x = lane < splits ? ml[lane * ml_step] : none;
            float m = x.x, l = 0.f;
            for (int s = 64 + lane; s < splits; s += 64) m = fmaxf(m, ml[s * ml_step].x);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
            v4f a0 = {}, a1 = {};
            for (int s0 = 0; s0 < splits; s0 += 64) {
                if (s0 > 0) x = s0 + lane < splits ? ml[(s0 + lane) * ml_step] : none;
                const float wt = x.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((x.x - m) * scale2);
                l += x.y * wt;
                const int end = min(64, splits - s0);
                auto add = [&](auto count, int s) {     // ranges s, s + per, ..
                    constexpr int U = decltype(count)::value;
                    v4f o[U][2];
                    const float* at = src + (s0 + s) * part;
#pragma unroll
                    for (int u = 0; u < U; ++u, at += per * part) { o[u][0] = *(const v4f*)at; o[u][1] = *(const v4f*)(at + kC / 2); }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const float k2 = u32_as_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_as_u32(wt), s + u * per));
                        a0 += o[u][0] * k2;
                        a1 += o[u][1] * k2;
                    }
                };
                int s = sub;
                for (; s + 5 * per < end; s += 6 * per) add(std::integral_constant<int, 6>(), s);
                if (s + 3 * per < end) { add(std::integral_constant<int, 4>(), s); s += 4 * per; }
                if (s + per < end) { add(std::integral_constant<int, 2>(), s); s += 2 * per; }
                if (s < end) add(std::integral_constant<int, 1>(), s);
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d);
            const float rl = PAGED && l == 0.f ? 0.f : 1.0f / l;        // (a row without any position: 0 * inf, NaN as softmax gives)
            if (per == 1) {
                put(k, lane * 4, a0 * rl);
                put(k, kC / 2 + lane * 4, a1 * rl);
            } else {
                v4f* dst = (v4f*)sums + wave * 128 + lane;
                dst[0] = a0;
                dst[64] = a1;
                if (lane == 0) norm[wave] = rl;
            }
        }
        if (per > 1) {
            __syncthreads();
            const int k = threadIdx.x >> 7, f4 = threadIdx.x & 127;
            if (k < n) {
                v4f x = ((const v4f*)sums)[k * per * 128 + f4];
                for (int w = 1; w < per; ++w) x += ((const v4f*)sums)[(k * per + w) * 128 + f4];
                put(k, f4 * 4, x * norm[k * per]);
            }
        }
        asm volatile("" :: "v"(touched));
        v4u raw[4][2];
        float sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int64_t r = (int64_t)h * 256 + 128 + dh * 64 + (i >> 2) * 16 + t * 4 + (i & 3);
            sc[t] = p.ws[(r >> 7) * (kC / 128) + kb];
            const v4u* src = (const v4u*)(p.w + r * kC + kb * 128 + g * 32);
            raw[t][0] = src[0];
            raw[t][1] = src[1];
        }
        barrier_no_fence();                             // the latents are there, and the partial sums have been read
        v4f acc[4] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint8_t* from = lat + i * 1024 + ((kb * 16 + ((g * 4 + s) ^ i)) << 4);
            const v4u x = *(const v4u*)from;
            v4u rest = {};
            if constexpr (PAGED) rest = *(const v4u*)(from + 16 * 1024);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t lo = raw[t][s >> 1][2 * (s & 1)], hi = raw[t][s >> 1][2 * (s & 1) + 1];
                const v2f x0 = fp8x2_lo_to_f32(lo), x1 = fp8x2_hi_to_f32(lo), x2 = fp8x2_lo_to_f32(hi), x3 = fp8x2_hi_to_f32(hi);
                const v4u A = { pack_bf16(x0.x * sc[t], x0.y * sc[t]), pack_bf16(x1.x * sc[t], x1.y * sc[t]),
                                pack_bf16(x2.x * sc[t], x2.y * sc[t]), pack_bf16(x3.x * sc[t], x3.y * sc[t]) };
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, A), __builtin_bit_cast(v8bf, x), acc[t], 0, 0, 0);
                if constexpr (PAGED) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, A), __builtin_bit_cast(v8bf, rest), acc[t], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);          // (no more operands at a time than registers)
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) sums[wave][t][lane] = acc[t];
        __syncthreads();
        // the lane's token is i, its features dh 64 + g 16 + kb 4 + [0, 4)
        v4f r = sums[dh * 4][kb][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) r += sums[dh * 4 + w][kb][lane];
        const int64_t out = (int64_t)(ms + i) * p.heads + h;
        const int f = dh * 64 + g * 16 + kb * 4;
        if constexpr (QUANT) {
            uint32_t abits = 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[e] = round_bf16(r[e]);
                abits = umax_u32(abits, abs_bits(r[e]));
            }
            abits = umax_u32(abits, (uint32_t)__shfl_xor((int)abits, 16));
            abits = umax_u32(abits, (uint32_t)__shfl_xor((int)abits, 32));
            if (g == 0) amax[wave][i] = abits;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; ++w) abits = umax_u32(abits, amax[w][i]);
            const float bs = block_scale(abits, false), rs = 1.0f / bs;
            const bool fast = block_is_finite(abits);
            if (i < n) {
                *(uint32_t*)((uint8_t*)p.y + out * 128 + f) = pack_fp8x4(block_quotient(r[0], bs, rs, fast), block_quotient(r[1], bs, rs, fast),
                                                                         block_quotient(r[2], bs, rs, fast), block_quotient(r[3], bs, rs, fast));
                if (wave == 0 && g == 0) p.ys[out] = bs;
            }
        } else if (i < n) {
            *(v2u*)((uint16_t*)p.y + out * 128 + f) = v2u{ pack_bf16(r[0], r[1]), pack_bf16(r[2], r[3]) };
        }
        __syncthreads();                                // everybody is done with this group's sums
    }
}

template <bool PAGED> int launch_fold(FoldArgs f, hipStream_t st) {
    // A head and four, eight or 16 tokens a workgroup, as few as leave a workgroup a compute unit (8 sequences at
    // 2000 positions: 19.5 us with eight tokens in 128 workgroups, 17.0 with four in 256, 18.3 with two in 512; 32 at 4096: 16.5 with
    // 16 in 256, 17.3 with eight in 512); then the groups are dealt over at most 1024.
    f.group = 4;
    while (f.group < 16 && ((int64_t)f.tokens + f.group - 1) / f.group * f.heads > 256) f.group *= 2;
    int64_t gz = ((int64_t)f.tokens + f.group - 1) / f.group, most = 1024 / f.heads;
    most = most < 1 ? 1 : most;
    gz = gz > most ? most : gz;
    const dim3 grid(f.heads, 1, (unsigned)gz);
    if (f.ys) hipLaunchKernelGGL((mla_fold_kernel<true, PAGED>), grid, dim3(512), 0, st, f);
    else hipLaunchKernelGGL((mla_fold_kernel<false, PAGED>), grid, dim3(512), 0, st, f);
    return launch_status();
}

}  // namespace
}  // namespace dsv3

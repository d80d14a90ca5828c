// The latent cache of MLA in pages of e4m3 rows: written behind the low-rank projections, read back as bf16, and an accepted draft's
// rows moved to the front.  (Reference: the caches of inference/model.py:443-444 and what fills them, :457-466, :480-483; it keeps them dense and in bf16.)
// A row is 512 latents as e4m3 codes, one binary32 power of two that multiplies them, 64 rotary elements in bf16: 644 bytes for 1152.
// One scale a row: the codes' own exponents span 2^-9 .. 448, so that an element is off by half a step of 2^-3 (a sixteenth of its
// value) down to 2^-13.8 of the row's largest (2^-6, the smallest normal code, where that is 224 .. 448); a scale per 128 would move that limit and nothing else.  A power of two: code times
// scale is a bf16 number, so that reading rounds nothing.
#include "mla.hpp"
#include "paged.hpp"

namespace dsv3 {
namespace {

constexpr int kC = 512, kRope = 64;
constexpr int64_t kMostItems = 0xffffffff;              // of a launch

struct WriteArgs {
    const uint16_t* a; int64_t a_stride;                // bf16 rows [q_rank | 512 | 64], stride in elements
    const uint16_t* q_w; const uint16_t* kv_w;          // norm weights
    const v2f* freqs;                                   // [batch * rows][32] (cos, sin)
    uint8_t* kv; float* scale; uint16_t* pe;            // pages
    const int32_t* table; int64_t width, pages; int page;
    const int32_t* starts; const int32_t* counts;
    uint8_t* y; float* ys;                              // e4m3 [batch * rows][q_rank], scales [batch * rows][q_rank / 128]
    int64_t total; int rows, q_rank;
    float q_eps, kv_eps;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ void unpack8(v4u p, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[2 * e] = bf16lo_to_f32(p[e]); f[2 * e + 1] = bf16hi_to_f32(p[e]); }
}
__device__ __forceinline__ double sum_sq8(const float (&f)[8]) {
    double s = 0.;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)f[e] * f[e];
    return s;
}
// The norm's factor.  Sums in binary64: the rows are rounded twice behind it (bf16, e4m3), and a factor that depended on the
// order of a binary32 sum would make the cached codes depend on it.
__device__ __forceinline__ float rms_factor(double sum, int n, float eps) { return (float)(1.0 / __builtin_sqrt(sum / n + eps)); }

// A wavefront: one row of the cache.
__device__ __forceinline__ void write_row(const WriteArgs& p, int64_t row, int lane) {
    const int b = (int)(row / p.rows), tok = (int)(row - (int64_t)b * p.rows);
    const int64_t start = p.starts[b];
    if (start < 0 || tok >= p.counts[b]) return;
    const int64_t at = page_row(p.table + b * p.width, p.width, p.pages, p.page, start + tok);
    if (at < 0) return;
    const uint16_t* src = p.a + row * p.a_stride + p.q_rank;
    const uint32_t key = lane < 32 ? *(const uint32_t*)(src + kC + lane * 2) : 0u;
    float x[8], w[8];
    unpack8(*(const v4u*)(src + lane * 8), x);
    unpack8(*(const v4u*)(p.kv_w + lane * 8), w);
    const float r = rms_factor(wave_sum(sum_sq8(x)), kC, p.kv_eps);
    uint32_t abits = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = round_bf16(x[e] * r * w[e]);
        abits = umax_u32(abits, abs_bits(x[e]));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) abits = umax_u32(abits, (uint32_t)__shfl_xor((int)abits, d));
    // a row that holds a NaN or an infinity: codes of zero and a scale of NaN, so that whoever reads it gets NaN, and whoever
    // multiplies it with a weight of zero gets zero
    const bool fine = block_is_finite(abits);
    const float s = fine ? block_scale(abits, true) : u32_as_f32(0x7fc00000u), rs = 1.0f / s;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fine ? x[e] * rs : 0.f;
    *(v2u*)(p.kv + at * kC + lane * 8) = v2u{ pack_fp8x4(x[0], x[1], x[2], x[3]), pack_fp8x4(x[4], x[5], x[6], x[7]) };
    if (lane == 0) p.scale[at] = s;
    if (lane < 32) {
        const v2f cs = p.freqs[row * (kRope / 2) + lane];
        const float re = bf16lo_to_f32(key), im = bf16hi_to_f32(key);
        *(uint32_t*)(p.pe + at * kRope + lane * 2) = pack_bf16(re * cs.x - im * cs.y, re * cs.y + im * cs.x);
    }
}

// Q: a workgroup a token, wavefronts 0 .. 3 its query latent (RMS norm, bf16, e4m3 per 128 values = 16 lanes), wavefront 4 the cache row.
// Otherwise four cache rows a workgroup.  A chain of three waits (start and page, row, sum): 3.5 us for one token, 5.4 for 32 x 21 with the query's
// latent, 5.5 for 4000 rows without it (8.2 MB); a call from Python takes 8.
template <bool Q>
__global__ __launch_bounds__(Q ? 320 : 256) void mla_write_kernel(WriteArgs p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (!Q) {
        const int64_t row = (int64_t)blockIdx.x * 4 + wave;
        if (row < p.total) write_row(p, row, lane);
        return;
    }
    __shared__ double part[4];
    const int64_t row = blockIdx.x;
    const int c = threadIdx.x * 8;
    float x[8], w[8];
    if (wave == 4) {
        write_row(p, row, lane);
    } else {
        v4u raw = {}, wr = {};
        if (c < p.q_rank) { raw = *(const v4u*)(p.a + row * p.a_stride + c); wr = *(const v4u*)(p.q_w + c); }    // whole 16-lane groups: q_rank is a multiple of 128
        unpack8(raw, x);
        unpack8(wr, w);
        const double sum = wave_sum(sum_sq8(x));
        if (lane == 0) part[wave] = sum;
    }
    __syncthreads();
    if (wave == 4) return;
    const float r = rms_factor(part[0] + part[1] + part[2] + part[3], p.q_rank, p.q_eps);
    uint32_t abits = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = round_bf16(x[e] * r * w[e]);
        abits = umax_u32(abits, abs_bits(x[e]));
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) abits = umax_u32(abits, (uint32_t)__shfl_xor((int)abits, d));
    const float sc = block_scale(abits, false), rs = 1.0f / sc;
    const bool fast = block_is_finite(abits);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = block_quotient(x[e], sc, rs, fast);
    if (c < p.q_rank) {
        *(v2u*)(p.y + row * p.q_rank + c) = v2u{ pack_fp8x4(v[0], v[1], v[2], v[3]), pack_fp8x4(v[4], v[5], v[6], v[7]) };
        if ((lane & 15) == 0) p.ys[row * (p.q_rank / 128) + c / 128] = sc;
    }
}

struct ReadArgs {
    const uint8_t* kv; const float* scale; const uint16_t* pe;
    const int32_t* table; int64_t width, pages; int page;
    const int32_t* lengths;
    uint16_t* out; uint16_t* out_pe;                    // bf16 [batch][positions][512], [.. 64]
    int64_t groups;                                     // of eight positions, of all sequences
    int positions, per_seq;                             // groups of a sequence
};

// A wavefront: eight positions, which lie in one page.  Eight bytes a lane and row in, 16 out.  16 sequences of up to 4096 positions (95 MB): 14.2 us,
// 6.7 TB/s, part of it from the caches in front of the memory; one of 700 3.5.
__global__ __launch_bounds__(256) void mla_read_kernel(ReadArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t group = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (group >= p.groups) return;
    const int b = (int)(group / p.per_seq), pos = (int)(group - (int64_t)b * p.per_seq) * 8;
    const int64_t row = page_row(p.table + b * p.width, p.width, p.pages, p.page, pos);
    const int have = row < 0 ? 0 : max(0, min(8, max(p.lengths[b], 0) - pos)), n = min(8, p.positions - pos);
    v2u raw[8] = {};
    float s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        s[k] = 0.f;
        if (k < have) { raw[k] = *(const v2u*)(p.kv + (row + k) * kC + lane * 8); s[k] = p.scale[row + k]; }
    }
    v4u key = {};
    if (lane >> 3 < have) key = *(const v4u*)(p.pe + (row + (lane >> 3)) * kRope + (lane & 7) * 8);
    const int64_t out = (int64_t)b * p.positions + pos;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (k >= n) break;
        const v2f a = fp8x2_lo_to_f32(raw[k][0]), c = fp8x2_hi_to_f32(raw[k][0]), d = fp8x2_lo_to_f32(raw[k][1]), e = fp8x2_hi_to_f32(raw[k][1]);
        *(v4u*)(p.out + (out + k) * kC + lane * 8) = v4u{ pack_bf16(a.x * s[k], a.y * s[k]), pack_bf16(c.x * s[k], c.y * s[k]),
                                                          pack_bf16(d.x * s[k], d.y * s[k]), pack_bf16(e.x * s[k], e.y * s[k]) };
    }
    if (lane >> 3 < n) *(v4u*)(p.out_pe + (out + (lane >> 3)) * kRope + (lane & 7) * 8) = key;
}

struct KeepArgs {
    uint8_t* kv; float* scale; uint16_t* pe;
    const int32_t* table; int64_t width, pages; int page;
    const int32_t* starts; const int32_t* path; const int32_t* kept;
    int most;                                           // entries of a path, up to 64
};

// A workgroup: one sequence.  All rows of its path are in registers before the first is written, so that they may be named in any
// order: 41 pieces a row (32 x 16 bytes of codes, 8 of the rotary key, the scale), up to six a thread.  3.6 us for 64 sequences of up to 61 rows, a
// launch and four dependent waits.
__global__ __launch_bounds__(512) void mla_keep_kernel(KeepArgs p) {
    constexpr int kPieces = 41, N = 6;
    const int b = blockIdx.x, total = max(0, min(p.kept[b], p.most)) * kPieces;
    const int64_t start = p.starts[b];
    const int32_t* entries = p.table + b * p.width;
    v4u hold[N] = {};
    int64_t to[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = threadIdx.x + n * 512, k = i / kPieces, c = i - k * kPieces;
        to[n] = -1;
        if (i < total && start >= 0) {
            const int from = p.path[(int64_t)b * p.most + k];
            const int64_t src = from < 0 ? -1 : page_row(entries, p.width, p.pages, p.page, start + from);
            if (src >= 0) {
                to[n] = page_row(entries, p.width, p.pages, p.page, start + k);
                if (c < 32) hold[n] = *(const v4u*)(p.kv + src * kC + c * 16);
                else if (c < 40) hold[n] = *(const v4u*)(p.pe + src * kRope + (c - 32) * 8);
                else hold[n][0] = f32_as_u32(p.scale[src]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+v"(hold[n]));       // (they have arrived: a barrier alone does not wait for loads)
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = threadIdx.x + n * 512, c = i % kPieces;
        if (to[n] < 0) continue;
        if (c < 32) *(v4u*)(p.kv + to[n] * kC + c * 16) = hold[n];
        else if (c < 40) *(v4u*)(p.pe + to[n] * kRope + (c - 32) * 8) = hold[n];
        else p.scale[to[n]] = u32_as_f32(hold[n][0]);
    }
}

}  // namespace

int launch_mla_latent_paged(const void* a, int64_t a_stride, const void* q_w, const void* kv_w, const void* freqs, const dsv3_mla_pages& cache,
                            const int32_t* starts, const int32_t* counts, void* y, float* ys, int64_t batch, int64_t rows, int q_rank,
                            float q_eps, float kv_eps, hipStream_t st) {
    WriteArgs p;
    p.a = (const uint16_t*)a; p.a_stride = a_stride; p.q_w = (const uint16_t*)q_w; p.kv_w = (const uint16_t*)kv_w; p.freqs = (const v2f*)freqs;
    p.kv = (uint8_t*)cache.kv; p.scale = cache.kv_scale; p.pe = (uint16_t*)cache.pe;
    p.table = cache.table; p.width = cache.table_width; p.pages = cache.pages; p.page = cache.page_size;
    p.starts = starts; p.counts = counts; p.y = (uint8_t*)y; p.ys = ys;
    p.total = batch * rows; p.rows = (int)rows; p.q_rank = q_rank; p.q_eps = q_eps; p.kv_eps = kv_eps;
    const int64_t grid = q_rank ? p.total : (p.total + 3) / 4, threads = q_rank ? 320 : 256;
    if (grid * threads > kMostItems) return DSV3_ERR_BAD_SHAPE;
    if (q_rank) hipLaunchKernelGGL(mla_write_kernel<true>, dim3((unsigned)grid), dim3((unsigned)threads), 0, st, p);
    else hipLaunchKernelGGL(mla_write_kernel<false>, dim3((unsigned)grid), dim3((unsigned)threads), 0, st, p);
    return launch_status();
}

int launch_mla_cache_read(const dsv3_mla_pages& cache, const int32_t* lengths, void* kv, void* pe, int64_t batch, int64_t positions, hipStream_t st) {
    ReadArgs p;
    p.kv = (const uint8_t*)cache.kv; p.scale = cache.kv_scale; p.pe = (const uint16_t*)cache.pe;
    p.table = cache.table; p.width = cache.table_width; p.pages = cache.pages; p.page = cache.page_size;
    p.lengths = lengths; p.out = (uint16_t*)kv; p.out_pe = (uint16_t*)pe;
    p.positions = (int)positions; p.per_seq = (int)((positions + 7) / 8); p.groups = batch * p.per_seq;
    if ((p.groups + 3) / 4 * 256 > kMostItems) return DSV3_ERR_BAD_SHAPE;
    hipLaunchKernelGGL(mla_read_kernel, dim3((unsigned)((p.groups + 3) / 4)), dim3(256), 0, st, p);
    return launch_status();
}

int launch_mla_cache_keep(const dsv3_mla_pages& cache, const int32_t* starts, const int32_t* path, const int32_t* kept, int64_t batch, int most,
                          hipStream_t st) {
    KeepArgs p;
    p.kv = (uint8_t*)cache.kv; p.scale = cache.kv_scale; p.pe = (uint16_t*)cache.pe;
    p.table = cache.table; p.width = cache.table_width; p.pages = cache.pages; p.page = cache.page_size;
    p.starts = starts; p.path = path; p.kept = kept; p.most = most;
    hipLaunchKernelGGL(mla_keep_kernel, dim3((unsigned)batch), dim3(512), 0, st, p);
    return launch_status();
}

}  // namespace dsv3

// mx4_gemm for many rows: tiles of activations and weight rows through LDS.
#include "mla.hpp"
#include "mx4_gemm.hpp"

namespace dsv3 {
namespace {

typedef const __attribute__((address_space(3))) v4u* lds_read16;
// the loaded value is looked at here
__device__ __forceinline__ void there(v2u& x) { asm volatile("" : "+v"(x)); }

struct TileArgs {
    const uint8_t* a; const uint8_t* b;
    const v2u* as; const v2u* bs;                       // scales as the instruction takes them, of 64 rows and 256 along k: a dword per lane for each 32 rows
    void* c; v4f* part;                                 // results, or sums of slices [slice][tile][wavefront][16-byte pieces][lane]
    int m, n, k, units, pack_units;                     // units: of 256 along k, the last one may be half; those that there are scales for
    int tiles_m, tiles_n, per_slice;                    // units of a slice, an even number
};

// ---- scales.  A lane (r, g) = (l % 32, l / 32) of v_mfma_scale_f32_32x32x64_f8f6f4 gives the scale of row r's block g of 32.  Four products
// u = 0 .. 3 take 256 along k; product u multiplies blocks 4 (u / 2) + u % 2 (g = 0) and two further (g = 1), so that its four scales are one dword:
// bytes 2 g, 2 g + 1 of the first 128 and of the second.  Rows and products that are not there get zeros.
struct PackArgs { const uint32_t* a; const uint32_t* b; v2u* as; v2u* bs; int64_t a_groups, b_groups; int m, n, cols, units; };
template <bool A8> __global__ __launch_bounds__(256) void mx4_pack_kernel(PackArgs p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, g = lane >> 5;
    int64_t group = blockIdx.x;
    const bool of_a = group < p.a_groups;
    if (!of_a) group -= p.a_groups;
    const uint32_t* src = of_a ? p.a : p.b;
    const int rows = of_a ? p.m : p.n;
    v2u* dst = (of_a ? p.as : p.bs) + group * p.units * 64 + lane;
    for (int unit = blockIdx.y * 16 + wave; unit < min(p.units, (int)blockIdx.y * 16 + 16); unit += 4) {
        v2u w = {};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int64_t row = group * 64 + t * 32 + r;
            if (row >= rows) continue;
            const uint32_t* s = src + row * p.cols + 2 * unit;
            uint32_t lo = 2 * unit < p.cols ? s[0] : 0u, hi = 2 * unit + 1 < p.cols ? s[1] : 0u;
            if (A8 && of_a) { lo = (lo >> 23 & 0xffu) * 0x01010101u; hi = (hi >> 23 & 0xffu) * 0x01010101u; }
            w[t] = (lo >> (16 * g) & 0xffffu) | (hi >> (16 * g)) << 16;
        }
        dst[(int64_t)unit * 64] = w;
    }
}

// The product of 32 weight rows and 32 activation rows over 64 along k, onto sums that stay in accumulation registers: as builtins with 16 of them the compiler
// moves and spills the sums.  It does not know that these are MFMAs, so what it would keep apart stands here: two wait states in front (an ordinary instruction
// may have written an operand); behind the last one, before a sum is read, sums_there.  SEL: the byte of both scales.
template <int SEL> __device__ __forceinline__ void mfma_codes(v16f& d, v4u w, v4u a, uint32_t sw, uint32_t sa) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
                 : "+a"(d) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SEL & 1), "n"(SEL >> 1));
}
template <int SEL> __device__ __forceinline__ void mfma_codes(v16f& d, v4u w, v8i a, uint32_t sw, uint32_t sa) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:0"
                 : "+a"(d) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SEL & 1), "n"(SEL >> 1));
}
__device__ __forceinline__ void sums_there(v16f& d) { asm volatile("s_nop 15\n\ts_nop 15" : "+a"(d)); }

// ---- the product.  Four wavefronts, 2 x 2, each 32 RT activation rows x 32 CT weight rows.  A stage of LDS holds 128 bytes of every activation row
// (256 codes, or 128 e4m3 ones) and the codes of the weight rows that meet them; chunks of 16 bytes stand at c ^ (row / 2 % 8), in rows of 64 bytes at
// c ^ (row / 4 % 4), so that 16 rows read at one place hit all banks.
template <bool A8, int RT, int CT> struct Geo {
    static constexpr int TM = 64 * RT, TN = 64 * CT;
    static constexpr int SUB = A8 ? 2 : 4;              // products along k of a stage
    static constexpr int WB = A8 ? 64 : 128;            // bytes of a weight row
    static constexpr int SA = TM * 128, SB = TN * WB;
    static constexpr int NA = TM / 32, NB = TN * WB / 4096;             // copies of a wavefront
    static constexpr int LDS = 2 * (SA + SB);
};

template <bool A8, int RT, int CT, int CD, bool SPLIT>
__global__ __launch_bounds__(256, RT * CT >= 16 ? 1 : 2) void mx4_tile_kernel(TileArgs p) {
    using G = Geo<A8, RT, CT>;
    constexpr int SUB = G::SUB, NA = G::NA, NB = G::NB, NC = NA + NB, X = RT * CT;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave & 1, wn = wave >> 1, r = lane & 31, g = lane >> 5;

    // workgroup -> tile: a contiguous run per XCD, in bands of 4 tile rows
    int m0, n0, tile;
    {
        const int T = p.tiles_m * p.tiles_n, x = blockIdx.x % 8, q = T / 8, rest = T % 8;
        tile = x * q + min(x, rest) + blockIdx.x / 8;
        const int band = tile / (4 * p.tiles_n), rows = min(4, p.tiles_m - 4 * band), in = tile - band * 4 * p.tiles_n;
        m0 = (4 * band + in % rows) * G::TM;
        n0 = in / rows * G::TN;
    }
    const int u0 = blockIdx.y * p.per_slice, units = min(p.per_slice, p.units - u0);
    const int steps128 = min(p.k / 128 - 2 * u0, 2 * units);            // of the slice
    const int last = (A8 ? steps128 : units) - 1, stages = last + 2 & ~1;   // an odd one out is followed by itself, with scales of zero

    // ---- copies into LDS
    const uint32_t lds0 = lds_addr_of(lds);
    const uint32_t a_row = A8 ? p.k : p.k / 2, b_row = p.k / 2;
    const uint8_t* a0 = p.a + (int64_t)m0 * a_row + (int64_t)u0 * (A8 ? 256 : 128);
    const uint8_t* b0 = p.b + (int64_t)n0 * b_row + (int64_t)u0 * 128;
    uint32_t a_off[NA], b_off[NB];                      // rows past the end repeat the last one
#pragma unroll
    for (int t = 0; t < NA; ++t) {
        const int row = (wave * NA + t) * 8 + (lane >> 3);
        a_off[t] = min(row, p.m - 1 - m0) * a_row + (((lane & 7) ^ (row >> 1 & 7)) << 4);
    }
#pragma unroll
    for (int t = 0; t < NB; ++t) {
        const int row = A8 ? (wave * NB + t) * 16 + (lane >> 2) : (wave * NB + t) * 8 + (lane >> 3);
        b_off[t] = min(row, p.n - 1 - n0) * b_row + (A8 ? ((lane & 3) ^ (row >> 2 & 3)) << 4 : ((lane & 7) ^ (row >> 1 & 7)) << 4);
    }
    // a last stage of half the codes: the other half is the first once more, its scales are zeros
    const int odd = !A8 && (steps128 & 1);
    auto copy = [&](int s, auto slot, auto which) {
        constexpr int n = decltype(which)::value, S = decltype(slot)::value;
        const int at = min(s, last);
        uint32_t back = 0u;
        if constexpr (!A8) {
            const int t = n < NA ? n : n - NA, row = (wave * (n < NA ? NA : NB) + t) * 8 + (lane >> 3);
            back = odd && at == last && (((lane & 7) ^ (row >> 1 & 7)) & 4) ? 64u : 0u;
        }
        if constexpr (n < NA) copy16(a0 + (int64_t)at * 128, a_off[n] - back, lds0 + S * G::SA + (wave * NA + n) * 1024);
        else copy16(b0 + (int64_t)at * G::WB, b_off[n - NA] - back, lds0 + 2 * G::SA + S * G::SB + (wave * NB + n - NA) * 1024);
    };

    // ---- fragments
    const uint32_t a_rd = lds0 + (wm * 32 * RT + r) * 128, b_rd = lds0 + 2 * G::SA + (wn * 32 * CT + r) * G::WB;
    auto read16 = [](uint32_t at) -> v4u { return *(lds_read16)(uintptr_t)at; };
    uint32_t a_ch[4], b_ch[SUB];               // where the lane's chunk of product u lies in its row
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        // e4m3: halves of blocks u (bytes 32 u + 16 g) and u + 2
        const int c = A8 ? 2 * (u & 1) + 4 * (u >> 1) + g : 4 * (u >> 1) + 2 * g + (u & 1);
        a_ch[u] = a_rd + ((c ^ (r >> 1 & 7)) << 4);
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        const int c = A8 ? 2 * g + u : 4 * (u >> 1) + 2 * g + (u & 1);
        b_ch[u] = b_rd + (A8 ? ((c ^ (r >> 2 & 3)) << 4) : ((c ^ (r >> 1 & 7)) << 4));
    }
    v4u fa[2][RT][A8 ? 2 : 1], fb[2][CT];
    constexpr int NR = (A8 ? 2 : 1) * RT + CT;          // reads of a product's fragments
    auto read = [&](auto slot, auto prod, auto buf, auto which) {
        constexpr int S = decltype(slot)::value, u = decltype(prod)::value, B = decltype(buf)::value, n = decltype(which)::value;
        if constexpr (n < CT) fb[B][n] = read16(b_ch[u] + S * G::SB + n * 32 * G::WB);
        else if constexpr (A8) fa[B][(n - CT) / 2][(n - CT) % 2] = read16(a_ch[u + 2 * ((n - CT) % 2)] + S * G::SA + (n - CT) / 2 * 4096);
        else fa[B][n - CT][0] = read16(a_ch[u] + S * G::SA + (n - CT) * 4096);
    };

    // ---- scales: of a unit, for 64 rows each
    constexpr int GA = (RT + 1) / 2, GB = (CT + 1) / 2;
    const v2u* as = p.as + ((int64_t)((m0 + wm * 32 * RT) / 64) * p.pack_units + u0) * 64 + lane;
    const v2u* bs = p.bs + ((int64_t)((n0 + wn * 32 * CT) / 64) * p.pack_units + u0) * 64 + lane;
    v2u sa[2][GA], sb[2][GB];                           // of the unit in use and the next
    auto load_scales = [&](int unit, auto buf) {
        constexpr int B = decltype(buf)::value;
        const int64_t at = (int64_t)min(unit, p.pack_units - 1 - u0) * 64;
#pragma unroll
        for (int t = 0; t < GA; ++t) sa[B][t] = as[(int64_t)t * p.pack_units * 64 + at];
#pragma unroll
        for (int t = 0; t < GB; ++t) sb[B][t] = bs[(int64_t)t * p.pack_units * 64 + at];
    };
    auto scales_there = [&](auto buf) {
        constexpr int B = decltype(buf)::value;
#pragma unroll
        for (int t = 0; t < GA; ++t) there(sa[B][t]);
#pragma unroll
        for (int t = 0; t < GB; ++t) there(sb[B][t]);
    };

    v16f acc[CT][RT] = {};
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, 1> I1;
    unrolled<NC>([&](auto n) { copy(0, I0(), n); });
    load_scales(0, I0());
    if constexpr (A8) load_scales(1, I1());
    __builtin_amdgcn_s_waitcnt(0x0f70);                 // vmcnt(0)
    scales_there(I0());
    scales_there(I1());
    unrolled<NC>([&](auto n) { copy(1, I1(), n); });
    if constexpr (!A8) load_scales(1, I1());
    barrier_no_fence();
    unrolled<NR>([&](auto n) { read(I0(), I0(), I0(), n); });

    // One stage.  Its last product's fragments are read during the one before; behind the barrier in front of that product the stage is free and the next
    // one is there.
    auto stage = [&](int s, auto slot, auto unit_buf) {
        constexpr int S = decltype(slot)::value, UB = decltype(unit_buf)::value;
        unrolled<SUB>([&](auto prod) {
            constexpr int u = decltype(prod)::value, B = u & 1;
            constexpr bool last = u == SUB - 1;
            if constexpr (last) {
                __builtin_amdgcn_s_waitcnt(0x0070);     // everything that was read and copied is there
                asm volatile("s_barrier" ::: "memory");
                if constexpr (!A8 || S == 0) scales_there(std::integral_constant<int, UB ^ 1>());
            }
            __builtin_amdgcn_sched_barrier(0);
            unrolled<X>([&](auto step) {
                constexpr int x = decltype(step)::value, ct = x / RT, rt = (ct & 1) ? RT - 1 - x % RT : x % RT;
                constexpr int sel = A8 ? 2 * S + u : u;
                const uint32_t ws = sb[UB][ct / 2][ct % 2], xs = sa[UB][rt / 2][rt % 2];
                if constexpr (A8) mfma_codes<sel>(acc[ct][rt], fb[B][ct], __builtin_bit_cast(v8i, __builtin_shufflevector(fa[B][rt][0], fa[B][rt][1], 0, 1, 2, 3, 4, 5, 6, 7)), ws, xs);
                else mfma_codes<sel>(acc[ct][rt], fb[B][ct], fa[B][rt][0], ws, xs);
                // beside it: the next product's fragments, the copies of the stage after the next
                unrolled<NR>([&](auto n) {
                    if constexpr (decltype(n)::value * X / NR == x) {
                        if constexpr (last) read(std::integral_constant<int, S ^ 1>(), I0(), std::integral_constant<int, B ^ 1>(), n);
                        else read(slot, std::integral_constant<int, u + 1>(), std::integral_constant<int, B ^ 1>(), n);
                    }
                });
                if constexpr (last) {
                    unrolled<NC>([&](auto n) {
                        if constexpr (decltype(n)::value * X / NC == x) copy(s + 2, slot, n);
                    });
                    if constexpr (!A8 && x == X - 1) load_scales(s + 2, unit_buf);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
    };
    // (one way out, at the end: otherwise the compiler moves the sums)
    int s = 0;
    do {
        stage(s, I0(), I0());
        stage(s + 1, I1(), std::integral_constant<int, A8 ? 0 : 1>());
        s += 2;
        if constexpr (A8) {
#pragma unroll
            for (int t = 0; t < GA; ++t) sa[0][t] = sa[1][t];
#pragma unroll
            for (int t = 0; t < GB; ++t) sb[0][t] = sb[1][t];
            load_scales(s / 2 + 1, I1());
        }
    } while (s < stages);
    __builtin_amdgcn_s_waitcnt(0x0070);                 // (copies past the end are still on their way into LDS)
    barrier_no_fence();

#pragma unroll
    for (int x = 0; x < X; ++x) sums_there(acc[x / RT][x % RT]);
    // ---- results.  A lane has activation row r, weight rows 8 (e / 4) + 4 g + e % 4 of 32.
    if constexpr (SPLIT) {
        v4f* dst = p.part + (((int64_t)blockIdx.y * p.tiles_m * p.tiles_n + tile) * 4 + wave) * (X * 4 * 64) + lane;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const v16f& o = acc[ct][rt];
                    dst[((ct * RT + rt) * 4 + e) * 64] = v4f{ o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3] };
                }
    } else if constexpr (CD == DSV3_F32) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int row = m0 + (wm * RT + rt) * 32 + r, col = n0 + (wn * CT + ct) * 32 + 4 * g;
                if (row >= p.m) continue;
                float* c = (float*)p.c + (int64_t)row * p.n + col;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (col + 8 * (e / 4) + e % 4 < p.n) c[8 * (e / 4) + e % 4] = acc[ct][rt][e];
            }
    } else {
        // 32 activation rows at a time through LDS, as rows of 64 CT bytes whose 16-byte chunks are xor-ed with the row
        constexpr int RB = CT * 64, CH = CT * 4;        // bytes and chunks of a row
        uint8_t* stg = lds + wave * (32 * RB * (RT > 1 ? 2 : 1));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            uint8_t* at = stg + (rt & 1) * (32 * RB);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const v16f& o = acc[ct][rt];
                    v2u x;
                    if constexpr (CD == DSV3_BF16) x = v2u{ pack_bf16(o[4 * e], o[4 * e + 1]), pack_bf16(o[4 * e + 2], o[4 * e + 3]) };
                    else x = v2u{ pack_f16(o[4 * e], o[4 * e + 1]), pack_f16(o[4 * e + 2], o[4 * e + 3]) };
                    *(v2u*)(at + r * RB + (((4 * ct + e) ^ (r & (CH - 1))) << 4) + 8 * g) = x;
                }
            const int row0 = m0 + (wm * RT + rt) * 32, col0 = n0 + wn * CT * 32;
            auto* c = (uint16_t*)p.c;
            if (p.n % 8 == 0) {
#pragma unroll
                for (int i = 0; i < 32 * CH / 64; ++i) {
                    const int x = i * 64 + lane, lr = x / CH, ch = x % CH;
                    const v4u v = *(const v4u*)(at + lr * RB + ((ch ^ (lr & (CH - 1))) << 4));
                    if (row0 + lr < p.m && col0 + ch * 8 < p.n) *(v4u*)(c + (int64_t)(row0 + lr) * p.n + col0 + ch * 8) = v;
                }
            } else {
                for (int i = 0; i < 32 * RB / 2 / 64; ++i) {
                    const int x = i * 64 + lane, lr = x / (RB / 2), j = x % (RB / 2);
                    const uint16_t v = *(const uint16_t*)(at + lr * RB + (((j >> 3) ^ (lr & (CH - 1))) << 4) + (j & 7) * 2);
                    if (row0 + lr < p.m && col0 + j < p.n) c[(int64_t)(row0 + lr) * p.n + col0 + j] = v;
                }
            }
        }
    }
}

// Slices' sums, added in their order: a thread has the four results of a lane's 16 bytes.
template <int RT, int CT, int CD>
__global__ __launch_bounds__(256) void mx4_join_kernel(const v4f* part, void* out, int m, int n, int tiles_m, int tiles_n, int slices) {
    constexpr int X = RT * CT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x, x = blockIdx.y;      // x: (ct, rt)
    const int band = tile / (4 * tiles_n), rows = min(4, tiles_m - 4 * band), in = tile - band * 4 * tiles_n;
    const int m0 = (4 * band + in % rows) * (64 * RT), n0 = in / rows * (64 * CT);
    const int ct = x / RT, rt = x % RT, wm = wave & 1, wn = wave >> 1;
    const int row = m0 + (wm * RT + rt) * 32 + (lane & 31), col0 = n0 + (wn * CT + ct) * 32 + 4 * (lane >> 5);
    if (row >= m) return;
    const int64_t step = (int64_t)tiles_m * tiles_n * 4 * (X * 4 * 64);
    const v4f* src = part + ((int64_t)tile * 4 + wave) * (X * 4 * 64) + x * 256 + lane;
    auto* c = (typename OutT<CD>::type*)out + (int64_t)row * n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int col = col0 + 8 * e;
        if (col >= n) break;
        v4f s = src[e * 64];
        for (int k = 1; k < slices; ++k) s += src[k * step + e * 64];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < n) c[col + j] = cvt_out<CD>(s[j]);
    }
}

struct Plan { int rt, ct, tiles_m, tiles_n, slices, per_slice, units, pack_units; };
Plan plan_of(int64_t m, int64_t n, int64_t k, bool a8) {
    Plan p;
    p.units = (int)((k + 255) / 256);
    p.pack_units = p.units + 1 & ~1;
    const int64_t big = ((m + 255) / 256) * ((n + 255) / 256);
    p.rt = p.ct = big >= 192 ? 4 : 2;
    p.tiles_m = (int)((m + 64 * p.rt - 1) / (64 * p.rt));
    p.tiles_n = (int)((n + 64 * p.ct - 1) / (64 * p.ct));
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    int64_t slices = tiles >= 192 ? 1 : 256 / tiles;
    slices = slices > p.units / 4 ? p.units / 4 : slices;
    if (slices < 1) slices = 1;
    p.per_slice = (int)((p.units + slices - 1) / slices) + 1 & ~1;
    p.slices = (p.units + p.per_slice - 1) / p.per_slice;
    return p;
}
struct Space { size_t bs, part, bytes; int64_t a_groups, b_groups; };
Space space_of(const Plan& p) {
    Space s;
    s.a_groups = (int64_t)p.tiles_m * p.rt; s.b_groups = (int64_t)p.tiles_n * p.ct;
    s.bs = (size_t)s.a_groups * p.pack_units * 512;
    s.part = s.bs + (size_t)s.b_groups * p.pack_units * 512;
    s.bytes = s.part + (p.slices > 1 ? (size_t)p.slices * p.tiles_m * p.tiles_n * p.rt * p.ct * 4096 * 4 : 0);
    return s;
}

template <bool A8, int RT, int CT, int CD> int launch_tiles(const TileArgs& a, const Plan& plan, hipStream_t st) {
    using G = Geo<A8, RT, CT>;
    static_assert(G::LDS <= 160 * 1024 && 4 * 32 * CT * 64 * (RT > 1 ? 2 : 1) <= G::LDS, "the results leave through the stages");
    const unsigned tiles = (unsigned)plan.tiles_m * plan.tiles_n;
    if (plan.slices == 1) {
        static LdsGrant grant;
        if (!grant.ensure((const void*)mx4_tile_kernel<A8, RT, CT, CD, false>, G::LDS)) return DSV3_ERR_LAUNCH;
        hipLaunchKernelGGL((mx4_tile_kernel<A8, RT, CT, CD, false>), dim3(tiles), dim3(256), G::LDS, st, a);
        return launch_status();
    }
    static LdsGrant grant;
    if (!grant.ensure((const void*)mx4_tile_kernel<A8, RT, CT, DSV3_F32, true>, G::LDS)) return DSV3_ERR_LAUNCH;
    hipLaunchKernelGGL((mx4_tile_kernel<A8, RT, CT, DSV3_F32, true>), dim3(tiles, plan.slices), dim3(256), G::LDS, st, a);
    hipLaunchKernelGGL((mx4_join_kernel<RT, CT, CD>), dim3(tiles, RT * CT), dim3(256), 0, st, (const v4f*)a.part, a.c, a.m, a.n, plan.tiles_m, plan.tiles_n, plan.slices);
    return launch_status();
}
template <bool A8, int CD> int launch_cd(const TileArgs& a, const Plan& plan, hipStream_t st) {
    if (plan.rt == 4) return launch_tiles<A8, 4, 4, CD>(a, plan, st);
    return launch_tiles<A8, 2, 2, CD>(a, plan, st);
}

}  // namespace

bool mx4_tile_takes(int64_t m, int64_t n, int64_t k) {
    // (offsets in a tile are 32 bits, launches and tiles are counted in 31)
    return k > 0 && k <= 1 << 22 && ((m + 127) / 128) * ((n + 127) / 128) <= 1 << 22 && (m + n) / 64 + 8 <= 1 << 24;
}

size_t mx4_tile_workspace_bytes(int64_t m, int64_t n, int64_t k, bool a8) { return space_of(plan_of(m, n, k, a8)).bytes; }

int launch_mx4_tile(const Mx4Args& q, bool a8, int c_dtype, void* workspace, hipStream_t st) {
    const Plan plan = plan_of(q.m, q.n, q.k, a8);
    const Space space = space_of(plan);
    uint8_t* ws = (uint8_t*)workspace;
    PackArgs pk = { (const uint32_t*)q.a_s, (const uint32_t*)q.b_s, (v2u*)ws, (v2u*)(ws + space.bs), space.a_groups, space.b_groups, (int)q.m, (int)q.n, (int)(q.k / 128), plan.pack_units };
    const dim3 grid((unsigned)(space.a_groups + space.b_groups), (unsigned)((plan.pack_units + 15) / 16));
    if (a8) hipLaunchKernelGGL(mx4_pack_kernel<true>, grid, dim3(256), 0, st, pk);
    else hipLaunchKernelGGL(mx4_pack_kernel<false>, grid, dim3(256), 0, st, pk);
    const TileArgs a = { q.a, q.b, pk.as, pk.bs, q.c, (v4f*)(ws + space.part), (int)q.m, (int)q.n, (int)q.k, plan.units, plan.pack_units, plan.tiles_m, plan.tiles_n, plan.per_slice };
    if (c_dtype == DSV3_BF16) return a8 ? launch_cd<true, DSV3_BF16>(a, plan, st) : launch_cd<false, DSV3_BF16>(a, plan, st);
    if (c_dtype == DSV3_F16) return a8 ? launch_cd<true, DSV3_F16>(a, plan, st) : launch_cd<false, DSV3_F16>(a, plan, st);
    return a8 ? launch_cd<true, DSV3_F32>(a, plan, st) : launch_cd<false, DSV3_F32>(a, plan, st);
}

// ---- which kernel takes which sizes

static bool tiles(int64_t m, int64_t n, int64_t k) { return m > 64 && mx4_tile_takes(m, n, k); }

size_t mx4_gemm_workspace_bytes(bool a8, int64_t m, int64_t n, int64_t k) { return tiles(m, n, k) ? mx4_tile_workspace_bytes(m, n, k, a8) : 0; }

int launch_mx4_gemm(const void* a, const void* a_s, bool a8, const void* b, const void* b_s, void* c, int c_dtype, int64_t m, int64_t n, int64_t k,
                    void* workspace, hipStream_t st) {
    const Mx4Args p = { (const uint8_t*)a, a_s, (const uint8_t*)b, (const uint8_t*)b_s, c, m, n, k };
    return tiles(m, n, k) ? launch_mx4_tile(p, a8, c_dtype, workspace, st) : launch_mx4_stream(p, a8, c_dtype, st);
}

}  // namespace dsv3

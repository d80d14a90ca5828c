// mx4_gemm for many rows: tiles of activations and weight rows through LDS.
#include <algorithm>

#include "mla.hpp"
#include "mx4_gemm.hpp"

namespace dsv3 {
namespace {

typedef const __attribute__((address_space(3))) v4u* lds_read16;
typedef const __attribute__((address_space(3))) v2u* lds_read8;

struct TileArgs {
    const uint8_t* a; const uint8_t* b;
    const uint8_t* as; const uint8_t* bs;               // scales as the instruction takes them
    void* c; v4f* part;                                 // results, or sums of slices [slice][tile][wavefront][16-byte pieces][lane]
    int m, n, k, steps, pack_cols;                      // steps: of 128 along k; those that there are scales for
    int tiles_m, tiles_n, per_slice;                    // steps of a slice, an even number
    int whole;                                          // tiles in front of those that two workgroups have
};

// ---- scales.  A lane (r, g) = (l % 32, l / 32) of v_mfma_scale_f32_32x32x64_f8f6f4 gives the scale of row r's block g of 32.  Two products
// u = 0, 1 take 128 along k; product u multiplies blocks u (g = 0) and u + 2 (g = 1), so that a lane's two scales are the bytes 2 g, 2 g + 1 of the row's four.
// They are laid out for 128 rows and 128 along k as 512 bytes, eight for each lane: two for each 32 rows.  Rows that are not there, and what lies behind k, get zeros.
struct PackArgs { const uint32_t* a; const uint32_t* b; v2u* as; v2u* bs; int64_t a_groups, b_groups; int m, n, cols, pack_cols; };
template <bool A8> __global__ __launch_bounds__(256) void mx4_pack_kernel(PackArgs p) {
    constexpr int COLS = 16;                            // of a workgroup
    __shared__ uint32_t rows[128][COLS + 1];
    int64_t group = blockIdx.x;
    const bool of_a = group < p.a_groups;
    if (!of_a) group -= p.a_groups;
    const uint32_t* src = of_a ? p.a : p.b;
    const int64_t have = of_a ? p.m : p.n;
    const int c0 = blockIdx.y * COLS, t = threadIdx.x;
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {                       // 16 rows at a time, a whole piece of each
        const int64_t row = group * 128 + i * 16 + (t >> 4);
        const int col = c0 + (t & 15);
        x[i] = row < have && col < p.cols ? src[row * p.cols + col] : 0u;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) rows[i * 16 + (t >> 4)][t & 15] = A8 && of_a ? (x[i] >> 23 & 0xffu) * 0x01010101u : x[i];
    __syncthreads();
    const int lane = t & 63, r = lane & 31, g = lane >> 5;
    v2u* dst = (of_a ? p.as : p.bs) + (group * p.pack_cols + c0) * 64 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = (t >> 6) + 4 * i;
        if (c0 + c >= p.pack_cols) break;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = rows[j * 32 + r][c] >> (16 * g) & 0xffffu;
        dst[(int64_t)c * 64] = v2u{ w[0] | w[1] << 16, w[2] | w[3] << 16 };
    }
}

// The product of 32 weight rows and 32 activation rows over 64 along k, onto sums that stay in accumulation registers: as builtins with 16 of them the compiler
// moves and spills the sums.  It does not know that these are MFMAs, so what it would keep apart stands here: two wait states in front (an ordinary instruction
// may have written an operand); behind the last one, before a sum is read, sums_there.  SW, SA: the bytes of their scales.
template <int SW, int SA> __device__ __forceinline__ void mfma_codes(v16f& d, v4u w, v4u a, uint32_t sw, uint32_t sa) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                 : "+a"(d) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SW & 1), "n"(SA & 1), "n"(SW >> 1), "n"(SA >> 1));
}
template <int SW, int SA> __device__ __forceinline__ void mfma_codes(v16f& d, v4u w, v8i a, uint32_t sw, uint32_t sa) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:0"
                 : "+a"(d) : "v"(w), "v"(a), "v"(sw), "v"(sa), "n"(SW & 1), "n"(SA & 1), "n"(SW >> 1), "n"(SA >> 1));
}
__device__ __forceinline__ void sums_there(v16f& d) { asm volatile("s_nop 15\n\ts_nop 15" : "+a"(d)); }

// Two copies of 1 KiB, to lds_addr and the KiB behind it (the second one's offset counts for both its addresses)
__device__ __forceinline__ void copy16_two(const void* base, uint32_t off, uint32_t off_less_1024, uint32_t lds_addr) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:1024"
                 :: "v"(off), "v"(off_less_1024), "s"(base), "s"(lds_addr) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_copies() {        // all but the N youngest
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
    asm volatile("" ::: "memory");
}

// ---- the product.  Four wavefronts, 2 x 2, each 32 RT activation rows x 32 CT weight rows.  A stage of LDS holds 128 along k: rows of 64 bytes, or 128 of
// e4m3 activations, whose chunks of 16 bytes stand at c ^ (row / 4 % 4) and c ^ (row / 2 % 8), so that 16 rows read at one place hit all banks.
//
// D stages, D - 1 on their way (more make no tile faster).  A compute unit has one tile of 256 x 256, or two of 128 x 128, whose barriers and copies stand beside each other's products.
//
// Measured, mx4 x mx4: 4096 x 7168 -> 18432 in 272 .. 294 us by card (3.7 .. 4.0 PFLOP/s), 4096 x 18432 -> 7168 in 262 .. 271 (4.0 .. 4.1); e4m3 x mx4
// 367 .. 389 and 360 .. 375.  1.75 rounds of tiles cost the second 12 %.  The products alone, with neither copies nor reads, would take
// 200 and 180 us at the 1.85 GHz that the chip's power leaves: the copies cost 50 us more, the reads 20.  More stages on their way change nothing there (three
// or four), nor do stages of twice the length.
// LAID: scales as mx4_pack_kernel lays them out; else a wavefront fetches 16 bytes of each of 64 rows every four stages, into one place of two.
template <bool A8, int RT, int CT, int D, bool LAID> struct Geo {
    static constexpr int TM = 64 * RT, TN = 64 * CT;
    static constexpr int AB = A8 ? 128 : 64, WB = 64;   // bytes of a row
    static constexpr int SA = TM * AB, SB = TN * WB;
    static constexpr int GA = (TM + 127) / 128, GB = (TN + 127) / 128;  // 128 rows whose scales come in as one
    static constexpr int SS = LAID ? (GA + GB + 1 & ~1) * 512 : 4096;
    static constexpr int NA = SA / 4096, NB = SB / 4096, NS = LAID ? (GA + GB + 1) / 2 : 1, NC = NA + NB + (LAID ? NS : 0);      // copies of a wavefront for each stage
    static constexpr int B0 = D * SA, S0 = B0 + D * SB, LDS = S0 + (LAID ? D : 2) * SS;
    static_assert(LAID || D <= 4, "two places for scales");
    static_assert(NA * 4096 == SA && NB * 4096 == SB, "whole copies for every wavefront");
    static_assert((D - 1) * NC < 64, "no more copies than can be counted");
};

// One of `blocks` workgroups, PARTS a tile of 64 RT x 64 CT PARTS, from tile `first` on.
template <bool A8, int RT, int CT, int D, bool LAID, int CD, bool SPLIT, int PARTS>
__device__ __forceinline__ void mx4_tile(const TileArgs& p, int block, int first, int blocks) {
    using G = Geo<A8, RT, CT, D, LAID>;
    constexpr int NA = G::NA, NB = G::NB, NC = G::NC, X = RT * CT;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave & 1, wn = wave >> 1, r = lane & 31, g = lane >> 5;

    // workgroup -> tile: a contiguous run per XCD, in bands of 4 tile rows (of 2 or 8 up to 5 % more, of 16 up to 6 %)
    int m0, n0, tile;
    {
        const int x = block % 8, q = blocks / 8, rest = blocks % 8, at = x * q + min(x, rest) + block / 8;
        tile = first + at / PARTS;
        const int band = tile / (4 * p.tiles_n), rows = min(4, p.tiles_m - 4 * band), in = tile - band * 4 * p.tiles_n;
        m0 = (4 * band + in % rows) * G::TM;
        n0 = (in / rows * PARTS + at % PARTS) * G::TN;
        if (PARTS > 1 && n0 >= p.n) return;
    }
    const int k0 = blockIdx.y * p.per_slice, last = min(p.per_slice, p.steps - k0) - 1;
    const int stages = last + 2 & ~1;                   // an odd one out (LAID) is followed by itself, with scales of zero

    // ---- copies into LDS
    const uint32_t lds0 = lds_addr_of(lds);
    const uint32_t a_row = A8 ? p.k : p.k / 2, b_row = p.k / 2;
    // (addresses from 1024 in front, which the second copy of two takes off)
    const uint8_t* a0 = p.a + (int64_t)m0 * a_row + (int64_t)k0 * G::AB - 1024;
    const uint8_t* b0 = p.b + (int64_t)n0 * b_row + (int64_t)k0 * G::WB - 1024;
    constexpr int AR = 1024 / G::AB, BR = 16;           // rows of a copy; those past the end repeat the last one
    uint32_t a_off[NA], b_off[NB];
#pragma unroll
    for (int t = 0; t < NA; ++t) {
        const int row = (wave * NA + t) * AR + lane / (64 / AR), c = A8 ? lane & 7 ^ row >> 1 & 7 : lane & 3 ^ row >> 2 & 3;
        a_off[t] = min(row, p.m - 1 - m0) * a_row + c * 16 + 1024 - (t & 1) * 1024;
    }
#pragma unroll
    for (int t = 0; t < NB; ++t) {
        const int row = (wave * NB + t) * BR + lane / 4, c = lane & 3 ^ row >> 2 & 3;
        b_off[t] = min(row, p.n - 1 - n0) * b_row + c * 16 + 1024 - (t & 1) * 1024;
    }
    // scales: 512 bytes for each 128 rows, wavefronts 0 and 1 (2 and 3) one group's halves; or four bytes of each of a wavefront's 64 rows, activations' first
    const uint8_t* sc0[G::NS];
    uint32_t sc_off = 0;
    if constexpr (LAID) {
#pragma unroll
        for (int i = 0; i < G::NS; ++i) {
            const int group = min(2 * i + (wave >> 1), G::GA + G::GB - 1);
            sc0[i] = (group < G::GA ? p.as + ((int64_t)(m0 / 128 + group) * p.pack_cols + k0) * 512 : p.bs + ((int64_t)(n0 / 128 + group - G::GA) * p.pack_cols + k0) * 512) + (wave & 1) * 256;
        }
    } else {
        const int row0 = wave < RT ? wave * 64 : min(wave - RT, CT - 1) * 64;
        sc0[0] = (wave < RT ? p.as + (int64_t)m0 * (p.k / 32) : p.bs + (int64_t)n0 * (p.k / 32)) + (int64_t)k0 * 4;
        sc_off = (uint32_t)min(row0 + lane, (wave < RT ? p.m - m0 : p.n - n0) - 1) * (uint32_t)(p.k / 32);
    }
    // requests of a stage: two copies each (or what is left), then the scales
    constexpr int QA = (NA + 1) / 2, QB = (NB + 1) / 2, NQ = QA + QB + G::NS;
    auto copy = [&](int s, int slot, auto phase, auto which) {          // phase: s % 4
        constexpr int n = decltype(which)::value;
        const int at = min(s, last);
        if constexpr (n < QA) {
            const uint32_t to = lds0 + slot * G::SA + (wave * NA + 2 * n) * 1024;
            if constexpr (2 * n + 1 < NA) copy16_two(a0 + (int64_t)at * G::AB, a_off[2 * n], a_off[2 * n + 1], to);
            else copy16(a0 + (int64_t)at * G::AB, a_off[2 * n], to);
        } else if constexpr (n < QA + QB) {
            constexpr int t = 2 * (n - QA);
            const uint32_t to = lds0 + G::B0 + slot * G::SB + (wave * NB + t) * 1024;
            if constexpr (t + 1 < NB) copy16_two(b0 + (int64_t)at * G::WB, b_off[t], b_off[t + 1], to);
            else copy16(b0 + (int64_t)at * G::WB, b_off[t], to);
        } else {                                        // (LAID: of the stage past an odd one out, zeros)
            constexpr int i = n - QA - QB;
            if constexpr (!LAID) {
                if constexpr (decltype(phase)::value % 4 == 0) copy16(sc0[0] + (int64_t)(at >> 2) * 16, sc_off, lds0 + G::S0 + (s >> 2 & 1) * G::SS + wave * 1024);
            }
            else copy4(sc0[i] + (int64_t)min(s, p.pack_cols - 1 - k0) * 512, lane * 4, lds0 + G::S0 + slot * G::SS + i * 1024 + wave * 256);
        }
    };
    // They are spread over the stage's last product and the next stage's first one: this many of them in the former
    auto early = [](int n) constexpr { return n * 2 * X / NQ < X; };

    // ---- fragments and scales
    auto read16 = [](uint32_t at) -> v4u { return *(lds_read16)(uintptr_t)at; };
    // where the lane's chunk of product u lies in a stage, beside the wavefront's first row
    uint32_t a_ch[A8 ? 4 : 2], b_ch[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) b_ch[u] = r * 64 + ((2 * g + u ^ r >> 2 & 3) << 4);
#pragma unroll
    for (int u = 0; u < (A8 ? 4 : 2); ++u)              // e4m3: halves g of blocks u and u + 2
        a_ch[u] = A8 ? r * 128 + ((2 * (u & 1) + 4 * (u >> 1) + g ^ r >> 1 & 7) << 4) : b_ch[u];
    const uint32_t a_rd = lds0 + wm * 32 * RT * G::AB, b_rd = lds0 + G::B0 + wn * 32 * CT * G::WB;
    // the wavefront's tiles in a lane's eight bytes of 128 rows (tiles of 64 rows may be the second half of them), or its rows' four bytes
    const uint32_t as_at = lds0 + G::S0 + (LAID ? (wm * RT / 4) * 512 + ((m0 / 32 + wm * RT) & 3) * 2 + lane * 8 : (wm * RT * 32 + r) * 16);
    const uint32_t bs_at = lds0 + G::S0 + (LAID ? (G::GA + wn * CT / 4) * 512 + ((n0 / 32 + wn * CT) & 3) * 2 + lane * 8 : (64 * RT + wn * CT * 32 + r) * 16);
    // Activations' fragments in two sets, the weight's too where there are few products; else each is read anew behind its last product, RT (CT - 1) of them before
    // it is needed.
    constexpr bool ONE = X >= 16;
    v4u fa[2][RT][A8 ? 2 : 1], fb[ONE ? 1 : 2][CT];
    constexpr int PER = LAID ? 2 : 1;                // tiles a dword of scales
    uint32_t sa[2][(RT + PER - 1) / PER], sb[2][(CT + PER - 1) / PER];  // of the stage in use and the next
    auto read_scales = [&](int s, int slot, auto phase) {               // of stage s
        constexpr int B = decltype(phase)::value & 1;
        const uint32_t place = LAID ? slot * G::SS : (s >> 2 & 1) * G::SS + (decltype(phase)::value & 3) * 4;
        auto some = [&](uint32_t at, auto& x, auto tiles) {
            constexpr int n = decltype(tiles)::value;
            if constexpr (!LAID) unrolled<n>([&](auto t) { x[decltype(t)::value] = *(lds_u32)(uintptr_t)(at + decltype(t)::value * 512); });
            else if constexpr (n == 4) { const v2u v = *(lds_read8)(uintptr_t)at; x[0] = v[0]; x[1] = v[1]; }
            else if constexpr (n == 2) x[0] = *(lds_u32)(uintptr_t)at;
            else x[0] = *(const __attribute__((address_space(3))) uint16_t*)(uintptr_t)at;
        };
        some(as_at + place, sa[B], std::integral_constant<int, RT>());
        some(bs_at + place, sb[B], std::integral_constant<int, CT>());
    };
    // (what is read as it lies: the lane's two bytes of four, the exponent of a binary32)
    auto turn_scales = [&](auto buf) {
        constexpr int B = decltype(buf)::value;
        if constexpr (!LAID) {
#pragma unroll
            for (int t = 0; t < RT; ++t) sa[B][t] = A8 ? sa[B][t] >> 23 & 0xffu : sa[B][t] >> (16 * g);
#pragma unroll
            for (int t = 0; t < CT; ++t) sb[B][t] >>= 16 * g;
        }
    };
    constexpr int NRA = (A8 ? 2 : 1) * RT, NR = NRA + CT;               // reads of a product's fragments
    auto read = [&](int slot, auto prod, auto buf, auto which) {
        constexpr int u = decltype(prod)::value, B = decltype(buf)::value, n = decltype(which)::value;
        if constexpr (n >= NRA) fb[ONE ? 0 : B][n - NRA] = read16(b_ch[u] + (b_rd + slot * G::SB) + (n - NRA) * 32 * G::WB);
        else if constexpr (A8) fa[B][n / 2][n % 2] = read16(a_ch[u + 2 * (n % 2)] + (a_rd + slot * G::SA) + n / 2 * 32 * G::AB);
        else fa[B][n][0] = read16(a_ch[u] + (a_rd + slot * G::SA) + n * 32 * G::AB);
    };
    // behind which product it is read
    auto read_at = [](int n) constexpr { return ONE ? (n < NRA ? n * 8 / NRA : (n - NRA) * RT + RT - 1) : n * X / NR; };

    v16f acc[CT][RT] = {};
    typedef std::integral_constant<int, 0> I0;
    typedef std::integral_constant<int, 1> I1;
    unrolled<D>([&](auto d) {
        constexpr int i = decltype(d)::value;
        unrolled<NQ>([&](auto n) {
            if constexpr (i < D - 1 || early(decltype(n)::value)) copy(i, i, d, n);
        });
    });
    wait_copies<(D - 2) * NC>();                        // (and of the last stage's those that are on their way)
    barrier_no_fence();
    read_scales(0, 0, I0());
    turn_scales(I0());
    unrolled<NR>([&](auto n) { read(0, I0(), I0(), n); });

    // One stage.  Its last product's fragments are read during the one before; behind the barrier in front of that product the stage is free and the next
    // one is there.
    int slot = 0, before = D - 1;                       // the stage's place and that of the one in front of it
    auto stage = [&](int s, auto phase) {               // phase: s % 4, or s % 2
        constexpr int F = decltype(phase)::value, P = F & 1;
        // requests for scales among those of the D - 2 stages behind the next one
        constexpr int MORE = LAID ? 0 : (D > 2 && (F + 2) % 4 == 0) + (D > 3 && (F + 3) % 4 == 0);
        const int next = slot + 1 == D ? 0 : slot + 1;
        unrolled<2>([&](auto prod) {
            constexpr int u = decltype(prod)::value, B = u & 1;
            constexpr bool last = u == 1;
            if constexpr (last) {
                wait_copies<(D - 2) * NC + MORE>();     // the next stage's, of this wavefront
                barrier_no_fence();                     // and of all; what was read is there
            }
            __builtin_amdgcn_sched_barrier(0);
            unrolled<X>([&](auto step) {
                constexpr int x = decltype(step)::value, ct = x / RT, rt = (ct & 1) ? RT - 1 - x % RT : x % RT;
                const uint32_t ws = sb[P][ct / PER], xs = sa[P][rt / PER];
                constexpr int ws_at = LAID ? 2 * (ct & 1) + u : u, xs_at = LAID ? 2 * (rt & 1) + u : A8 ? 0 : u;
                if constexpr (A8) mfma_codes<ws_at, xs_at>(acc[ct][rt], fb[ONE ? 0 : B][ct], __builtin_bit_cast(v8i, __builtin_shufflevector(fa[B][rt][0], fa[B][rt][1], 0, 1, 2, 3, 4, 5, 6, 7)), ws, xs);
                else mfma_codes<ws_at, xs_at>(acc[ct][rt], fb[ONE ? 0 : B][ct], fa[B][rt][0], ws, xs);
                // beside it: the next product's fragments, the copies of the stage that takes this one's place
                if constexpr (last && x == 0) read_scales(s + 1, next, std::integral_constant<int, F + 1>());
                if constexpr (last && x == X - 1) turn_scales(std::integral_constant<int, P ^ 1>());
                unrolled<NR>([&](auto n) {
                    if constexpr (read_at(decltype(n)::value) == x) {
                        if constexpr (last) read(next, I0(), std::integral_constant<int, B ^ 1>(), n);
                        else read(slot, std::integral_constant<int, u + 1>(), std::integral_constant<int, B ^ 1>(), n);
                    }
                });
                unrolled<NQ>([&](auto n) {
                    constexpr int y = decltype(n)::value * 2 * X / NQ;
                    if constexpr (last && y == x) copy(s + D, slot, std::integral_constant<int, F + D>(), n);
                    if constexpr (!last && y == X + x) copy(s - 1 + D, before, std::integral_constant<int, F - 1 + D>(), n);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        before = slot;
        slot = next;
    };
    // (one way out, at the end: otherwise the compiler moves the sums)
    int s = 0;
    do {
        stage(s, I0());
        stage(s + 1, I1());
        if constexpr (!LAID) {
            stage(s + 2, std::integral_constant<int, 2>());
            stage(s + 3, std::integral_constant<int, 3>());
        }
        s += LAID ? 2 : 4;
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

template <bool A8, int RT, int CT, int D, bool LAID, int CD, bool SPLIT>
__global__ __launch_bounds__(256, 1) void mx4_tile_kernel(TileArgs p) {
    if constexpr (RT == 4) {
        if ((int)blockIdx.x >= p.whole) {
            mx4_tile<A8, 4, 2, D, LAID, CD, SPLIT, 2>(p, blockIdx.x - p.whole, p.whole, gridDim.x - p.whole);
            return;
        }
        mx4_tile<A8, RT, CT, D, LAID, CD, SPLIT, 1>(p, blockIdx.x, 0, p.whole);
    } else {
        mx4_tile<A8, RT, CT, D, LAID, CD, SPLIT, 1>(p, blockIdx.x, 0, gridDim.x);
    }
}

// Slices' sums, added in their order: a thread has the four results of a lane's 16 bytes.
template <int RT, int CT, int CD>
__global__ __launch_bounds__(256) void mx4_join_kernel(const v4f* part, void* out, int m, int n, int tiles_m, int tiles_n, int slices) {
    constexpr int X = RT * CT, MOST = 8;                // loads at once
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x, x = blockIdx.y >> 2, e = blockIdx.y & 3;    // x: (ct, rt)
    const int band = tile / (4 * tiles_n), rows = min(4, tiles_m - 4 * band), in = tile - band * 4 * tiles_n;
    const int m0 = (4 * band + in % rows) * (64 * RT), n0 = in / rows * (64 * CT);
    const int ct = x / RT, rt = x % RT, wm = wave & 1, wn = wave >> 1;
    const int row = m0 + (wm * RT + rt) * 32 + (lane & 31), col = n0 + (wn * CT + ct) * 32 + 8 * e + 4 * (lane >> 5);
    if (row >= m || col >= n) return;
    const int64_t step = (int64_t)tiles_m * tiles_n * 4 * (X * 4 * 64);
    const v4f* src = part + ((int64_t)tile * 4 + wave) * (X * 4 * 64) + x * 256 + e * 64 + lane;
    v4f s = {};
    for (int k = 0; k < slices; k += MOST) {
        v4f v[MOST];
#pragma unroll
        for (int j = 0; j < MOST; ++j) v[j] = src[min(k + j, slices - 1) * step];
#pragma unroll
        for (int j = 0; j < MOST; ++j)
            if (k + j < slices) s = k + j ? s + v[j] : v[j];
    }
    auto* c = (typename OutT<CD>::type*)out + (int64_t)row * n + col;
    if (CD != DSV3_F32 && n % 4 == 0) {
        *(v2u*)c = CD == DSV3_BF16 ? v2u{ pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]) } : v2u{ pack_f16(s[0], s[1]), pack_f16(s[2], s[3]) };
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < n) c[j] = cvt_out<CD>(s[j]);
}

struct Plan { int rt, ct, tiles_m, tiles_n, whole, slices, per_slice, steps, pack_cols; bool laid; double time; };
Plan plan_of(int64_t m, int64_t n, int64_t k, bool a8) {
    Plan p;
    p.steps = (int)(k / 128);
    p.pack_cols = p.steps + 1 & ~1;
    // Tiles of 256 where their rounds take less time: a round of one each takes 1.03 us a step (e4m3 1.40), one of two small ones 0.78 (1.0), of one half of that,
    // and where there are no whole rounds of those the next ones fill them.  Of a last round that is half empty each tile goes to two workgroups, 0.58 of the
    // time: 4096 x 7168 -> 18432 (4.5 rounds) 272 us in place of 284, e4m3 367 for 379, 2304 x 7168 -> 9216 (1.27) 91 for 116.  2000 x 7168 -> 7168: 61 us with 224
    // tiles of 256 and 82 with 896 small ones; 1024 x 7168 -> 18432 98 with 256 tiles and 32 in halves, 116 with small ones (e4m3: 123 and 135); 2048 x 7168 -> 4096
    // 43 with 128 in halves and 49; 1024 x 7168 -> 4096 32 with 64 in halves and 26 with 256 small ones.  The costs are of k = 7168 and count steps alone: 4096 x 2048 -> 7168 takes 47
    // and 52, 4096 x 512 -> 32768 111 and 129, but 1024 x 512 -> 32768 29 and 26, and 512 x 7168 -> 18432 gets small tiles, 73, where large ones take 57.
    const int64_t large = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128), left = large % 256;
    const bool halves = left > 0 && left <= 128;
    const double rounds = (double)((large + 255) / 256) - (halves ? 0.42 : 0.0), some = small > 512 ? small / 512.0 : small > 256 ? 1.0 : 0.5;
    p.rt = p.ct = rounds * (a8 ? 1.40 : 1.03) < some * (a8 ? 1.0 : 0.78) ? 4 : 2;
    if (m <= 64) p.rt = 1;
    p.tiles_m = (int)((m + 64 * p.rt - 1) / (64 * p.rt));
    p.tiles_n = (int)((n + 64 * p.ct - 1) / (64 * p.ct));
    p.whole = (int)((int64_t)p.tiles_m * p.tiles_n - (p.rt == 4 && halves ? left : 0));
    // Slices of k where compute units would have no tile, if the shorter way pays for their sums, a launch that adds them and 8 bytes an element and slice, written and
    // read at 5 TB/s: with scales laid out in front, 300 x 7168 -> 2304 in 19.2 us with four and 21.0 without, 128 x 16384 -> 7168 29.4 and 54; 256 x 2048 ->
    // 7168 9.9 without, 18.4 with two, 300 x 4096 -> 4096 14.7 and 18.1.  A step of a tile by itself on its unit takes 0.38 us (e4m3 0.47).
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    const double step = a8 ? 0.47 : 0.38;
    double least = 1e30;
    int64_t slices = 1;
    for (int64_t x = 1; x == 1 || (p.rt != 4 && x * tiles <= 256 && x * 2 <= p.steps); ++x) {
        const double time = (double)((p.steps + x - 1) / x) * step + (x > 1 ? 5.0 + (double)x * m * n * 8 / 5e6 : 0.0);
        if (time < least) { least = time; slices = x; }
    }
    const int whole = k % 512 != 0 ? 2 : 4;             // stages that the kernel does at once
    p.per_slice = ((int)((p.steps + slices - 1) / slices) + whole - 1) / whole * whole;
    p.slices = (p.steps + p.per_slice - 1) / p.per_slice;
    // Small tiles fetch their scales from where they lie, 16 bytes a row, where rows begin at multiples of that: without the launch that lays them out 64 x 512 ->
    // 32768 takes 5.1 us in place of 8.2, 500 x 7168 -> 4096 19.2 for 21.8, 64 x 16384 -> 7168 21 for 27, 1024 x 7168 -> 4096 24.8 for 25.0 (four bytes a row every
    // stage would take 34 there).
    p.laid = p.rt == 4 || k % 512 != 0;
    p.time = 3.0 + (p.laid ? 5.0 : 0.0) + (p.rt == 4 ? rounds * p.steps * (a8 ? 1.40 : 1.03) : tiles > 256 ? std::max(1.0, tiles / 512.0) * p.steps * (a8 ? 1.0 : 0.78) : least);
    return p;
}
struct Space { size_t bs, part, bytes; int64_t a_groups, b_groups; };
Space space_of(const Plan& p) {
    Space s;
    s.a_groups = p.laid ? ((int64_t)p.tiles_m * p.rt + 1) / 2 : 0; s.b_groups = p.laid ? ((int64_t)p.tiles_n * p.ct + 1) / 2 : 0;
    s.bs = (size_t)s.a_groups * p.pack_cols * 512;
    s.part = s.bs + (size_t)s.b_groups * p.pack_cols * 512;
    s.bytes = s.part + (p.slices > 1 ? (size_t)p.slices * p.tiles_m * p.tiles_n * p.rt * p.ct * 4096 * 4 : 0);
    return s;
}

template <bool A8, int RT, int CT, int D, bool LAID, int CD> int launch_tiles(const TileArgs& a, const Plan& plan, hipStream_t st) {
    using G = Geo<A8, RT, CT, D, LAID>;
    static_assert(G::LDS <= 160 * 1024 && 4 * 32 * CT * 64 * (RT > 1 ? 2 : 1) <= G::LDS, "the results leave through the stages");
    const unsigned tiles = (unsigned)plan.tiles_m * plan.tiles_n;
    if (plan.slices == 1) {
        static LdsGrant grant;
        if (!grant.ensure((const void*)mx4_tile_kernel<A8, RT, CT, D, LAID, CD, false>, G::LDS)) return DSV3_ERR_LAUNCH;
        hipLaunchKernelGGL((mx4_tile_kernel<A8, RT, CT, D, LAID, CD, false>), dim3(2 * tiles - plan.whole), dim3(256), G::LDS, st, a);
        return launch_status();
    }
    if constexpr (RT < 4) {
        static LdsGrant grant;
        if (!grant.ensure((const void*)mx4_tile_kernel<A8, RT, CT, D, LAID, DSV3_F32, true>, G::LDS)) return DSV3_ERR_LAUNCH;
        hipLaunchKernelGGL((mx4_tile_kernel<A8, RT, CT, D, LAID, DSV3_F32, true>), dim3(tiles, plan.slices), dim3(256), G::LDS, st, a);
        hipLaunchKernelGGL((mx4_join_kernel<RT, CT, CD>), dim3(tiles, RT * CT * 4), dim3(256), 0, st, (const v4f*)a.part, a.c, a.m, a.n, plan.tiles_m, plan.tiles_n, plan.slices);
    }
    return launch_status();
}
template <bool A8, int CD> int launch_cd(const TileArgs& a, const Plan& plan, hipStream_t st) {
    if (plan.rt == 4) return launch_tiles<A8, 4, 4, A8 ? 3 : 4, true, CD>(a, plan, st);
    if (plan.rt == 1) return plan.laid ? launch_tiles<A8, 1, 2, A8 ? 4 : 6, true, CD>(a, plan, st) : launch_tiles<A8, 1, 2, 4, false, CD>(a, plan, st);
    return plan.laid ? launch_tiles<A8, 2, 2, A8 ? 3 : 4, true, CD>(a, plan, st) : launch_tiles<A8, 2, 2, A8 ? 3 : 4, false, CD>(a, plan, st);
}

}  // namespace

size_t mx4_tile_workspace_bytes(int64_t m, int64_t n, int64_t k, bool a8) { return space_of(plan_of(m, n, k, a8)).bytes; }

int launch_mx4_tile(const Mx4Args& q, bool a8, int c_dtype, void* workspace, hipStream_t st) {
    const Plan plan = plan_of(q.m, q.n, q.k, a8);
    const Space space = space_of(plan);
    // (what launches hold)
    if ((int64_t)plan.tiles_m * plan.tiles_n > 0xffffff || space.a_groups + space.b_groups > 0xffffff) return DSV3_ERR_BAD_SHAPE;
    uint8_t* ws = (uint8_t*)workspace;
    TileArgs a = { q.a, q.b, (const uint8_t*)q.a_s, q.b_s, q.c, (v4f*)(ws + space.part), (int)q.m, (int)q.n, (int)q.k, plan.steps, plan.pack_cols, plan.tiles_m, plan.tiles_n, plan.per_slice, plan.whole };
    if (plan.laid) {
        PackArgs pk = { (const uint32_t*)q.a_s, (const uint32_t*)q.b_s, (v2u*)ws, (v2u*)(ws + space.bs), space.a_groups, space.b_groups, (int)q.m, (int)q.n, (int)(q.k / 128), plan.pack_cols };
        const dim3 grid((unsigned)(space.a_groups + space.b_groups), (unsigned)((plan.pack_cols + 15) / 16));
        if (a8) hipLaunchKernelGGL(mx4_pack_kernel<true>, grid, dim3(256), 0, st, pk);
        else hipLaunchKernelGGL(mx4_pack_kernel<false>, grid, dim3(256), 0, st, pk);
        a.as = ws;
        a.bs = ws + space.bs;
    }
    if (c_dtype == DSV3_BF16) return a8 ? launch_cd<true, DSV3_BF16>(a, plan, st) : launch_cd<false, DSV3_BF16>(a, plan, st);
    if (c_dtype == DSV3_F16) return a8 ? launch_cd<true, DSV3_F16>(a, plan, st) : launch_cd<false, DSV3_F16>(a, plan, st);
    return a8 ? launch_cd<true, DSV3_F32>(a, plan, st) : launch_cd<false, DSV3_F32>(a, plan, st);
}

// ---- which kernel takes which sizes

// Up to 32 rows the weight is streamed, and beyond where that takes less time: every workgroup of mx4_stream_kernel reads its weight rows and 32 activation rows, all
// of them at some 12 TB/s.  64 x 7168 -> 2112: 8.5 us streamed and 9.5 in tiles; 100 x 7168 -> 2112 10.0 and 11.6; 128 x 7168 -> 576 5.3 and 9.9; 300 x 2048 -> 7168
// 16.9 and 8.2; 64 x 512 -> 32768, many workgroups, 9.7 and 5.0; 128 x 2048 -> 7168 9.1 and 8.2, e4m3 13.7 and 9.3.  Of 40 sizes with both kinds of activations 77 of 80 get a way
// within 5 % of the better one; 90 x 4096 -> 4096 of e4m3 does not, 12.4 in tiles and 9.5 streamed, and 200 x 7168 -> 2112, 16.0 and 12.9.
static bool tiles(int64_t m, int64_t n, int64_t k, bool a8) {
    if (m <= 32 || k == 0) return false;
    const int64_t strip = n >= 6144 ? 32 : 16, groups = (n + strip - 1) / strip * ((m + 31) / 32);
    const double time = 3.0 + groups * 0.0015 + (double)groups * (strip * (k / 2) + 32 * (a8 ? k : k / 2)) / 12e6;
    return groups > 65535 || plan_of(m, n, k, a8).time < time;
}

size_t mx4_gemm_workspace_bytes(bool a8, int64_t m, int64_t n, int64_t k) { return tiles(m, n, k, a8) ? mx4_tile_workspace_bytes(m, n, k, a8) : 0; }

int launch_mx4_gemm(const void* a, const void* a_s, bool a8, const void* b, const void* b_s, void* c, int c_dtype, int64_t m, int64_t n, int64_t k,
                    void* workspace, hipStream_t st) {
    const Mx4Args p = { (const uint8_t*)a, a_s, (const uint8_t*)b, (const uint8_t*)b_s, c, m, n, k };
    return tiles(m, n, k, a8) ? launch_mx4_tile(p, a8, c_dtype, workspace, st) : launch_mx4_stream(p, a8, c_dtype, st);
}

}  // namespace dsv3

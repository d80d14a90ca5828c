// Attention of MLA.forward for one new token or a tree of drafted ones per sequence (reference: inference/model.py:480-497), on the cache
// in pages of e4m3 rows (mla_paged.hip), in the absorbed form of mla_decode.hip: behind the query's fold through wkv_b
//   attend   one range of a sequence's positions for 128 or 64 of its (token, head) rows: scores, softmax, weighted sum; binary32 partial sums
//   fold     mla_fold.hpp
// Codes are turned into bf16 operands in front of the matrix cores, exactly (a power of two times four bits): the folded query and
// the exponentials are rounded to bf16, scores and sums stay in binary32.
#include <type_traits>

#include "mla.hpp"
#include "mla_fold.hpp"
#include "paged.hpp"

namespace dsv3 {
namespace {

constexpr int kTile = 32;                               // positions per tile
constexpr int kRopeOff = kTile * kC;                    // a stage: 32 rows of 512 codes, 32 rotary keys of 128 B, four groups of eight scales, 256 B each
constexpr int kScaleOff = kRopeOff + kTile * kRope * 2;
constexpr int kStage = kScaleOff + 1024;
constexpr int kStages = 6;                              // tiles in LDS, computed or on their way
constexpr int kCopies = 6;                              // of a tile, by each of the four wavefronts
constexpr int kKeys = 4, kValues = 6;                   // reads from LDS ahead of the MFMAs that take them: keys (a read is two K steps), values
constexpr int kSync = 27;                               // the value step behind which a tile's stage is free and the next tile's keys are read

struct PagedArgs {
    const void* ql;                                     // folded queries [batch][rows][512], rows = tokens * heads, or in operand order
    const uint16_t* q;                                  // queries [batch][rows][192]: their rotary part is read here
    const v2f* freqs;                                   // [batch][tokens][32] (cos, sin)
    const uint8_t* kv; const float* scales; const uint8_t* pe;
    const int32_t* table; int64_t width, pages;
    const int32_t* starts; const int32_t* counts;
    const int64_t* tree;                                // [batch][tokens], or nullptr: a token sees those in front of it and itself
    float* part;                                        // [range][row block][row][512]
    v2f* ml;                                            // [range][row block][row] (maximum, sum)
    v2i* plan;                                          // [batch] (first range, ranges)
    int batch, tokens, rows, heads, positions, page, groups, blocks, ranges;        // groups: of 32 rows, in whole 128s; ranges: at most
    uint32_t page_magic;                                // for quotient()
    float scale;
};

// Rows that are no page's: zeros, with a scale that no row has.
struct alignas(16) Nothing { uint8_t kv[8 * kC]; uint8_t pe[8 * kRope * 2]; float scale[8]; };
__device__ const Nothing nothing = { {}, {}, { -1.f, -1.f, -1.f, -1.f, -1.f, -1.f, -1.f, -1.f } };

// Loads that the compiler may make scalar: `p` is written by nobody while the kernel runs.
typedef const __attribute__((address_space(4))) int32_t* const_ints;
__device__ __forceinline__ int scalar_load(const int32_t* p, int64_t at) { return ((const_ints)(uintptr_t)p)[at]; }

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// sums of lanes 0 .. l
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xf>(v);                         // row_shr 1, 2, 4, 8; then the rows' last values (row_bcast 15, 31)
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Which positions a workgroup takes.  The lengths are on the device, so every workgroup divides the work by itself: `per` tiles a
// range, the fewest with which all sequences' ranges are at most p.ranges, ranges numbered through the sequences.
struct Share { int b, first, ranges, per, used; };      // sequence (-1: none), its first range and ranges, tiles a range, ranges of all
template <class F> __device__ __forceinline__ Share share_of(const PagedArgs& p, int lane, F which, bool write_plan) {
    auto tiles = [&](int b) -> int {
        if (b >= p.batch) return 0;
        const SeqSpan s = seq_span(p.starts[b], p.counts[b], p.tokens, p.positions);
        return s.count > 0 ? (s.end + kTile - 1) / kTile : 0;
    };
    const int mine = tiles(lane);
    auto sum = [&](auto f) -> int {
        int n = f(mine);
        for (int b0 = 64; b0 < p.batch; b0 += 64) n += f(tiles(b0 + lane));
        return wave_total(n);
    };
    const int all = sum([](int t) { return t; });
    Share s = { -1, 0, 0, max(1, (all + p.ranges - 1) / p.ranges), 0 };
    for (;;) {
        const int per = s.per;
        s.used = sum([per](int t) { return (t + per - 1) / per; });
        if (s.used <= p.ranges) break;
        // a sequence's last range is half full on average: what these take off the ranges does not change with `per`
        const int lost = s.used - all / per, left = max(1, p.ranges - lost);
        s.per = max(per + 1, min(all / left, per + per / 4));
    }
    const int range = which(s.used);
    int base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const int t = b0 ? tiles(b0 + lane) : mine, n = (t + s.per - 1) / s.per, upto = base + wave_scan(n);
        if (write_plan && b0 + lane < p.batch) p.plan[b0 + lane] = v2i{ upto - n, n };
        const uint64_t past = __ballot(upto > range);
        if (past && s.b < 0 && range >= 0) {
            const int l = __builtin_ctzll(past);
            s.b = b0 + l;
            s.ranges = __builtin_amdgcn_readlane(n, l);
            s.first = __builtin_amdgcn_readlane(upto, l) - s.ranges;
            if (!write_plan) break;
        }
        base = __builtin_amdgcn_readlane(upto, 63);
    }
    return s;
}

// two codes of a dword times a power of two, as bf16
template <bool HI> __device__ __forceinline__ uint32_t codes_to_bf16(uint32_t c, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)c, s, HI));
}
__device__ __forceinline__ v4u operand(uint32_t lo, uint32_t hi, float s) {
    return v4u{ codes_to_bf16<false>(lo, s), codes_to_bf16<true>(lo, s), codes_to_bf16<false>(hi, s), codes_to_bf16<true>(hi, s) };
}

// mla_decode_kernel's maps (mla_decode.hip) on codes: four wavefronts, 32 rows' queries and 32 x 512 sums each; S^T = K Q^T, O^T += V^T P^T.
// A lane's 16 bytes of a key row are the operands of two K steps: step 2 n takes features 32 n + 16 g .. + 7 of lane half g, step 2 n + 1
// the eight behind them.  Values are read transposed, eight positions of a feature per lane; the positions' scales go into the
// exponentials (before these are rounded).
// G tiles side by side: the G wavefronts of a group of 32 rows take every G-th tile and add their sums in LDS at the end.
template <bool PACK, int G>
__global__ __launch_bounds__(256, 1) void mla_paged_kernel(PagedArgs p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int RB = 4 / G, R = kStages / G;          // row groups of a workgroup; steps that the stages hold
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 31, g = lane >> 5, rg = wave % RB, par = wave / RB;
    // a contiguous run of the ranges in use per XCD, the row blocks of a range next to each other: its rows are in the XCD's L2
    int unit = -1;
    const Share mine = share_of(p, lane, [&](int used) -> int {
        const int T = used * p.blocks, q = T / 8, r = T % 8, x = blockIdx.x % 8, k = blockIdx.x / 8;
        if (k < q + (x < r)) unit = x * q + min(x, r) + k;
        return unit < 0 ? -1 : unit / p.blocks;
    }, blockIdx.x == 0 && wave == 0);
    if (mine.b < 0) return;
    const int range = unit / p.blocks, blk = unit - range * p.blocks, b = mine.b;
    const SeqSpan seq = seq_span(scalar_load(p.starts, b), scalar_load(p.counts, b), p.tokens, p.positions);
    const int live = seq.count * p.heads;               // rows behind these are of tokens that the sequence does not have
    if (blk * (RB * 32) >= live) return;
    const int t0 = (range - mine.first) * mine.per, t1 = min((seq.end + kTile - 1) / kTile, t0 + mine.per);
    const int row0 = blk * (RB * 32) + rg * 32;
    const int row = min(row0 + i, p.rows - 1);          // rows past the end repeat the last one; fold leaves them out

    // A wavefront copies eight rows of a tile, which lie in one page: four KiB of latents, a KiB of rotary keys, the scales (by
    // all lanes, for what the first eight fetch).  Rows past the sequence's end are its last one again; what is no page's comes from `nothing`,
    // so that every tile is as many copies, whose outstanding ones can be counted.
    const uint32_t lds0 = lds_addr_of(lds);
    const int32_t* entries = p.table + b * p.width;
    struct Source { const uint8_t* kv; const uint8_t* pe; const float* scales; int last; uint32_t at; };
    auto entry_of = [&](int t) -> int {                 // the page number of the wavefront's rows of tile t (past the end: of the last ones)
        return scalar_load(entries, quotient(min(t * kTile + wave * 8, seq.end - 1), p.page, p.page_magic));
    };
    auto source = [&](int t, int entry, int stage) -> Source {
        const int pos = t * kTile + wave * 8;
        Source s = { nothing.kv, nothing.pe, nothing.scale, 0, lds0 + stage * kStage };
        if (t < t1 && pos < seq.end && (uint32_t)entry < (uint64_t)p.pages) {
            const int64_t r = (int64_t)entry * p.page + (pos - quotient(pos, p.page, p.page_magic) * p.page);
            s.kv = p.kv + r * kC;
            s.pe = p.pe + r * (kRope * 2);
            s.scales = p.scales + r;
            s.last = min(7, seq.end - 1 - pos);
        }
        return s;
    };
    auto issue = [&](const Source& s, auto which) {
        constexpr int n = decltype(which)::value;
        if constexpr (n < 4) {                          // row r's chunk c of 16 bytes lies at c ^ r (low four bits)
            const int r = 2 * n + (lane >> 5);
            copy16(s.kv, min(r, s.last) * kC + (((lane & 31) ^ ((wave * 8 + r) & 15)) << 4), s.at + wave * 4096 + n * 1024);
        } else if constexpr (n == 4) {                  // chunk c at c ^ r / 2 (low three bits)
            const int r = lane >> 3;
            copy16(s.pe, min(r, s.last) * (kRope * 2) + (((lane & 7) ^ (((wave * 8 + r) >> 1) & 7)) << 4), s.at + kRopeOff + wave * 1024);
        } else {
            copy4(s.scales, min(lane & 7, s.last) * 4, s.at + kScaleOff + wave * 256);
        }
    };
    for (int n = 0; n < (R - 1) * G; ++n) {
        const Source s = source(t0 + n, entry_of(t0 + n), n);
        unrolled<kCopies>([&](auto k) { issue(s, k); });
    }

    v4u Q[36];
    {
        // (packed, a last block's missing rows hold anything; nobody reads their results)
        const v4u* src = (const v4u*)p.ql + (PACK ? ((int64_t)b * p.groups + row0 / 32) * (kC / 16) * 64 + i : ((int64_t)b * p.rows + row) * (kC / 8));
#pragma unroll
        for (int n = 0; n < 16; ++n) {
            Q[2 * n] = src[PACK ? (2 * n + g) * 64 : 4 * n + 2 * g];
            Q[2 * n + 1] = src[PACK ? (2 * n + g) * 64 + 32 : 4 * n + 2 * g + 1];
        }
        const uint16_t* rsrc = p.q + ((int64_t)b * p.rows + row) * kQd + kNope + 8 * g;
        const v2f* fr = p.freqs + ((int64_t)b * p.tokens + row / p.heads) * (kRope / 2) + 4 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            Q[32 + s] = *(const v4u*)(rsrc + 16 * s);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const v2f cs = fr[8 * s + e];
                const float re = bf16lo_to_f32(Q[32 + s][e]), im = bf16hi_to_f32(Q[32 + s][e]);
                Q[32 + s][e] = pack_bf16(re * cs.x - im * cs.y, re * cs.y + im * cs.x);
            }
        }
    }

    const uint32_t kaddr = i * kC + ((g ^ (i & 15)) << 4);                      // pair n: ^ (2 n mod 16) << 4
    const uint32_t raddr = kRopeOff + i * 128 + ((g ^ ((i >> 1) & 7)) << 4);    // ^ 2 s << 4
    // transposed reads: lane group q2 of a half takes 16 features; its lane l fetches eight of row l / 2 of 4 g .. + 3, 8 + 4 g .. + 3
    const int l15 = lane & 15, q2 = (lane >> 4) & 1, vrow = 8 * (l15 >> 3) + 4 * g + ((l15 >> 1) & 3);
    const uint32_t vaddr = vrow * kC + ((q2 ^ vrow) << 4) + 8 * (l15 & 1);

    v16f O[16] = {};
    float m = -__builtin_inff(), l = 0.f;               // running maximum of the scores, this lane's share of the sum
    const float scale2 = p.scale * 1.44269504088896340736f;
    // The reads' order and place are those that are written here (sched_barrier); a step's operand is made from its codes beside the MFMA
    // in front of it: four conversions take no time there (33.6 cycles instead of 33.1), six do (38.6).
    v4u keys[kKeys];
    float sc;                                           // the scale of position i
    auto key = [&](const uint8_t* base, int x) -> v4u {
        return x < 16 ? *(const v4u*)(base + (kaddr ^ ((x & 7) << 5)) + (x >> 3) * 256) : *(const v4u*)(base + (raddr ^ ((x - 16) << 5)));
    };
    auto scale_at = [&](const uint8_t* base) { return *(const float*)(base + kScaleOff + (i >> 3) * 256 + (i & 7) * 4); };
    // the next step's tiles are there, once this wavefront's copies of them are (those of the steps behind it stay in flight) and everybody's
    auto arrived = [&] {
        constexpr int left = (R - 2) * kCopies * G;
        __builtin_amdgcn_s_waitcnt(0x0f70 | (left & 15) | (left >> 4) << 14);   // vmcnt
        barrier_no_fence();
    };
    // One tile.  copy: beside the MFMA just issued.  The last value steps read the next tile's first keys.
    auto tile = [&](int t, const uint8_t* base, const uint8_t* next, auto copy) {
        const uint32_t vbase = lds_addr_of(base) + vaddr;
        v2i values[kValues];
        auto value = [&](int y) -> v2i {                // positions 16 (y / 16) .. of features 32 (y % 16) ..
            return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(uintptr_t)((vbase ^ ((y & 7) << 5)) + ((y >> 3) & 1) * 256 + (y >> 4) * 8192));
        };
        v4f w[4];
        v16f T[1];
        v16f& S = T[0];
        v4u cur = operand(keys[0][0], keys[0][1], sc);
        __builtin_amdgcn_sched_barrier(0);
        unrolled<36>([&](auto step) {
            constexpr int s = decltype(step)::value;
            if constexpr (s == 0) mfma32_first(S, cur, Q[0]);
            else mfma32_next(S, cur, Q[s]);
            if constexpr (s < 31 && s % 2 == 0) cur = operand(keys[s / 2 % kKeys][2], keys[s / 2 % kKeys][3], sc);
            else if constexpr (s < 31) cur = operand(keys[(s + 1) / 2 % kKeys][0], keys[(s + 1) / 2 % kKeys][1], sc);
            else if constexpr (s < 35) cur = keys[(s - 15) % kKeys];
            if constexpr (s < 32 && s % 2 == 0 && s / 2 + kKeys < 20) keys[s / 2 % kKeys] = key(base, s / 2 + kKeys);
            if constexpr (s >= 26 && s < 26 + 4) w[s - 26] = *(const v4f*)(base + kScaleOff + (s - 26) * 256 + g * 16);
            if constexpr (s >= 30) values[s - 30] = value(s - 30);
            copy(step);
            __builtin_amdgcn_sched_barrier(0);
        });
        scores_ready(S);
        // positions that nobody sees: past the end, of no page (a row that was not finite has scores of NaN already)
        const int left = seq.end - t * kTile;
        uint32_t there = ~(uint32_t)__ballot(sc < 0.f);
        if (left < kTile) there &= left > 0 ? (1u << left) - 1u : 0u;
        if (there != ~0u || t * kTile + kTile > seq.start) {
            const int j0 = t * kTile - seq.start;       // the tile's first position among the new ones
            uint32_t seen = there;
            if (j0 > -kTile) {
                int tok = row / p.heads;
                asm volatile("" : "+v"(tok));           // (formed here: there are no registers to keep it in)
                const uint64_t bits = p.tree ? (uint64_t)p.tree[(int64_t)b * p.tokens + tok] : (2ull << tok) - 1;
                seen &= j0 >= 64 ? 0u : j0 >= 0 ? (uint32_t)(bits >> j0) : (uint32_t)(bits << -j0) | ((1u << -j0) - 1u);
            }
            seen >>= 4 * g;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!(seen >> (8 * (e >> 2) + (e & 3)) & 1)) S[e] = -__builtin_inff();
        }
        float mx = S[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, S[e]);
        const v2f both = halves32(mx);
        mx = fmaxf(both.x, both.y);
        // the maximum is raised as in mla_decode_kernel: when it grows by more than 2^64, and not for rows that nobody reads
        const bool raise = row0 + i < live && ((mx - m) * scale2 > 64.f || (m == -__builtin_inff() && mx > m));
        if (__any(raise)) {
            const float mn = fmaxf(m, mx);
            const float a = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m - mn) * scale2);
            l *= a;
            m = mn;
            if (t >= t0 + G) {
#pragma unroll
                for (int d = 0; d < 16; ++d) scale_agprs(O[d], a);
                asm volatile("s_nop 7" ::: "memory");
            }
        }
        const float off = softmax_offset(T, m, scale2);
        if (__any(sc != sc)) {                          // NaN times an exponential of zero: these rows' codes are zeros, the scores say who sees them
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e >> 2][e & 3] = w[e >> 2][e & 3] == w[e >> 2][e & 3] ? w[e >> 2][e & 3] : 0.f;
        }
        float sum = 0.f;
        v4u P[2];
        auto weights = [&](int e) {                     // two positions' exponentials
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e], scale2, -off));
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e + 1], scale2, -off));
            sum += x + y;
            P[e >> 3][(e & 7) >> 1] = pack_bf16(x * w[e >> 2][e & 3], y * w[e >> 2][(e & 3) + 1]);
        };
#pragma unroll
        for (int e = 0; e < 8; e += 2) weights(e);
        cur = operand((uint32_t)values[0][0], (uint32_t)values[0][1], 1.0f);
        __builtin_amdgcn_sched_barrier(0);
        unrolled<32>([&](auto step) {
            constexpr int s = decltype(step)::value;
            O[s & 15] = mfma32(cur, P[s >> 4], O[s & 15]);
            if constexpr (s < 31) cur = operand((uint32_t)values[(s + 1) % kValues][0], (uint32_t)values[(s + 1) % kValues][1], 1.0f);
            if constexpr (s + kValues < 32) values[s % kValues] = value(s + kValues);
            if constexpr (s < 12 && s % 3 == 2) weights(8 + s / 3 * 2);         // the second half's, beside the first half's products
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (s == kSync) {                 // this tile's last codes are in registers: its stage is free behind the barrier
                arrived();
                sc = scale_at(next);
            }
            if constexpr (s >= kSync && s - kSync < kKeys) {
                keys[s - kSync] = key(next, s - kSync);
                __builtin_amdgcn_sched_barrier(0);
            }
        });
        l += sum;
#pragma unroll
        for (int d = 0; d < 16; ++d) asm volatile("" : "+a"(O[d]));     // (the sums stay where they are)
    };

    arrived();
    sc = scale_at(lds + par * kStage);
#pragma unroll
    for (int x = 0; x < kKeys; ++x) keys[x] = key(lds + par * kStage, x);
    int st = 0, entry[G];
#pragma unroll
    for (int j = 0; j < G; ++j) entry[j] = entry_of(t0 + (R - 1) * G + j);
    for (int t = t0; t < t1; t += G) {
        const int st_next = st + 1 == R ? 0 : st + 1, st_free = st == 0 ? R - 1 : st - 1;
        // Copies into the stage of the step before, which is free, every few MFMAs: the four wavefronts take turns on the compute unit's load
        // path.  Page numbers are loaded a step ahead of the copies that need them.
        Source ahead[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            ahead[j] = source(t + (R - 1) * G + j, entry[j], st_free * G + j);
            entry[j] = entry_of(t + R * G + j);
        }
        tile(t + par, lds + (st * G + par) * kStage, lds + (st_next * G + par) * kStage, [&](auto step) {
            constexpr int s = decltype(step)::value, E = 4 / G;
            if constexpr (s % E == E - 1 && s / E < kCopies * G) issue(ahead[s / E / kCopies], std::integral_constant<int, s / E % kCopies>());
        });
        st = st_next;
    }

    const v2f parts = halves32(l);
    l = parts.x + parts.y;
    const int64_t slot = ((int64_t)range * p.blocks + blk) * (RB * 32);         // the workgroup's rows among all
    __builtin_amdgcn_s_waitcnt(0x0f70);                 // (copies of the tiles past the range are still on their way into the stages)
    barrier_no_fence();
    // The sums leave as in mla_decode_kernel: 64 features of 32 rows at a time through LDS (16-byte chunks xor-ed with the row); the G
    // wavefronts of a row group first add theirs, each for 32 / G of the rows.
    v2f* const table = (v2f*)(lds + 65536);             // (maximum, sum) [wavefront][row]
    constexpr int N = 8 / G;
    float wt[N][G];
    if constexpr (G == 1) {
        if (g == 0) p.ml[slot + rg * 32 + i] = v2f{ m, l };
    } else {
        if (g == 0) table[wave * 32 + i] = v2f{ m, l };
        barrier_no_fence();
        auto weigh = [&](int r, float (&w)[G]) -> v2f { // row r's weights; its maximum and sum
            v2f x[G];
            float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
            for (int j = 0; j < G; ++j) { x[j] = table[(rg + RB * j) * 32 + r]; top = fmaxf(top, x[j].x); }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                w[j] = x[j].x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((x[j].x - top) * scale2);
                sum += x[j].y * w[j];
            }
            return v2f{ top, sum };
        };
#pragma unroll
        for (int n = 0; n < N; ++n) weigh(4 * (par * N + n) + (lane >> 4), wt[n]);
        if (par == 0) {
            float w[G];
            const v2f ml = weigh(i, w);
            if (g == 0) p.ml[slot + rg * 32 + i] = ml;
        }
    }
    float* dst = p.part + (slot + rg * 32 + par * (4 * N) + (lane >> 4)) * kC + (lane & 15) * 4;
    auto put = [&](int d2) {                            // two buffers a wavefront: the next 64 features are written while these are read
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const v16f& o = O[2 * d2 + (c >> 2)];
            const int e = 4 * (c & 3);
            *(v4f*)(lds + wave * 16384 + (d2 & 1) * 8192 + i * 256 + (((2 * c + g) ^ (i & 15)) << 4)) = v4f{ o[e], o[e + 1], o[e + 2], o[e + 3] };
        }
    };
    put(0);
#pragma unroll
    for (int d2 = 0; d2 < 8; ++d2) {
        if constexpr (G > 1) barrier_no_fence();        // everybody's are there, and the buffers written next have been read
        v4f x[N][G];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const int r = 4 * (par * N + n) + (lane >> 4);
                x[n][j] = *(const v4f*)(lds + (rg + RB * j) * 16384 + (d2 & 1) * 8192 + r * 256 + (((lane & 15) ^ (r & 15)) << 4));
            }
        if (d2 < 7) put(d2 + 1);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v4f v = x[n][0];
            if constexpr (G > 1) {
                v = v * wt[n][0];
#pragma unroll
                for (int j = 1; j < G; ++j) v += x[n][j] * wt[n][j];
            }
            *(v4f*)(dst + n * 4 * kC + d2 * 64) = v;
        }
    }
}

// Row blocks of 128 (token, head) rows, or of 64 with two tiles side by side; one workgroup a compute unit (its registers take a whole one).
struct PagedPlan { int side, groups; int64_t blocks, ranges; };
PagedPlan paged_plan(int64_t batch, int64_t rows) {
    PagedPlan a;
    a.side = rows <= 64 ? 2 : 1;
    a.groups = (int)((rows + 127) / 128 * 4);
    a.blocks = (rows + 128 / a.side - 1) / (128 / a.side);
    // Ranges of all sequences: as many as there are compute units for the row blocks; where the sequences alone are more than half of
    // these, room for the longer ones to be cut.
    const int64_t units = a.blocks < 256 ? 256 / a.blocks : 1;
    a.ranges = batch <= units / 2 ? units : batch + units / 2;
    return a;
}
// Folded queries, partial sums, their maxima and sums, the division of the work
struct PagedSpace { size_t part, ml, plan, bytes; };
PagedSpace paged_space(const PagedPlan& a, int64_t batch) {
    const int64_t rows = a.ranges * a.blocks * (128 / a.side);
    PagedSpace s;
    s.part = (size_t)(batch * a.groups * (32 * kC * 2));
    s.ml = s.part + (size_t)(rows * kC * 4);
    s.plan = s.ml + (size_t)(rows * 8);
    s.bytes = s.plan + (size_t)(batch * 8);
    return s;
}

template <int G> int launch_paged(const PagedArgs& a, bool pack, unsigned grid, hipStream_t st) {
    static void (*const kernels[2])(PagedArgs) = { mla_paged_kernel<false, G>, mla_paged_kernel<true, G> };
    static LdsGrant grant[2];
    constexpr int bytes = kStages * kStage;
    static_assert(bytes >= 65536 + 1024 && bytes <= 160 * 1024, "the sums leave through the stages");
    if (!grant[pack].ensure((const void*)kernels[pack], bytes)) return DSV3_ERR_LAUNCH;
    hipLaunchKernelGGL(kernels[pack], dim3(grid), dim3(256), bytes, st, a);
    return DSV3_OK;
}

}  // namespace

size_t mla_decode_paged_workspace_bytes(int64_t batch, int64_t tokens, int heads) { return paged_space(paged_plan(batch, tokens * heads), batch).bytes; }

int launch_mla_decode_paged(const void* q, const void* freqs, const dsv3_mla_pages& cache, const int32_t* starts, const int32_t* counts,
                            const int64_t* tree, const void* w, const float* ws, void* y, float* ys, int64_t batch, int64_t tokens,
                            int64_t positions, int heads, float scale, void* workspace, hipStream_t st) {
    const int64_t rows = tokens * heads;
    const PagedPlan plan = paged_plan(batch, rows);
    const PagedSpace space = paged_space(plan, batch);
    if (plan.ranges * plan.blocks > 0xfffff0 || batch * tokens > 0x7fffffff - 16) return DSV3_ERR_BAD_SHAPE;
    PagedArgs a;
    uint8_t* wsp = (uint8_t*)workspace;
    a.ql = wsp; a.q = (const uint16_t*)q; a.freqs = (const v2f*)freqs;
    a.kv = (const uint8_t*)cache.kv; a.scales = cache.kv_scale; a.pe = (const uint8_t*)cache.pe;
    a.table = cache.table; a.width = cache.table_width; a.pages = cache.pages;
    a.starts = starts; a.counts = counts; a.tree = tree;
    a.part = (float*)(wsp + space.part); a.ml = (v2f*)(wsp + space.ml); a.plan = (v2i*)(wsp + space.plan);
    a.batch = (int)batch; a.tokens = (int)tokens; a.rows = (int)rows; a.heads = heads; a.positions = (int)positions;
    a.page = cache.page_size; a.groups = plan.groups; a.blocks = (int)plan.blocks; a.ranges = (int)plan.ranges;
    a.page_magic = magic_of(positions, cache.page_size);
    a.scale = scale;
    // operand order up to 16 tokens in all, which is what the kernel that writes it takes (mla_decode.hip)
    const bool pack = batch * tokens <= 16;
    const int rc = pack ? launch_wkv_b_absorb_q_packed(q, (int64_t)heads * kQd, kQd, w, ws, wsp, batch, tokens, a.groups / 4, heads, kNope, kNope, st)
                        : launch_wkv_b_absorb(q, (int64_t)heads * kQd, kQd, w, ws, wsp, DSV3_ABSORB_Q, batch * tokens, heads, kNope, kNope, kC, st);
    if (rc != DSV3_OK) return rc;
    const unsigned grid = (unsigned)((plan.ranges * plan.blocks + 7) / 8 * 8);
    const int launched = plan.side == 1 ? launch_paged<1>(a, pack, grid, st) : launch_paged<2>(a, pack, grid, st);
    if (launched != DSV3_OK) return launched;
    FoldArgs f = {};
    f.part = a.part; f.ml = a.ml; f.plan = a.plan; f.counts = counts; f.w = (const uint8_t*)w; f.ws = ws; f.y = y; f.ys = ys;
    f.tokens = (int)(batch * tokens); f.per_seq = (int)tokens; f.heads = heads; f.rows = 128 / plan.side; f.blocks = a.blocks;
    f.scale = scale;
    return launch_fold<true>(f, st);
}

}  // namespace dsv3

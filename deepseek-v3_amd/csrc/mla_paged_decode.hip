// Attention of MLA.forward for one new token or a tree of drafted ones per sequence (reference: inference/model.py:480-497), on the cache
// in pages of e4m3 rows (mla_paged.hip), in the absorbed form of mla_decode.hip: behind the query's fold through wkv_b
//   attend   one range of a sequence's positions for 128 of its (token, head) rows: scores, softmax, weighted sum; binary32 partial sums
//   fold     mla_fold.hpp
// The matrix cores take the codes as they are.  What meets them is two codes an element as well (split_codes), with scales of powers of two that
// the products apply: the folded query, split by the kernel that folds it (wkv_b_absorb.hip), and the exponentials times their
// position's scale, split here.  A pair of codes is off by 2^-9 of the value, where bf16 would be by 2^-8, and of the smallest values by
// 2^-21 of the largest beside them.  Scores and sums are binary32.
#include <type_traits>

#include "mla.hpp"
#include "mla_fold.hpp"
#include "paged.hpp"

namespace dsv3 {
namespace {

constexpr int kTile = 64;                               // positions per tile
// A stage: 64 rows of 512 codes, 64 rotary keys of 128 B, eight groups of eight scales, 256 B each.  Two neighbouring rows are a KiB, as they are
// copied, the odd one with its chunks of 16 bytes c at c ^ 4; the eight pairs of 16 rows stand 32 bytes further apart than that, pairs 2, 3, 6 and 7
// another 16.  Sixteen rows read at the same place (the scores) then hit sixteen different chunks of 256 bytes, and so do the eight rows of two
// neighbouring chunks that half a wavefront's transposed read takes (0 .. 3 and 8 .. 11, or 4 .. 7 and 12 .. 15 of sixteen), all from a few
// addresses a phase with constants added.
constexpr int kPair = 2 * kC + 32, kRows16 = 34 * 256;
constexpr int pair_off(int p) { return p * kPair + ((p >> 1) & 1) * 16; }       // of 0 .. 7
static_assert(pair_off(7) + 2 * kC <= kRows16, "16 rows");
constexpr int kRopeOff = 4 * kRows16;
constexpr int kScaleOff = kRopeOff + kTile * kRope * 2;
constexpr int kStage = kScaleOff + 8 * 256;
constexpr int kStages = 3;                              // tiles in LDS: the one whose values and the one whose keys are read, one on its way
constexpr int kLds = kStages * kStage;
// A stage of a wavefront by itself: the rotary keys of its last 32 rows only, the others come into registers.
constexpr int kFewScaleOff = kRopeOff + kTile / 2 * kRope * 2;
constexpr int kFewStage = kFewScaleOff + 8 * 256;
constexpr int kFewLds = 4 * kFewStage;

struct PagedArgs {
    const uint8_t* ql;                                  // folded queries in codes [batch][rows][first, second][512], rows = tokens * heads, or in operand order
    const uint8_t* qe;                                  // their exponents [batch][rows][8]
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
    uint32_t page_magic;                                // 2^31 / (page / 8) rounded up: pos / page = (pos / 8 * page_magic) / 2^31 for the positions that there are
    float scale;                                        // of the softmax, times log2 e
};

// The scale of rows that are no page's, which no row has (positive: exponentials times it keep their sign).
constexpr float kNothing = 0x1p-126f;
constexpr float kNoScore = -0x1.fffffep127f;            // the exponents' offset in front of a row's first score
__device__ const float nothing[8] = { kNothing, kNothing, kNothing, kNothing, kNothing, kNothing, kNothing, kNothing };
__device__ const v4u nothing_key[kRope / 8] = {};

// Loads that the compiler may make scalar: `p` is written by nobody while the kernel runs.
typedef const __attribute__((address_space(4))) int32_t* const_ints;
__device__ __forceinline__ int scalar_load(const int32_t* p, uint32_t at) { return ((const_ints)(uintptr_t)p)[at]; }

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
// range, with which all sequences' ranges are at most p.ranges, ranges numbered through the sequences.  The search for it goes upwards in steps of up to a
// quarter and does not go back: with many more ranges than sequences it finds the fewest, with few (8 sequences of 250 .. 2001 positions, 10 ranges) in a fifth
// of the cases only, elsewhere up to a fifth more.  A range counts for p.blocks workgroups, also where its sequence has fewer rows than the widest; those
// without any return at once.
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
    // (uniform, which the compiler does not see)
    return Share{ __builtin_amdgcn_readfirstlane(s.b), __builtin_amdgcn_readfirstlane(s.first), __builtin_amdgcn_readfirstlane(s.ranges),
                  __builtin_amdgcn_readfirstlane(s.per), s.used };
}

// v_mfma_scale_f32_32x32x64_f8f6f4 of codes with its result in ordinary registers (mla.hpp: mfma32_first).  a's scale: byte 0 of sa; b's: byte B of sb.
// Bytes 0 .. 15 of both lane halves share the scale that the low lanes hold, bytes 16 .. 31 that of the high lanes.  (As a builtin with a sum of zero
// the compiler puts the result over the operands, which are still being read.)
template <int B> __device__ __forceinline__ void mfma64_first(v16f& d, v8i a, v8i b, int sa, int sb) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel:[0,%5,0] op_sel_hi:[0,%6,0] cbsz:0 blgp:0"
                 : "=&v"(d) : "v"(a), "v"(b), "v"(sa), "v"(sb), "n"(B & 1), "n"(B >> 1));
}
template <int B> __device__ __forceinline__ void mfma64_next(v16f& d, v8i a, v8i b, int sa, int sb) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[0,%5,0] op_sel_hi:[0,%6,0] cbsz:0 blgp:0"
                 : "+v"(d) : "v"(a), "v"(b), "v"(sa), "v"(sb), "n"(B & 1), "n"(B >> 1));
}
// the same with its sum in accumulation registers, byte 0 of both scales
__device__ __forceinline__ void mfma64_sum(v16f& d, v8i a, v8i b, int sa, int sb) {
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:0 blgp:0" : "+a"(d) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}
// a * b, and zero where a or b is (v_mul_legacy_f32): also beside a scale of NaN (the codes of such a row are zeros, the scores say who sees it)
extern "C" __device__ float dsv3_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
// the lane's number, formed where it is needed: nothing that goes by it stays in a register for the loop
__device__ __forceinline__ int lane_now() {
    int l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(l));
    return l;
}
__device__ __forceinline__ v8i join(v4u a, v4u b) {
    return __builtin_bit_cast(v8i, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Four wavefronts with all 512 registers of their SIMD lane each: a wavefront holds 32 rows' folded queries as pairs of codes (128 registers) and their
// 32 x 512 weighted sums (256).  Transposed products as in mla_decode_kernel (mla_decode.hip): S^T = K Q^T leaves a row in one lane and the lane
// 32 further (position 8 (e / 4) + 4 g + e % 4 of 32 in register e of lane half g), O^T += V^T P^T takes it from there.  Per tile of 64 positions, in two
// halves of 32: 2 x (16 products of 64 features with the two codes of the query, 4 of the rotary part in bf16), 16 x 2 products of 64
// positions: 72 MFMAs, 4350 cycles.
// One wavefront a SIMD issues an instruction every 5 cycles or so: turning each code into a bf16 operand in every wavefront (256 conversions per 32
// positions beside 68 MFMAs, the form before this one) bound it at 4200 cycles per 32 positions.
// Three phases a tile, in which the exponentials of one half stand beside the other half's or the next tile's scores:
//   C  scores of the second half      | exponentials of the first half
//   A  scores of the next tile's first half | exponentials of the second half
//   B  weighted sums of the tile      | copies of the tile after the next
// Measured: one sequence of 61 tokens x 128 heads at 32768 positions 403 .. 435 us by card, up to 1.29 PFLOP/s of the bf16 products that the pairs stand for in
// the whole call (the form before: 542); the matrix cores are busy 57 .. 64 % of the time.  Without the copies of all but the first rows it would be 40 us less wherever they
// are issued, without the exponentials and their codes 65.  A compute unit that does one tile takes 12 us: 1.2 to find it, 3.2 until it is there with
// the queries, 4 for the products, 3.2 for writing 128 x 512 sums.
//
// FEW (up to 32 rows a sequence, 16 heads of one token say): the wavefronts share the positions in place of the rows, each with a stage for
// itself and no barrier; the products of one stand beside the copies and exponentials of the others, and the four sums meet in LDS.  64
// sequences x 16 heads at up to 8192 positions (147 MB): 50 us, 2.9 TB/s; with one wavefront at work
// and the others copying for it 61.  Blocks of 32 rows do not pay where there are more: 32 sequences x 128 heads at up to 4096 positions 57.4 us for the
// whole call and 56.5 with blocks of 128, one sequence at 700 26.6 and 26.3.
template <bool PACK, bool FEW>
__global__ __launch_bounds__(256, 1) void mla_paged_kernel(PagedArgs p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 31, g = lane >> 5;
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
    if (blk * 128 >= live) return;
    const int t0 = (range - mine.first) * mine.per, t1 = min((seq.end + kTile - 1) / kTile, t0 + mine.per);
    const int row0 = FEW ? 0 : blk * 128 + wave * 32;
    const int row = min(row0 + i, p.rows - 1);          // rows past the end repeat the last one; fold leaves them out

    // A wavefront copies two groups of eight rows of a tile, of which each lies in one page: four KiB of latents, a KiB of rotary keys, the scales (by
    // all lanes, for what the first eight fetch).  A group is a buffer of the rows that it has: rows past the sequence's end, and all that
    // is no page's, are zeros; the scales of the latter come from `nothing`.
    const uint32_t lds0 = lds_addr_of(lds);
    const int32_t* entries = p.table + b * p.width;
    struct Source { v4i kv, pe; const float* scales; int last; uint32_t at; };
    constexpr int kScaleAt = FEW ? kFewScaleOff : kScaleOff, kGroups = FEW ? 8 : 2;
    const int first_row = FEW ? 0 : wave * 16;          // the wavefront's rows in a tile
    auto first_of = [&](int t, int h) -> uint32_t {     // group h of the wavefront's rows of tile t (past the end: the last group)
        return min(t * kTile + first_row + h * 8, (seq.end - 1) & ~7);
    };
    auto row_of = [&](uint32_t entry, uint32_t pos) -> uint64_t {       // where position pos, whose page is `entry`, lies in the pool
        return (uint64_t)entry * (uint32_t)p.page + (pos - __umulhi((pos & ~7u) >> 2, p.page_magic) * p.page);
    };
    // page number of group `lane % kGroups`, as a load of vectors: one by scalars would make every wait for LDS behind it wait for it as well
    auto page_of = [&](int t) -> int { return entries[__umulhi(first_of(t, lane_now() & (kGroups - 1)) >> 2, p.page_magic)]; };
    auto source = [&](int t, int h, int page, uint32_t stage) -> Source {
        const int entry = __builtin_amdgcn_readlane(page, h), left = min(seq.end, t1 * kTile) - (t * kTile + first_row + h * 8);
        // without branches, which would part the products that this stands beside (an empty buffer's address is not looked at)
        const int64_t some = -(int64_t)((left > 0) & ((uint32_t)entry < (uint32_t)p.pages));
        const uint64_t r = row_of(entry, first_of(t, h));
        const int rows = min(8, left) & (int)some;
        const uint64_t scales = (((uint64_t)(uintptr_t)p.scales + r * 4) & some) | ((uint64_t)(uintptr_t)nothing & ~some);
        return Source{ buffer_of(p.kv + r * kC, rows * kC), buffer_of(p.pe + r * (kRope * 2), rows * (kRope * 2)), (const float*)(uintptr_t)scales,
                       max(rows, 1) - 1, stage };
    };
    // where a lane reads of two rows of latents
    auto latent_off = [&]() -> uint32_t { const int lane = lane_now(); return (lane >> 5) * kC + (((lane & 31) ^ (lane >> 5 << 2)) << 4); };
    auto issue = [&](const Source& s, uint32_t latents, auto group, auto which) {
        constexpr int n = decltype(which)::value, h = decltype(group)::value;
        if constexpr (n < 4) {
            copy16_buffer_at(s.kv, latents, n * (2 * kC), s.at + (FEW ? h >> 1 : wave) * kRows16 + pair_off(4 * (h & 1) + n));
        } else if constexpr (n == 4) {                  // a key's chunk c at c ^ r / 2 (low three bits)
            const int lane = lane_now();
            if constexpr (!FEW || h >= 4)
                copy16_buffer_at(s.pe, (lane >> 3) * (kRope * 2) + (((lane & 7) ^ (4 * (h & 1) + (lane >> 4))) << 4), 0,
                                 s.at + kRopeOff + (FEW ? 8 * (h - 4) : wave * 16 + 8 * h) * (kRope * 2));
        } else {
            copy4(s.scales, min(lane_now() & 7, s.last) * 4, s.at + kScaleAt + (FEW ? h : wave * 2 + h) * 256);
        }
    };
    auto copy_tile = [&](int t, uint32_t stage, int page) {
        unrolled<kGroups>([&](auto h) {
            const Source s = source(t, h, page, stage);
            const uint32_t latents = latent_off();
            unrolled<6>([&](auto n) { issue(s, latents, h, n); });
        });
    };
    // this wavefront's copies have landed, and everybody's
    auto arrived = [&] {
        __builtin_amdgcn_s_waitcnt(0x0f70);             // vmcnt(0)
        barrier_no_fence();
    };
    uint32_t own = lds0 + wave * kFewStage;             // FEW: the wavefront's stage
    int page = 0;
    if constexpr (FEW) {
        page = page_of(t0 + wave);
        if (t0 + wave < t1) copy_tile(t0 + wave, own, page);
    } else {
        copy_tile(t0, lds0, page_of(t0));
        copy_tile(t0 + 1, lds0 + kStage, page_of(t0 + 1));
        if (row0 >= live) {                             // no rows: the others' copies
            arrived();
            for (int t = t0, st = 2; t < t1; ++t, st = st == 2 ? 0 : st + 1) {
                arrived();
                copy_tile(t + 2, lds0 + st * kStage, page_of(t + 2));
            }
            arrived();
            return;
        }
    }

    v8i Q[2][8];                                        // first and second codes; K step n: features 64 n + 32 g .. + 31
    int qs[2][2];                                       // their scales, K steps 0 .. 3 and 4 .. 7
    v4u turned[4];                                      // rotary query, K steps of 16: rounded to bf16, as apply_rotary_emb leaves it and as its keys are
    {
        // (packed, a last block's missing rows hold anything; nobody reads their results)
        const uint8_t* src = PACK ? p.ql + ((int64_t)b * p.groups + row0 / 32) * 32768 + lane * 16 : p.ql + ((int64_t)b * p.rows + row) * 1024 + g * 32;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int n = 0; n < 8; ++n)
                Q[c][n] = PACK ? join(*(const v4u*)(src + c * 16384 + n * 2048), *(const v4u*)(src + c * 16384 + n * 2048 + 1024))
                               : join(*(const v4u*)(src + c * 512 + n * 64), *(const v4u*)(src + c * 512 + n * 64 + 16));
        const v2u e = *(const v2u*)(p.qe + ((int64_t)b * p.rows + row) * 8);
#pragma unroll
        for (int k = 0; k < 2; ++k) { qs[0][k] = (int)e[k]; qs[1][k] = (int)(e[k] - 0x04040404u); }
        const uint16_t* rsrc = p.q + ((int64_t)b * p.rows + row) * kQd + kNope + 8 * g;
        const v2f* fr = p.freqs + ((int64_t)b * p.tokens + row / p.heads) * (kRope / 2) + 4 * g;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            v4u x = *(const v4u*)(rsrc + 16 * s);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const v2f cs = fr[8 * s + e];
                const float re = bf16lo_to_f32(x[e]), im = bf16hi_to_f32(x[e]);
                x[e] = pack_bf16(re * cs.x - im * cs.y, re * cs.y + im * cs.x);
            }
            turned[s] = x;
        }
    }

    const auto row_off = [](int r) { return (r >> 1) * kPair + ((r >> 2) & 1) * 16 + (r & 1) * kC; };      // of 0 .. 15
    // K step n is 64 bytes; of an odd row, steps n and n + 1 of even n are exchanged.  Values: 32 bytes for 32 features, in odd rows two and two exchanged.
    const uint32_t kaddr = (i >> 4) * kRows16 + row_off(i & 15) + 32 * g;
    const uint32_t raddr = kRopeOff - (FEW ? 32 * kRope * 2 : 0) + i * 128 + ((g ^ ((i >> 1) & 7)) << 4);    // ^ 2 s << 4
    // transposed reads: lane group q2 of a half takes 16 features; its lane l fetches eight of row l / 2 of 4 g .. + 3, 8 + 4 g .. + 3 of 16 rows
    const int l15 = lane & 15, q2 = (lane >> 4) & 1, vrow = 8 * (l15 >> 3) + 4 * g + ((l15 >> 1) & 3);
    const uint32_t vaddr = row_off(vrow) + 16 * q2 + 8 * (l15 & 1);
    const uint32_t kodd = (i & 1) * 64, vodd = (vrow & 1) * 64;
    auto read16 = [](uint32_t at) -> v4u { return *(lds_v4u)(uintptr_t)at; };
    // `at`: a stage's address with the lane's place, the even and the odd ones of what an odd row exchanges
    struct Two { uint32_t at[2]; };
    auto keys_at = [&](uint32_t stage) -> Two { return Two{ { stage + kaddr + kodd, stage + kaddr - kodd } }; };
    auto values_at = [&](uint32_t stage) -> Two { return Two{ { stage + vaddr + vodd, stage + vaddr - vodd } }; };
    auto key = [&](const Two& a, int half, int n) -> v8i {
        const uint32_t at = a.at[n & 1] + half * (2 * kRows16) + n * 64;
        return join(read16(at), read16(at + 16));
    };
    auto rope_key = [&](uint32_t at, int half, int s) -> v4u { return read16((at ^ (s << 5)) + half * (32 * kRope * 2)); };
    auto value = [&](const Two& a, int f) -> v8i {      // features 32 f .. of all 64 positions
        v8i v;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(uintptr_t)(a.at[(f >> 1) & 1] + f * 32 + k * kRows16));
            v[2 * k] = x[0];
            v[2 * k + 1] = x[1];
        }
        return v;
    };

    v16f O[16] = {};
    v16f S[2];
    v8i ring[2];                                        // keys of two K steps, or values of 64 features: read two to four MFMAs ahead
    v4u rope[4];                                        // rotary keys
    v8i P[2];                                           // exponentials, first and second codes; dwords 4 h .. of half h
    int pe[2];                                          // their exponents, by halves
    float off = kNoScore, l = 0.f;                      // exponentials are of 2^(score - off), off a whole number; this lane's share of their sum
    int ks[2];                                          // scale byte of position i, by halves
    uint32_t none[2];                                   // positions that nobody sees for want of a page, by halves
    float sc;                                           // the scale that the next scores need
    auto scale_at = [&](uint32_t stage, int half) -> float {
        const int i = lane_now() & 31;
        return *(lds_f32)(uintptr_t)(stage + (i >> 3) * 256 + (i & 7) * 4 + kScaleAt + half * 1024);
    };
    auto look_at_scale = [&](int half) {
        ks[half] = (int)(f32_as_u32(sc) >> 23 & 0xff);  // (NaN: 255, which makes the products NaN)
        none[half] = (uint32_t)__ballot(sc == kNothing);
    };

    // The exponentials of half h, in 17 steps that stand beside the MFMAs of 20.
    v4f w[4];
    uint32_t largest = 0u;                              // bits of the largest exponential times its scale
    float pm = 0.f, shrink = 1.f, ex[2], times = 0.f, less = 0.f;       // exponentials are of 2^(score * times - less)
    uint32_t scales_at = 0u;
    const uint64_t alive = __ballot(row0 + i < live);
    bool behind = false, far = false;                   // the sums are still to be multiplied with `shrink`; some row's offset is beyond 2^24
    auto soften = [&](int t, uint32_t stage, auto half, auto step) {
        constexpr int h = decltype(half)::value, x = decltype(step)::value;
        v16f& s = S[h];
        if constexpr (x == 0) scales_at = stage + (lane_now() >> 5) * 16 + kScaleAt;
        if constexpr (x < 8 && x % 2 == 0) w[x / 2] = *(lds_v4f)(uintptr_t)(scales_at + (4 * h + x / 2) * 256);
        if constexpr (x == 1) {
            asm volatile("" : "+v"(s));                 // (behind two more MFMAs: the scores are there)
            const int at = t * kTile + 32 * h;
            if (none[h] || at + 32 > seq.start) {       // (the sequence's end lies behind its start)
                const int left = seq.end - at, j0 = at - seq.start;            // j0: the first position among the new ones
                uint32_t seen = ~none[h];
                if (left < 32) seen &= left > 0 ? (1u << left) - 1u : 0u;
                if (j0 > -32) {
                    const int tok = min(row0 + (lane_now() & 31), p.rows - 1) / p.heads;
                    const uint64_t bits = p.tree ? (uint64_t)p.tree[(int64_t)b * p.tokens + tok] : (2ull << tok) - 1;
                    seen &= j0 >= 64 ? 0u : j0 >= 0 ? (uint32_t)(bits >> j0) : (uint32_t)(bits << -j0) | ((1u << -j0) - 1u);
                }
                seen >>= (lane_now() >> 5) * 4;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(seen >> (8 * (e >> 2) + (e & 3)) & 1)) s[e] = -__builtin_inff();
            }
            pm = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) pm = __builtin_elementwise_maximum(pm, s[e]);
        }
        if constexpr (x == 2) {
            const v2f both = halves32(pm);
            const float top = fmaxf(both.x, both.y) * p.scale;
            // `off` is only raised when a score passes it by more than 2^64: exponentials and sums have room for that in binary32, and so the 256
            // multiplications are needed in the rarest of cases.  By whole powers of two: the first half's codes change their exponent only.
            // (Rows that nobody reads do not ask for it.)
            const uint64_t raise = __ballot(top - off > 64.f) & alive;
            if (raise) {
                const bool mine = raise >> lane_now() & 1;
                const float on = mine ? __builtin_ceilf(top) : off, a = __builtin_amdgcn_exp2f(off - on);
                l *= a;
                if constexpr (h == 1) pe[0] = max(5, pe[0] - (int)fminf(on - off, 300.f));
                off = on;
                shrink = behind ? shrink * a : a;       // (the sums follow in front of phase B)
                behind = true;
                far = __ballot(__builtin_fabsf(off) > 0x1p24f && off != kNoScore) & alive;
            }
            times = p.scale;
            less = off;
            if (far) {
                // `off` is a rounded score: up to 2^24 it is a whole number that a fused product minus it differs from by 1 at most, but far beyond, the
                // difference would be any power of two.  There the score's product is rounded as the offset was, so that the largest exponential is 1.
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = s[e] * p.scale;
                    s[e] = __builtin_fabsf(off) > 0x1p24f ? x - off : __builtin_fmaf(s[e], p.scale, -off);
                }
                times = 1.f;
                less = 0.f;
            }
            largest = 0u;
        }
        if constexpr (x >= 4 && x < 12) {               // (a step behind their exponentials: those results take a while)
            constexpr int e = 2 * (x - 4);
            l += ex[0];
            l += ex[1];
            s[e] = dsv3_mul_legacy(ex[0], w[e >> 2][e & 3]);
            s[e + 1] = dsv3_mul_legacy(ex[1], w[e >> 2][(e & 3) + 1]);
            largest = umax_u32(largest, umax_u32(f32_as_u32(s[e]), f32_as_u32(s[e + 1])));
            asm volatile("" : "+v"(l), "+v"(largest));                          // (here, not where they are next looked at)
        }
        if constexpr (x >= 3 && x < 11) {
#pragma unroll
            for (int e = 0; e < 2; ++e) ex[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * (x - 3) + e], times, -less));
        }
        if constexpr (x == 12) {                        // (the halves' bytes share a scale)
            const v2u both = __builtin_amdgcn_permlane32_swap(largest, largest, false, false);
            pe[h] = split_exponent(umax_u32(both[0], both[1]));
        }
        if constexpr (x >= 13 && x < 17) {
            constexpr int k = x - 13;
            uint32_t first, second;
            split_codes(s[4 * k], s[4 * k + 1], s[4 * k + 2], s[4 * k + 3], u32_as_f32((uint32_t)pe[h] << 23), u32_as_f32((uint32_t)(pe[h] - 4) << 23), first, second);
            asm volatile("" : "+v"(first), "+v"(second));                       // (made here, not where they are used)
            P[0][4 * h + k] = (int)first;
            P[1][4 * h + k] = (int)second;
        }
    };
    // The scores of half h of the tile at `stage`, whose first two keys are in the ring.  beside(step): what stands behind the step's MFMA;
    // tail(0 / 1): the ring's place is free for what the next phase reads first.
    auto score = [&](uint32_t stage, auto half, auto beside, auto tail) {
        constexpr int h = decltype(half)::value;
        v16f& s = S[h];
        uint32_t ropes = raddr;
        asm volatile("" : "+v"(ropes));                 // (formed ahead of the loop, what the reads' places xor to would take the registers that there are not)
        ropes += stage;
        const Two keys = keys_at(stage);
        unrolled<20>([&](auto step) {
            constexpr int x = decltype(step)::value, n = x >> 1;
            if constexpr (x == 0) mfma64_first<0>(s, ring[0], Q[0][0], ks[h], qs[0][0]);
            else if constexpr (x < 16) mfma64_next<(n & 3)>(s, ring[n & 1], Q[x & 1][n], ks[h], qs[x & 1][n >> 2]);
            else mfma32_next(s, rope[x - 16], turned[x - 16]);
            if constexpr (x < 12 && (x & 1)) ring[n & 1] = key(keys, h, n + 2);
            if constexpr (x >= 12 && x < 16 && !(FEW && h == 0)) rope[x - 12] = rope_key(ropes, h, x - 12);
            beside(step);
            if constexpr (x == 14) tail(std::integral_constant<int, 0>());
            if constexpr (x == 16) tail(std::integral_constant<int, 1>());
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    // The weighted sums of the tile at `base`, whose first two values are in the ring
    auto weigh = [&](bool first, uint32_t base, auto beside) {
        const Two values = values_at(base);
        const int one = 127, g = lane_now() >> 5, e[2] = { g ? pe[1] : pe[0], (g ? pe[1] : pe[0]) - 4 };
        if (behind) {
            behind = false;
            if (!first) {
#pragma unroll
                for (int d = 0; d < 16; ++d) scale_agprs(O[d], shrink);
                asm volatile("s_nop 7" ::: "memory");
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        unrolled<32>([&](auto step) {
            constexpr int x = decltype(step)::value, f = x >> 1;
            mfma64_sum(O[f], ring[f & 1], P[x & 1], one, e[x & 1]);
            if constexpr ((x & 1) && f < 14) ring[f & 1] = value(values, f + 2);
            beside(step);
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int d = 0; d < 16; ++d) asm volatile("" : "+a"(O[d]));     // (the sums stay where they are)
    };

    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, 1> Second;
    if constexpr (FEW) {
        // A wavefront by itself takes every fourth tile, from its own stage, without barriers: the scores of the first half, those of the second
        // beside the first's exponentials, the second's exponentials, the weighted sums.
        for (int t = t0 + wave; t < t1; t += 4) {
            asm volatile("" : "+s"(own));               // (what is formed from it is not kept through the loop: there are no registers for that)
            {
                const int lane = lane_now(), i = lane & 31, entry = __shfl(page, i >> 3);
                const uint32_t pos = t * kTile + i;
                const bool there = (int)pos < seq.end && (uint32_t)entry < (uint32_t)p.pages;
                const v4u* src = there ? (const v4u*)(p.pe + row_of(entry, pos) * (kRope * 2)) : nothing_key;
#pragma unroll
                for (int s = 0; s < 4; ++s) rope[s] = src[2 * s + (lane >> 5)];
            }
            page = page_of(t + 4);
            __builtin_amdgcn_s_waitcnt(0x0f70);         // vmcnt(0)
            asm volatile("" ::: "memory");
            sc = scale_at(own, 0);
            ring[0] = key(keys_at(own), 0, 0);
            ring[1] = key(keys_at(own), 0, 1);
            look_at_scale(0);
            sc = scale_at(own, 1);
            score(own, First(), [](auto) {}, [&](auto k) { ring[k] = key(keys_at(own), 1, k); });
            look_at_scale(1);
            score(own, Second(), [&](auto step) { soften(t, own, First(), step); }, [&](auto k) { ring[k] = value(values_at(own), k); });
            scores_ready(S[1]);
            scores_ready(S[1]);
            unrolled<17>([&](auto step) {
                soften(t, own, Second(), step);
                __builtin_amdgcn_sched_barrier(0);
            });
            weigh(t == t0 + wave, own, [](auto) {});
            if (t + 4 < t1) copy_tile(t + 4, own, page);                // (every read of the stage has been used)
        }
    } else {
        page = page_of(t0 + 2);
        arrived();
        sc = scale_at(lds0, 0);
        ring[0] = key(keys_at(lds0), 0, 0);
        ring[1] = key(keys_at(lds0), 0, 1);
        look_at_scale(0);
        sc = scale_at(lds0, 1);
        score(lds0, First(), [](auto) {}, [&](auto k) { ring[k] = key(keys_at(lds0), 1, k); });
        look_at_scale(1);
        int st = 0;
        for (int t = t0;; ++t) {
            const int st_next = st == 2 ? 0 : st + 1, st_free = st_next == 2 ? 0 : st_next + 1;
            const uint32_t base = lds0 + st * kStage, next = lds0 + st_next * kStage;
            const int page_now = page;
            // C.  Behind its barrier the next tile is there, and the stage of the one before is free.
            score(base, Second(), [&](auto step) {
                soften(t, base, First(), step);
                if constexpr (decltype(step)::value == 13) {
                    arrived();
                    page = page_of(t + 3);
                    sc = scale_at(next, 0);
                }
            }, [&](auto k) { ring[k] = key(keys_at(next), 0, k); });
            // A, also behind the last tile (of zeros: a path without it would let the compiler copy scores before they are there)
            look_at_scale(0);
            score(next, First(), [&](auto step) { soften(t, base, Second(), step); }, [&](auto k) { ring[k] = value(values_at(base), k); });
            // B
            Source ahead;
            uint32_t latents;
            weigh(t == t0, base, [&](auto step) {
                constexpr int x = decltype(step)::value;
                if constexpr (x == 29 || x == 31) ring[x >> 1 & 1] = key(keys_at(next), 1, (x >> 1) - 14);
                // copies of the tile after the next, one behind a product
                if constexpr (x == 0 || x == 8) {
                    ahead = source(t + 2, x / 8, page_now, lds0 + st_free * kStage);
                    latents = latent_off();
                }
                if constexpr (x >= 1 && x < 7) issue(ahead, latents, First(), std::integral_constant<int, x - 1>());
                if constexpr (x >= 9 && x < 15) issue(ahead, latents, Second(), std::integral_constant<int, x - 9>());
                if constexpr (x == 20) sc = scale_at(next, 1);
            });
            if (t + 1 == t1) break;
            look_at_scale(1);
            st = st_next;
        }
    }

    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // (the last sums are there)
#pragma unroll
    for (int d = 0; d < 16; ++d) asm volatile("" : "+a"(O[d]));
    const v2f parts = halves32(l);
    l = parts.x + parts.y;
    const int last_lane = lane_now(), i2 = last_lane & 31, g2 = last_lane >> 5;
    const int64_t slot = ((int64_t)range * p.blocks + blk) * 128 + (FEW ? 0 : wave * 32);       // the wavefront's rows among all
    float factor = 1.f;                                 // FEW: to the wavefronts' common offset
    if constexpr (FEW) {
        __syncthreads();                                // the stages are free
        v2f* stats = (v2f*)lds;
        if (g2 == 0) stats[wave * 32 + i2] = v2f{ off, l };
        __syncthreads();
        float top = kNoScore, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stats[w * 32 + i2].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += stats[w * 32 + i2].y * __builtin_amdgcn_exp2f(stats[w * 32 + i2].x - top);
        factor = __builtin_amdgcn_exp2f(off - top);
        if (wave == 0 && g2 == 0) p.ml[slot + i2] = v2f{ top, sum };
    } else {
        if (g2 == 0) p.ml[slot + i2] = v2f{ off, l };
        arrived();                                      // (copies past the range are still on their way into the stages)
    }
    // The sums leave as rows, which fold reads whole: 64 features of 32 rows at a time through LDS (16-byte chunks xor-ed with the row), so that a
    // store writes four pieces of 256 bytes; rows that nobody reads stay here.
    auto put = [&](int d2, uint8_t* at) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const v16f& o = O[2 * d2 + (c >> 2)];
            const int e = 4 * (c & 3);
            v4f x = { o[e], o[e + 1], o[e + 2], o[e + 3] };
            if constexpr (FEW) x *= factor;
            *(v4f*)(at + i2 * 256 + (((2 * c + g2) ^ (i2 & 15)) << 4)) = x;
        }
    };
    auto taken = [&](const uint8_t* at, int r, int c) -> v4f { return *(const v4f*)(at + r * 256 + ((c ^ (r & 15)) << 4)); };
    if constexpr (FEW) {                                // the four wavefronts' sums meet there
        const int r0 = wave * 4 + (last_lane >> 4), c = last_lane & 15;
        float* dst = p.part + (slot + r0) * kC + c * 4;
        uint8_t* sums = lds + 4096;
        put(0, sums + wave * 8192);
#pragma unroll
        for (int d2 = 0; d2 < 8; ++d2) {                // two buffers a wavefront: the next 64 features are written while these are read
            const uint8_t* at = sums + (d2 & 1) * 32768;
            __syncthreads();
            v4f x[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                x[n] = taken(at, r0 + 16 * n, c);
#pragma unroll
                for (int w = 1; w < 4; ++w) x[n] += taken(at + w * 8192, r0 + 16 * n, c);
            }
            if (d2 < 7) put(d2 + 1, sums + (~d2 & 1) * 32768 + wave * 8192);
#pragma unroll
            for (int n = 0; n < 2; ++n)
                if (r0 + 16 * n < live) *(v4f*)(dst + n * 16 * kC + d2 * 64) = x[n];
        }
    } else {
        float* dst = p.part + (slot + (last_lane >> 4)) * kC + (last_lane & 15) * 4;
        uint8_t* at = lds + wave * 16384;
        put(0, at);
#pragma unroll
        for (int d2 = 0; d2 < 8; ++d2) {
            v4f x[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = taken(at + (d2 & 1) * 8192, 4 * n + (last_lane >> 4), last_lane & 15);
            if (d2 < 7) put(d2 + 1, at + (~d2 & 1) * 8192);
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (row0 + 4 * n + (last_lane >> 4) < live) *(v4f*)(dst + n * 4 * kC + d2 * 64) = x[n];
        }
    }
}

// Row blocks of 128 (token, head) rows; one workgroup a compute unit (its registers take a whole one).
struct PagedPlan { int groups; int64_t blocks, ranges; };
PagedPlan paged_plan(int64_t batch, int64_t rows) {
    PagedPlan a;
    a.blocks = (rows + 127) / 128;
    a.groups = (int)(a.blocks * 4);
    // Ranges of all sequences: as many as there are compute units for the row blocks of the widest, so that all run at once (8 sequences x 25 tokens x 128
    // heads, 10 to 2001 positions: 10 ranges of up to 22 tiles 84 us, 13 of up to 18 in two rounds 105); where the sequences alone are
    // more than these, room for the longer ones to be cut.
    const int64_t units = a.blocks < 256 ? 256 / a.blocks : 1;
    a.ranges = batch <= units ? units : batch + units / 2;
    return a;
}
// Folded queries, their exponents, partial sums, their maxima and sums, the division of the work
struct PagedSpace { size_t exponents, part, ml, plan, bytes; };
PagedSpace paged_space(const PagedPlan& a, int64_t batch) {
    const int64_t rows = a.ranges * a.blocks * 128;
    PagedSpace s;
    s.exponents = (size_t)(batch * a.groups * (32 * kC * 2));
    s.part = s.exponents + (size_t)(batch * a.groups * (32 * 8));
    s.ml = s.part + (size_t)(rows * kC * 4);
    s.plan = s.ml + (size_t)(rows * 8);
    s.bytes = s.plan + (size_t)(batch * 8);
    return s;
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
    a.ql = wsp; a.qe = wsp + space.exponents; a.q = (const uint16_t*)q; a.freqs = (const v2f*)freqs;
    a.kv = (const uint8_t*)cache.kv; a.scales = cache.kv_scale; a.pe = (const uint8_t*)cache.pe;
    a.table = cache.table; a.width = cache.table_width; a.pages = cache.pages;
    a.starts = starts; a.counts = counts; a.tree = tree;
    a.part = (float*)(wsp + space.part); a.ml = (v2f*)(wsp + space.ml); a.plan = (v2i*)(wsp + space.plan);
    a.batch = (int)batch; a.tokens = (int)tokens; a.rows = (int)rows; a.heads = heads; a.positions = (int)positions;
    a.page = cache.page_size; a.groups = plan.groups; a.blocks = (int)plan.blocks; a.ranges = (int)plan.ranges;
    a.page_magic = (uint32_t)(((1ll << 31) + cache.page_size / 8 - 1) / (cache.page_size / 8));
    a.scale = scale * 1.44269504088896340736f;
    // operand order up to 16 tokens in all, which is what the kernel that writes it takes (mla_decode.hip)
    const bool pack = batch * tokens <= 16;
    const int rc = launch_wkv_b_absorb_q_codes(q, (int64_t)heads * kQd, kQd, w, ws, wsp, wsp + space.exponents, pack, batch, tokens, (int)plan.blocks, heads, st);
    if (rc != DSV3_OK) return rc;
    const bool few = rows <= 32;
    static void (*const kernels[2][2])(PagedArgs) = { { mla_paged_kernel<false, false>, mla_paged_kernel<true, false> },
                                                      { mla_paged_kernel<false, true>, mla_paged_kernel<true, true> } };
    static LdsGrant grant[2][2];
    static_assert(kLds <= 160 * 1024 && kFewLds <= 160 * 1024 && 4 * 16384 <= kStages * kStage && 4096 + 2 * 32768 <= kFewLds, "the sums leave through the stages");
    const int lds = few ? kFewLds : kLds;
    if (!grant[few][pack].ensure((const void*)kernels[few][pack], lds)) return DSV3_ERR_LAUNCH;
    const unsigned grid = (unsigned)((plan.ranges * plan.blocks + 7) / 8 * 8);
    hipLaunchKernelGGL(kernels[few][pack], dim3(grid), dim3(256), lds, st, a);
    FoldArgs f = {};
    f.part = a.part; f.ml = a.ml; f.plan = a.plan; f.counts = counts; f.w = (const uint8_t*)w; f.ws = ws; f.y = y; f.ys = ys;
    f.tokens = (int)(batch * tokens); f.per_seq = (int)tokens; f.heads = heads; f.rows = 128; f.blocks = a.blocks;
    return launch_fold<true>(f, st);
}

}  // namespace dsv3

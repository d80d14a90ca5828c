// Where a position of a sequence lies in a cache of pages.  Plain C++: kernels and host-side checks share it.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define DSV3_HD __host__ __device__ __forceinline__
#else
#define DSV3_HD inline
#endif

namespace dsv3 {

// The cache row of position `pos`, or -1 where the sequence has none: `entries` are the sequence's `width` page numbers, of which
// those outside [0, pages) name no page.  Eight positions from a multiple of eight on lie in one page (page sizes are multiples of eight).
DSV3_HD int64_t page_row(const int32_t* entries, int64_t width, int64_t pages, int page, int64_t pos) {
    if (pos < 0) return -1;
    const int64_t k = (uint64_t)pos >> 31 ? pos / page : (int64_t)((uint32_t)pos / (uint32_t)page);
    if (k >= width) return -1;
    const int64_t entry = entries[k];
    if (entry < 0 || entry >= pages) return -1;
    return entry * page + (pos - k * page);
}

// A sequence's part in a step of `rows` rows at most: positions in front of it and behind it, rows.  Nothing lies behind `most`; a negative
// start or count leaves nothing.
struct SeqSpan { int start, end, count; };
DSV3_HD SeqSpan seq_span(int start, int count, int rows, int most) {
    if (start < 0 || count <= 0) return SeqSpan{ 0, 0, 0 };
    const int s = start > most ? most : start, n = count > rows ? rows : count;
    return SeqSpan{ s, n < most - s ? s + n : most, n };
}

}  // namespace dsv3

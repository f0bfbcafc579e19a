// Where the tokens of a paged batch sit: plain C++, so that the bounds of every index a kernel forms from device data (starts, lengths,
// block tables, all of which a caller can get wrong) can be checked on the host.
#pragma once
#include <cstdint>

#include "../../include/tts_amd.h"

#if defined(__HIPCC__)
#define TTSAMD_HD __host__ __device__ __forceinline__
#else
#define TTSAMD_HD inline
#endif

namespace ttsamd {

// n / d for 0 <= n < 2^31 by one multiply and shift (magic = ceil(2^(31+s) / d), s = ceil(log2 d): exact over that range).
struct FastDiv {
    uint32_t d, magic, shift;
    TTSAMD_HD uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * magic) >> 31) >> shift; }
};
inline FastDiv fast_div(uint32_t d)
{
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return FastDiv{d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

// One sequence of a call, bounded: tokens [start, start + n) of [0, tokens), `len` tokens in all (new token i at position len - n + i),
// of which the first `keys` have a column in the table.
struct Sequence {
    int start, n, len, keys;
};
TTSAMD_HD int bounded(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
TTSAMD_HD Sequence sequence_of(const ttsamd_paged_batch &bt, int tokens, int page_size, int b)
{
    Sequence s;
    s.start = bounded(bt.q_starts[b], 0, tokens);
    s.n = bounded(bt.q_starts[b + 1], s.start, tokens) - s.start;
    s.len = bt.seq_lens[b] < 0 ? 0 : bt.seq_lens[b];
    const int64_t room = (int64_t)bt.table_width * page_size;
    s.keys = (int)(s.len < room ? s.len : room);
    return s;
}

// The keys new token `pos` sees: [begin, end) within [0, s.keys) (empty where begin >= end).
struct Range {
    int begin, end;
};
TTSAMD_HD Range seen_by(const Sequence &s, int pos, int causal, int window)
{
    const int64_t from = (int64_t)pos - window + 1;
    return Range{window > 0 && from > 0 ? (int)from : 0, causal && pos + 1 < s.keys ? (pos + 1 < 0 ? 0 : pos + 1) : s.keys};
}

// The table's entry for position j of sequence b, j in [0, s.keys), and the row in its page.  What the entry holds is checked where it is
// used (held), so that a kernel can leave the load on its way.
TTSAMD_HD int entry_of(const ttsamd_paged_batch &bt, const FastDiv &by_page, int b, int j, int &row)
{
    const uint32_t col = by_page.div((uint32_t)j);
    row = j - (int)(col * by_page.d);
    return bt.block_table[b * bt.table_stride + col];
}
TTSAMD_HD bool held(int page, int pages) { return (unsigned)page < (unsigned)pages; }

// The page of sequence b that holds position j in [0, s.keys), or -1; `row`: the row in it.
TTSAMD_HD int page_of(const ttsamd_paged_batch &bt, const FastDiv &by_page, int pages, int b, int j, int &row)
{
    const int page = entry_of(bt, by_page, b, j, row);
    return held(page, pages) ? page : -1;
}

}  // namespace ttsamd

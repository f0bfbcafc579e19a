// Host check of csrc/decode_overlap.h against brute force: every byte of small row sets, written out.
#include <cstdio>
#include <random>
#include <set>

#include "../../tts_amd/csrc/decode_overlap.h"

using namespace ttsamd;

#define CHECK(c) do { if (!(c)) { std::printf("failed: %s (line %d)\n", #c, __LINE__); return 1; } } while (0)

static bool bytes_of(const RowSet &s, std::set<int64_t> &to)
{
    bool twice = false;
    for (int64_t i = 0; i < s.tokens; ++i)
        for (int64_t j = 0; j < s.heads; ++j)
            for (int64_t k = 0; k < s.bytes; ++k) twice |= !to.insert((int64_t)(uintptr_t)s.at + i * s.t + j * s.h + k).second;
    return twice;
}

int main()
{
    std::mt19937 rng(7);
    auto in = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    int met = 0, apart = 0, alike = 0;
    for (int round = 0; round < 40000; ++round) {
        RowSet a = {(void *)(uintptr_t)(4096 + in(0, 40)), in(-24, 24), in(-24, 24), in(1, 5), in(1, 5), in(1, 8)};
        RowSet b = {(void *)(uintptr_t)(4096 + in(0, 40)), in(-24, 24), in(-24, 24), in(1, 5), in(1, 5), in(1, 8)};
        if (rng() % 2) b.t = a.t;
        if (rng() % 2) b.h = a.h;
        std::set<int64_t> x, y;
        const bool twice = bytes_of(a, x);
        bytes_of(b, y);
        CHECK(rows_meet(a) == twice);
        bool meet = false;
        for (int64_t v : x) meet |= y.count(v) != 0;
        const bool same = (a.t == b.t || a.tokens == 1 || b.tokens == 1) && (a.h == b.h || a.heads == 1 || b.heads == 1);
        if (meet) CHECK(sets_meet(a, b));
        if (same) CHECK(sets_meet(a, b) == meet);
        met += meet && same, apart += !meet && same, alike += !meet && !sets_meet(a, b);
    }
    CHECK(met > 2000 && apart > 2000 && alike > 2000);
    // a fused projection: queries, keys and values side by side in each token's row, and heads taken in turns
    RowSet q = {(void *)4096, 768, 64, 1000, 8, 64}, k = {(void *)(4096 + 512), 768, 64, 1000, 2, 64};
    CHECK(!sets_meet(q, k) && !sets_meet(k, q) && !rows_meet(q) && same_rows(q, q));
    k.at = (void *)(4096 + 448);
    CHECK(sets_meet(q, k) && sets_meet(k, q));
    RowSet even = {(void *)4096, 1024, 128, 1 << 20, 4, 64}, odd = {(void *)(4096 + 64), 1024, 128, 1 << 20, 4, 64};
    CHECK(!sets_meet(even, odd) && !rows_meet(even));
    CHECK(rows_meet({(void *)4096, 0, 64, 2, 1, 64}) && rows_meet({(void *)4096, 64, 0, 1, 2, 64}) && !rows_meet({(void *)4096, 0, 0, 1, 1, 64}));
    CHECK(!rows_meet({(void *)4096, 64, 64 << 20, 1 << 20, 512, 64}));             // heads outermost
    std::printf("overlap OK\n");
    return 0;
}

// Host check of csrc/decode_places.h: whatever starts, lengths and tables hold, every index formed from them is in bounds.
// Built with address and undefined-behaviour sanitizers; the tables are allocated at their exact size.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../tts_amd/csrc/decode_places.h"

using namespace ttsamd;

#define CHECK(c) do { if (!(c)) { std::printf("failed: %s (line %d)\n", #c, __LINE__); return 1; } } while (0)

int main()
{
    std::mt19937 rng(1);
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 13u, 16u, 24u, 100u, 4095u, 65536u, 65537u, 1u << 30, (1u << 30) + 1, 0x7fffffffu}) {
        const FastDiv f = fast_div(d);
        for (uint32_t n : {0u, 1u, d - 1, d, d + 1, 2 * d - 1, 0x7fffffffu, 0x7ffffffeu, 0x40000000u})
            if (n <= 0x7fffffffu) CHECK(f.div(n) == n / d);
        for (int i = 0; i < 20000; ++i) {
            const uint32_t n = rng() & 0x7fffffffu;
            CHECK(f.div(n) == n / d);
        }
    }
    const int hostile[] = {0, 1, -1, INT_MIN, INT_MAX, INT_MAX - 1, 5, 17, 64, 1000, -1000};
    auto any = [&] { return hostile[rng() % 11]; };
    for (int round = 0; round < 20000; ++round) {
        const int batch = 1 + rng() % 4, width = rng() % 5, page = 1 + rng() % 40, pages = 1 + rng() % 8, tokens = rng() % 50;
        std::vector<int32_t> starts(batch + 1), lens(batch), table(batch * width);
        for (auto &v : starts) v = rng() % 2 ? any() : (int)(rng() % 60);
        for (auto &v : lens) v = rng() % 2 ? any() : (int)(rng() % 200);
        for (auto &v : table) v = rng() % 3 ? (int)(rng() % pages) : any();
        ttsamd_paged_batch b = {table.data(), width, lens.data(), starts.data(), width, batch, 1, 1};
        const FastDiv by_page = fast_div(page);
        for (int s = 0; s < batch; ++s) {
            const Sequence q = sequence_of(b, tokens, page, s);
            CHECK(q.start >= 0 && q.n >= 0 && q.start + q.n <= tokens && q.keys >= 0 && q.keys <= q.len && (int64_t)q.keys <= (int64_t)width * page);
            for (int i = 0; i < q.n; ++i) {
                const int pos = q.len - q.n + i;
                for (int window : {0, 1, 3, INT_MAX})
                    for (int causal : {0, 1}) {
                        const Range r = seen_by(q, pos, causal, window);
                        CHECK(r.begin >= 0 && r.end <= q.keys);
                        if (causal) CHECK(r.end <= (pos + 1 < 0 ? 0 : pos + 1));
                        if (window) CHECK(r.begin > (int64_t)pos - window);
                    }
            }
            for (int j = 0; j < q.keys; ++j) {
                int row = -1;
                const int p = page_of(b, by_page, pages, s, j, row);
                CHECK(p >= -1 && p < pages && row >= 0 && row < page && row == j % page);
                CHECK(p == -1 || p == table[s * width + j / page]);
            }
        }
    }
    std::printf("places OK\n");
    return 0;
}

// Every position that a row sees lies in exactly one step of its tile's span,
// no step lies behind what the tile sees, and the parts of a call's work are
// its steps, each in one part.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../qwenqwen3.js_amd/csrc/kv_plan.h"

using namespace qq;

#define CHECK(c)                                                                      \
    do {                                                                              \
        if (!(c)) {                                                                   \
            std::printf("%s: len %d rows %d t %d cols %d group %d cap %d window %d sinks %d slog %d\n", #c, len, rows, t, \
                        cols, group, cap, window, sinks, slog);                       \
            std::exit(1);                                                             \
        }                                                                             \
    } while (0)

int main()
{
    std::mt19937 rng(1);
    auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
    for (int it = 0; it < 60000; it++) {
        const int len = upto(upto(3) ? 300 : 40), rows = 1 + upto(upto(2) ? 3 : 60), group = 1 + upto(upto(1) ? 3 : 23);
        const int cols = upto(1) ? 16 : 128, slog = 4 + upto(2), cap = upto(3) ? 100000 : 16 * (1 + upto(20));
        const int window = upto(2) ? 1 + upto(200) : 0, sinks = window && upto(1) ? upto(100) : 0;
        const int tiles = kv_tiles(rows, group, cols);
        int t = 0;
        CHECK((int64_t)tiles * cols >= rows * group && (int64_t)(tiles - 1) * cols < rows * group);
        for (t = 0; t < tiles; t++) {
            const KvSpan s = kv_tile_span(len, rows, t, cols, group, cap, window, sinks, slog);
            CHECK(s.n >= 1 && s.sinks >= 0 && s.sinks < s.n + (s.n == 1));
            std::vector<int> times(400 + (1 << slog), 0);
            int last = -1, top = -1;
            for (int i = 0; i < s.n; i++) {
                const int base = kv_base(s, i, slog);
                CHECK(base > last && base % (1 << slog) == 0);
                last = base;
                for (int e = 0; e < 1 << slog; e++)
                    if (base + e < (int)times.size()) times[base + e]++;
            }
            for (int c = t * cols; c < (t + 1) * cols && c < rows * group; c++) {
                const int p = len - rows + c / group;
                for (int x = 0; x <= p && x < cap; x++)
                    if (!window || x > p - window || x < sinks) {
                        CHECK(times[x] == 1);
                        top = x > top ? x : top;
                    }
            }
            CHECK(s.n == 1 || last <= top);
        }
    }
    // the ends of the ranges
    int len = 0, rows = 0, t = 0, cols = 0, group = 0, cap = 1 << 30, window = 0, sinks = 0, slog = 4;
    for (int p : {-2147483647 - 1, -1, 0, (1 << 30) - 1, 1 << 30, 2147483646, 2147483647})
        for (int w : {0, 1, 2147483647})
            for (int k : {0, 1, 2147483647}) {
                const KvSpan s = kv_span(p, p, cap, w, k, slog);
                const int hi = p < 0 ? 0 : p < cap ? p + 1 : cap;
                CHECK(s.n >= 1 && s.n <= (1 << 26) && kv_base(s, s.n - 1, slog) <= (hi ? hi - 1 : 0));
                CHECK(w || s.n == (hi ? (hi + 15) / 16 : 1));
            }
    for (int it = 0; it < 20000; it++) {
        const uint64_t W = 1 + rng() % (it % 3 ? 5000 : 50);
        const uint32_t n = kv_parts(W, 1 + rng() % 600, 1 + rng() % 8);
        CHECK(n >= 1 && n <= W && kv_cut(W, n, 0) == 0 && kv_cut(W, n, n) == W);
        for (uint32_t w = 0; w < n; w++) {
            CHECK(kv_cut(W, n, w) < kv_cut(W, n, w + 1));
            for (uint64_t x = kv_cut(W, n, w); x < kv_cut(W, n, w + 1); x++) CHECK(kv_part(W, n, x) == w);
        }
    }
    const uint64_t W = (uint64_t)1 << 50;
    CHECK(kv_part(W, 4095, W - 1) == 4094 && kv_cut(W, 4095, 4095) == W && kv_part(W, 4095, 0) == 0);
    std::puts("ok");
    return 0;
}

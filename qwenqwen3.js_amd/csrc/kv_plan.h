// kv_plan.h -- which positions a tile of attention columns goes through, and
// how a call's work is cut into equal parts.  Plain integer arithmetic, the
// same on the host (its test) and in the kernels.
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define QQ_HD __host__ __device__ __forceinline__
#else
#define QQ_HD inline
#endif

namespace qq {

QQ_HD int kv_min(int a, int b) { return a < b ? a : b; }
QQ_HD int kv_max(int a, int b) { return a > b ? a : b; }

// A tile's columns are pairs (row, query head) of one sequence and one
// key/value head: column c of the sequence is row c / group, head c % group.
QQ_HD int kv_tiles(int rows, int group, int cols) { return (int)(((int64_t)rows * group + cols - 1) / cols); }

// The steps of 1 << slog positions that rows at positions p0 .. p1 see
// together, p1 < cap or not: steps 0 .. sinks - 1, then first .. (n in all).
// A tile that sees nothing has one step all the same: it writes its zeros.
struct KvSpan {
    int first, sinks, n;
};
QQ_HD KvSpan kv_span(int p0, int p1, int cap, int window, int sinks, int slog)
{
    KvSpan s = {0, 0, 1};
    const int hi = kv_min(p1, cap - 1) + 1;   // past the last position seen
    if (hi <= 0) return s;
    const int end = (int)(((int64_t)hi + (1 << slog) - 1) >> slog);
    const int lo = window ? kv_min(kv_max(kv_max(p0, 0) - window + 1, 0), hi) : 0;
    const int sk = window ? kv_min(sinks, lo) : 0;
    const int ns = (int)(((int64_t)sk + (1 << slog) - 1) >> slog);
    if (window && lo == hi) {   // the window lies past the last page: sinks alone
        s.n = kv_max(ns, 1);
        return s;
    }
    if (ns < (lo >> slog)) {
        s.sinks = ns;
        s.first = lo >> slog;
    }
    s.n = kv_max(s.sinks + end - s.first, 1);
    return s;
}
// First position of a span's step i.
QQ_HD int kv_base(const KvSpan &s, int i, int slog) { return (i < s.sinks ? i : s.first + i - s.sinks) << slog; }

// Tile t of a sequence of `len` positions whose last `rows` are the call's.
QQ_HD KvSpan kv_tile_span(int len, int rows, int t, int cols, int group, int cap, int window, int sinks, int slog)
{
    const int c0 = t * cols;
    const int r0 = c0 / group, r1 = kv_min((c0 + cols - 1) / group, rows - 1);
    return kv_span(len - rows + r0, len - rows + r1, cap, window, sinks, slog);
}

// (32 bits where they do: the quotient of 64 takes a few hundred clocks)
QQ_HD uint64_t kv_div(uint64_t a, uint64_t b) { return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b; }
// W steps over n parts: part w has [w W / n, (w + 1) W / n), and step x lies in
// part kv_part(x).  W < 2^50, n < 2^12.
QQ_HD uint64_t kv_cut(uint64_t W, uint32_t n, uint32_t w) { return kv_div(W * w, n); }
QQ_HD uint32_t kv_part(uint64_t W, uint32_t n, uint64_t x) { return (uint32_t)kv_div((x + 1) * n - 1, W); }
// How many parts: at least `least` steps each.
QQ_HD uint32_t kv_parts(uint64_t W, uint32_t most, uint32_t least)
{
    const uint64_t n = kv_div(W, least);
    return n < 1 ? 1 : n < most ? (uint32_t)n : most;
}

}  // namespace qq

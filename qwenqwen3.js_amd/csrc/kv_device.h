// kv_device.h -- how the kernels address a paged key/value cache.
#pragma once
#include "qq_device.h"

namespace qq {

// The cache's types: F32, and the 16-bit ones by their tag.
struct KvF32 {
    typedef float T;
    static constexpr int U = 4;   // values in a 16-byte unit
};
struct KvF16 {
    typedef uint16_t T;
    static constexpr int U = 8;
};
struct KvBf16 {
    typedef uint16_t T;
    static constexpr int U = 8;
};

__device__ __forceinline__ float kv_to_f32(KvF32, float v) { return v; }
__device__ __forceinline__ float kv_to_f32(KvF16, uint16_t v) { return __half2float(__ushort_as_half(v)); }
__device__ __forceinline__ float kv_to_f32(KvBf16, uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

// One rounding to the nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ float kv_from_f32(KvF32, float v) { return v; }
__device__ __forceinline__ uint16_t kv_from_f32(KvF16, float v) { return __half_as_ushort(__float2half_rn(v)); }
__device__ __forceinline__ uint16_t kv_from_f32(KvBf16, float v)
{
    const uint32_t u = __float_as_uint(v);
    if (v != v) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

// Sequence b's new rows [r0, r1), clipped to the call's rows.
__device__ __forceinline__ void kv_rows(const KvBatch &b, int seq, int &r0, int &r1)
{
    if (!b.row_start) {
        r0 = seq;
        r1 = seq + 1;
        return;
    }
    r0 = min(max(b.row_start[seq], 0), b.n_rows);
    r1 = min(max(b.row_start[seq + 1], r0), b.n_rows);
}

// Row t's sequence and position; false when no sequence has the row or the
// position is negative.
__device__ __forceinline__ bool kv_row(const KvBatch &b, int t, int &seq, int &pos)
{
    int end = t + 1;
    if (!b.row_start) {
        seq = t;
    } else {
        int lo = 0, hi = b.n_seqs - 1;   // the last sequence that starts at or ahead of t
        if (b.n_seqs <= WAVE) {          // by one load of the wave's (all of its lanes are here, for one t)
            const int l = threadIdx.x & (WAVE - 1);
            const uint64_t ahead = __ballot(b.row_start[min(l, hi)] <= t && l <= hi);
            lo = hi = ahead ? 63 - __builtin_clzll(ahead) : 0;
        }
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (b.row_start[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        seq = lo;
        end = b.row_start[seq + 1];
        if (t < b.row_start[seq] || t >= end) return false;
    }
    pos = max(b.len[seq], 0) - (end - t);
    return pos >= 0;
}

// The table's entry for position pos >= 0 of a sequence, read without a
// condition (a load under a branch is waited for where the branch ends, and
// everything in flight with it), and the page that it is, -1 for none.
__device__ __forceinline__ int kv_entry(const KvBatch &b, int seq, int pos)
{
    return b.table[(size_t)seq * b.stride + min(pos >> b.s.page_log, b.stride - 1)];
}
__device__ __forceinline__ int kv_page_of(const KvBatch &b, int pos, int entry)
{
    return (pos >> b.s.page_log) < b.stride && (unsigned)entry < (unsigned)b.s.n_pages ? entry : -1;
}
__device__ __forceinline__ int kv_page(const KvBatch &b, int seq, int pos)
{
    return kv_page_of(b, pos, kv_entry(b, seq, pos));
}

}  // namespace qq

// kv.hip -- filling and moving the pages of a key/value cache.
//
// Store: per-head RMSNorm (src/tensor.js:117-129) and split-half RoPE
// (:132-147) of the new rows' q and k, rounding to the cache's type, and the
// writes into pages.  A lane holds the pair (x[i], x[i + h]), h = D / 2, that
// RoPE turns together, so a wave holds 64 / h heads (one of D = 96 with 16
// lanes idle) and the sum of squares is a shuffle tree over h lanes.  The
// angle belongs to (row, i), not to the head: a lane forms its binary64 sine
// and cosine once and goes through the row's heads with them.
#include "kv_device.h"

// binary64 expressions of the reference stay separate multiplies and adds
#pragma clang fp contract(off)

namespace qq {

constexpr int KV_STORE_THREADS = 256;

template <class E, int D>
__global__ __launch_bounds__(KV_STORE_THREADS) void kv_store_kernel(KvBatch b, KvStore st)
{
    typedef typename E::T T;
    constexpr int U = E::U, H = D / 2;
    constexpr int HPW = H <= 32 ? WAVE / H : 1;   // heads a wave holds
    constexpr int NW = KV_STORE_THREADS / WAVE;
    const int t = blockIdx.x;
    int seq, pos;
    if (!kv_row(b, t, seq, pos)) return;
    const int page = kv_page(b, seq, pos);
    const int nkv = b.s.n_kv_heads, ps = b.s.page_size, slot = pos & (ps - 1);
    T *const kp = reinterpret_cast<T *>(b.pool + (size_t)max(page, 0) * b.s.page_bytes);
    T *const vp = kp + (size_t)nkv * ps * D;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = blockIdx.y * NW + threadIdx.x / WAVE, waves = gridDim.y * NW;
    const int i = lane % H;                        // this lane's pair ...
    const int sub = lane / H;                      // ... of the wave's head `sub`
    const bool in = sub < HPW;
    double c = 1.0, s = 0.0;
    if (st.rope) sincos((double)pos * st.freq[i], &s, &c);
    const int nh = st.n_heads + nkv;
    for (int g = wave; g * HPW < nh; g += waves) {
        const int head = g * HPW + sub;
        const bool live = in && head < nh;
        const bool is_k = head >= st.n_heads;
        const float *src = is_k ? st.k + ((size_t)t * nkv + (head - st.n_heads)) * D
                                : st.q + ((size_t)t * st.n_heads + head) * D;
        const float *nw = is_k ? st.kn : st.qn;
        float x0 = 0.0f, x1 = 0.0f;
        if (live) {
            x0 = src[i];
            x1 = src[i + H];
        }
        double ss = (double)x0 * (double)x0 + (double)x1 * (double)x1;
#pragma unroll
        for (int o = 1; o < (H <= 32 ? H : WAVE); o <<= 1) ss = ss + __shfl_xor(ss, o, WAVE);
        if (!live) continue;
        if (nw) {
            const double inv = 1.0 / sqrt(ss / (double)D + st.eps);
            x0 = (float)((double)nw[i] * (double)x0 * inv);
            x1 = (float)((double)nw[i + H] * (double)x1 * inv);
        }
        if (st.rope) {
            const double a = (double)x0, z = (double)x1;
            x0 = (float)(a * c - z * s);
            x1 = (float)(a * s + z * c);
        }
        if (!is_k) {
            float *dst = st.q_out + ((size_t)t * st.n_heads + head) * D;
            dst[i] = x0;
            dst[i + H] = x1;
        } else if (page >= 0) {
            T *dst = kp + (size_t)(head - st.n_heads) * ps * D;
            dst[((i / U) * ps + slot) * U + i % U] = kv_from_f32(E{}, x0);
            dst[(((i + H) / U) * ps + slot) * U + (i + H) % U] = kv_from_f32(E{}, x1);
        }
    }
    if (page < 0) return;
    for (int e = blockIdx.y * KV_STORE_THREADS + threadIdx.x; e < nkv * D; e += gridDim.y * KV_STORE_THREADS) {
        const int head = e / D, d = e % D;
        vp[(size_t)head * ps * D + ((slot / U) * D + d) * U + slot % U] = kv_from_f32(E{}, st.v[(size_t)t * nkv * D + e]);
    }
}

template <class E>
static void store_launch(qq_ctx *ctx, dim3 grid, const KvBatch &b, const KvStore &st)
{
    switch (b.s.head_dim) {
    case 32: QQ_LAUNCH(ctx, (kv_store_kernel<E, 32>), grid, dim3(KV_STORE_THREADS), 0, b, st); break;
    case 64: QQ_LAUNCH(ctx, (kv_store_kernel<E, 64>), grid, dim3(KV_STORE_THREADS), 0, b, st); break;
    case 96: QQ_LAUNCH(ctx, (kv_store_kernel<E, 96>), grid, dim3(KV_STORE_THREADS), 0, b, st); break;
    default: QQ_LAUNCH(ctx, (kv_store_kernel<E, 128>), grid, dim3(KV_STORE_THREADS), 0, b, st); break;
    }
}

int launch_kv_store(qq_ctx *ctx, const KvBatch &b, const KvStore &st)
{
    const int half = b.s.head_dim / 2, hpw = half <= 32 ? WAVE / half : 1;
    const int waves = (st.n_heads + b.s.n_kv_heads + hpw - 1) / hpw;
    const int gy = std::max(1, std::min((waves + 3) / 4, 512 / b.n_rows));
    const dim3 grid(b.n_rows, gy);
    prof_begin(ctx, K_KV_STORE);
    if (b.s.type == QQ_TYPE_F32) store_launch<KvF32>(ctx, grid, b, st);
    else if (b.s.type == QQ_TYPE_F16) store_launch<KvF16>(ctx, grid, b, st);
    else store_launch<KvBf16>(ctx, grid, b, st);
    prof_end(ctx);
    QQ_HIP(ctx, hipGetLastError());
    return QQ_OK;
}

// ---- pages ---------------------------------------------------------------------

// Grid (pair, layer): a page of one layer is one run of page_bytes (a multiple
// of 512), copied 16 bytes a lane.
__global__ __launch_bounds__(256) void kv_copy_kernel(char *pool, size_t page_bytes, int n_pages,
                                                      const int32_t *__restrict__ pairs)
{
    const int src = pairs[2 * blockIdx.x], dst = pairs[2 * blockIdx.x + 1];
    if ((unsigned)src >= (unsigned)n_pages || (unsigned)dst >= (unsigned)n_pages || src == dst) return;
    char *layer = pool + (size_t)blockIdx.y * n_pages * page_bytes;
    const uint4 *s = reinterpret_cast<const uint4 *>(layer + (size_t)src * page_bytes);
    uint4 *d = reinterpret_cast<uint4 *>(layer + (size_t)dst * page_bytes);
    for (size_t i = threadIdx.x; i < page_bytes / 16; i += 256) d[i] = s[i];
}

int launch_kv_copy(qq_ctx *ctx, const KvShape &s, char *pool, const int32_t *pairs, int n)
{
    prof_begin(ctx, K_KV_PAGES);
    QQ_LAUNCH(ctx, kv_copy_kernel, dim3(n, s.n_layers), dim3(256), 0, pool, s.page_bytes, s.n_pages, pairs);
    prof_end(ctx);
    QQ_HIP(ctx, hipGetLastError());
    return QQ_OK;
}

__global__ __launch_bounds__(256) void kv_remap_kernel(int32_t *__restrict__ table, int n,
                                                       const int32_t *__restrict__ map, int n_map)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int g = table[i];
    if ((unsigned)g < (unsigned)n_map) table[i] = map[g];
}

int launch_kv_remap(qq_ctx *ctx, int32_t *table, int n, const int32_t *map, int n_map)
{
    prof_begin(ctx, K_KV_PAGES);
    QQ_LAUNCH(ctx, kv_remap_kernel, dim3((unsigned)(((size_t)n + 255) / 256)), dim3(256), 0, table, n, map, n_map);
    prof_end(ctx);
    QQ_HIP(ctx, hipGetLastError());
    return QQ_OK;
}

}  // namespace qq

// kv.hip -- filling and moving the pages of a key/value cache.
//
// Store: per-head RMSNorm (src/tensor.js:117-129) and split-half RoPE
// (:132-147) of the new rows' q and k, rounding to the cache's type, and the
// writes into pages.  A lane holds the pair (x[i], x[i + h]), h = D / 2, that
// RoPE turns together, so a wave holds 64 / h heads (one of D = 96 with 16
// lanes idle) and the sum of squares is a shuffle tree over h lanes.  The
// angle belongs to (row, i), not to the head: a workgroup forms its row's
// binary64 sines and cosines once, and its waves go through the row's heads.
// Measured: 64 rows of 32 + 4 heads of 128 5.2 us, a launch and three loads
// one behind the other; 1470 rows of 32 + 8 heads of 64 13.1 us, 2.5 TB/s,
// waves waiting two thirds of the time and binary64 half of the rest.
#include "kv_device.h"

// binary64 expressions of the reference stay separate multiplies and adds
#pragma clang fp contract(off)

namespace qq {

constexpr int KV_STORE_THREADS = 256;

__device__ __forceinline__ double f64_of(uint32_t lo, uint32_t hi)
{
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// Sum over a head's lanes (16, 32 or, with more, all 64), in every lane:
// rotations within rows of 16, then rows and halves of the wave swapped, where
// shuffles would go through LDS.
template <int LANES>
__device__ __forceinline__ double lanes_sum(double v)
{
    v = v + dpp_f64<0x128>(v);
    v = v + dpp_f64<0x124>(v);
    v = v + dpp_f64<0x122>(v);
    v = v + dpp_f64<0x121>(v);
    if (LANES > 16) {
        const uint64_t b = __double_as_longlong(v);
        auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
        auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        v = f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]);
    }
    if (LANES > 32) {
        const uint64_t b = __double_as_longlong(v);
        auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
        auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        v = f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]);
    }
    return v;
}

template <class E, int D>
__global__ __launch_bounds__(KV_STORE_THREADS) void kv_store_kernel(KvBatch b, KvStore st)
{
    typedef typename E::T T;
    constexpr int U = E::U, H = D / 2;
    constexpr int HPW = H <= 32 ? WAVE / H : 1;   // heads a wave holds
    constexpr int NW = KV_STORE_THREADS / WAVE;
    const int t = blockIdx.x;
    const int nkv = b.s.n_kv_heads, ps = b.s.page_size;
    const int lane = threadIdx.x & (WAVE - 1);
    const int wave = blockIdx.y * NW + threadIdx.x / WAVE, waves = gridDim.y * NW;
    const int i = lane % H;                        // this lane's pair ...
    const int sub = lane / H;                      // ... of the wave's head `sub`
    const bool in = sub < HPW;
    const int nh = st.n_heads + nkv;
    // a head's pair is loaded while the one before it is worked on, the first
    // ahead of all that says where the row stands
    auto source = [&](int g) {
        const int head = min(g * HPW + min(sub, HPW - 1), nh - 1);
        return (head < st.n_heads ? st.q + ((size_t)t * st.n_heads + head) * D
                                  : st.k + ((size_t)t * nkv + (head - st.n_heads)) * D) + i;
    };
    const float *src = source(wave);
    float n0 = src[0], n1 = src[H];
    int seq, pos;
    if (!kv_row(b, t, seq, pos)) return;
    const int page = kv_page(b, seq, pos), slot = pos & (ps - 1);
    T *const kp = reinterpret_cast<T *>(b.pool + (size_t)max(page, 0) * b.s.page_bytes);
    T *const vp = kp + (size_t)nkv * ps * D;
    __shared__ double turn[2][H];
    if (st.rope) {
        if ((int)threadIdx.x < H) sincos((double)pos * st.freq[threadIdx.x], &turn[0][threadIdx.x], &turn[1][threadIdx.x]);
        __syncthreads();
    }
    const double s = turn[0][i], c = turn[1][i];   // used only with RoPE
    for (int g = wave; g * HPW < nh; g += waves) {
        const int head = g * HPW + sub;
        const bool live = in && head < nh;
        const bool is_k = head >= st.n_heads;
        const float *nw = is_k ? st.kn : st.qn;
        float x0 = live ? n0 : 0.0f, x1 = live ? n1 : 0.0f;
        src = source(g + waves);
        n0 = src[0];
        n1 = src[H];
        const double ss = lanes_sum<H>((double)x0 * (double)x0 + (double)x1 * (double)x1);
        if (!live) continue;
        if (nw) {
            const double inv = rsqrt(ss / (double)D + st.eps);
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
    // V: a unit holds U positions, so the first row of a unit that the call
    // has writes for all of them, whole units with one store of 16 bytes
    // (rows one by one: 2 bytes each, 16 apart).
    int first = seq, end = seq + 1;
    if (b.row_start) kv_rows(b, seq, first, end);
    const int at = slot % U;
    if (page < 0 || (at && t > first && pos > 0)) return;
    const int n = min(U - at, end - t);
    const float *v = st.v + (size_t)t * nkv * D;
    for (int e = blockIdx.y * KV_STORE_THREADS + threadIdx.x; e < nkv * D; e += gridDim.y * KV_STORE_THREADS) {
        T *dst = vp + (size_t)(e / D) * ps * D + ((slot / U) * D + e % D) * U;
        union {
            T x[U];
            uint4 w;
        } u;
#pragma unroll
        for (int r = 0; r < U; r++) u.x[r] = kv_from_f32(E{}, v[(size_t)min(r, n - 1) * nkv * D + e]);
        if (n == U) {
            *reinterpret_cast<uint4 *>(dst) = u.w;
        } else {
#pragma unroll
            for (int r = 0; r < U; r++)
                if (r < n) dst[at + r] = u.x[r];
        }
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
    // one pass of a workgroup's waves over the row's heads while rows are few (64 rows 5.2 us, a workgroup a row 10; 1470 rows the same)
    const int gy = std::max(1, std::min((waves + 3) / 4, 1024 / b.n_rows));
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

// Grid (pair, layer, piece): a page of one layer is one run of page_bytes (a
// multiple of 512), copied in pieces of 16 KiB, four 16-byte loads of a lane in
// flight: 5.0 TB/s, read and written, for 100 MB, the rate of a large copy.
constexpr int KV_PIECE = 16384;
__global__ __launch_bounds__(256) void kv_copy_kernel(char *pool, size_t page_bytes, int n_pages,
                                                      const int32_t *__restrict__ pairs)
{
    const int src = pairs[2 * blockIdx.x], dst = pairs[2 * blockIdx.x + 1];
    if ((unsigned)src >= (unsigned)n_pages || (unsigned)dst >= (unsigned)n_pages || src == dst) return;
    char *layer = pool + (size_t)blockIdx.y * n_pages * page_bytes;
    const size_t off = (size_t)blockIdx.z * KV_PIECE;
    typedef unsigned int v4u __attribute__((ext_vector_type(4)));
    const v4u *s = reinterpret_cast<const v4u *>(layer + (size_t)src * page_bytes + off);
    v4u *d = reinterpret_cast<v4u *>(layer + (size_t)dst * page_bytes + off);
    const int n = (int)(std::min<size_t>(KV_PIECE, page_bytes - off) / 16);
    v4u v[KV_PIECE / 4096];
#pragma unroll
    for (int i = 0; i < KV_PIECE / 4096; i++) v[i] = __builtin_nontemporal_load(s + min(256 * i + (int)threadIdx.x, n - 1));
#pragma unroll
    for (int i = 0; i < KV_PIECE / 4096; i++)
        if (256 * i + (int)threadIdx.x < n) __builtin_nontemporal_store(v[i], d + 256 * i + threadIdx.x);
}

int launch_kv_copy(qq_ctx *ctx, const KvShape &s, char *pool, const int32_t *pairs, int n)
{
    const unsigned pieces = (unsigned)((s.page_bytes + KV_PIECE - 1) / KV_PIECE);   // at most 2^12
    prof_begin(ctx, K_KV_PAGES);
    QQ_LAUNCH(ctx, kv_copy_kernel, dim3(n, s.n_layers, pieces), dim3(256), 0, pool, s.page_bytes, s.n_pages, pairs);
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

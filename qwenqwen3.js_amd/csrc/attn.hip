// attn.hip -- attention of new rows over the pages of a key/value cache.
//
// One wave per (row, query head): 64 positions a step, a lane each for the
// scores, then a lane per dimension for the sum over values, with the running
// maximum and sum of a softmax (fp32).
#include "kv_device.h"

namespace qq {

__device__ __forceinline__ float wave_maxf(float v)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, WAVE));
    return v;
}

template <class E, int D>
__global__ __launch_bounds__(WAVE) void kv_attn_simple_kernel(KvBatch b, KvAttn a)
{
    typedef typename E::T T;
    constexpr int U = E::U, ND = (D + WAVE - 1) / WAVE;
    __shared__ float ql[D];
    __shared__ float pl[WAVE];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    int seq, pos;
    const bool live = kv_row(b, t, seq, pos);
    if (!live) {
        // a padding row gives zeros; a row of no sequence stays
        bool own = !b.row_start;
        for (int s = 0; !own && s < b.n_seqs; s++) {
            int r0, r1;
            kv_rows(b, s, r0, r1);
            own = t >= r0 && t < r1;
        }
        if (own)
            for (int d = lane; d < D; d += WAVE) a.out[((size_t)t * a.n_heads + h) * D + d] = 0.0f;
        return;
    }
    const int nkv = b.s.n_kv_heads, ps = b.s.page_size, kvh = h / a.group;
    for (int d = lane; d < D; d += WAVE) ql[d] = a.q[((size_t)t * a.n_heads + h) * D + d];
    __syncthreads();
    const int cap = b.stride << b.s.page_log;
    const int hi = min(pos, cap - 1) + 1;                       // sees [0, sinks) and [lo, hi)
    const int lo = a.window ? max(0, pos - a.window + 1) : 0;
    const int sinks = min(a.sinks, hi);
    float m = -INFINITY, l = 0.0f, acc[ND] = {};
    for (int base = 0; base < hi; base += WAVE) {
        if (base >= sinks && base + WAVE <= lo) {
            base = (lo & ~(WAVE - 1)) - WAVE;
            continue;
        }
        const int p = base + lane;
        const int page = p < hi ? kv_page(b, seq, p) : -1;
        const bool see = page >= 0 && (p >= lo || p < sinks);
        float s = -INFINITY;
        if (see) {
            const T *k = reinterpret_cast<const T *>(b.pool + (size_t)page * b.s.page_bytes) + (size_t)kvh * ps * D;
            float dot = 0.0f;
            for (int c = 0; c < D / U; c++)
                for (int e = 0; e < U; e++)
                    dot = fmaf(ql[c * U + e], kv_to_f32(E{}, k[(c * ps + (p & (ps - 1))) * U + e]), dot);
            s = dot * (float)a.scale;
        }
        const float mn = fmaxf(m, wave_maxf(s));
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float pr = see ? expf(s - ms) : 0.0f, f = expf(m - ms);
        m = mn;
        l = l * f + wave_sum(pr);
        __syncthreads();
        pl[lane] = see ? pr : -1.0f;   // -1: not seen
        __syncthreads();
        for (int j = 0; j < ND; j++) acc[j] *= f;
        for (int j = 0; j < WAVE && base + j < hi; j++) {
            const float w = pl[j];
            if (w < 0.0f) continue;
            const int g = kv_page(b, seq, base + j), slot = (base + j) & (ps - 1);
            const T *v = reinterpret_cast<const T *>(b.pool + (size_t)g * b.s.page_bytes) + (size_t)(nkv + kvh) * ps * D;
            for (int n = 0; n < ND; n++) {
                const int d = n * WAVE + lane;
                if (d < D) acc[n] = fmaf(w, kv_to_f32(E{}, v[((slot / U) * D + d) * U + slot % U]), acc[n]);
            }
        }
    }
    for (int n = 0; n < ND; n++) {
        const int d = n * WAVE + lane;
        if (d < D) a.out[((size_t)t * a.n_heads + h) * D + d] = l == 0.0f ? 0.0f : acc[n] / l;
    }
}

template <class E>
static void attn_launch(qq_ctx *ctx, const KvBatch &b, const KvAttn &a)
{
    const dim3 grid(b.n_rows, a.n_heads);
    switch (b.s.head_dim) {
    case 32: QQ_LAUNCH(ctx, (kv_attn_simple_kernel<E, 32>), grid, dim3(WAVE), 0, b, a); break;
    case 64: QQ_LAUNCH(ctx, (kv_attn_simple_kernel<E, 64>), grid, dim3(WAVE), 0, b, a); break;
    case 96: QQ_LAUNCH(ctx, (kv_attn_simple_kernel<E, 96>), grid, dim3(WAVE), 0, b, a); break;
    default: QQ_LAUNCH(ctx, (kv_attn_simple_kernel<E, 128>), grid, dim3(WAVE), 0, b, a); break;
    }
}

int launch_kv_attn(qq_ctx *ctx, const qq_kv *, const KvBatch &b, const KvAttn &a)
{
    prof_begin(ctx, K_KV_ATTN);
    if (b.s.type == QQ_TYPE_F32) attn_launch<KvF32>(ctx, b, a);
    else if (b.s.type == QQ_TYPE_F16) attn_launch<KvF16>(ctx, b, a);
    else attn_launch<KvBf16>(ctx, b, a);
    prof_end(ctx);
    QQ_HIP(ctx, hipGetLastError());
    return QQ_OK;
}

}  // namespace qq

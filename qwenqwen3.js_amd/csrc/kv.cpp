// kv.cpp -- the host side of the paged key/value cache (include/qq_moe.h):
// pool handles, the checks of the device calls, and the book-keeping of pages.
#include <cmath>
#include <new>
#include <vector>

#include "qq_internal.h"

using namespace qq;

// ---- pages: who uses which -----------------------------------------------------

// Free pages are kept as a stack with the lowest numbers on top at the start,
// so a pool fills from its front; a page's users are the sequences whose rows
// hold it.  A sequence holds exactly the pages of its length.
struct qq_pages {
    struct Seq {
        bool live = false;
        int len = 0;
        std::vector<int32_t> pages;
    };
    int n_pages = 0, page_size = 0;
    std::vector<int32_t> users, free;
    std::vector<Seq> seqs;
    std::vector<int> idle;   // numbers of ended sequences
};

namespace {

int pages_error(const char *what) { return set_error(nullptr, "%s", what); }

int no_memory()
{
    set_error(nullptr, "host allocation failed");
    return QQ_E_NOMEM;
}

int pages_of(const qq_pages *p, int len) { return (int)(((long long)len + p->page_size - 1) / p->page_size); }

bool is_seq(const qq_pages *p, int seq) { return p && seq >= 0 && (size_t)seq < p->seqs.size() && p->seqs[seq].live; }

int no_seq(int seq) { return set_error(nullptr, "qq_pages: no sequence %d", seq); }

// The last pages of a sequence, from count n on, lose this user.  (The stack
// has room for every page: nothing here allocates.)
void drop(qq_pages *p, qq_pages::Seq &s, size_t n)
{
    while (s.pages.size() > n) {
        const int32_t g = s.pages.back();
        s.pages.pop_back();
        if (--p->users[g] == 0) p->free.push_back(g);
    }
}

// A number for a new sequence.
int new_seq(qq_pages *p)
{
    if (!p->idle.empty()) {
        const int id = p->idle.back();
        p->idle.pop_back();
        return id;
    }
    p->seqs.emplace_back();
    p->idle.reserve(p->seqs.size());   // ending it then allocates nothing
    return (int)p->seqs.size() - 1;
}

}  // namespace

extern "C" {

int qq_pages_create(int n_pages, int page_size, qq_pages **out)
{
    if (!out) return pages_error("qq_pages_create: out is NULL");
    *out = nullptr;
    if (n_pages < 1 || n_pages > 1 << 24 || page_size < 1) return set_error(nullptr, "qq_pages_create: %d pages of %d", n_pages, page_size);
    qq_pages *p = new (std::nothrow) qq_pages();
    if (!p) return no_memory();
    try {
        p->n_pages = n_pages;
        p->page_size = page_size;
        p->users.assign(n_pages, 0);
        p->free.resize(n_pages);
        for (int i = 0; i < n_pages; i++) p->free[i] = n_pages - 1 - i;
    } catch (...) {
        delete p;
        return no_memory();
    }
    *out = p;
    return QQ_OK;
}

int qq_pages_release(qq_pages *p)
{
    delete p;
    return QQ_OK;
}

int qq_pages_new(qq_pages *p, int *seq)
{
    if (!p || !seq) return pages_error("qq_pages_new: NULL argument");
    try {
        const int id = new_seq(p);
        p->seqs[id].live = true;
        *seq = id;
    } catch (...) {
        return no_memory();
    }
    return QQ_OK;
}

int qq_pages_extend(qq_pages *p, int seq, int n, int32_t *pair, int *n_pairs)
{
    if (!p || !pair || !n_pairs) return pages_error("qq_pages_extend: NULL argument");
    if (!is_seq(p, seq)) return no_seq(seq);
    qq_pages::Seq &s = p->seqs[seq];
    if (n < 0 || n > INT32_MAX - s.len) return set_error(nullptr, "qq_pages_extend: %d positions behind %d", n, s.len);
    *n_pairs = 0;
    if (n == 0) return QQ_OK;
    const int want = pages_of(p, s.len + n);
    // the page that holds the next position, when others use it too
    const bool own = s.len % p->page_size != 0 && p->users[s.pages.back()] > 1;
    const size_t need = (size_t)want - s.pages.size() + (own ? 1 : 0);
    if (need > p->free.size()) {
        set_error(nullptr, "qq_pages_extend: %zu pages needed, %zu free", need, p->free.size());
        return QQ_E_NOMEM;
    }
    try {
        s.pages.reserve(want);
    } catch (...) {
        return no_memory();
    }
    auto take = [&] {
        const int32_t g = p->free.back();
        p->free.pop_back();
        p->users[g] = 1;
        return g;
    };
    if (own) {
        pair[0] = s.pages.back();
        p->users[pair[0]]--;
        pair[1] = s.pages.back() = take();
        *n_pairs = 1;
    }
    while ((int)s.pages.size() < want) s.pages.push_back(take());
    s.len += n;
    return QQ_OK;
}

int qq_pages_fork(qq_pages *p, int seq, int len, int *out_seq)
{
    if (!p || !out_seq) return pages_error("qq_pages_fork: NULL argument");
    if (!is_seq(p, seq)) return no_seq(seq);
    if (len < 0 || len > p->seqs[seq].len)
        return set_error(nullptr, "qq_pages_fork: %d positions of a sequence of %d", len, p->seqs[seq].len);
    try {
        std::vector<int32_t> pages(p->seqs[seq].pages.begin(), p->seqs[seq].pages.begin() + pages_of(p, len));
        const int id = new_seq(p);   // may move the sequences
        for (int32_t g : pages) p->users[g]++;
        p->seqs[id].live = true;
        p->seqs[id].len = len;
        p->seqs[id].pages.swap(pages);
        *out_seq = id;
    } catch (...) {
        return no_memory();
    }
    return QQ_OK;
}

int qq_pages_truncate(qq_pages *p, int seq, int len)
{
    if (!is_seq(p, seq)) return no_seq(seq);
    qq_pages::Seq &s = p->seqs[seq];
    if (len < 0 || len > s.len) return set_error(nullptr, "qq_pages_truncate: %d positions of %d", len, s.len);
    drop(p, s, pages_of(p, len));
    s.len = len;
    return QQ_OK;
}

int qq_pages_free(qq_pages *p, int seq)
{
    if (!is_seq(p, seq)) return no_seq(seq);
    qq_pages::Seq &s = p->seqs[seq];
    drop(p, s, 0);
    s.len = 0;
    s.live = false;
    p->idle.push_back(seq);
    return QQ_OK;
}

int qq_pages_table(const qq_pages *p, int seq, int32_t *row, int cap, int *n, int *len)
{
    if (!is_seq(p, seq)) return no_seq(seq);
    const qq_pages::Seq &s = p->seqs[seq];
    if (row && (cap < 0 || (size_t)cap < s.pages.size()))
        return set_error(nullptr, "qq_pages_table: %zu pages, room for %d", s.pages.size(), cap);
    if (n) *n = (int)s.pages.size();
    if (len) *len = s.len;
    if (row)
        for (int i = 0; i < cap; i++) row[i] = (size_t)i < s.pages.size() ? s.pages[i] : -1;
    return QQ_OK;
}

int qq_pages_compact(qq_pages *p, int32_t *pairs, int cap, int *n_pairs, int32_t *map)
{
    if (!p || !n_pairs || (cap > 0 && !pairs)) return pages_error("qq_pages_compact: NULL argument");
    const int used = p->n_pages - (int)p->free.size();
    int moves = 0;
    for (int g = used; g < p->n_pages; g++) moves += p->users[g] > 0;
    if (cap < moves) return set_error(nullptr, "qq_pages_compact: %d pages move, room for %d", moves, cap);
    std::vector<int32_t> to;
    try {
        to.resize(p->n_pages);
    } catch (...) {
        return no_memory();
    }
    // the used pages past the first `used` numbers, in order, into the free ones among those
    int hole = 0, k = 0;
    for (int g = 0; g < p->n_pages; g++) {
        to[g] = g;
        if (g < used || !p->users[g]) continue;
        while (p->users[hole]) hole++;
        to[g] = hole;
        p->users[hole] = p->users[g];
        p->users[g] = 0;
        pairs[2 * k] = g;
        pairs[2 * k + 1] = hole;
        k++;
    }
    for (qq_pages::Seq &s : p->seqs)
        for (int32_t &g : s.pages) g = to[g];
    for (size_t i = 0; i < p->free.size(); i++) p->free[i] = p->n_pages - 1 - (int)i;
    if (map) memcpy(map, to.data(), to.size() * sizeof(int32_t));
    *n_pairs = k;
    return QQ_OK;
}

int qq_pages_count(const qq_pages *p, int *n_free, int *n_used)
{
    if (!p) return pages_error("qq_pages_count: NULL argument");
    if (n_free) *n_free = (int)p->free.size();
    if (n_used) *n_used = p->n_pages - (int)p->free.size();
    return QQ_OK;
}

// ---- pools ----------------------------------------------------------------------

static int pool_shape(qq_ctx *ctx, int n_layers, int n_pages, int page_size, int n_kv_heads, int head_dim, int type,
                      KvShape *s)
{
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
        return set_error(ctx, "kv: page size %d (16, 32, 64, 128 or 256)", page_size);
    if (head_dim != 32 && head_dim != 64 && head_dim != 96 && head_dim != 128)
        return set_error(ctx, "kv: head size %d (32, 64, 96 or 128)", head_dim);
    if (type != QQ_TYPE_F32 && type != QQ_TYPE_F16 && type != QQ_TYPE_BF16)
        return set_error(ctx, "kv: cache type %d (F32, F16 or BF16)", type);
    if (n_layers < 1 || n_layers > 4096 || n_pages < 1 || n_pages > 1 << 24 || n_kv_heads < 1 || n_kv_heads > 256)
        return set_error(ctx, "kv: bad shape (%d layers, %d pages, %d heads)", n_layers, n_pages, n_kv_heads);
    s->n_layers = n_layers;
    s->n_pages = n_pages;
    s->page_size = page_size;
    s->page_log = __builtin_ctz(page_size);
    s->n_kv_heads = n_kv_heads;
    s->head_dim = head_dim;
    s->type = type;
    // at most 2^26 bytes a page, 2^36 pages: no overflow
    s->page_bytes = (size_t)2 * n_kv_heads * page_size * head_dim * (type == QQ_TYPE_F32 ? 4 : 2);
    return QQ_OK;
}

int qq_kv_pool_bytes(int n_layers, int n_pages, int page_size, int n_kv_heads, int head_dim, int type, size_t *nbytes)
{
    if (!nbytes) return set_error(nullptr, "kv: NULL argument");
    KvShape s;
    if (int rc = pool_shape(nullptr, n_layers, n_pages, page_size, n_kv_heads, head_dim, type, &s)) return rc;
    *nbytes = s.page_bytes * n_pages * n_layers;
    return QQ_OK;
}

int qq_kv_create(qq_ctx *ctx, void *pool_dev, size_t nbytes, int n_layers, int n_pages, int page_size, int n_kv_heads,
                 int head_dim, int type, qq_kv **out)
{
    if (!ctx) return QQ_E_ARG;
    if (!out) return set_error(ctx, "kv_create: NULL argument");
    *out = nullptr;
    if (int rc = no_capture(ctx, "qq_kv_create")) return rc;
    KvShape s;
    if (int rc = pool_shape(ctx, n_layers, n_pages, page_size, n_kv_heads, head_dim, type, &s)) return rc;
    const size_t need = s.page_bytes * n_pages * n_layers;
    if (pool_dev && nbytes < need) return set_error(ctx, "kv_create: the pool needs %zu bytes, got %zu", need, nbytes);
    if ((uintptr_t)pool_dev % 16) return set_error(ctx, "kv_create: the pool is not 16-byte aligned");
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    qq_kv *kv = new (std::nothrow) qq_kv();
    if (!kv) return set_error(ctx, "host allocation failed");
    kv->ctx = ctx;
    kv->s = s;
    kv->nbytes = need;
    kv->pool = static_cast<char *>(pool_dev);
    hipError_t e = hipSuccess;
    if (!pool_dev) {
        void *v = nullptr;
        e = hipMalloc(&v, need);
        kv->pool = static_cast<char *>(v);
        kv->own_pool = true;
        if (e == hipSuccess) e = hipMemsetAsync(v, 0, need, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    }
    if (e == hipSuccess && !ctx->kv_work) {
        void *v = nullptr;
        e = hipMalloc(&v, kv_attn_work_bytes(ctx));
        if (e == hipSuccess) e = hipMemsetAsync(v, 0, kv_attn_counter_bytes(), ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
        if (e == hipSuccess) ctx->kv_work = static_cast<uint32_t *>(v);
        else if (v) (void)hipFree(v);
    }
    if (e != hipSuccess) {
        if (kv->own_pool && kv->pool) (void)hipFree(kv->pool);
        delete kv;
        return check_hip(ctx, e, "kv_create");
    }
    *out = kv;
    return QQ_OK;
}

static int kv_check(qq_ctx *ctx, const qq_kv *kv, const char *what)
{
    if (!ctx) return QQ_E_ARG;
    if (!kv) return set_error(ctx, "%s: NULL cache", what);
    if (kv->ctx != ctx) return set_error(ctx, "%s: the cache belongs to another context", what);
    return QQ_OK;
}

int qq_kv_release(qq_ctx *ctx, qq_kv *kv)
{
    if (!kv) return QQ_OK;
    if (int rc = kv_check(ctx, kv, "kv_release")) return rc;
    if (int rc = no_capture(ctx, "qq_kv_release")) return rc;
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    QQ_HIP(ctx, hipStreamSynchronize(ctx->stream));
    if (kv->own_pool) (void)hipFree(kv->pool);
    delete kv;
    return QQ_OK;
}

int qq_kv_pool(const qq_kv *kv, void **pool_dev, size_t *nbytes)
{
    if (!kv || !pool_dev || !nbytes) return set_error(nullptr, "kv_pool: NULL argument");
    *pool_dev = kv->pool;
    *nbytes = kv->nbytes;
    return QQ_OK;
}

// ---- device calls -----------------------------------------------------------------

static int batch_check(qq_ctx *ctx, const qq_kv *kv, int layer, const qq_kv_batch *b, const char *what)
{
    if (int rc = kv_check(ctx, kv, what)) return rc;
    if (layer < 0 || layer >= kv->s.n_layers)
        return set_error(ctx, "%s: layer %d of %d", what, layer, kv->s.n_layers);
    if (!b) return set_error(ctx, "%s: NULL batch", what);
    if (b->n_seqs < 0 || b->n_seqs > QQ_KV_MAX_SEQS)
        return set_error(ctx, "%s: %d sequences (at most %d)", what, b->n_seqs, QQ_KV_MAX_SEQS);
    // (a launch's first dimension: below 2^32 threads, 256 a row)
    if (b->n_rows < 0 || b->n_rows >= 1 << 24) return set_error(ctx, "%s: %d rows", what, b->n_rows);
    if (b->n_seqs == 0 || b->n_rows == 0) return QQ_OK;
    if (!b->table_dev || !b->len_dev) return set_error(ctx, "%s: NULL table or lengths", what);
    if (b->table_stride < 1 || (long long)b->table_stride * kv->s.page_size > 1 << 30)
        return set_error(ctx, "%s: a table row of %d pages of %d", what, b->table_stride, kv->s.page_size);
    if (!b->row_start_dev && b->n_rows != b->n_seqs)
        return set_error(ctx, "%s: %d rows of %d sequences without row_start", what, b->n_rows, b->n_seqs);
    return QQ_OK;
}

static KvBatch device_batch(const qq_kv *kv, int layer, const qq_kv_batch *b)
{
    KvBatch d;
    d.s = kv->s;
    d.pool = kv->pool + kv->s.page_bytes * kv->s.n_pages * layer;
    d.table = b->table_dev;
    d.len = b->len_dev;
    d.row_start = b->row_start_dev;
    d.n_seqs = b->n_seqs;
    d.n_rows = b->n_rows;
    d.stride = b->table_stride;
    return d;
}

static int heads_check(qq_ctx *ctx, const qq_kv *kv, int n_heads, const char *what)
{
    if (n_heads < 1 || n_heads > 4096 || n_heads % kv->s.n_kv_heads)
        return set_error(ctx, "%s: %d query heads over %d key/value heads", what, n_heads, kv->s.n_kv_heads);
    return QQ_OK;
}

static bool overlap(const void *a, const void *b, size_t nbytes)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nbytes && y < x + nbytes;
}

int qq_kv_store_dev(qq_ctx *ctx, qq_kv *kv, int layer, const qq_kv_batch *batch, const float *q_dev, int n_heads,
                    const float *k_dev, const float *v_dev, const float *q_norm_dev, const float *k_norm_dev,
                    double eps, double rope_base, float *q_out_dev)
{
    if (int rc = batch_check(ctx, kv, layer, batch, "kv_store")) return rc;
    if (!q_dev != !q_out_dev) return set_error(ctx, "kv_store: q and q_out go together");
    if (q_dev)
        if (int rc = heads_check(ctx, kv, n_heads, "kv_store")) return rc;
    if (!(eps >= 0.0) || !std::isfinite(eps)) return set_error(ctx, "kv_store: eps %g", eps);
    if (!(rope_base >= 0.0) || !std::isfinite(rope_base)) return set_error(ctx, "kv_store: rope_base %g", rope_base);
    if (batch->n_seqs == 0 || batch->n_rows == 0) return QQ_OK;
    if (!k_dev || !v_dev) return set_error(ctx, "kv_store: NULL buffer");
    if (q_dev && q_out_dev != q_dev &&
        overlap(q_dev, q_out_dev, (size_t)batch->n_rows * n_heads * kv->s.head_dim * sizeof(float)))
        return set_error(ctx, "kv_store: q_out overlaps q but is not q");
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    KvStore st;
    st.q = q_dev;
    st.q_out = q_out_dev;
    st.k = k_dev;
    st.v = v_dev;
    st.qn = q_norm_dev;
    st.kn = k_norm_dev;
    st.n_heads = q_dev ? n_heads : 0;
    st.eps = eps;
    st.rope = rope_base != 0.0;
    const int half = kv->s.head_dim / 2;
    for (int i = 0; i < KV_MAX_DIM / 2; i++)
        st.freq[i] = st.rope && i < half ? 1.0 / std::pow(rope_base, (double)i / half) : 0.0;
    return launch_kv_store(ctx, device_batch(kv, layer, batch), st);
}

int qq_kv_attn_dev(qq_ctx *ctx, qq_kv *kv, int layer, const qq_kv_batch *batch, const float *q_dev, int n_heads,
                   double scale, int window, int sinks, float *out_dev)
{
    if (int rc = batch_check(ctx, kv, layer, batch, "kv_attn")) return rc;
    if (int rc = heads_check(ctx, kv, n_heads, "kv_attn")) return rc;
    // (the kernels take powers of two, in fp32)
    if (!std::isfinite((float)(scale * 1.4426950408889634))) return set_error(ctx, "kv_attn: scale %g", scale);
    if (window < 0 || sinks < 0) return set_error(ctx, "kv_attn: window %d, sinks %d", window, sinks);
    if (batch->n_seqs == 0 || batch->n_rows == 0) return QQ_OK;
    if (!q_dev || !out_dev) return set_error(ctx, "kv_attn: NULL buffer");
    // steps of 16 positions, at the most that the tables allow: their count in 50 bits (kv_plan.h)
    const uint64_t tiles = ((uint64_t)batch->n_rows * n_heads + 15) / 16 + (uint64_t)batch->n_seqs * kv->s.n_kv_heads;
    if ((uint64_t)batch->n_rows * n_heads > 1u << 30 || tiles * ((uint64_t)batch->table_stride * kv->s.page_size / 16) >> 50)
        return set_error(ctx, "kv_attn: %d rows of %d heads over tables of %d pages", batch->n_rows, n_heads,
                         batch->table_stride);
    if (overlap(q_dev, out_dev, (size_t)batch->n_rows * n_heads * kv->s.head_dim * sizeof(float)))
        return set_error(ctx, "kv_attn: out overlaps q");
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    KvAttn a;
    a.q = q_dev;
    a.out = out_dev;
    a.n_heads = n_heads;
    a.group = n_heads / kv->s.n_kv_heads;
    a.scale = scale;
    a.window = window;
    a.sinks = window ? sinks : 0;
    return launch_kv_attn(ctx, device_batch(kv, layer, batch), a);
}

int qq_kv_copy_pages_dev(qq_ctx *ctx, qq_kv *kv, const int32_t *pairs_dev, int n)
{
    if (int rc = kv_check(ctx, kv, "kv_copy_pages")) return rc;
    if (n < 0 || n >= 1 << 24) return set_error(ctx, "kv_copy_pages: %d pairs", n);
    if (n == 0) return QQ_OK;
    if (!pairs_dev) return set_error(ctx, "kv_copy_pages: NULL buffer");
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    return launch_kv_copy(ctx, kv->s, kv->pool, pairs_dev, n);
}

int qq_kv_remap_dev(qq_ctx *ctx, int32_t *table_dev, int n, const int32_t *map_dev, int n_map)
{
    if (!ctx) return QQ_E_ARG;
    if (n < 0 || n_map < 0) return set_error(ctx, "kv_remap: %d entries, %d pages", n, n_map);
    if (n == 0 || n_map == 0) return QQ_OK;
    if (!table_dev || !map_dev) return set_error(ctx, "kv_remap: NULL buffer");
    QQ_HIP(ctx, hipSetDevice(ctx->device));
    return launch_kv_remap(ctx, table_dev, n, map_dev, n_map);
}

}  // extern "C"

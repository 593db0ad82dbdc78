// attn.hip -- attention of new rows over the pages of a key/value cache:
// softmax(scale q K^T) V with the running maximum and sum of a softmax, in
// one pass over the keys and values a row sees.
//
// A key/value head's query heads and rows are the 16 columns of one matrix
// product: a wave takes a step of 4 U positions (U values in 16 bytes: 16
// positions of fp32, 32 of the 16-bit types) and forms
//     S^T [positions x columns] = K Q^T,   O^T [dimensions x columns] += V^T P^T
// with 16x16 matrix instructions.  Lane l of a wave stands for column l % 16;
// j = l / 16 picks the unit of the inner index.  The result of the first
// product leaves lane (column, j) with the scores of 4 positions per
// instruction, and the second wants, in the same lane, the probabilities of U
// consecutive positions, unit j of the step.  Which position is which row of
// K's operand is free, so row m of instruction x is position U (m / 4) + 4 x +
// m % 4 of the step: the scores then are in the lane that needs them, and
// nothing moves between lanes but a maximum over j.  The operands come
// straight from the pool, 16 bytes a lane: its layout is the instructions'.
//
// Precision: a product of a 16-bit key with an fp32 query is exact where the
// query is taken as planes of that type (three of bf16, cut, 24 bits; two of
// fp16, rounded, 22 bits beside the column's largest, which is scaled to
// 2^14), and the same goes for probabilities (fp16: scaled by 2^14) and
// values; sums are fp32.  The matrix pipes are far from the bound here: the
// cache's bytes are.
//
// Work: all steps of the call in a row -- sequences, key/value heads, column
// tiles, each tile's span -- are cut into equal parts, one a workgroup,
// wherever the cuts fall (kv_plan.h); lengths are read on the device.  A tile
// counts AT_LEAD steps more than it has, ahead of its own: what its query,
// its first loads and its end cost a workgroup.  A workgroup's waves take its
// steps in turn and join in LDS; what a cut separates goes to the workspace,
// two slots a workgroup (a tile it goes on with from the workgroup before it,
// and one it leaves to the next), and the last workgroup to bring a tile's
// part joins them, in the order of the parts.
//
// Measured: 64 ragged sequences of up to 4096 positions, fp16, 8 heads of 64
// (312 MB) 56.5 us, 5.5 TB/s, bound by the reads and the ends of tiles; one
// of 100001 positions, bf16, 4 heads of 128 (205 MB) 44.3 us, the join of 128
// parts a head among them; one short sequence 8.9 us, a chain of latencies.
#include "kv_device.h"
#include "kv_plan.h"

#include <type_traits>

namespace qq {

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));

constexpr int AT_COLS = 16;      // columns of a tile
constexpr int AT_WAVES = 4;      // waves of a workgroup
constexpr int AT_THREADS = AT_WAVES * WAVE;
constexpr int AT_LEAD = 4;       // steps that a tile's beginning and end are worth (6: 64 ragged sequences 1 % longer)
constexpr int AT_LEAST = 4;      // steps a part has at least
constexpr int AT_MAX_PARTS = 4096;
constexpr int AT_GROUP = 16;     // parts of a tile that one workgroup joins (8, 32: 100001 positions 2 and 4 % longer)
// Workgroups of a CU.  Registers allow no more with heads of 128 (a wave keeps
// two steps of values and one of keys, q's planes and the sums); smaller heads
// fit three, but larger parts are worth more (heads of 64, 64 sequences of 1024
// and of 4096 positions 25 and 86 us, with three 33 and 92).
constexpr int AT_PER_CU = 2;

static int attn_parts(const qq_ctx *ctx) { return std::min(ctx->num_cus * AT_PER_CU, AT_MAX_PARTS - 1); }
// The form for many rows: 128 columns, 32 a wave
constexpr int AW_COLS = 128;
constexpr int AW_LEAD = 2;
constexpr int AW_GROUP = 8;
constexpr int AW_PER_CU = 2;
constexpr int AW_TILES = 32;     // tiles a call has at least
static int wide_parts(const qq_ctx *ctx) { return std::min(ctx->num_cus * AW_PER_CU, AT_MAX_PARTS - 1); }

// The workspace, one a context: counters of arrived parts, zero between
// launches (who finds its tile complete clears them), three for every
// workgroup; then its slots,
// in words of two floats: the columns' D sums (two planes of half of every
// four, or each thread's), then maximum and sum of probabilities of a column,
// or of each thread's.
__host__ __device__ constexpr int attn_slot(int cols, int dim) { return cols * (dim / 2 + 2); }
constexpr int AT_COUNTERS = 3 * AT_MAX_PARTS;   // their place depends on no launch: no slot may lie where another's counters do
size_t kv_attn_counter_bytes() { return sizeof(uint32_t) * AT_COUNTERS; }
size_t kv_attn_work_bytes(const qq_ctx *ctx)
{
    size_t words = 0;
    for (int dim = 32; dim <= KV_MAX_DIM; dim += 32)
        words = std::max({words, (size_t)attn_parts(ctx) * 2 * attn_slot(AT_COLS, dim),
                          (size_t)wide_parts(ctx) * 2 * attn_slot(AW_COLS, dim)});
    return kv_attn_counter_bytes() + sizeof(uint64_t) * words;
}

// Two fp32 rounded to fp16 in one register, and what rounding left of either
// (by the instructions: the compiler converts twice to take the pair apart).
__device__ __forceinline__ uint32_t f16_pair(float a, float b)
{
    uint32_t r;
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float f16_rest0(uint32_t h, float x)
{
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float f16_rest1(uint32_t h, float x)
{
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

// ---- operands by cache type: q's planes, a step's probabilities -------------------

// Fp32 keys and values: 16x16x4 instructions, one per element of the 16 bytes.
template <class E>
struct AtOps {
    static constexpr float PSHIFT = 0.0f;
    struct Q {
        float v[4];
    };
    typedef Q P;
    static __device__ __forceinline__ Q split(const float (&x)[4]) { return Q{{x[0], x[1], x[2], x[3]}}; }
    static __device__ __forceinline__ f4_t mul(const uint4 &a, const Q &q, f4_t c)
    {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[i]), q.v[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ f16_t mul(const uint4 &a, const Q &q, f16_t c)
    {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(w[i]), q.v[i], c, 0, 0, 0);
        return c;
    }
};

template <>
struct AtOps<KvBf16> {
    static constexpr float PSHIFT = 0.0f;
    struct Q {
        b8_t h, m, l;   // x = h + m + l
    };
    typedef Q P;
    static __device__ __forceinline__ Q split(const float (&x)[8])
    {
        uint32_t h[4], m[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
            float ra = x[2 * i] - __uint_as_float(a & 0xffff0000u), rb = x[2 * i + 1] - __uint_as_float(b & 0xffff0000u);
            h[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);   // the high halves
            a = __float_as_uint(ra);
            b = __float_as_uint(rb);
            ra -= __uint_as_float(a & 0xffff0000u);
            rb -= __uint_as_float(b & 0xffff0000u);
            m[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            l[i] = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
        }
        Q q;
        q.h = __builtin_bit_cast(b8_t, make_uint4(h[0], h[1], h[2], h[3]));
        q.m = __builtin_bit_cast(b8_t, make_uint4(m[0], m[1], m[2], m[3]));
        q.l = __builtin_bit_cast(b8_t, make_uint4(l[0], l[1], l[2], l[3]));
        return q;
    }
    static __device__ __forceinline__ f4_t mul(const uint4 &a, const Q &q, f4_t c)
    {
        const b8_t v = __builtin_bit_cast(b8_t, a);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, q.l, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, q.m, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, q.h, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16_t mul(const uint4 &a, const Q &q, f16_t c)
    {
        const b8_t v = __builtin_bit_cast(b8_t, a);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, q.l, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, q.m, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, q.h, c, 0, 0, 0);
    }
};

template <>
struct AtOps<KvF16> {
    static constexpr float PSHIFT = 14.0f;   // probabilities up to 2^14: 2^-39 of the largest is still told apart
    struct Q {
        h8_t h, l;   // x = h + l to 22 bits
    };
    typedef Q P;
    static __device__ __forceinline__ Q split(const float (&x)[8])
    {
        uint32_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            h[i] = f16_pair(x[2 * i], x[2 * i + 1]);
            l[i] = f16_pair(f16_rest0(h[i], x[2 * i]), f16_rest1(h[i], x[2 * i + 1]));
        }
        Q q;
        q.h = __builtin_bit_cast(h8_t, make_uint4(h[0], h[1], h[2], h[3]));
        q.l = __builtin_bit_cast(h8_t, make_uint4(l[0], l[1], l[2], l[3]));
        return q;
    }
    static __device__ __forceinline__ f4_t mul(const uint4 &a, const Q &q, f4_t c)
    {
        const h8_t v = __builtin_bit_cast(h8_t, a);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, q.l, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v, q.h, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f16_t mul(const uint4 &a, const Q &q, f16_t c)
    {
        const h8_t v = __builtin_bit_cast(h8_t, a);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, q.l, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(v, q.h, c, 0, 0, 0);
    }
};

// ---- lanes ------------------------------------------------------------------------

__device__ __forceinline__ float f_of(uint32_t v) { return __uint_as_float(v); }

// Maximum, or sum, over the four lanes of one column (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float col_max(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(f_of(a[0]), f_of(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(f_of(b[0]), f_of(b[1]));
}
__device__ __forceinline__ float col_sum(float v)
{
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f_of(a[0]) + f_of(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f_of(b[0]) + f_of(b[1]);
}

// A value from its bits.
__device__ __forceinline__ float at_value(KvF32, uint32_t b) { return __uint_as_float(b); }
template <class E>
__device__ __forceinline__ float at_value(E e, uint32_t b)
{
    return kv_to_f32(e, (uint16_t)b);
}

// 16 bytes of the pool, read once by the call or nearly so: not kept (four
// draft rows of 16 sequences 43.2 us, 46.0 kept).
__device__ __forceinline__ uint4 at_load(const char *p)
{
    typedef unsigned int v4u __attribute__((ext_vector_type(4)));
    const v4u v = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}

// The same over the two lanes of one column (l, l ^ 32).
__device__ __forceinline__ float half_max(float v)
{
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(f_of(b[0]), f_of(b[1]));
}
__device__ __forceinline__ float half_sum(float v)
{
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f_of(b[0]) + f_of(b[1]);
}

// ---- the plan, in every workgroup ---------------------------------------------------

// Tiles count by sequence, then column tile, the same for every key/value
// head; heads are the outer order.  A thread weighs T / NT tiles in a row; a
// step is found by a search over those runs and a walk through one of them.
// Up to 64 tiles of one row each, every wave has for itself, one a lane (one
// short sequence 9.6 us, 10.6 by runs).
struct AtTile {
    int seq, head, t;        // sequence, key/value head, column tile
    int row0, rows, len;     // the sequence's new rows and length
    uint64_t start;          // the tile's first step among the call's (LEAD of them ahead of its own)
    KvSpan span;
};

template <int NT>
struct AtPlan {
    uint64_t runs[NT + 1];   // steps of one head ahead of every thread's run
    uint64_t red[NT / WAVE];
};
// ... and in dynamic LDS, per sequence: its length, and where a sequence may
// have other than one row, its tiles' number among all, its first row, its rows
static size_t at_plan_bytes(const KvBatch &b) { return (size_t)(b.row_start ? 4 * b.n_seqs + 1 : b.n_seqs) * sizeof(int); }

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uni64(uint64_t v)
{
    return (uint64_t)(uint32_t)uni((int)(v >> 32)) << 32 | (uint32_t)uni((int)v);
}

// Exclusive prefix of one value a thread over the workgroup, and the total.
template <class V, int NT>
__device__ __forceinline__ V at_scan(V v, V &total, uint64_t *red)
{
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    V inc = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const V up = __shfl_up(inc, o, WAVE);
        if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == WAVE - 1) red[wave] = inc;
    __syncthreads();
    V off = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / WAVE; w++) {
        if (w < wave) off += (V)red[w];
        total += (V)red[w];
    }
    return off;
}

template <bool ROWS, int COLS, int LEAD, int SLOG, int NT>
struct AtWork {
    const KvBatch &b;
    const KvAttn &a;
    AtPlan<NT> &p;
    int *const len, *const first, *const row0, *const rows;
    int per;          // tiles of a run
    int each;         // tiles of a sequence of one row
    uint64_t S;       // steps of one head
    bool few;         // a tile a lane: its first step and its sequence's length
    uint32_t lane_start;
    int lane_len;

    __device__ AtWork(const KvBatch &b_, const KvAttn &a_, AtPlan<NT> &p_, int *lds)
        : b(b_), a(a_), p(p_), len(lds), first(lds + b_.n_seqs), row0(lds + 2 * b_.n_seqs + 1),
          rows(lds + 3 * b_.n_seqs + 1)
    {
        each = kv_tiles(1, a.group, COLS);
    }
    __device__ __forceinline__ KvSpan span(int ln, int rw, int t) const
    {
        return kv_tile_span(ln, rw, t, COLS, a.group, b.stride << b.s.page_log, a.window, a.sinks, SLOG);
    }
    // The sequence of tile g and its tile there.
    __device__ __forceinline__ void place(int g, int &seq, int &t) const
    {
        if (!ROWS) {
            seq = each == 1 ? g : g / each;
            t = each == 1 ? 0 : g - seq * each;
            return;
        }
        int lo = 0, hi = b.n_seqs - 1;   // the last sequence that starts at or ahead of g
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= g) lo = mid;
            else hi = mid - 1;
        }
        seq = lo;
        t = g - first[lo];
    }
    __device__ __forceinline__ void next(int &seq, int &t) const
    {
        t++;
        if (!ROWS) {
            if (t == each) {
                t = 0;
                seq++;
            }
            return;
        }
        if (t < first[seq + 1] - first[seq]) return;
        t = 0;
        do seq++;
        while (seq < b.n_seqs && first[seq + 1] == first[seq]);
    }
    // All steps of the call (the whole workgroup).
    __device__ __forceinline__ uint64_t plan()
    {
        const int tid = threadIdx.x;
        int T = b.n_seqs * each;
        few = !ROWS && T <= WAVE && ((int64_t)b.stride << b.s.page_log) <= 1 << 28;   // steps in 32 bits
        if (few) {
            const int g = tid & (WAVE - 1);
            int seq, t;
            place(min(g, T - 1), seq, t);
            lane_len = max(b.len[seq], 0);
            const uint32_t own = g < T ? span(lane_len, 1, t).n + LEAD : 0;
            uint32_t inc = own;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const uint32_t up = __shfl_up(inc, o, WAVE);
                if (g >= o) inc += up;
            }
            lane_start = inc - own;
            S = (uint32_t)__builtin_amdgcn_readlane((int)inc, WAVE - 1);
            return S * b.s.n_kv_heads;
        }
        for (int s = tid; s < b.n_seqs; s += NT) len[s] = max(b.len[s], 0);
        if (ROWS) {
            const int run = (b.n_seqs + NT - 1) / NT, s0 = min(tid * run, b.n_seqs), s1 = min(s0 + run, b.n_seqs);
            uint64_t sum = 0, all;
            for (int s = s0; s < s1; s++) {
                int r0, r1;
                kv_rows(b, s, r0, r1);
                row0[s] = r0;
                rows[s] = r1 - r0;
                first[s] = (int)sum;
                sum += kv_tiles(r1 - r0, a.group, COLS);
            }
            const uint64_t off = at_scan<uint64_t, NT>(sum, all, p.red);
            for (int s = s0; s < s1; s++) first[s] += (int)off;
            // more tiles than rows make: row_start falls, and the call does nothing
            T = all <= ((uint64_t)b.n_rows * a.group + COLS - 1) / COLS + b.n_seqs ? (int)all : 0;
            if (tid == 0) first[b.n_seqs] = T;
        }
        __syncthreads();
        T = uni(T);
        per = (T + NT - 1) / NT;
        const int g0 = min(tid * per, T), g1 = min(g0 + per, T);
        uint64_t sum = 0;
        if (g0 < g1) {
            int seq, t;
            place(g0, seq, t);
            for (int g = g0;;) {
                sum += span(len[seq], ROWS ? rows[seq] : 1, t).n + LEAD;
                if (++g == g1) break;
                next(seq, t);
            }
        }
        const uint64_t off = at_scan<uint64_t, NT>(sum, S, p.red);
        p.runs[tid] = off;
        if (tid == 0) p.runs[NT] = S;
        __syncthreads();
        S = uni64(S);
        return S * b.s.n_kv_heads;
    }
    // The tile that holds step x.
    __device__ __forceinline__ AtTile find(uint64_t x) const
    {
        AtTile t;
        t.head = (int)kv_div(x, S);
        const uint64_t base = S * t.head, r = x - base;
        if (few) {
            // the last tile that starts at or ahead of r (those behind the last start at S)
            const int g = 63 - __builtin_clzll(__ballot(lane_start <= (uint32_t)r));
            place(g, t.seq, t.t);
            t.len = __builtin_amdgcn_readlane(lane_len, g);
            t.rows = 1;
            t.row0 = t.seq;
            t.span = span(t.len, 1, t.t);
            t.start = base + (uint32_t)__builtin_amdgcn_readlane((int)lane_start, g);
            return t;
        }
        int lo = 0, hi = NT - 1;         // the last run that starts at or ahead of r
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (uni64(p.runs[mid]) <= r) lo = mid;
            else hi = mid - 1;
        }
        uint64_t start = uni64(p.runs[lo]);
        place(lo * per, t.seq, t.t);
        for (;;) {
            t.seq = uni(t.seq);
            t.t = uni(t.t);
            t.len = uni(len[t.seq]);
            t.rows = ROWS ? uni(rows[t.seq]) : 1;
            t.span = span(t.len, t.rows, t.t);
            if (r < start + LEAD + t.span.n) break;
            start += LEAD + t.span.n;
            next(t.seq, t.t);
        }
        t.row0 = ROWS ? uni(row0[t.seq]) : t.seq;
        t.start = base + start;
        return t;
    }
};

// ---- tiles in parts -------------------------------------------------------------------

// Slots are written through to memory and read from there (relaxed atomics of
// device scope), so that a workgroup on another XCD needs no cache written
// back or thrown away before it reads one: with fences in their place 64
// ragged sequences took 127 us, not 57.
// A slot is words of two floats, consecutive lanes' words side by side.
__device__ __forceinline__ void slot_put(uint64_t *p, float a, float b)
{
    __hip_atomic_store(p, (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 slot_get(const uint64_t *p)
{
    const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// A tile's parts w0 .. w0 + count - 1, this workgroup's the k-th.  Up to GROUP
// are joined by whoever brings the last; more in groups of so many first, by
// the last of each, into the group's first slot.
struct AtSplit {
    uint32_t *counters;
    uint64_t *slots;
    uint32_t w0;
    int k, count, slot;     // slot: words of one

    __device__ __forceinline__ AtSplit(uint32_t *work, int slot_, uint64_t W, uint32_t n, uint32_t part,
                                       uint64_t own, uint64_t tend)
        : counters(work), slots(reinterpret_cast<uint64_t *>(work + AT_COUNTERS)), slot(slot_)
    {
        w0 = kv_part(W, n, own);
        count = (int)(kv_part(W, n, tend - 1) - w0) + 1;
        k = (int)(part - w0);
    }
    __device__ __forceinline__ uint64_t *at(int i) const
    {
        return slots + (size_t)(2 * (w0 + i) + (i == 0)) * slot;
    }
    // Whether this workgroup is the last of `all` to count itself in: every
    // wave's stores to the slot are acknowledged first.
    __device__ __forceinline__ bool last(uint32_t *counter, int all, uint32_t *said) const
    {
        wait_vm<0>();
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if ((int)before == all - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *said = (int)before == all - 1;
        }
        __syncthreads();
        return *said;
    }
    // join(first, step, number, into): the parts first, first + step, ... into a slot, or the result (NULL)
    template <int GROUP, class F>
    __device__ __forceinline__ void bring(uint32_t *said, F join) const
    {
        if (count <= GROUP) {
            if (last(counters + w0, count, said)) join(0, 1, count, nullptr);
            return;
        }
        const int g = k / GROUP, first = g * GROUP, size = min(GROUP, count - first);
        // (a workgroup may be the first of one tile and in the middle of another)
        if (!last(counters + (g == 0 ? 1 : 2) * AT_MAX_PARTS + w0 + first, size, said)) return;
        join(first, 1, size, at(first));
        if (last(counters + w0, (count + GROUP - 1) / GROUP, said)) join(0, GROUP, (count + GROUP - 1) / GROUP, nullptr);
    }
};

// ---- the kernel ---------------------------------------------------------------------

// ROWS: a tile's columns may be several rows, that see different positions.
template <class E, int D, bool ROWS>
__global__ __launch_bounds__(AT_THREADS, AT_PER_CU) void kv_attn_kernel(KvBatch b, KvAttn a, uint32_t *work)
{
    typedef AtOps<E> Ops;
    constexpr int U = E::U, TK = U / 4, DS = D / (4 * U), DT = D / 16;
    constexpr int STEP = 4 * U, SLOG = U == 4 ? 4 : 5;
    constexpr uint32_t EXP = U == 4 ? 0x7f800000u : Ops::PSHIFT != 0.0f ? 0x7c00u : 0x7f80u;   // all ones: not finite
    constexpr int LDO = D + 4;   // floats of a column in LDS: the four lanes of a column 16 bytes apart, columns over all banks
    extern __shared__ int seqs[];
    __shared__ __align__(16) float so[AT_WAVES][AT_COLS][LDO];
    __shared__ float sm[AT_WAVES][AT_COLS], sl[AT_WAVES][AT_COLS];
    __shared__ AtPlan<AT_THREADS> plan;
    AtWork<ROWS, AT_COLS, AT_LEAD, SLOG, AT_THREADS> wk(b, a, plan, seqs);
    __shared__ uint32_t said;
    const uint64_t W = wk.plan();
    const uint32_t n = kv_parts(W, gridDim.x, AT_LEAST);
    // (no steps, or fewer parts than workgroups: none for this one)
    const uint64_t x0 = W && blockIdx.x < n ? kv_cut(W, n, blockIdx.x) : 0;
    const uint64_t x1 = W && blockIdx.x < n ? kv_cut(W, n, blockIdx.x + 1) : 0;

    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = uni(tid / WAVE);
    const int col = lane & 15, j = lane >> 4;
    const int nkv = b.s.n_kv_heads, ps = b.s.page_size, nh = a.n_heads, grp = a.group;
    // K's operand row `col` is a position of unit ku; its unit of dimensions is j + 4 s
    const int ku = col >> 2, kp = U * ku + (col & 3);
    const size_t vbase = (size_t)nkv * ps * D * (16 / U);
    const float qscale = (float)(a.scale * 1.4426950408889634);   // probabilities are powers of two

    for (uint64_t x = x0; x < x1;) {
        const AtTile t = wk.find(x);
        const uint64_t own = t.start + AT_LEAD, tend = own + t.span.n;
        x = tend;
        if (own >= x1) break;    // the next workgroup's
        const int i0 = x0 > own ? (int)(x0 - own) : 0;
        const int i1 = (int)((tend < x1 ? tend : x1) - own);
        const int c0 = t.t * AT_COLS, ncol = min(AT_COLS, t.rows * grp - c0);
        // rows of the tile's columns, and their positions
        const int p0 = t.len - t.rows + c0 / grp, p1 = t.len - t.rows + (c0 + ncol - 1) / grp;
        // columns behind the tile's last do what that one does, and are not stored
        const int cc = c0 + min(col, ncol - 1), cr = cc / grp;
        const int pos = t.len - t.rows + cr;
        const int low = a.window && pos >= 0 ? max(pos - a.window + 1, 0) : 0;
        const int low0 = a.window && p0 >= 0 ? max(p0 - a.window + 1, 0) : 0;   // what the tile's first ...
        const int low1 = a.window && p1 >= 0 ? max(p1 - a.window + 1, 0) : 0;   // ... and last row's windows start with
        const int sinks = a.sinks;

        float m = -INFINITY, l = 0.0f;
        f4_t o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};

        // Keys and values of the next step are loaded once this step's scores
        // are formed: a step is in flight all the time.  (Table entries are
        // read a step ahead of the loads that need them.)
        uint4 fk[TK][DS], fva[DT], fvb[DT];
        auto entries = [&](int i, int &gk, int &gv) {
            const int base = kv_base(t.span, min(i, i1 - 1), SLOG);
            gk = kv_entry(b, t.seq, base + U * ku);
            gv = kv_entry(b, t.seq, base + U * j);
        };
        auto load_k = [&](int i, int g) {
            const int at = kv_base(t.span, min(i, i1 - 1), SLOG) + kp, ks = at & (ps - 1);
            const char *src = b.pool + (size_t)max(kv_page_of(b, at, g), 0) * b.s.page_bytes + ((size_t)(t.head * (D / U) + j) * ps + ks) * 16;
#pragma unroll
            for (int s = 0; s < DS; s++)
#pragma unroll
                for (int xx = 0; xx < TK; xx++)
                    fk[xx][s] = at_load(src + (size_t)s * 64 * ps + 64 * xx);
        };
        auto load_v = [&](uint4 (&fv)[DT], int i, int g) {
            const int at = kv_base(t.span, min(i, i1 - 1), SLOG) + U * j, vs = at & (ps - 1);
            const char *src = b.pool + (size_t)max(kv_page_of(b, at, g), 0) * b.s.page_bytes + vbase +
                              ((size_t)(t.head * (ps / U) + vs / U) * D + col) * 16;
#pragma unroll
            for (int d = 0; d < DT; d++) fv[d] = at_load(src + 256 * d);
        };
        auto sums = [&](uint4 (&fv)[DT], float (&sc)[U], int base, int entry) {
            const int g = kv_page_of(b, base + U * j, entry);
            // every column sees every position of the step, or some do not
            const bool whole = base + STEP - 1 <= p0 && (base >= low1 || base + STEP <= sinks) &&
                               __all(g >= 0);
            const int up = base + U * j;    // this lane's first position
            bool odd = false;               // a value that is not finite, in a step that some rows see and others do not
            if (!whole) {
                uint32_t keep[U];
#pragma unroll
                for (int e = 0; e < U; e++) {
                    const int p = up + e;
                    const bool page = g >= 0;
                    sc[e] = page & (p <= pos) & ((p >= low) | (p < sinks)) ? sc[e] : -INFINITY;
                    // what no row of the tile sees may hold anything
                    keep[e] = page & (p <= p1) & ((p >= low0) | (p < sinks)) ? 0xffffffffu : 0u;
                }
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    uint32_t w[4] = {fv[d].x, fv[d].y, fv[d].z, fv[d].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        w[i] &= U == 4 ? keep[i % U] : (keep[(2 * i) % U] & 0xffffu) | (keep[(2 * i + 1) % U] & 0xffff0000u);
                        if (ROWS) odd |= (w[i] & EXP) == EXP || (U == 8 && (w[i] & (EXP << 16)) == EXP << 16);
                    }
                    fv[d] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            float mx = sc[0];
#pragma unroll
            for (int e = 1; e < U; e++) mx = fmaxf(mx, sc[e]);
            mx = fmaxf(m, col_max(mx));
            if (__any(mx > m)) {
                const float r = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.0f : mx));
                l *= r;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= r;
                m = mx;
            }
            const float sub = (m == -INFINITY ? 0.0f : m) - Ops::PSHIFT;
            float p[U];
#pragma unroll
            for (int e = 0; e < U; e++) {
                p[e] = __builtin_amdgcn_exp2f(sc[e] - sub);
                l += p[e];
            }
            if (ROWS && p0 != p1 && __any(odd)) {
                // Such values leave the product, where 0 times one would reach
                // the rows that do not see it, and are added one by one: lane
                // L holds dimension L % 16 of unit L / 16, and its probability
                // for this lane's column is in lane (column, unit).
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    uint32_t w[4] = {fv[d].x, fv[d].y, fv[d].z, fv[d].w};
#pragma unroll
                    for (int e = 0; e < U; e++) {
                        const int sh = U == 4 ? 0 : 16 * (e & 1);
                        const uint32_t bits = U == 4 ? w[e % 4] : (w[e / 2] >> sh) & 0xffffu;
                        const bool bad = (bits & EXP) == EXP;
                        for (uint64_t who = __ballot(bad); who; who &= who - 1) {
                            const int L = __builtin_ctzll(who);
                            const float v = at_value(E{}, __builtin_amdgcn_readlane(bits, L));
                            const float pr = __shfl(p[e], (L & 48) | col, WAVE);
                            const int at = base + U * (L >> 4) + e;
                            const bool sees = at <= pos && (at >= low || at < sinks);
                            const float add = sees && (L & 15) >> 2 == j ? pr * v : 0.0f;
#pragma unroll
                            for (int r = 0; r < 4; r++) o[d][r] += (L & 3) == r ? add : 0.0f;
                        }
                        if (bad) w[U == 4 ? e % 4 : e / 2] &= U == 4 ? 0u : 0xffff0000u >> sh;
                    }
                    fv[d] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            const typename Ops::P pp = Ops::split(p);
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] = Ops::mul(fv[d], pp, o[d]);
        };

        // ---- the first loads, then q in planes ----
        int i = i0 + wave;
        int gk, gv, now, gk1, gv1;
        entries(i, gk, now);
        entries(i + AT_WAVES, gk1, gv1);
        typename Ops::Q q[DS];
        float unscale = 1.0f;
        {
            f4_t v[DS][U / 4];
            const float *src = a.q + ((size_t)(t.row0 + cr) * nh + t.head * grp + cc % grp) * D + j * U;
#pragma unroll
            for (int s = 0; s < DS; s++)
#pragma unroll
                for (int e = 0; e < U / 4; e++) v[s][e] = *reinterpret_cast<const f4u_t *>(src + 4 * U * s + 4 * e);
            if (i < i1) {
                load_k(i, gk);
                load_v(fva, i, now);
            }
            gk = gk1;
            gv = gv1;
            __builtin_amdgcn_sched_barrier(0);
            float up = qscale;
            if (Ops::PSHIFT != 0.0f) {
                // the largest to [2^14, 2^15)
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < DS; s++)
#pragma unroll
                    for (int e = 0; e < U; e++) big = fmaxf(big, fabsf(v[s][e / 4][e % 4] * qscale));
                const int f = min(268 - (int)(__float_as_uint(col_max(big)) >> 23), 253);
                unscale = __uint_as_float((uint32_t)(254 - f) << 23);
                up = __uint_as_float((uint32_t)f << 23);
            }
#pragma unroll
            for (int s = 0; s < DS; s++) {
                float x[U];
#pragma unroll
                for (int e = 0; e < U; e++)
                    x[e] = Ops::PSHIFT != 0.0f ? v[s][e / 4][e % 4] * qscale * up : v[s][e / 4][e % 4] * qscale;
                q[s] = Ops::split(x);
            }
        }

        auto scores = [&](float (&sc)[U]) {
            f4_t s4[TK];
#pragma unroll
            for (int xx = 0; xx < TK; xx++) s4[xx] = f4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < DS; s++)
#pragma unroll
                for (int xx = 0; xx < TK; xx++) s4[xx] = Ops::mul(fk[xx][s], q[s], s4[xx]);
#pragma unroll
            for (int e = 0; e < U; e++) sc[e] = s4[e / 4][e % 4] * unscale;
        };
        auto step = [&](uint4 (&cur)[DT], uint4 (&next)[DT]) {
            float sc[U];
            scores(sc);
            __builtin_amdgcn_sched_barrier(0);
            if (i + AT_WAVES < i1) {
                load_k(i + AT_WAVES, gk);
                load_v(next, i + AT_WAVES, gv);
            }
            entries(i + 2 * AT_WAVES, gk, gv1);
            __builtin_amdgcn_sched_barrier(0);
            sums(cur, sc, kv_base(t.span, i, SLOG), now);
            __builtin_amdgcn_sched_barrier(0);
            now = gv;
            gv = gv1;
            i += AT_WAVES;
        };
        while (i < i1) {
            step(fva, fvb);
            if (i >= i1) break;
            step(fvb, fva);
        }

        // ---- the waves together ----
        l = col_sum(l);
        if (j == 0) {
            sm[wave][col] = m;
            sl[wave][col] = l;
        }
#pragma unroll
        for (int d = 0; d < DT; d++) *reinterpret_cast<f4_t *>(&so[wave][col][16 * d + 4 * j]) = o[d];
        __syncthreads();
        // whole: the result; else this workgroup's part of it
        const bool mine = i0 == 0 && i1 == t.span.n;
        const AtSplit split(work, attn_slot(AT_COLS, D), W, n, blockIdx.x, own, tend);
        auto result = [&](int c, int d, const f4_t &sum, float L) {
            const int row = t.row0 + (c0 + c) / grp, head = t.head * grp + (c0 + c) % grp;
            // nothing seen: L = 0 and a sum of zeros
            *reinterpret_cast<f4u_t *>(a.out + ((size_t)row * nh + head) * D + d) = L == 0.0f ? sum : sum / L;
        };
        auto keep = [&](uint64_t *slot, int c, int d, const f4_t &sum, float M, float L) {
            slot_put(slot + (c * D + d) / 4, sum[0], sum[1]);
            slot_put(slot + (AT_COLS * D + c * D + d) / 4, sum[2], sum[3]);
            if (d == 0) slot_put(slot + AT_COLS * D / 2 + c, M, L);
        };
        for (int e = tid; e < ncol * (D / 4); e += AT_THREADS) {
            const int c = e / (D / 4), d = e % (D / 4) * 4;
            float M = sm[0][c];
#pragma unroll
            for (int w = 1; w < AT_WAVES; w++) M = fmaxf(M, sm[w][c]);
            const float ms = M == -INFINITY ? 0.0f : M;
            f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
            float L = 0.0f;
#pragma unroll
            for (int w = 0; w < AT_WAVES; w++) {
                const float r = __builtin_amdgcn_exp2f(sm[w][c] - ms);
                sum += *reinterpret_cast<const f4_t *>(&so[w][c][d]) * r;
                L += sl[w][c] * r;
            }
            if (mine) result(c, d, sum, L);
            else keep(split.at(split.k), c, d, sum, M, L);
        }
        if (!mine)
            split.template bring<AT_GROUP>(&said, [&](int first, int by, int num, uint64_t *into) {
                // Whole columns a pass: a pass may leave the joined maximum and
                // sum of its columns where the parts' were.
                constexpr int PER = AT_THREADS / (D / 4), AHEAD = 8;
                for (int cp = 0; cp < ncol; cp += PER) {
                    // (threads behind the last column do its work and store nothing)
                    const bool live = tid < PER * (D / 4) && cp + tid / (D / 4) < ncol;
                    const int c = min(cp + min(tid / (D / 4), PER - 1), ncol - 1), d = tid % (D / 4) * 4;
                    float M = -INFINITY, L = 0.0f;
                    f4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int k = 0; k < num; k += AHEAD) {
                        float m[AHEAD], l[AHEAD];
                        f4_t v[AHEAD];
#pragma unroll
                        for (int u = 0; u < AHEAD; u++) {
                            const uint64_t *s = split.at(first + by * min(k + u, num - 1));
                            const float2 ml = slot_get(s + AT_COLS * D / 2 + c);
                            const float2 x = slot_get(s + (c * D + d) / 4), y = slot_get(s + (AT_COLS * D + c * D + d) / 4);
                            m[u] = ml.x;
                            l[u] = ml.y;
                            v[u] = f4_t{x.x, x.y, y.x, y.y};
                        }
                        float top = M;
#pragma unroll
                        for (int u = 0; u < AHEAD; u++) top = fmaxf(top, m[u]);
                        const float ts = top == -INFINITY ? 0.0f : top, r = __builtin_amdgcn_exp2f(M - ts);
                        sum *= r;
                        L *= r;
#pragma unroll
                        for (int u = 0; u < AHEAD; u++)
                            if (k + u < num) {
                                const float w = __builtin_amdgcn_exp2f(m[u] - ts);
                                sum += v[u] * w;
                                L += l[u] * w;
                            }
                        M = top;
                    }
                    __syncthreads();    // `into` is one of these slots
                    if (!live) continue;
                    if (into) keep(into, c, d, sum, M, L);
                    else result(c, d, sum, L);
                }
            });
        __syncthreads();   // LDS is used again
    }
}

// ---- many rows ----------------------------------------------------------------------

// The same over tiles of 128 columns, 32 a wave, for calls whose columns are
// many: keys and values go through LDS, where the four waves read them, and
// 32x32 instructions.  A stage is P positions of K, [D / U][P] units, and of
// V, [P / U][D] units, copied straight from the pool (asynchronously, 16 bytes
// a lane) while the stage before it is worked on; K's positions are stored in
// the order of the instruction's rows, so that every read of LDS is of
// consecutive units.  Row m = 8 a + 4 h + b of 32 is position 16 (a / 2) + 8 h
// + 4 (a % 2) + b of 16-bit types, m of fp32: the scores of a lane's half h
// then are those of whole units of V.
// Measured: a 4096-token prompt, fp16, 32 query heads of 64 over 8, 172 us, 400
// TFLOP/s of products with one plane counted of the two that are formed; the
// matrix and the vector pipes take turns there.
// ONE: pages of a stage or more.
template <class E, int D, bool ONE>
__global__ __launch_bounds__(AT_THREADS, AW_PER_CU) void kv_attn_wide_kernel(KvBatch b, KvAttn a, uint32_t *work)
{
    typedef AtOps<E> Ops;
    constexpr int U = E::U, P = U == 4 ? 32 : 64, SLOG = U == 4 ? 5 : 6;
    constexpr int KU = D / U * P, VU = P / U * D;          // units of a stage
    constexpr int NK = KU / AT_THREADS, NV = VU / AT_THREADS;
    constexpr int DS = D / (2 * U), DT = D / 32, HALVES = P / 32, NI = 16 / U;
    constexpr int JH = HALVES == 2 && D <= 64 ? 2 : 1;
    constexpr uint32_t EXP = U == 4 ? 0x7f800000u : Ops::PSHIFT != 0.0f ? 0x7c00u : 0x7f80u;
    static_assert(KU % AT_THREADS == 0 && VU % AT_THREADS == 0, "copies by whole workgroups");
    extern __shared__ int seqs[];
    __shared__ __align__(16) uint4 sk[2][KU], sv[2][VU];
    __shared__ AtPlan<AT_THREADS> plan;
    AtWork<true, AW_COLS, AW_LEAD, SLOG, AT_THREADS> wk(b, a, plan, seqs);
    __shared__ uint32_t said;
    const uint64_t W = wk.plan();
    const uint32_t n = kv_parts(W, gridDim.x, AT_LEAST);
    // parts in a row on one XCD (workgroups go to the eight in turn): they read the same keys and values
    const uint32_t per = (gridDim.x + 7) / 8;
    const uint32_t part = gridDim.x % 8 ? blockIdx.x : blockIdx.x % 8 * per + blockIdx.x / 8;
    const uint64_t x0 = W && part < n ? kv_cut(W, n, part) : 0;
    const uint64_t x1 = W && part < n ? kv_cut(W, n, part + 1) : 0;

    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = uni(tid / WAVE);
    const int col = lane & 31, h = lane >> 5;
    const int nkv = b.s.n_kv_heads, ps = b.s.page_size, nh = a.n_heads, grp = a.group;
    const size_t vbase = (size_t)nkv * ps * D * (16 / U);
    const float qscale = (float)(a.scale * 1.4426950408889634);
    // the position that this lane copies of K (unit tid of AT_THREADS: position tid % P in the rows' order)
    const int kr = tid % P % 32;
    const int kp = tid % P / 32 * 32 + (U == 4 ? kr : 16 * (kr >> 4) + 8 * (kr >> 2 & 1) + 4 * (kr >> 3 & 1) + (kr & 3));
    const uint32_t koff = (uint32_t)(tid / P * ps + kp) * 16;   // ... and its place behind the first one's
    // the position of register r among 32
    auto at = [&](int r) { return U == 4 ? 8 * (r >> 2) + 4 * h + (r & 3) : 16 * (r >> 3) + 8 * h + (r & 7); };
    const uint32_t lk = lds_u32(&sk[0][wave * WAVE]), lv = lds_u32(&sv[0][wave * WAVE]);

    for (uint64_t x = x0; x < x1;) {
        const AtTile t = wk.find(x);
        const uint64_t own = t.start + AW_LEAD, tend = own + t.span.n;
        x = tend;
        if (own >= x1) break;    // the next workgroup's
        const int i0 = x0 > own ? (int)(x0 - own) : 0;
        const int i1 = (int)((tend < x1 ? tend : x1) - own);
        const int c0 = t.t * AW_COLS, ncol = min(AW_COLS, t.rows * grp - c0);
        // this wave's columns, those behind the tile's last doing what that one does
        const bool any = wave * 32 < ncol;
        const int w0 = min(wave * 32, ncol - 1), w1 = min(wave * 32 + 31, ncol - 1);
        const int cc = c0 + min(wave * 32 + col, ncol - 1), cr = cc / grp;
        const int p0 = t.len - t.rows + (c0 + w0) / grp, p1 = t.len - t.rows + (c0 + w1) / grp;
        const int pos = t.len - t.rows + cr;
        const int low = a.window && pos >= 0 ? max(pos - a.window + 1, 0) : 0;
        const int low0 = a.window && p0 >= 0 ? max(p0 - a.window + 1, 0) : 0;
        const int low1 = a.window && p1 >= 0 ? max(p1 - a.window + 1, 0) : 0;
        const int sinks = a.sinks;
        // ... and of the whole tile: its first row, and where its last row's window starts
        const int tp0 = t.len - t.rows + c0 / grp, tp1 = t.len - t.rows + (c0 + ncol - 1) / grp;
        const int tl1 = a.window && tp1 >= 0 ? max(tp1 - a.window + 1, 0) : 0;

        // Table entries of the next copies, and the copies (which return which
        // of the stage's positions, in the rows' order, have a page).  With one
        // page a stage its number is a scalar, and lanes differ by a constant: a
        // 4096-token prompt 171 us, not 174.  (No load under a branch: it would be
        // waited for where the branch ends.)
        typedef const int32_t __attribute__((address_space(4))) *scalar_t;    // read by the scalar unit
        const scalar_t row = (scalar_t)(uintptr_t)(b.table + (size_t)t.seq * b.stride);
        int ek, ev[NV];
        auto entries = [&](int i) {
            const int base = kv_base(t.span, min(i, i1 - 1), SLOG);
            if constexpr (ONE) {
                ek = row[min(base >> b.s.page_log, b.stride - 1)];
            } else {
                ek = kv_entry(b, t.seq, base + kp);
#pragma unroll
                for (int k = 0; k < NV; k++) ev[k] = kv_entry(b, t.seq, base + (k * AT_THREADS + tid) / D * U);
            }
        };
        auto copy = [&](int i, int buf) -> uint64_t {
            const int base = kv_base(t.span, i, SLOG);
            if constexpr (ONE) {
                const int g = kv_page_of(b, base, ek), slot = base & (ps - 1);
                const char *page = b.pool + (size_t)max(g, 0) * b.s.page_bytes;
                const char *kb = page + ((size_t)t.head * (D / U) * ps + slot) * 16;
                const char *vb = page + vbase + ((size_t)t.head * ps + slot) * (D / U) * 16;
#pragma unroll
                for (int k = 0; k < NK; k++)
                    dma16s(koff, kb + (size_t)k * (AT_THREADS / P) * ps * 16, lk + (buf * KU + k * AT_THREADS) * 16);
#pragma unroll
                for (int k = 0; k < NV; k++)
                    dma16s(tid * 16, vb + k * AT_THREADS * 16, lv + (buf * VU + k * AT_THREADS) * 16);
                return g >= 0 ? ~(uint64_t)0 : 0;
            }
            const int at = base + kp, kg = kv_page_of(b, at, ek);
            const char *src = b.pool + (size_t)max(kg, 0) * b.s.page_bytes +
                              ((size_t)(t.head * (D / U) + tid / P) * ps + (at & (ps - 1))) * 16;
#pragma unroll
            for (int k = 0; k < NK; k++)
                dma16(src + (size_t)k * (AT_THREADS / P) * ps * 16, lk + (buf * KU + k * AT_THREADS) * 16);
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int g = k * AT_THREADS + tid, v = base + g / D * U;
                dma16(b.pool + (size_t)max(kv_page_of(b, v, ev[k]), 0) * b.s.page_bytes + vbase +
                          ((size_t)(t.head * (ps / U) + (v & (ps - 1)) / U) * D + g % D) * 16,
                      lv + (buf * VU + k * AT_THREADS) * 16);
            }
            return __ballot(kg >= 0);
        };
        entries(i0);
        lds_barrier();       // the stages are free: every wave is done with the tile before
        uint64_t pages = copy(i0, 0), pages_next = 0;
        entries(i0 + 1);

        // ---- q in planes ----
        typename Ops::Q q[DS];
        float unscale = 1.0f;
        {
            f4_t v[DS][U / 4];
            const float *src = a.q + ((size_t)(t.row0 + cr) * nh + t.head * grp + cc % grp) * D + h * U;
#pragma unroll
            for (int s = 0; s < DS; s++)
#pragma unroll
                for (int e = 0; e < U / 4; e++) v[s][e] = *reinterpret_cast<const f4u_t *>(src + 2 * U * s + 4 * e);
            float up = 1.0f;
            if (Ops::PSHIFT != 0.0f) {
                // the largest to [2^14, 2^15)
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < DS; s++)
#pragma unroll
                    for (int e = 0; e < U; e++) big = fmaxf(big, fabsf(v[s][e / 4][e % 4] * qscale));
                const int f = min(268 - (int)(__float_as_uint(half_max(big)) >> 23), 253);
                unscale = __uint_as_float((uint32_t)(254 - f) << 23);
                up = __uint_as_float((uint32_t)f << 23);
            }
#pragma unroll
            for (int s = 0; s < DS; s++) {
                float xs[U];
#pragma unroll
                for (int e = 0; e < U; e++) xs[e] = v[s][e / 4][e % 4] * qscale * up;
                q[s] = Ops::split(xs);
            }
        }

        float m = -INFINITY, l = 0.0f;
        f16_t o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = f16_t{};

        // A stage that some column of the tile does not see whole: what none of
        // them sees may hold anything, and leaves V for zeros.  So do values
        // that are not finite where some rows see them and others do not (0
        // times one would reach those): true, and they are added one by one.
        auto clean = [&](int base, int buf, uint64_t got) {
            const int ql = a.window && tp0 >= 0 ? max(tp0 - a.window + 1, 0) : 0;
            bool odd = false;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int g = k * AT_THREADS + tid, u = g / D;    // unit u of the stage: its row in K's order
                const int row = U == 4 ? 4 * u : 32 * (u >> 2) + 16 * (u >> 1 & 1) + 4 * (u & 1);
                const bool page = got >> row & 1;
                uint4 &v = sv[buf][g];
                uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < U; e++) {
                    const int p = base + u * U + e, sh = U == 4 ? 0 : 16 * (e & 1);
                    uint32_t &x = w[U == 4 ? e % 4 : e / 2];
                    const bool sees = page & (p <= tp1) & ((p >= ql) | (p < sinks));
                    const bool bad = ((x >> sh & EXP) == EXP) & (tp0 != tp1);
                    odd |= sees & bad;
                    x = (!sees | bad) ? x & (U == 4 ? 0u : 0xffff0000u >> sh) : x;
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
            return odd;
        };
        // 32 JH positions from `base` on: halves hf .. of the stage in `buf`.
        // (Together where registers allow: the sums of one half then run
        // beside the exponentials of the other.)
        auto work_half = [&](int base, int buf, int hf, uint64_t got, bool whole, bool odd) {
            f16_t sc[JH];
#pragma unroll
            for (int g = 0; g < JH; g++) sc[g] = f16_t{};
#pragma unroll
            for (int s = 0; s < DS; s++)
#pragma unroll
                for (int g = 0; g < JH; g++)
                    sc[g] = Ops::mul(sk[buf][(2 * s + h) * P + 32 * (hf + g) + col], q[s], sc[g]);
            if (!whole) {
#pragma unroll
                for (int g = 0; g < JH; g++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int p = base + 32 * g + at(r);
                        const bool page = (uint32_t)(got >> 32 * g) >> (8 * (r >> 2) + 4 * h + (r & 3)) & 1;
                        sc[g][r] = page & (p <= pos) & ((p >= low) | (p < sinks)) ? sc[g][r] : -INFINITY;
                    }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int g = 0; g < JH; g++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, sc[g][r]);
            mx = fmaxf(m, half_max(mx * unscale));
            if (__any(mx > m)) {
                const float f = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.0f : mx));
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= f;
                m = mx;
            }
            const float sub = Ops::PSHIFT - (m == -INFINITY ? 0.0f : m);
#pragma unroll
            for (int g = 0; g < JH; g++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    sc[g][r] = __builtin_amdgcn_exp2f(fmaf(sc[g][r], unscale, sub));
                    l += sc[g][r];
                }
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    float pr[U];
#pragma unroll
                    for (int e = 0; e < U; e++) pr[e] = sc[g][i * U + e];
                    const typename Ops::P pp = Ops::split(pr);
#pragma unroll
                    for (int d = 0; d < DT; d++)
                        o[d] = Ops::mul(sv[buf][(32 / U * (hf + g) + 2 * i + h) * D + 32 * d + col], pp, o[d]);
                }
            }
            if (odd) {
                // from the pool again: lane L holds a unit's dimension L of
                // 64, and position (unit u, e) is register U (u / 2) + e of half u % 2
#pragma unroll 1
                for (int u = 0; u < 32 * JH / U; u++) {
                    const int p0u = base + u * U, g = kv_page(b, t.seq, p0u);
                    if (g < 0) continue;
#pragma unroll 1
                    for (int d0 = 0; d0 < D; d0 += WAVE) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(
                            b.pool + (size_t)g * b.s.page_bytes + vbase +
                            ((size_t)(t.head * (ps / U) + (p0u & (ps - 1)) / U) * D + min(d0 + lane, D - 1)) * 16);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < U; e++) {
                            const uint32_t bits = U == 4 ? w[e % 4] : w[e / 2] >> 16 * (e & 1) & 0xffffu;
                            const bool sees = p0u + e <= pos && (p0u + e >= low || p0u + e < sinks);
                            float pr = 0.0f;
#pragma unroll
                            for (int i = 0; i < NI * JH; i++) pr = (u >> 1) == i ? sc[i / NI][i % NI * U + e] : pr;
                            pr = __shfl(pr, (u & 1) * 32 + col, WAVE);
                            for (uint64_t who = __ballot((bits & EXP) == EXP && d0 + lane < D); who; who &= who - 1) {
                                const int L = __builtin_ctzll(who), dim = d0 + L;
                                const float val = at_value(E{}, __builtin_amdgcn_readlane(bits, L));
                                // dimension `dim` is register 4 (dim / 8 % 4) + dim % 4 of half dim / 4 % 2, tile dim / 32
                                const float add = sees && (dim >> 2 & 1) == h ? pr * val : 0.0f;
#pragma unroll
                                for (int d = 0; d < DT; d++)
#pragma unroll
                                    for (int r = 0; r < 16; r++)
                                        o[d][r] += dim >> 5 == d && (dim >> 3 & 3) * 4 + (dim & 3) == r ? add : 0.0f;
                            }
                        }
                    }
                }
            }
        };
        for (int i = i0; i < i1; i++) {
            const int buf = (i - i0) & 1;
            wait_vm<0>();
            lds_barrier();       // this stage is there, and the other one free
            if (i + 1 < i1) {
                pages_next = copy(i + 1, buf ^ 1);
                entries(i + 2);
            }
            const int base = kv_base(t.span, i, SLOG);
            bool odd = false;
            if (!(base + P - 1 <= tp0 && (base >= tl1 || base + P <= sinks) && pages == ~(uint64_t)0))
                odd = __syncthreads_or(clean(base, buf, pages));
#pragma unroll 1
            for (int hf = 0; hf < HALVES; hf += JH) {
                const int hb = base + 32 * hf, he = hb + 32 * JH;
                if (!any || hb > p1 || (he <= low0 && hb >= sinks)) continue;   // nobody's
                const uint64_t all = JH == 2 ? ~(uint64_t)0 : 0xffffffffu, got = pages >> 32 * hf & all;
                work_half(hb, buf, hf, got, he - 1 <= p0 && (hb >= low1 || he <= sinks) && got == all, odd);
            }
            pages = pages_next;
        }

        // ---- results, or this workgroup's part of them ----
        l = half_sum(l);
        const int c = wave * 32 + col;      // this lane's column, dimensions 32 d + 8 k + 4 h ..
        auto result = [&](int d, const auto &v, float L) {
            float *dst = a.out + ((size_t)(t.row0 + cr) * nh + t.head * grp + cc % grp) * D + 32 * d;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const f4_t x = {v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                *reinterpret_cast<f4u_t *>(dst + 8 * k + 4 * h) = L == 0.0f ? x : x / L;
            }
        };
        if (i0 == 0 && i1 == t.span.n) {
            if (c < ncol)
#pragma unroll
                for (int d = 0; d < DT; d++) result(d, o[d], l);
            continue;
        }
        const AtSplit split(work, attn_slot(AW_COLS, D), W, n, part, own, tend);
        if (c < ncol) {
            uint64_t *slot = split.at(split.k) + tid;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int k = 0; k < 8; k++) slot_put(slot + (8 * d + k) * AT_THREADS, o[d][2 * k], o[d][2 * k + 1]);
            slot_put(slot + 8 * DT * AT_THREADS, m, l);
        }
        split.template bring<AW_GROUP>(&said, [&](int first, int by, int num, uint64_t *into) {
            if (c >= ncol) return;
            // A thread reads and leaves its own words alone, 16 dimensions at
            // a time, so many parts' in flight at once.
            constexpr int AHEAD = 4;
            float M = -INFINITY, L = 0.0f;
#pragma unroll 1
            for (int d = 0; d < DT; d++) {
                M = -INFINITY;
                L = 0.0f;
                float sum[16] = {};
#pragma unroll 1
                for (int i = 0; i < num; i += AHEAD) {
                    float2 ml[AHEAD], v[AHEAD][8];
#pragma unroll
                    for (int u = 0; u < AHEAD; u++) {
                        const uint64_t *s =    // (a scalar: lanes differ by tid)
                            reinterpret_cast<const uint64_t *>(uni64((uintptr_t)split.at(first + by * min(i + u, num - 1))));
                        ml[u] = slot_get(s + 8 * DT * AT_THREADS + tid);
#pragma unroll
                        for (int k = 0; k < 8; k++) v[u][k] = slot_get(s + (8 * d + k) * AT_THREADS + tid);
                    }
                    float top = M;
#pragma unroll
                    for (int u = 0; u < AHEAD; u++) top = fmaxf(top, ml[u].x);
                    const float ts = top == -INFINITY ? 0.0f : top, r = __builtin_amdgcn_exp2f(M - ts);
                    M = top;
                    L *= r;
#pragma unroll
                    for (int k = 0; k < 16; k++) sum[k] *= r;
#pragma unroll
                    for (int u = 0; u < AHEAD; u++)
                        if (i + u < num) {
                            const float w = __builtin_amdgcn_exp2f(ml[u].x - ts);
                            L += ml[u].y * w;
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                sum[2 * k] += v[u][k].x * w;
                                sum[2 * k + 1] += v[u][k].y * w;
                            }
                        }
                }
                if (into) {
#pragma unroll
                    for (int k = 0; k < 8; k++) slot_put(into + (8 * d + k) * AT_THREADS + tid, sum[2 * k], sum[2 * k + 1]);
                } else {
                    result(d, sum, L);
                }
            }
            if (into) slot_put(into + 8 * DT * AT_THREADS + tid, M, L);   // (behind every read of the parts')
        });
    }
}

template <class E, int D>
static void attn_launch_d(qq_ctx *ctx, const KvBatch &b, const KvAttn &a)
{
    const size_t shm = at_plan_bytes(b);
    uint32_t *work = ctx->kv_work;
    // The form by what the host knows, columns (lengths are on the device): a
    // quarter of a wide tile or more a sequence, as sequences with few leave it
    // idle, and AW_TILES tiles or more in all, as fewer are cut into many parts
    // whose joins cost more than reading keys again for every 16 columns.
    // Narrow and wide form, us (bf16, 4 heads of 128; fp16, 8 heads of 64):
    //   64 sequences of 1024, 16 columns each          -          29 and 37
    //   64 of 1024, 32 columns                     61 and 51      52 and 37
    //   1 of 2048, 16 tiles / 32 tiles       30 and 63 / 49 and 63    17 and 32 / 28 and 35
    //   1 of 8192, 16 tiles / 32 tiles       63 and 70 / 137 and 83   35 and 39 / 69 and 45
    //   1 of 32768, 8 tiles / 32 tiles      108 and 85 / 478 and 173  59 and 47 / 234 and 87
    //   4 of 8192, 32 tiles                       154 and 84      82 and 48
    const int64_t columns = (int64_t)b.n_rows * a.group;
    const bool wide = b.row_start && columns >= (int64_t)AW_COLS / 4 * b.n_seqs &&
                      columns * b.s.n_kv_heads >= (int64_t)AW_TILES * AW_COLS;
    const int parts = wide ? wide_parts(ctx) : attn_parts(ctx);
    prof_begin(ctx, K_KV_ATTN);
    if (wide && b.s.page_size >= (E::U == 4 ? 32 : 64))
        QQ_LAUNCH(ctx, (kv_attn_wide_kernel<E, D, true>), dim3(parts), dim3(AT_THREADS), shm, b, a, work);
    else if (wide)
        QQ_LAUNCH(ctx, (kv_attn_wide_kernel<E, D, false>), dim3(parts), dim3(AT_THREADS), shm, b, a, work);
    else if (b.row_start)
        QQ_LAUNCH(ctx, (kv_attn_kernel<E, D, true>), dim3(parts), dim3(AT_THREADS), shm, b, a, work);
    else
        QQ_LAUNCH(ctx, (kv_attn_kernel<E, D, false>), dim3(parts), dim3(AT_THREADS), shm, b, a, work);
    prof_end(ctx);
}

template <class E>
static void attn_launch(qq_ctx *ctx, const KvBatch &b, const KvAttn &a)
{
    switch (b.s.head_dim) {
    case 32: attn_launch_d<E, 32>(ctx, b, a); break;
    case 64: attn_launch_d<E, 64>(ctx, b, a); break;
    case 96: attn_launch_d<E, 96>(ctx, b, a); break;
    default: attn_launch_d<E, 128>(ctx, b, a); break;
    }
}

int launch_kv_attn(qq_ctx *ctx, const KvBatch &b, const KvAttn &a)
{
    if (b.s.type == QQ_TYPE_F32) attn_launch<KvF32>(ctx, b, a);
    else if (b.s.type == QQ_TYPE_F16) attn_launch<KvF16>(ctx, b, a);
    else attn_launch<KvBf16>(ctx, b, a);
    QQ_HIP(ctx, hipGetLastError());
    return QQ_OK;
}

}  // namespace qq

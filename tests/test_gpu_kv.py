"""The paged key/value cache on the device (qq_kv_*) against binary64.

Pools start out full of NaN: only what a row may see is finite, so a value
read from an unwritten slot, a page's end, a page of nobody or a position
outside the window shows in the result.
"""
import ctypes

import numpy as np
import pytest

import qq_hip
from _kv import BF16, EPS_HALF, F16, F32, NAMES, Pool, attention, from_bits, norm_rope, rounded, seen
from _util import gpu_context

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    return torch


def _up(a):
    torch = _torch()
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint16:
        return torch.from_numpy(a.view(np.int16)).cuda()
    return torch.from_numpy(a).cuda()


class Batch:
    """Sequences with random keys and values in a pool of scattered pages, and their device copies.

    news: new rows per sequence (None: one row each, without row_start)."""
    PAD = 0     # rows of no sequence behind the others

    def __init__(self, lens, news, nq, nkv, dim, typ, ps, seed=0, window=0, sinks=0, fill=np.nan, layers=1, layer=0,
                 spare=3, width=None, qscale=2.0):
        torch = _torch()
        rng = np.random.default_rng([seed, nq, nkv, dim, typ, ps, len(lens), sum(lens)])
        self.lens, self.news = list(lens), [1] * len(lens) if news is None else list(news)
        self.nq, self.nkv, self.dim, self.window, self.sinks = nq, nkv, dim, window, sinks
        need = [-(-l // ps) for l in lens]
        n_pages = sum(need) + spare
        order = rng.permutation(n_pages).astype(np.int32)
        self.width = width or max(1, max(need))
        self.table = np.full((len(lens), self.width), -1, np.int32)
        self.pool = Pool(layers, n_pages, ps, nkv, dim, typ, fill)
        self.k, self.v, at = [], [], 0
        for b, l in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            k = rounded(rng.standard_normal((l, nkv, dim)), typ)
            v = rounded(rng.standard_normal((l, nkv, dim)), typ)
            self.k.append(k)
            self.v.append(v)
            pos = l - self.news[b] + np.arange(self.news[b])
            vis = seen(pos[:, None], np.arange(l)[None], window, sinks).any(0) if self.news[b] else np.zeros(l, bool)
            for p in range(l):
                if vis[p] or np.isfinite(fill):
                    self.pool.put(layer, self.table[b, p // ps], p % ps, k[p], v[p])
        self.starts = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.n = int(self.starts[-1])
        self.q = (rng.standard_normal((self.n, nq, dim)) * qscale).astype(np.float32)
        self.d_pool, self.d_table = _up(self.pool.raw), _up(self.table)
        self.d_lens, self.d_starts = _up(np.array(lens, np.int32)), _up(self.starts)
        self.rows = self.n + (self.PAD if news is not None else 0)
        self.d_q = torch.zeros((self.rows, nq, dim), device="cuda")[:self.n]
        self.d_q.copy_(_up(self.q))
        self.d_out = torch.full((self.rows + 2, nq, dim), 77.0, device="cuda")   # two rows of nobody
        self.no_starts = news is None
        torch.cuda.synchronize()

    def kv(self, ctx):
        p = self.pool
        return ctx.kv_pool(p.layers, p.pages, p.ps, p.nkv, p.dim, p.typ, ptr=self.d_pool.data_ptr(), nbytes=p.raw.nbytes)

    def batch(self, **over):
        f = dict(n_seqs=len(self.lens), table_ptr=self.d_table.data_ptr(), table_stride=self.width,
                 len_ptr=self.d_lens.data_ptr(), row_start_ptr=None if self.no_starts else self.d_starts.data_ptr(),
                 n_rows=self.rows)
        f.update(over)
        return qq_hip.KvBatch(**f)

    def ref(self, scale, known=None):
        out, bound = np.zeros((self.n, self.nq, self.dim)), np.zeros((self.n, self.nq, self.dim))
        for b, l in enumerate(self.lens):
            r0, r1 = self.starts[b], self.starts[b + 1]
            if l and r1 > r0:
                pos = l - (r1 - r0) + np.arange(r1 - r0)
                out[r0:r1], bound[r0:r1] = attention(self.q[r0:r1], self.k[b], self.v[b], pos, scale, self.window,
                                                     self.sinks, None if known is None else known[b])
        return out, bound

    def attn(self, ctx, kv, scale, batch=None, layer=0, out=None):
        kv.attn_dev(layer, batch or self.batch(), self.d_q.data_ptr(), self.nq, (self.d_out if out is None else out).data_ptr(),
                    scale, self.window, self.sinks)
        ctx.synchronize()
        return (self.d_out if out is None else out)[:self.n].cpu().numpy()


def _check(got, ref, bound, what=""):
    assert np.isfinite(got).all(), (what, np.argwhere(~np.isfinite(got))[:4])
    err = np.abs(got - ref)
    # 2^-24 |ref| more: the result's own rounding
    lim = bound + 2.0 ** -24 * np.abs(ref)
    worst = np.argmax(err - lim)
    assert (err <= lim).all(), (what, np.unravel_index(worst, err.shape), err.max(), (err / np.maximum(lim, 1e-30)).max())


def _run(lens, news, heads, typ, ps, window=0, sinks=0, **more):
    nq, nkv, dim = heads
    print("kv", lens if len(lens) < 12 else len(lens), news if news is None or len(news) < 12 else len(news), heads, typ, ps,
          window, sinks, flush=True)
    ctx = gpu_context()
    b = Batch(lens, news, nq, nkv, dim, NAMES[typ], ps, window=window, sinks=sinks, **more)
    kv = b.kv(ctx)
    try:
        scale = 1.0 / np.sqrt(dim)
        got = b.attn(ctx, kv, scale)
        ref, bound = b.ref(scale)
        _check(got, ref, bound)
        assert (b.d_out[b.n:] == 77.0).all()      # rows of no sequence
        # the same call again gives the same bits
        assert (b.attn(ctx, kv, scale) == got).all()
    finally:
        kv.release()


HEADS = [(4, 1, 64), (8, 2, 128), (3, 3, 32), (24, 1, 96), (5, 1, 64), (32, 2, 32), (14, 2, 96)]


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_decode(heads, typ):
    # lengths on either side of units, steps, pages and a wave's share; an idle slot
    _run([1, 0, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 130, 700], None, heads, typ, 16)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
def test_decode_page_sizes(ps, typ):
    _run([5, 257, 512, 1000], None, (8, 2, 64), typ, ps)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("lens", [[1], [3], [0], [5000], [9000, 1, 1, 1], [33] * 40, [0, 0, 700]], ids=str)
def test_decode_shapes(lens, typ):
    _run(lens, None, (4, 1, 64), typ, 64)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 33), (100, 700), (1000, 4), (31, 129)])
def test_decode_window(window, sinks, typ):
    _run([1, 6, 40, 200, 901, 0, 3000], None, (8, 2, 64), typ, 32, window=window, sinks=sinks)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_rows(heads, typ):
    # whole prompts, chunks behind a prefix, single rows, none, an idle slot
    _run([1, 40, 100, 0, 130, 300, 64], [1, 40, 3, 0, 130, 33, 0], heads, typ, 16)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (64, 4), (100, 40), (250, 1)])
def test_rows_window(window, sinks, typ):
    _run([257, 30, 700], [257, 30, 200], (8, 2, 64), typ, 32, window=window, sinks=sinks)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("heads,ps", [((8, 2, 128), 64), ((2, 2, 32), 256), ((4, 1, 96), 16), ((16, 1, 64), 128)], ids=str)
def test_rows_long(heads, ps, typ):
    _run([900, 2600], [900, 140], heads, typ, ps)


@pytest.mark.parametrize("typ", sorted(NAMES))
def test_few_rows_each(typ):
    # draft tokens: 2 to 6 rows a sequence
    _run([100, 33, 1000, 6, 64, 17], [4, 2, 6, 6, 3, 4], (8, 1, 128), typ, 32)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("heads", [(24, 1, 96), (11, 1, 96), (16, 1, 128), (13, 1, 64), (16, 1, 32)], ids=str)
@pytest.mark.parametrize("news", [None, [2, 1]], ids=str)
def test_joined_in_groups(news, heads, typ):
    # one tile in more parts than a workgroup joins, its columns in more than one pass
    _run([9000, 30], news, heads, typ, 64)


def test_many_sequences():
    rng = np.random.default_rng(5)
    _run([int(x) for x in rng.integers(0, 40, 4096)], None, (2, 1, 32), "f16", 16)


@pytest.mark.parametrize("heads,news", [((2, 1, 128), 2), ((16, 1, 128), 3), ((1, 1, 32), 1)], ids=str)
def test_many_sequences_with_rows(heads, news):
    """As many sequences as a call takes, several rows each (either form), with row_start."""
    torch, ctx = _torch(), gpu_context()
    n, ps, (nq, nkv, dim) = 4096, 16, heads
    rng = np.random.default_rng(6)
    lens = rng.integers(news, 2 * ps, n)
    kv = ctx.kv_pool(1, 2 * n, ps, nkv, dim, F32)
    try:
        table = _up(rng.permutation(2 * n).reshape(n, 2).astype(np.int32))
        every = np.concatenate([[0], np.cumsum(lens)])
        k, v = (rng.standard_normal((int(every[-1]), nkv, dim)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((n * news, nq, dim)).astype(np.float32)
        dk, dv, dq, dl, de = _up(k), _up(v), _up(q), _up(lens.astype(np.int32)), _up(every.astype(np.int32))
        ds = _up((np.arange(n + 1) * news).astype(np.int32))
        out = torch.full((n * news, nq, dim), 77.0, device="cuda")
        torch.cuda.synchronize()
        kv.store_dev(0, qq_hip.KvBatch(n, table.data_ptr(), 2, dl.data_ptr(), de.data_ptr(), int(every[-1])), dk.data_ptr(),
                     dv.data_ptr())
        kv.attn_dev(0, qq_hip.KvBatch(n, table.data_ptr(), 2, dl.data_ptr(), ds.data_ptr(), n * news), dq.data_ptr(), nq,
                    out.data_ptr(), 0.1)
        ctx.synchronize()
        got = out.cpu().numpy()
        assert np.isfinite(got).all() and (got != 77.0).all()
        for b in list(range(0, n, 97)) + [n - 1]:
            r = slice(b * news, (b + 1) * news)
            ref, bound = attention(q[r], k[every[b]:every[b + 1]], v[every[b]:every[b + 1]], lens[b] - news + np.arange(news),
                                   0.1, 0, 0)
            _check(got[r], ref, bound, b)
        # row_start that falls again and again: nothing is written outside the rows, and the next call is right
        bad = _up(np.where(np.arange(n + 1) % 2, n * news, 0).astype(np.int32))
        torch.cuda.synchronize()
        kv.attn_dev(0, qq_hip.KvBatch(n, table.data_ptr(), 2, dl.data_ptr(), bad.data_ptr(), n * news), dq.data_ptr(), nq,
                    out.data_ptr(), 0.1)
        kv.attn_dev(0, qq_hip.KvBatch(n, table.data_ptr(), 2, dl.data_ptr(), ds.data_ptr(), n * news), dq.data_ptr(), nq,
                    out.data_ptr(), 0.1)
        ctx.synchronize()
        assert (out.cpu().numpy() == got).all()
    finally:
        kv.release()


def test_wide_scores():
    """Scores of some hundreds: all the weight on few positions, exponentials that vanish elsewhere."""
    for typ in sorted(NAMES):
        _run([300, 40], None, (8, 2, 64), typ, 32, qscale=200.0)


def test_magnitudes():
    """Queries and values far from 1: tiny and huge in one row, fp16's subnormals among keys and values."""
    ctx = gpu_context()
    for typ in sorted(NAMES):
        for qs, vs in ((2.0 ** -20, 1.0), (1.0, 2.0 ** -18), (2.0 ** 10, 2.0 ** 10)):
            print("magnitudes", typ, qs, vs, flush=True)
            b = Batch([90, 400], None, 8, 2, 64, NAMES[typ], 32, qscale=qs)
            for i, l in enumerate(b.lens):
                # keys down to 2^-24 and queries the other way, so that scores stay moderate
                b.k[i] = rounded(b.k[i] * (1.0 if qs <= 1 else 2.0 ** -10), NAMES[typ])
                b.v[i] = rounded(b.v[i] * vs, NAMES[typ])
                for p in range(l):
                    b.pool.put(0, b.table[i, p // 32], p % 32, b.k[i][p], b.v[i][p])
            b.q[:, :, ::7] *= 2.0 ** -6
            b.d_pool, b.d_q = _up(b.pool.raw), _up(b.q)
            _torch().cuda.synchronize()
            kv = b.kv(ctx)
            try:
                got = b.attn(ctx, kv, 0.125)
                ref, bound = b.ref(0.125)
                _check(got, ref, bound, (typ, qs, vs))
            finally:
                kv.release()


@pytest.mark.parametrize("rows", [False, True])
def test_pages_that_are_none(rows):
    """Entries outside the pool, and lengths past the table, hide their positions and are never read."""
    ctx = gpu_context()
    for typ in sorted(NAMES):
        print("bad pages", typ, rows, flush=True)
        lens = [200, 130, 64, 500, 100]
        b = Batch(lens, [40, 3, 64, 17, 100] if rows else None, 8, 2, 64, NAMES[typ], 16)
        known = [np.ones(l, bool) for l in lens]
        for seq, i, g in ((0, 1, -1), (0, 2, b.pool.pages), (1, 0, 2 ** 31 - 1), (3, 4, -2 ** 31), (3, 31, -1)):
            b.table[seq, i] = g
            known[seq][16 * i:16 * i + 16] = False
        b.table[4, :] = -1                      # nothing at all: zeros
        known[4][:] = False
        b.d_table = _up(b.table)
        # a sequence whose length lies past its row of the table (32 pages): len 500 -> 512 + 300 with 300 unseen
        _torch().cuda.synchronize()
        kv = b.kv(ctx)
        try:
            got = b.attn(ctx, kv, 0.125)
            ref, bound = b.ref(0.125, known)
            _check(got, ref, bound, typ)
            assert (got[b.starts[4]:b.starts[5]] == 0).all()
        finally:
            kv.release()


def test_length_past_the_table():
    ctx = gpu_context()
    b = Batch([96, 96], None, 4, 1, 64, F16, 32)
    scale = 0.125
    ref, bound = b.ref(scale)
    kv = b.kv(ctx)
    try:
        for far in (97, 5000, 2 ** 31 - 1):
            b.d_lens.copy_(_torch().tensor([far, 96], dtype=_torch().int32))
            _torch().cuda.synchronize()
            _check(b.attn(ctx, kv, scale), ref, bound, far)
        # negative lengths are idle slots
        b.d_lens.copy_(_torch().tensor([-5, -2 ** 31], dtype=_torch().int32))
        _torch().cuda.synchronize()
        assert (b.attn(ctx, kv, scale) == 0).all()
    finally:
        kv.release()


def test_rows_ahead_of_position_zero():
    """More new rows than positions: the first rows are padding and give zeros."""
    ctx = gpu_context()
    b = Batch([10, 50], [10, 20], 8, 2, 64, BF16, 16)
    scale = 0.125
    ref, bound = b.ref(scale)
    b.d_lens.copy_(_torch().tensor([4, 50], dtype=_torch().int32))     # rows 0..5 at -6..-1, rows 6..9 at 0..3
    _torch().cuda.synchronize()
    kv = b.kv(ctx)
    try:
        got = b.attn(ctx, kv, scale)
        assert (got[:6] == 0).all()
        r, bd = attention(b.q[6:10], b.k[0], b.v[0], np.arange(4), scale, 0, 0)
        _check(got[6:10], r, bd)
        _check(got[10:], ref[10:], bound[10:])
    finally:
        kv.release()


def test_uncovered_rows_and_empty_calls():
    """row_start that leaves rows out, ahead and behind; calls of nothing."""
    ctx = gpu_context()
    for typ in sorted(NAMES):
        b = Batch([40, 60], [7, 9], 4, 2, 64, NAMES[typ], 16)
        scale = 0.125
        ref, bound = b.ref(scale)
        kv = b.kv(ctx)
        try:
            # rows 2..6 belong to sequence 0 (its last five), 7..11 to sequence 1's first 5 of 9 ... as its last five
            b.d_starts.copy_(_torch().tensor([2, 7, 12], dtype=_torch().int32))
            _torch().cuda.synchronize()
            got = b.attn(ctx, kv, scale)
            assert (got[:2] == 77.0).all() and (got[12:] == 77.0).all()
            _check(got[2:7], ref[2:7], bound[2:7])
            r, bd = attention(b.q[7:12], b.k[1], b.v[1], np.arange(55, 60), scale, 0, 0)
            _check(got[7:12], r, bd)
            # starts past the rows or falling: clipped, nothing outside is touched
            b.d_out.fill_(77.0)
            b.d_starts.copy_(_torch().tensor([14, 3, 900], dtype=_torch().int32))
            _torch().cuda.synchronize()
            b.attn(ctx, kv, scale)
            assert (b.d_out[:3] == 77.0).all() and (b.d_out[b.n:] == 77.0).all()
            b.d_out.fill_(77.0)
            for over in (dict(n_seqs=0, n_rows=0), dict(n_rows=0)):
                kv.attn_dev(0, b.batch(**over), None, 4, None, scale)
            ctx.synchronize()
            assert (b.d_out == 77.0).all()
        finally:
            kv.release()


def test_shared_pages_and_unaligned_rows():
    """Two sequences over the same pages, one page twice in a table, q and out at any 4-byte alignment."""
    torch, ctx = _torch(), gpu_context()
    for typ in sorted(NAMES):
        b = Batch([100, 100], None, 8, 2, 128, NAMES[typ], 16)
        b.table[1] = b.table[0]
        b.table[1, 3] = b.table[1, 1]
        b.k[1], b.v[1] = b.k[0].copy(), b.v[0].copy()
        b.k[1][48:64], b.v[1][48:64] = b.k[0][16:32], b.v[0][16:32]
        b.d_table = _up(b.table)
        q = torch.zeros(b.d_q.numel() + 1, device="cuda")
        q[1:] = b.d_q.reshape(-1)
        out = torch.full((b.d_out.numel() + 3,), 77.0, device="cuda")
        torch.cuda.synchronize()
        kv = b.kv(ctx)
        try:
            kv.attn_dev(0, b.batch(), q[1:].data_ptr(), 8, out[3:].data_ptr(), 0.09)
            ctx.synchronize()
            ref, bound = b.ref(0.09)
            _check(out[3:3 + b.n * 8 * 128].view(b.n, 8, 128).cpu().numpy(), ref, bound, typ)
            assert (out[:3] == 77.0).all() and (out[3 + b.n * 8 * 128:] == 77.0).all()
        finally:
            kv.release()


def test_values_that_are_not_finite():
    """Infinities and NaN at visible positions reach their own heads and rows alone."""
    ctx = gpu_context()
    for typ in sorted(NAMES):
        for kind in ("k", "v"):
            for bad in (np.nan, np.inf):
                b = Batch([80, 80], [80, 1], 4, 2, 64, NAMES[typ], 16)
                ref, bound = b.ref(0.125)
                k, v = b.k[0][50].copy(), b.v[0][50].copy()
                (k if kind == "k" else v)[1, 5] = bad
                b.pool.put(0, b.table[0, 3], 2, k, v)
                b.d_pool = _up(b.pool.raw)
                _torch().cuda.synchronize()
                kv = b.kv(ctx)
                try:
                    got = b.attn(ctx, kv, 0.125)
                    _check(got[:50], ref[:50], bound[:50])          # rows that do not see it
                    _check(got[:, :2], ref[:, :2], bound[:, :2])    # the other head
                    _check(got[80:], ref[80:], bound[80:])          # the other sequence
                    hit = got[50:80, 2:]
                    if kind == "v":
                        assert not np.isfinite(hit[:, :, 5]).any()
                    elif np.isnan(bad):
                        assert np.isnan(hit).all()
                finally:
                    kv.release()


def test_far_pages():
    """Pages past 2^32 bytes of a pool, in the second layer."""
    torch, ctx = _torch(), gpu_context()
    nkv, dim, ps, pages = 4, 128, 64, 20000
    kv = ctx.kv_pool(2, pages, ps, nkv, dim, F32)        # 2 x 5.2 GB
    try:
        assert kv.nbytes == 2 * pages * 2 * nkv * ps * dim * 4
        rng = np.random.default_rng(3)
        n = 150
        table = _up(np.array([[pages - 1, 0, pages - 2]], np.int32))
        lens = _up(np.array([n], np.int32))
        starts = _up(np.array([0, n], np.int32))
        k = rng.standard_normal((n, nkv, dim)).astype(np.float32)
        v = rng.standard_normal((n, nkv, dim)).astype(np.float32)
        q = rng.standard_normal((1, 8, dim)).astype(np.float32)
        dk, dv, dq, out = _up(k), _up(v), _up(q), torch.zeros((1, 8, dim), device="cuda")
        torch.cuda.synchronize()
        kv.store_dev(1, qq_hip.KvBatch(1, table.data_ptr(), 3, lens.data_ptr(), starts.data_ptr(), n), dk.data_ptr(), dv.data_ptr())
        kv.attn_dev(1, qq_hip.KvBatch(1, table.data_ptr(), 3, lens.data_ptr()), dq.data_ptr(), 8, out.data_ptr(), 0.1)
        ctx.synchronize()
        ref, bound = attention(q, k, v, [n - 1], 0.1, 0, 0)
        _check(out.cpu().numpy(), ref, bound)
    finally:
        kv.release()


# ---------------------------------------------------------------- store

@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("nq,nkv,dim", [(4, 1, 64), (8, 2, 128), (3, 3, 32), (24, 1, 96), (0, 5, 64), (21, 7, 96)])
@pytest.mark.parametrize("base", [0.0, 1e6])
def test_store(nq, nkv, dim, base, typ):
    """Every row's q, k and v, whole prompts and single tokens, and nothing else in the pool touched.

    Tolerance: binary64 arithmetic rounded to fp32 ahead of RoPE (2^-24 of each of the pair), to fp32 behind it and to
    the cache's type once."""
    torch, ctx, t = _torch(), gpu_context(), NAMES[typ]
    print("store", nq, nkv, dim, base, typ, flush=True)
    lens, news, ps = [1, 0, 40, 33, 17, 5, 64], [1, 1, 40, 2, 1, 0, 64], 16
    b = Batch(lens, news, max(nq, 1), nkv, dim, t, ps, fill=3.0, layers=2, layer=1)
    b.pool.raw[:] = Pool(1, 1, ps, nkv, dim, t, 3.0).raw.flat[0]
    b.d_pool = _up(b.pool.raw)
    rng = np.random.default_rng(9)
    k, v = (rng.standard_normal((b.n, nkv, dim)).astype(np.float32) * s for s in (3.0, 1.0))
    qn, kn = (rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2))
    d = [_up(x) for x in (k, v, qn, kn)]
    q_out = torch.full_like(b.d_q, 77.0)
    torch.cuda.synchronize()
    kv = b.kv(ctx)
    pos = np.concatenate([l - n + np.arange(n) for l, n in zip(lens, news)])
    seq = np.repeat(np.arange(len(lens)), news)
    try:
        if nq:
            kv.store_dev(1, b.batch(), d[0].data_ptr(), d[1].data_ptr(), b.d_q.data_ptr(), nq, d[2].data_ptr(), d[3].data_ptr(),
                         1e-5, base, q_out.data_ptr())
        else:
            kv.store_dev(1, b.batch(), d[0].data_ptr(), d[1].data_ptr(), k_norm_ptr=d[3].data_ptr(), eps=1e-5, rope_base=base)
        ctx.synchronize()
        raw = b.d_pool.cpu().numpy()
        b.pool.raw = raw if t == F32 else raw.view(np.uint16)
        want_k = norm_rope(k, kn, pos, 1e-5, base)
        pair = np.abs(norm_rope(k, kn, pos, 1e-5, 0.0))
        pair = pair + np.roll(pair, dim // 2, -1)
        touched = np.zeros(b.pool.raw.shape, bool)
        mark = Pool(2, b.pool.pages, ps, nkv, dim, t, 0.0)
        for i in range(b.n):
            if pos[i] < 0:
                continue
            g, s = b.table[seq[i], pos[i] // ps], pos[i] % ps
            gk, gv = b.pool.get(1, g, s)
            lim = EPS_HALF[t] * (np.abs(want_k[i]) + 2.0 ** -22 * pair[i]) + 2.0 ** -22 * pair[i] + 2.0 ** -25 * (t == F16)
            assert (np.abs(gk - want_k[i]) <= lim).all(), (i, np.abs(gk - want_k[i]).max())
            assert (np.abs(gv - v[i]) <= EPS_HALF[t] * np.abs(v[i]) + 2.0 ** -25 * (t == F16)).all()
            mark.put(1, g, s, np.ones((nkv, dim), np.float32), np.ones((nkv, dim), np.float32))
        touched = mark.raw != 0
        assert (b.pool.raw[~touched] == Pool(1, 1, ps, nkv, dim, t, 3.0).raw.flat[0]).all()
        if nq:
            got = q_out.cpu().numpy()
            want = norm_rope(b.q, qn, pos, 1e-5, base)
            size = np.abs(norm_rope(b.q, qn, pos, 1e-5, 0.0))
            size = size + np.roll(size, dim // 2, -1)
            live = pos >= 0
            assert (np.abs(got - want) <= 2.0 ** -22 * size)[live].all()
            assert (got[~live] == 77.0).all()
            # in place
            kv.store_dev(1, b.batch(), d[0].data_ptr(), d[1].data_ptr(), b.d_q.data_ptr(), nq, d[2].data_ptr(),
                         d[3].data_ptr(), 1e-5, base, b.d_q.data_ptr())
            ctx.synchronize()
            same = b.d_q.cpu().numpy()
            assert (same[live] == got[live]).all() and (same[~live] == b.q[~live]).all()
    finally:
        kv.release()


def test_store_far_positions_and_bad_pages():
    """Angles of a million positions; positions without a page write nothing, their q is turned all the same."""
    torch, ctx = _torch(), gpu_context()
    ps, nkv, dim, nq = 256, 2, 64, 4
    far = [1000001, 250, 300, 2 ** 30, 900]
    width = (1 << 30) // ps
    pool = Pool(1, 6, ps, nkv, dim, F32, 5.0)
    table = torch.full((len(far), width), -1, dtype=torch.int32, device="cuda")
    for b, (l, g) in enumerate(zip(far, [2, 6, 1, 0, -3])):
        table[b, (l - 1) // ps] = g
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal((5, h, dim)).astype(np.float32) for h in (nq, nkv, nkv))
    dq, dk, dv, dp, dl = _up(q), _up(k), _up(v), _up(pool.raw), _up(np.array(far, np.int32))
    torch.cuda.synchronize()
    kv = ctx.kv_pool(1, 6, ps, nkv, dim, F32, ptr=dp.data_ptr(), nbytes=pool.raw.nbytes)
    try:
        kv.store_dev(0, qq_hip.KvBatch(5, table.data_ptr(), width, dl.data_ptr()), dk.data_ptr(), dv.data_ptr(), dq.data_ptr(),
                     nq, rope_base=5e6, q_out_ptr=dq.data_ptr())
        ctx.synchronize()
        pos = np.array(far) - 1
        got, want = dq.cpu().numpy(), norm_rope(q, None, pos, 0.0, 5e6)
        size = np.abs(q) + np.abs(np.roll(q, dim // 2, -1))
        # the angle itself, up to 2^30, carries 2^-53 of its size (a few times: power, product, reduction)
        assert (np.abs(got - want) <= (2.0 ** -23 + 2.0 ** -20) * size).all()
        assert (np.abs(got - want)[:3] <= 2.0 ** -22 * size[:3]).all()
        pool.raw = dp.cpu().numpy()
        kept = 0
        for b, g in ((0, 2), (2, 1), (3, 0)):
            gk, gv = pool.get(0, g, int(pos[b] % ps))
            assert np.abs(gv - v[b]).max() == 0 and np.abs(gk).max() < 8
            kept += 2 * nkv * dim
        assert (pool.raw != 5.0).sum() == kept       # no drawn value is 5
    finally:
        kv.release()


# ---------------------------------------------------------------- pages

@pytest.mark.parametrize("typ,ps,nkv,dim,layers", [("f32", 16, 1, 32, 3), ("f16", 64, 2, 64, 2), ("bf16", 256, 3, 96, 1),
                                                  ("f16", 16, 1, 32, 40)])
def test_copy_pages(typ, ps, nkv, dim, layers):
    torch, ctx, pages = _torch(), gpu_context(), 37
    shape = (layers, pages, 2, nkv, ps * dim)
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(-2 ** 15, 2 ** 15, shape, generator=g).to(torch.int16)
    if typ == "f32":
        raw = raw.float()
    d = raw.cuda()
    pairs = [(0, 36), (5, 1), (5, 2), (-1, 3), (4, -1), (pages, 6), (7, pages), (8, 8), (2 ** 31 - 1, 9), (20, -2 ** 31)]
    dp = torch.tensor(pairs, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    kv = ctx.kv_pool(layers, pages, ps, nkv, dim, NAMES[typ], ptr=d.data_ptr(), nbytes=d.numel() * d.element_size())
    try:
        kv.copy_pages_dev(dp.data_ptr(), 0)
        kv.copy_pages_dev(dp.data_ptr(), len(pairs))
        ctx.synchronize()
        want = raw.clone()
        for a, b in ((0, 36), (5, 1), (5, 2)):
            want[:, b] = raw[:, a]
        assert torch.equal(d.cpu(), want)
    finally:
        kv.release()


def test_remap():
    torch, ctx = _torch(), gpu_context()
    for n in (1, 63, 257, 100001):
        g = torch.Generator().manual_seed(n)
        table = torch.randint(-3, 60, (n + 5,), generator=g, dtype=torch.int32)
        to = torch.randperm(50, generator=g).to(torch.int32)
        dt, dm = table.cuda(), to.cuda()
        torch.cuda.synchronize()
        ctx.kv_remap_dev(dt.data_ptr(), n, dm.data_ptr(), 50)
        ctx.synchronize()
        want = table.clone()
        ok = (table[:n] >= 0) & (table[:n] < 50)
        want[:n][ok] = to[table[:n][ok].long()]
        assert torch.equal(dt.cpu(), want)


# ---------------------------------------------------------------- captured, other streams, refusals

def test_graphs_follow_lengths_and_tables():
    """Two captured graphs over one cache, replayed in turn while lengths and tables change, and eager calls between."""
    torch, ctx = _torch(), gpu_context()
    ps, nkv, dim, nq = 32, 2, 64, 8
    b = Batch([600, 31, 300], None, nq, nkv, dim, F16, ps, fill=0.25)
    c = Batch([600, 31, 300], [200, 31, 60], nq, nkv, dim, F16, ps, fill=0.25)
    c.d_pool = b.d_pool
    table = b.table.copy()
    dk, dv = (torch.randn((c.rows, nkv, dim), device="cuda") for _ in range(2))
    kv = b.kv(ctx)
    out = torch.zeros((3, nq, dim), device="cuda")
    torch.cuda.synchronize()
    try:
        ctx.capture_begin()
        b.attn_args = (0, b.batch(), b.d_q.data_ptr(), nq, b.d_out.data_ptr(), 0.125)
        kv.attn_dev(*b.attn_args)
        one = ctx.capture_end()
        ctx.capture_begin()
        kv.store_dev(0, c.batch(), dk.data_ptr(), dv.data_ptr())
        kv.attn_dev(0, c.batch(), c.d_q.data_ptr(), nq, c.d_out.data_ptr(), 0.125)
        two = ctx.capture_end()
        rng = np.random.default_rng(0)
        for step in range(4):
            lens = [int(x) for x in rng.integers(1, 600, 3)]
            row, own = table.copy(), table.copy()
            for i in range(3):
                row[i] = rng.permutation(table[0])      # read: every sequence on the first one's pages, in another order
                n = (table[i] >= 0).sum()               # written: each on its own
                own[i, :n] = rng.permutation(table[i, :n])
            b.d_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            b.d_table.copy_(torch.from_numpy(row))
            c.d_lens.copy_(torch.tensor(lens[::-1], dtype=torch.int32))
            c.d_table.copy_(torch.from_numpy(own))
            b.d_out.fill_(77.0)
            c.d_out.fill_(77.0)
            torch.cuda.synchronize()
            one.launch()
            ctx.synchronize()
            first = b.d_out.clone()
            kv.attn_dev(0, b.batch(), b.d_q.data_ptr(), nq, out.data_ptr(), 0.125)
            ctx.synchronize()
            same = torch.equal(first[:3], out)
            assert same, step
            two.launch()
            ctx.synchronize()
            second, stored = c.d_out.clone(), b.d_pool.clone()
            kv.store_dev(0, c.batch(), dk.data_ptr(), dv.data_ptr())
            kv.attn_dev(0, c.batch(), c.d_q.data_ptr(), nq, c.d_out.data_ptr(), 0.125)
            ctx.synchronize()
            same = torch.equal(second, c.d_out), torch.equal(stored, b.d_pool)
            assert same == (True, True), step
        one.release()
        two.release()
    finally:
        kv.release()


def test_calls_of_every_form_in_turn():
    """Calls that split their work differently share the context's workspace: whatever ran before, the next is right."""
    ctx = gpu_context()
    forms = [Batch([9000], None, 4, 1, 64, F16, 64, fill=0.5), Batch([2000], [300], 4, 1, 64, F16, 64, fill=0.5, seed=1),
             Batch([9000, 30], None, 8, 2, 128, BF16, 32, fill=0.5), Batch([5000], [40], 8, 1, 128, F32, 64, fill=0.5),
             Batch([9000, 100, 7], [3, 1, 2], 4, 1, 32, F16, 16, fill=0.5), Batch([1500], [1500], 2, 2, 96, BF16, 16, fill=0.5)]
    kvs = [b.kv(ctx) for b in forms]
    refs = [b.ref(0.1) for b in forms]
    try:
        for i in (0, 1, 0, 2, 3, 0, 4, 5, 2, 4, 1, 0, 5, 3, 2):
            forms[i].d_out.fill_(77.0)
            _torch().cuda.synchronize()
            _check(forms[i].attn(ctx, kvs[i], 0.1), *refs[i], i)
    finally:
        for kv in kvs:
            kv.release()


def test_on_the_callers_stream():
    torch = _torch()
    with qq_hip.Context(0) as ctx:
        s = torch.cuda.Stream()
        ctx.set_stream(s.cuda_stream)
        b = Batch([500, 40], None, 8, 2, 64, BF16, 16)
        kv = b.kv(ctx)
        ref, bound = b.ref(0.125)
        with torch.cuda.stream(s):      # ordered behind the caller's own work, ahead of its next
            q = torch.zeros_like(b.d_q)
            q.copy_(b.d_q)
            kv.attn_dev(0, b.batch(), q.data_ptr(), 8, b.d_out.data_ptr(), 0.125)
            got = b.d_out[:2] * 1.0
        s.synchronize()
        _check(got.cpu().numpy(), ref, bound)
        kv.release()


def test_refusals():
    torch, ctx = _torch(), gpu_context()
    b = Batch([40, 20], None, 8, 2, 64, F16, 16)
    kv, P = b.kv(ctx), b.pool
    good = dict(n_layers=1, n_pages=P.pages, page_size=16, n_kv_heads=2, head_dim=64, type=F16)
    ptr, nbytes = b.d_pool.data_ptr(), P.raw.nbytes
    q, o = b.d_q.data_ptr(), b.d_out.data_ptr()

    def no(match, call, *a, **k):
        with pytest.raises(qq_hip.QQError, match=match):
            call(*a, **k)

    try:
        for over in (dict(page_size=48), dict(page_size=0), dict(head_dim=80), dict(head_dim=160), dict(type=8), dict(n_layers=0),
                     dict(n_pages=0), dict(n_kv_heads=0)):
            no("kv:", ctx.kv_pool, **dict(good, **over))
        no("bytes", ctx.kv_pool, ptr=ptr, nbytes=nbytes - 1, **good)
        no("aligned", ctx.kv_pool, ptr=ptr + 8, nbytes=nbytes, **good)
        for layer in (-1, 1):
            no("layer", kv.attn_dev, layer, b.batch(), q, 8, o, 0.1)
            no("layer", kv.store_dev, layer, b.batch(), q, q)
        for nq in (0, -2, 7, 8192):
            no("heads", kv.attn_dev, 0, b.batch(), q, nq, o, 0.1)
        for over in (dict(n_seqs=-1), dict(n_seqs=4097), dict(n_rows=-1), dict(n_rows=3), dict(table_ptr=None), dict(len_ptr=None),
                     dict(table_stride=0), dict(table_stride=(1 << 26) + 1)):
            no("kv_attn", kv.attn_dev, 0, b.batch(**over), q, 8, o, 0.1)
            no("kv_store", kv.store_dev, 0, b.batch(**over), q, q)
        no("NULL", kv.attn_dev, 0, b.batch(), None, 8, o, 0.1)
        no("NULL", kv.attn_dev, 0, b.batch(), q, 8, None, 0.1)
        no("overlaps", kv.attn_dev, 0, b.batch(), q, 8, q, 0.1)
        no("overlaps", kv.attn_dev, 0, b.batch(), q, 8, q + 4 * 8 * 64, 0.1)
        no("scale", kv.attn_dev, 0, b.batch(), q, 8, o, float("nan"))
        no("window", kv.attn_dev, 0, b.batch(), q, 8, o, 0.1, -1, 0)
        no("sinks", kv.attn_dev, 0, b.batch(), q, 8, o, 0.1, 4, -1)
        no("NULL", kv.store_dev, 0, b.batch(), None, q)
        no("NULL", kv.store_dev, 0, b.batch(), q, None)
        no("go together", kv.store_dev, 0, b.batch(), q, q, q_ptr=q, n_heads=8)
        no("go together", kv.store_dev, 0, b.batch(), q, q, q_out_ptr=o)
        no("heads", kv.store_dev, 0, b.batch(), q, q, q_ptr=q, n_heads=3, q_out_ptr=o)
        no("overlaps", kv.store_dev, 0, b.batch(), o, o, q_ptr=q, n_heads=8, q_out_ptr=q + 4)
        for eps, base in ((-1.0, 0.0), (float("nan"), 0.0), (float("inf"), 0.0), (1e-5, -1.0), (1e-5, float("nan")), (1e-5, float("inf"))):
            no("eps|rope_base", kv.store_dev, 0, b.batch(), q, q, eps=eps, rope_base=base)
        no("pairs", kv.copy_pages_dev, q, -1)
        no("NULL", kv.copy_pages_dev, None, 1)
        no("kv_remap", ctx.kv_remap_dev, q, -1, q, 1)
        no("NULL", ctx.kv_remap_dev, None, 1, q, 1)
        L = ctx.L
        assert L.qq_kv_attn_dev(ctx.h, kv.h, 0, None, q, 8, 0.1, 0, 0, o) == -1
        assert L.qq_kv_attn_dev(ctx.h, None, 0, ctypes.byref(b.batch()), q, 8, 0.1, 0, 0, o) == -1
        with qq_hip.Context(0) as other:
            assert L.qq_kv_attn_dev(other.h, kv.h, 0, ctypes.byref(b.batch()), q, 8, 0.1, 0, 0, o) == -1
            assert L.qq_kv_release(other.h, kv.h) == -1
        ctx.capture_begin()
        no("capture", ctx.kv_pool, **good)
        no("capture", kv.release)
        ctx.capture_end().release()
        # and it still works
        ref, bound = b.ref(0.125)
        _check(b.attn(ctx, kv, 0.125), ref, bound)
    finally:
        kv.release()


def test_refusals_of_what_does_not_fit():
    torch, ctx = _torch(), gpu_context()
    b = Batch([40, 20], [1, 1], 8, 2, 64, F16, 16)
    kv = b.kv(ctx)
    q, o = b.d_q.data_ptr(), b.d_out.data_ptr()
    try:
        many = b.batch(n_rows=1 << 24)       # 2^32 threads
        for call in (lambda: kv.store_dev(0, many, q, q), lambda: kv.attn_dev(0, many, q, 8, o, 0.1),
                     lambda: kv.copy_pages_dev(q, 1 << 24), lambda: kv.attn_dev(0, b.batch(), q, 8, o, 3e38),
                     lambda: kv.attn_dev(0, b.batch(), q, 8, o, -1e39)):
            with pytest.raises(qq_hip.QQError, match="rows|pairs|scale"):
                call()
        ref, bound = b.ref(0.125)
        _check(b.attn(ctx, kv, 0.125), ref, bound)
    finally:
        kv.release()


def test_scores_of_minus_infinity():
    """A key whose score is -infinity weighs nothing; a row that sees no other gives zeros."""
    ctx = gpu_context()
    for news in (None, [2], [20]):
        b = Batch([20], news, 4, 1, 64, F32, 16)
        b.q[:] = np.abs(b.q) + 0.5
        b.d_q.copy_(_up(b.q))
        kept = [p for p in range(20) if p % 3]
        for p in range(20):
            if p % 3 == 0:
                k = b.k[0][p].copy()
                k[0, 7] = -np.inf
                b.pool.put(0, b.table[0, p // 16], p % 16, k, b.v[0][p])
        b.d_pool.copy_(_up(b.pool.raw))
        _torch().cuda.synchronize()
        kv = b.kv(ctx)
        try:
            got = b.attn(ctx, kv, 0.125)
        finally:
            kv.release()
        pos = 20 - b.n + np.arange(b.n)
        for r in range(b.n):
            at = [p for p in kept if p <= pos[r]]
            if not at:
                assert (got[r] == 0.0).all()
                continue
            ref, bound = attention(b.q[r:r + 1], b.k[0][at], b.v[0][at], np.array([len(at) - 1]), 0.125, 0, 0)
            _check(got[r:r + 1], ref, bound, (news, r))


# ---------------------------------------------------------------- the form of large calls

@pytest.fixture
def large(monkeypatch):
    """Rows of no sequence fill the calls up to the size that takes the form for many rows."""
    monkeypatch.setattr(Batch, "PAD", 4096)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_large_rows(large, heads, typ):
    test_rows(heads, typ)
    test_rows(heads[:2] + (160 - heads[2],), typ)      # another head size, the other page form
    _run([5, 257, 512, 1000], [5, 1, 12, 200], heads, typ, 128)


@pytest.mark.parametrize("typ", sorted(NAMES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (64, 4), (100, 40), (250, 1), (31, 700)])
def test_large_rows_window(large, window, sinks, typ):
    test_rows_window(window, sinks, typ)
    _run([257, 30, 700], [257, 30, 200], (4, 1, 128), typ, 64, window=window, sinks=sinks)


@pytest.mark.parametrize("typ", sorted(NAMES))
def test_large_rows_long(large, typ):
    test_rows_long((4, 1, 96), 16, typ)
    test_rows_long((2, 2, 32), 256, typ)
    test_joined_in_groups([2, 1], (16, 1, 128), typ)
    test_joined_in_groups([40, 1], (11, 1, 96), typ)
    test_few_rows_each(typ)


@pytest.mark.parametrize("case", [test_rows_ahead_of_position_zero, test_values_that_are_not_finite,
                                  test_scores_of_minus_infinity, test_graphs_follow_lengths_and_tables,
                                  lambda: test_pages_that_are_none(True)],
                         ids=["ahead_of_zero", "not_finite", "minus_infinity", "graphs", "no_pages"])
def test_large_edges(large, case):
    case()


def test_large_calls_in_turn(monkeypatch):
    """Both forms, split in many parts, by turns over one workspace."""
    ctx, forms = gpu_context(), []
    for i, (lens, news, heads, typ, ps) in enumerate((
            ([2000], [300], (4, 1, 64), F16, 64), ([9000], None, (4, 1, 64), F16, 64), ([5000], [40], (8, 1, 128), F32, 64),
            ([9000, 30], None, (8, 2, 128), BF16, 32), ([9000, 100, 7], [3, 1, 2], (4, 1, 32), F16, 16),
            ([1500], [500], (2, 2, 96), BF16, 16))):
        monkeypatch.setattr(Batch, "PAD", 4096 if i % 2 == 0 else 0)
        forms.append(Batch(lens, news, *heads, typ, ps, fill=0.5, seed=i))
    kvs = [b.kv(ctx) for b in forms]
    refs = [b.ref(0.1) for b in forms]
    try:
        for i in (0, 1, 0, 2, 3, 0, 4, 5, 2, 4, 1, 0, 5, 3, 2):
            forms[i].d_out.fill_(77.0)
            _torch().cuda.synchronize()
            _check(forms[i].attn(ctx, kvs[i], 0.1), *refs[i], i)
            assert (forms[i].d_out[forms[i].n:] == 77.0).all()
    finally:
        for kv in kvs:
            kv.release()


# ---------------------------------------------------------------- together

def test_serving_run():
    """What a server does with it all: prompts in chunks, batched decode, forks that share pages, a truncation, freed sequences,
    a compaction in between -- every step's attention against binary64 over the sequences' own histories."""
    torch, ctx = _torch(), gpu_context()
    rng = np.random.default_rng(8)
    nq, nkv, dim, ps, n_pages, layers, width = 8, 2, 64, 16, 90, 2, 12
    scale, base = dim ** -0.5, 1e4
    pages = qq_hip.Pages(n_pages, ps)
    kv = ctx.kv_pool(layers, n_pages, ps, nkv, dim, BF16)
    hist = {}                                                # sequence -> [k, v] of each layer, as stored
    qn, kn = (rng.uniform(0.5, 1.5, dim).astype(np.float32) for _ in range(2))
    dqn, dkn = _up(qn), _up(kn)

    def copies(pairs):
        if pairs:
            d = _up(np.array(pairs, np.int32))
            torch.cuda.synchronize()
            kv.copy_pages_dev(d.data_ptr(), len(pairs))
            ctx.synchronize()

    def step(seqs, news):
        copies([p for p in (pages.extend(s, n) for s, n in zip(seqs, news)) if p])
        table = np.stack([pages.table(s, width) for s in seqs])
        lens, starts = [pages.length(s) for s in seqs], np.concatenate([[0], np.cumsum(news)])
        n = int(starts[-1])
        dt, dl, ds = _up(table), _up(np.array(lens, np.int32)), _up(starts.astype(np.int32))
        one = all(x == 1 for x in news)
        batch = qq_hip.KvBatch(len(seqs), dt.data_ptr(), width, dl.data_ptr(), None if one else ds.data_ptr(), n)
        pos = np.concatenate([l - m + np.arange(m) for l, m in zip(lens, news)])
        for layer in range(layers):
            q, k, v = (rng.standard_normal((n, h, dim)).astype(np.float32) for h in (nq, nkv, nkv))
            dq, dk, dv = _up(q), _up(k), _up(v)
            out = torch.full((n, nq, dim), 77.0, device="cuda")
            torch.cuda.synchronize()
            kv.store_dev(layer, batch, dk.data_ptr(), dv.data_ptr(), dq.data_ptr(), nq, dqn.data_ptr(), dkn.data_ptr(), 1e-6,
                         base, dq.data_ptr())
            kv.attn_dev(layer, batch, dq.data_ptr(), nq, out.data_ptr(), scale, window=60, sinks=3)
            ctx.synchronize()
            want_q = norm_rope(q, qn, pos, 1e-6, base)
            want_k = norm_rope(k, kn, pos, 1e-6, base)
            got_q, got = dq.cpu().numpy(), out.cpu().numpy()
            assert np.abs(got_q - want_q).max() < 1e-5
            raw = torch.zeros(kv.nbytes // 2, dtype=torch.int16)
            ctx.buffer_read(kv.ptr, raw.numpy())
            view = Pool(layers, n_pages, ps, nkv, dim, BF16)
            view.raw = raw.numpy().view(np.uint16).reshape(view.raw.shape)
            for i, s in enumerate(seqs):
                r = slice(int(starts[i]), int(starts[i + 1]))
                for j in range(*r.indices(n)):
                    gk, gv = view.get(layer, table[i, pos[j] // ps], pos[j] % ps)
                    assert np.abs(gk - want_k[j]).max() < 2.0 ** -8 * 6 and np.abs(gv - v[j]).max() < 2.0 ** -8 * 6
                    hist[s][layer].append((gk, gv))
                hk = np.stack([a for a, _ in hist[s][layer]])
                hv = np.stack([a for _, a in hist[s][layer]])
                ref, bound = attention(got_q[r], hk, hv, pos[r], scale, 60, 3)
                _check(got[r], ref, bound, (s, layer))

    def new():
        s = pages.new()
        hist[s] = [[] for _ in range(layers)]
        return s

    def fork(s, n):
        f = pages.fork(s, n)
        hist[f] = [list(h[:n]) for h in hist[s]]
        return f

    try:
        a, b, c = new(), new(), new()
        step([a, b, c], [37, 5, 64])                # prompts
        step([c, a], [50, 3])                       # a second chunk, and a few draft tokens
        step([a, b, c], [1, 1, 1])
        d, e = fork(a, pages.length(a)), fork(c, 70)
        step([a, b, c, d, e], [1, 1, 1, 1, 1])      # the forks' shared last pages are copied
        pages.truncate(a, 38)                       # drafts rejected
        hist[a] = [h[:38] for h in hist[a]]
        step([a, d], [1, 1])
        pages.free(c)
        del hist[c]
        pairs, _ = pages.compact()
        assert len(pairs)
        copies(pairs.tolist())
        step([e, a, b, d], [1, 1, 1, 1])
        step([b, e], [70, 2])
        f = new()
        step([f, a], [1, 30])
    finally:
        kv.release()
        pages.release()


def test_attention_block():
    """An attention block of a batch as a server runs it -- rmsnorm, the Q8_0 products, the cache, attention, the output
    product -- against the same block in binary64 over the cache's fp32 values."""
    import synth
    torch, ctx = _torch(), gpu_context()
    H, nq, nkv, dim, ps = 256, 8, 2, 64, 32
    rng = np.random.default_rng(12)

    def dense(w, i, o):
        blk = np.asarray(w).view(synth.Q8_DTYPE).reshape(o, -1)
        return (blk["qs"].astype(np.float64) * blk["d"].astype(np.float64)[..., None]).reshape(o, -1)[:, :i]

    shapes = {"q": (H, nq * dim), "k": (H, nkv * dim), "v": (H, nkv * dim), "o": (nq * dim, H)}
    w = {n: synth.q8_0_tensor(rng, *s) for n, s in shapes.items()}
    t = {n: ctx.upload_q8_0(w[n], *s) for n, s in shapes.items()}
    dn = {n: dense(w[n], *s) for n, s in shapes.items()}
    norm, qn, kn = (rng.uniform(0.5, 1.5, n).astype(np.float32) for n in (H, dim, dim))
    lens, news = [50, 9, 33], [50, 1, 20]
    before = [l - n for l, n in zip(lens, news)]
    n = sum(news)
    x = rng.standard_normal((sum(lens), H)).astype(np.float32)       # every position's input, sequence by sequence
    first = np.concatenate([[0], np.cumsum(lens)])
    kv = ctx.kv_pool(1, 12, ps, nkv, dim, F32)
    table = _up(np.array([[3, 9], [0, -1], [7, 1]], np.int32))
    dnorm, dqn, dkn = _up(norm), _up(qn), _up(kn)

    def run(rows, lens_now, counts):
        m = rows.shape[0]
        starts = _up(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        dl, dx = _up(np.array(lens_now, np.int32)), _up(rows)
        buf = {k: torch.zeros((m, s[1]), device="cuda") for k, s in shapes.items()}
        attn = torch.zeros((m, nq * dim), device="cuda")
        torch.cuda.synchronize()
        ctx.rmsnorm_dev(dx.data_ptr(), dnorm.data_ptr(), dx.data_ptr(), m, H, 1e-5)
        for name in "qkv":
            t[name].matvec_dev(dx.data_ptr(), buf[name].data_ptr(), m)
        batch = qq_hip.KvBatch(3, table.data_ptr(), 2, dl.data_ptr(), starts.data_ptr(), m)
        kv.store_dev(0, batch, buf["k"].data_ptr(), buf["v"].data_ptr(), buf["q"].data_ptr(), nq, dqn.data_ptr(), dkn.data_ptr(),
                     1e-5, 5e6, buf["q"].data_ptr())
        kv.attn_dev(0, batch, buf["q"].data_ptr(), nq, attn.data_ptr(), dim ** -0.5)
        t["o"].matvec_dev(attn.data_ptr(), buf["o"].data_ptr(), m)
        ctx.synchronize()
        return buf["o"].cpu().numpy()

    try:
        run(np.concatenate([x[first[i]:first[i] + before[i]] for i in range(3)]), before, before)
        got = run(np.concatenate([x[first[i] + before[i]:first[i + 1]] for i in range(3)]), lens, news)
        at = 0
        for i in range(3):
            xi = x[first[i]:first[i + 1]].astype(np.float64)
            xi = xi / np.sqrt((xi * xi).mean(-1, keepdims=True) + 1e-5) * norm
            pos = np.arange(lens[i])
            q = norm_rope((xi @ dn["q"].T).reshape(-1, nq, dim), qn, pos, 1e-5, 5e6)
            k = norm_rope((xi @ dn["k"].T).reshape(-1, nkv, dim), kn, pos, 1e-5, 5e6)
            v = (xi @ dn["v"].T).reshape(-1, nkv, dim)
            o, _ = attention(q[before[i]:], k, v, pos[before[i]:], dim ** -0.5, 0, 0)
            want = o.reshape(news[i], -1) @ dn["o"].T
            err = np.linalg.norm(got[at:at + news[i]] - want) / np.linalg.norm(want)
            # fp32 sums of 256 and 512 products, then scores and sums over at most 50 positions: ~1e-6 of each step
            assert err < 1e-5, (i, err)
            at += news[i]
    finally:
        kv.release()
        for h in t.values():
            h.release()

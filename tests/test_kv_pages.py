"""The page book-keeping (qq_pages_*) against a model that names every value,
and the refusals that need no device."""
import ctypes
import random


import pytest

import qq_hip


class Model:
    """Every sequence's own list of values, and the pool of values its pages hold."""

    def __init__(self, n_pages, ps):
        self.ps = ps
        self.pool = [[None] * ps for _ in range(n_pages)]
        self.seqs = {}

    def write(self, pages, seq, values):
        """Extend through the book-keeping, follow its copy, then write the new values into the pages."""
        old = len(self.seqs[seq])
        pair = pages.extend(seq, len(values))
        if pair is not None:
            self.pool[pair[1]] = list(self.pool[pair[0]])
        row = pages.table(seq)
        for i, v in enumerate(values):
            self.pool[row[(old + i) // self.ps]][(old + i) % self.ps] = v
        self.seqs[seq] = self.seqs[seq] + list(values)

    def check(self, pages):
        users = {}
        for seq, want in self.seqs.items():
            row = pages.table(seq)
            assert pages.length(seq) == len(want) and len(row) == -(-len(want) // self.ps)
            got = [self.pool[row[i // self.ps]][i % self.ps] for i in range(len(want))]
            assert got == want, seq
            assert len(set(row.tolist())) == len(row)
            for g in row.tolist():
                users.setdefault(g, set()).add(seq)
        free, used = pages.count()
        assert used == len(users) and free + used == len(self.pool)


@pytest.mark.parametrize("seed,n_pages,ps", [(s, n, p) for s, (n, p) in enumerate([(1, 1), (3, 4), (12, 2), (40, 16), (200, 3), (64, 5)])])
def test_random_use(seed, n_pages, ps):
    rng = random.Random(seed)
    pages, m, stamp = qq_hip.Pages(n_pages, ps), Model(n_pages, ps), 0
    for step in range(600):
        what = rng.random()
        live = sorted(m.seqs)
        if what < 0.15 or not live:
            seq = pages.new()
            assert seq not in m.seqs
            m.seqs[seq] = []
        elif what < 0.55:
            seq, n = rng.choice(live), rng.randint(0, 3 * ps)
            before = {s: pages.table(s).tolist() for s in live}
            try:
                m.write(pages, seq, list(range(stamp, stamp + n)))
                stamp += n
            except qq_hip.QQError as e:
                assert "free" in str(e)
                assert before == {s: pages.table(s).tolist() for s in live}
                # it did not fit: more pages were needed than were free
                old = len(m.seqs[seq])
                more = -(-(old + n) // ps) - -(-old // ps) + (1 if old % ps else 0)
                assert more > pages.count()[0]
        elif what < 0.7:
            seq = rng.choice(live)
            n = rng.randint(0, len(m.seqs[seq]))
            dst = pages.fork(seq, n)
            assert dst not in m.seqs
            m.seqs[dst] = m.seqs[seq][:n]
        elif what < 0.8:
            seq = rng.choice(live)
            n = rng.randint(0, len(m.seqs[seq]))
            pages.truncate(seq, n)
            m.seqs[seq] = m.seqs[seq][:n]
        elif what < 0.92:
            seq = rng.choice(live)
            pages.free(seq)
            del m.seqs[seq]
            with pytest.raises(qq_hip.QQError, match="no sequence"):
                pages.table(seq)
        else:
            before = {s: pages.table(s) for s in live}
            pairs, to = pages.compact()
            used = pages.count()[1]
            src, dst = set(pairs[:, 0].tolist()), set(pairs[:, 1].tolist())
            assert len(src) == len(dst) == len(pairs) and not src & dst
            for a, b in pairs.tolist():
                m.pool[b] = list(m.pool[a])
                assert to[a] == b and a >= used > b
            for s in live:
                assert (to[before[s]] == pages.table(s)).all()
                assert (pages.table(s) < used).all()
        m.check(pages)
    pages.release()


def test_shared_last_page_is_copied_once():
    p = qq_hip.Pages(8, 4)
    a = p.new()
    assert p.extend(a, 6) is None
    b = p.fork(a, 6)
    assert p.count() == (6, 2)
    pair = p.extend(a, 1)                 # the page of positions 4, 5 has two users
    assert pair[0] == p.table(b)[1] and pair[1] == p.table(a)[1]
    assert p.extend(b, 1) is None         # now its own
    c = p.fork(a, 4)                      # shares whole pages alone
    assert p.extend(c, 1) is None
    assert p.table(c, 5).tolist()[2:] == [-1, -1, -1]
    p.release()


def test_refusals():
    for n, ps in ((0, 4), (-1, 4), (4, 0)):
        with pytest.raises(qq_hip.QQError, match="qq_pages_create"):
            qq_hip.Pages(n, ps)
    p = qq_hip.Pages(4, 4)
    s = p.new()
    p.extend(s, 5)
    for call in (lambda: p.extend(7, 1), lambda: p.extend(-1, 1), lambda: p.extend(s, -1), lambda: p.extend(s, 2 ** 31 - 1),
                 lambda: p.fork(s, 6), lambda: p.fork(s, -1), lambda: p.truncate(s, 6), lambda: p.table(s, 1),
                 lambda: p.extend(s, 12)):
        with pytest.raises(qq_hip.QQError):
            call()
        assert p.length(s) == 5 and p.count() == (2, 2)
    L, n = p.L, ctypes.c_int()
    assert L.qq_pages_create(1, 1, None) == -1
    assert L.qq_pages_new(None, ctypes.byref(n)) == -1
    assert L.qq_pages_extend(p.h, s, 1, None, ctypes.byref(n)) == -1
    assert L.qq_pages_compact(p.h, None, 4, ctypes.byref(n), None) == -1
    assert L.qq_pages_release(None) == 0
    # a compaction that does not fit changes nothing
    t = p.new()
    p.extend(t, 1)
    p.free(s)
    assert L.qq_pages_compact(p.h, None, 0, ctypes.byref(n), None) == -1
    assert p.table(t).tolist() == [2]
    assert p.compact()[0].tolist() == [[2, 0]] and p.table(t).tolist() == [0]
    p.release()


def test_more_pages_than_a_pool_has():
    L, h = qq_hip.load(), ctypes.c_void_p()
    assert L.qq_pages_create((1 << 24) + 1, 16, ctypes.byref(h)) == -1 and not h.value
    assert b"pages" in L.qq_last_error(None)


def test_pool_bytes():
    L, n = qq_hip.load(), ctypes.c_size_t()
    assert L.qq_kv_pool_bytes(6, 100, 64, 8, 64, qq_hip.TYPE_F16, ctypes.byref(n)) == 0
    assert n.value == 6 * 100 * 64 * 8 * 64 * 2 * 2
    assert L.qq_kv_pool_bytes(4096, 1 << 24, 256, 256, 128, qq_hip.TYPE_F32, ctypes.byref(n)) == 0
    assert n.value == 4096 * (1 << 24) * 256 * 256 * 128 * 8
    for bad in ((0, 1, 64, 8, 64, 0), (1, 0, 64, 8, 64, 0), (1, 1, 48, 8, 64, 0), (1, 1, 512, 8, 64, 0),
                (1, 1, 64, 0, 64, 0), (1, 1, 64, 257, 64, 0), (1, 1, 64, 8, 80, 0), (1, 1, 64, 8, 64, 8),
                (1, (1 << 24) + 1, 64, 8, 64, 0), (4097, 1, 64, 8, 64, 0), (1, 1, -64, 8, 64, 0)):
        assert L.qq_kv_pool_bytes(*bad, ctypes.byref(n)) == -1, bad
        assert b"kv" in L.qq_last_error(None)
    assert L.qq_kv_pool_bytes(1, 1, 64, 8, 64, 0, None) == -1


def test_null_context_is_rejected():
    L = qq_hip.load()
    h = ctypes.c_void_p()
    b = qq_hip.KvBatch(1, 0, 1, 0)
    assert L.qq_kv_create(None, None, 0, 1, 1, 64, 8, 64, 0, ctypes.byref(h)) == -1
    assert L.qq_kv_store_dev(None, None, 0, ctypes.byref(b), None, 0, None, None, None, None, 0.0, 0.0, None) == -1
    assert L.qq_kv_attn_dev(None, None, 0, ctypes.byref(b), None, 8, 1.0, 0, 0, None) == -1
    assert L.qq_kv_copy_pages_dev(None, None, None, 1) == -1
    assert L.qq_kv_remap_dev(None, None, 1, None, 1) == -1
    assert L.qq_kv_release(None, None) == 0


def test_header_constants():
    import os
    import re
    from _util import ROOT
    text = open(os.path.join(ROOT, "include", "qq_moe.h")).read()
    consts = dict(re.findall(r"#define\s+(QQ_[A-Z0-9_]+)\s+(-?\d+)", text))
    assert int(consts["QQ_TYPE_F16"]) == qq_hip.TYPE_F16 and int(consts["QQ_TYPE_BF16"]) == qq_hip.TYPE_BF16
    assert int(consts["QQ_KV_MAX_SEQS"]) == qq_hip.KV_MAX_SEQS
    # int, int, pointer, int and 4 bytes of padding, two pointers
    assert ctypes.sizeof(qq_hip.KvBatch) == 4 + 4 + 8 + 8 + 8 + 8

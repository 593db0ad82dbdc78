"""Operators of a paged key/value cache: what a serving loop calls between the
Q8_0 products of its attention blocks, at the sizes it calls them.

A case is one of three kinds of call:

  store   KvPool.store_dev: the new rows of a batch of sequences -- per-head
          RMSNorm and rotary positions on q and k, k and v written into pages
  attn    KvPool.attn_dev: attention of a batch's new rows over their
          sequences' pages, causal, optionally within a window beside a few
          first tokens; one row a sequence (decode) or several (prompt chunks)
  pages   KvPool.copy_pages_dev, and Context.kv_remap_dev when tables change:
          forked tails, or a compaction

Head layouts (query heads, key/value heads, head size): LFM2-8B-A1B's 32/8/64,
Qwen3-30B-A3B's 32/4/128, and others of any grouping in the drawn cases.  The
pool's layout is the one include/qq_moe.h documents; its values are the inputs
(a context's keys and values), so that both forms read the same memory.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-5
ROPE_BASE = 1000000.0
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEADS = {"lfm2": (32, 8, 64), "qwen3": (32, 4, 128), "small": (16, 8, 128), "mha": (6, 6, 32), "mqa": (24, 1, 96)}


# ---------------------------------------------------------------- the cases

def _case(name, kind, heads, typ, page, seqs, length, rows=1, mix=0, window=0, sinks=0, **more):
    """seqs sequences of up to `length` positions, the last up to `rows` of them new; mix > 0: ragged."""
    c = {"kind": kind, "heads": heads, "type": typ, "page": page, "seqs": seqs, "length": length, "rows": rows,
         "mix": mix, "window": window, "sinks": sinks}
    c.update(more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # interactive decode: the new token's row of one block
        _case("store_1", "store", "lfm2", "f32", 64, 1, 700),
        # a serving batch's rows, long contexts
        _case("store_64", "store", "qwen3", "bf16", 64, 64, 4000, mix=1),
        # the prompts of five requests in one chunk
        _case("store_prompts", "store", "lfm2", "f16", 32, 5, 900, rows=900, mix=2),
        # interactive decode at a moderate context, the cache in the engine's own type
        _case("decode_1", "attn", "lfm2", "f32", 64, 1, 700),
        # one conversation with a very long context
        _case("decode_long", "attn", "qwen3", "bf16", 64, 1, 100001),
        # a serving batch of ragged contexts (one slot idle)
        _case("decode_64", "attn", "lfm2", "f16", 64, 64, 4096, mix=3),
        # many sequences, a sliding window with four sink tokens
        _case("decode_window", "attn", "qwen3", "bf16", 16, 32, 20000, mix=4, window=1024, sinks=4),
        # the draft tokens of speculative decoding, checked in one call
        _case("verify_4", "attn", "small", "f16", 32, 16, 3000, rows=4, mix=0),
        # a whole prompt
        _case("prompt_4096", "attn", "lfm2", "f16", 64, 1, 4096, rows=4096),
        # chunks of ragged prompts over a cached prefix, window and sinks
        _case("chunks_window", "attn", "qwen3", "bf16", 64, 6, 3000, rows=1100, mix=5, window=1000, sinks=4),
        # a fork into beams: every sequence's last page in all layers of a model
        _case("fork_tails", "pages", "lfm2", "f16", 64, 64, 1, layers=6, pool=160),
        # a compaction: the live pages of the pool's upper half move into holes, the tables follow
        _case("compact", "pages", "qwen3", "bf16", 16, 600, 1, layers=4, pool=2001, remap=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choices(["store", "attn", "pages"], [2, 6, 1])[0]
    heads, typ = rng.choice(sorted(HEADS)), rng.choice(sorted(TYPES))
    page, mix = rng.choice([16, 32, 64, 128]), rng.randint(1, 10 ** 6)
    if kind == "pages":
        layers = rng.randint(1, 3)
        size = layers * 2 * math.prod(HEADS[heads][1:]) * page * (4 if typ == "f32" else 2)
        pool = _log_int(rng, 8, min(2001, int(1.0e9 / size)))
        return _case(None, kind, heads, typ, page, _log_int(rng, 1, max(1, min(pool // 4, int(7.0e7 / size)))), 1,
                     mix=mix, layers=layers, pool=pool, remap=rng.random() < 0.5)
    if kind == "store":
        rows = rng.choice([1, 1, _log_int(rng, 2, 1500)])
        seqs = _log_int(rng, 1, 64 if rows == 1 else 5)
        return _case(None, kind, heads, typ, page, seqs, max(rows, _log_int(rng, 1, 4000)), rows=rows,
                     mix=rng.choice([0, mix]))
    window = rng.choice([0, 0, _log_int(rng, 1, 4000)])
    sinks = rng.choice([0, 4, rng.randint(1, 40)]) if window else 0
    nq, nkv, dim = HEADS[heads]
    if rng.random() < 0.6:      # one new token a sequence
        seqs = _log_int(rng, 1, 128)
        length = _log_int(rng, 1, min(100001, int((0.7e8 if typ == "f32" else 1.4e8) / (2 * seqs * nkv * dim))))
        rows = 1
    else:
        seqs = _log_int(rng, 1, 16)
        rows = _log_int(rng, 2, 1500)
        length = max(rows, _log_int(rng, 2, 6000))
        rows = max(1, min(rows, int(2.5e8 / (seqs * nq * length))))
    return _case(None, kind, heads, typ, page, seqs, length, rows=rows, mix=rng.choice([0, mix, mix]),
                 window=window, sinks=sinks)


# ---------------------------------------------------------------- shapes and seeded inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _lens(case):
    """(length, new rows) of each sequence: ragged ones by the case's own numbers, one idle slot among four or more."""
    n, m, r = case["seqs"], case["length"], case["rows"]
    lens, news = [m] * n, [min(r, m)] * n
    if case["mix"]:
        rng = random.Random(case["mix"])
        lens = [max(1, int(m * rng.uniform(0.02, 1.0))) for _ in range(n)]
        lens[rng.randrange(n)] = m
        if n >= 4:
            lens[rng.randrange(n)] = 0
        news = [min(l, 1 if r == 1 else rng.randint(1, r)) for l in lens]
    if r == 1:
        news = [1] * n      # one row each, an idle slot's too
    return lens, news


def _gen(seed, salt):
    g = torch.Generator(device=_device())
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _unit(typ):
    """Values in 16 bytes of the cache: the pool's unit."""
    return 4 if typ == "f32" else 8


def _pool(case, seed, n_layers, n_pages):
    """[layer][page][K, V][head][page size * head size] values of a context."""
    _, nkv, dim = HEADS[case["heads"]]
    shape = (n_layers, n_pages, 2, nkv, case["page"] * dim)
    return torch.randn(shape, generator=_gen(seed, 1), device=_device(), dtype=TYPES[case["type"]])


# ---------------------------------------------------------------- states

_CTX = None


def _lib():
    """The library's Python binding."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwenqwen3.js_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qq_hip
    return qq_hip


def _ctx():
    """The program's one context."""
    global _CTX
    if _CTX is None:
        _CTX = _lib().Context(0)
    return _CTX


class State:
    """What a program holds for one case; the library's handle is given back with it."""

    def __init__(self, case):
        self.case, self.kv, self.batch = case, None, None

    def __del__(self):
        if self.kv is not None:
            self.kv.release()


def _handle(st):
    """The library's handle over the pool, and the batch's description."""
    case, pool = st.case, st.pool
    nq, nkv, dim = HEADS[case["heads"]]
    qq_hip = _lib()
    typ = {"f32": qq_hip.TYPE_F32, "f16": qq_hip.TYPE_F16, "bf16": qq_hip.TYPE_BF16}[case["type"]]
    st.kv = _ctx().kv_pool(pool.shape[0], pool.shape[1], case["page"], nkv, dim, typ, ptr=pool.data_ptr(),
                           nbytes=pool.numel() * pool.element_size())
    if case["kind"] != "pages":
        st.batch = qq_hip.KvBatch(case["seqs"], st.table.data_ptr(), st.table.shape[1], st.lens.data_ptr(),
                                  None if st.starts is None else st.starts.data_ptr(), st.n_rows)


def prepare(case, seed):
    st = State(case)
    dev = _device()
    nq, nkv, dim = HEADS[case["heads"]]
    if case["kind"] == "pages":
        st.pool = _pool(case, seed, case["layers"], case["pool"])
        order = torch.randperm(case["pool"], generator=_gen(seed, 2), device=dev).int()
        n = case["seqs"]
        # every source and every destination once
        st.pairs = torch.stack([order[:n], order[n:2 * n]], 1).contiguous()
        st.map = torch.arange(case["pool"], device=dev, dtype=torch.int32)
        st.map[st.pairs[:, 0].long()] = st.pairs[:, 1]
        # tables of the live pages (the sources and the pages that stay), some shared
        live = torch.cat([order[:n], order[2 * n:]])
        pick = torch.randint(0, live.numel(), (256, 64), generator=_gen(seed, 3), device=dev)
        st.table = live[pick].contiguous()
    else:
        lens, news = _lens(case)
        ps = case["page"]
        need = [-(-l // ps) for l in lens]
        width = max(max(need), 1)
        n_pages = sum(need) + 3
        order = torch.randperm(n_pages, generator=_gen(seed, 2), device=dev).int().cpu()
        table, at = torch.zeros((case["seqs"], width), dtype=torch.int32), 0
        for b, k in enumerate(need):
            table[b, :k] = order[at:at + k]
            at += k
        st.table = table.to(dev)
        st.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        starts = [0]
        for k in news:
            starts.append(starts[-1] + k)
        st.n_rows = starts[-1]
        st.max_rows, st.max_len = max(news), max(lens)
        st.starts = None if case["rows"] == 1 else torch.tensor(starts, dtype=torch.int32, device=dev)
        store = case["kind"] == "store"
        st.pool = _pool(case, seed, 2 if store else 1, n_pages)
        g = _gen(seed, 4)
        # scores of a trained head spread over a few units
        st.q = torch.randn((st.n_rows, nq * dim), generator=g, device=dev) * (1.0 if store else 2.0)
        st.out = torch.zeros_like(st.q)
        if store:
            st.k = torch.randn((st.n_rows, nkv * dim), generator=g, device=dev) * 3.0
            st.v = torch.randn((st.n_rows, nkv * dim), generator=g, device=dev)
            st.qn = torch.rand(dim, generator=g, device=dev) + 0.5
            st.kn = torch.rand(dim, generator=g, device=dev) + 0.5
    if torch.cuda.is_available():
        torch.cuda.synchronize()
    if own:
        _handle(st)
    return st


# ---------------------------------------------------------------- the plain forms

def _rows_of(st):
    """(sequence, position) of every row of the batch."""
    t = torch.arange(st.n_rows, device=st.lens.device)
    if st.starts is None:
        return t, st.lens.long() - 1
    seq = torch.searchsorted(st.starts[1:].long(), t, right=True)
    return seq, st.lens.long()[seq] - st.starts.long()[seq + 1] + t


def _norm_rope(x, w, pos, dim):
    """Per-head RMSNorm and split-half rotation of [rows, heads * dim]."""
    x = x.view(x.shape[0], -1, dim)
    x = w * x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    half = dim // 2
    i = torch.arange(half, device=x.device, dtype=torch.float64)
    angle = pos.double()[:, None] * ROPE_BASE ** (-i / half)      # far positions need 64 bits
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _plain_store(st):
    case, pool = st.case, st.pool
    nq, nkv, dim = HEADS[case["heads"]]
    ps, u = case["page"], _unit(case["type"])
    seq, pos = _rows_of(st)
    live = pos >= 0
    st.out.copy_(torch.where(live[:, None], _norm_rope(st.q, st.qn, pos, dim).view(st.n_rows, -1), st.out))
    k = _norm_rope(st.k, st.kn, pos, dim)[live].to(pool.dtype)
    v = st.v.view(st.n_rows, nkv, dim)[live].to(pool.dtype)
    seq, pos = seq[live], pos[live]
    page = st.table.long()[seq, pos // ps]
    slot = pos % ps
    n = page.numel()
    layer = pool[1].view(pool.shape[1], 2, nkv, -1)
    keys = layer[:, 0].view(-1, nkv, dim // u, ps, u)
    keys[page, :, :, slot] = k.view(n, nkv, dim // u, u)
    vals = layer[:, 1].view(-1, nkv, ps // u, dim, u)
    vals[page, :, slot // u, :, slot % u] = v
    return {"q": st.out, "pool": pool}


def _plain_attn(st):
    case, pool = st.case, st.pool
    nq, nkv, dim = HEADS[case["heads"]]
    ps, u, grp = case["page"], _unit(case["type"]), nq // nkv
    n, width, m = case["seqs"], st.table.shape[1], st.max_rows
    pages = st.table.long()
    keys = pool[0, :, 0].view(-1, nkv, dim // u, ps, u)[pages]         # [n, width, nkv, dim/u, ps, u]
    keys = keys.permute(0, 2, 3, 5, 1, 4).reshape(n, nkv, dim, width * ps).float()
    vals = pool[0, :, 1].view(-1, nkv, ps // u, dim, u)[pages]
    vals = vals.permute(0, 2, 1, 3, 5, 4).reshape(n, nkv, width * ps, dim).float()
    # the batch's rows, padded to the longest sequence's count
    seq, pos = _rows_of(st)
    first = torch.arange(n, device=pages.device) if st.starts is None else st.starts.long()[:-1]
    at = torch.arange(st.n_rows, device=pages.device) - first[seq]
    q = torch.zeros((n, m, nkv, grp, dim), device=pages.device)
    q[seq, at] = st.q.view(st.n_rows, nkv, grp, dim)
    p = torch.full((n, m), -1, device=pages.device)
    p[seq, at] = pos
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(n, nkv, m * grp, dim), keys) * (1.0 / math.sqrt(dim))
    s = torch.arange(width * ps, device=pages.device)
    seen = s <= p[..., None]
    if case["window"]:
        seen &= (s > p[..., None] - case["window"]) | (s < case["sinks"])
    seen = seen[:, None, :, None].expand(n, 1, m, grp, width * ps).reshape(n, 1, m * grp, width * ps)
    score = score.masked_fill(~seen, float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    # positions that no row of a sequence sees hold no values of it
    vals = vals.masked_fill(~seen.any(2)[..., None], 0.0)
    o = torch.matmul(e, vals) / torch.where(total == 0, 1.0, total)
    o = o.view(n, nkv, m, grp, dim).permute(0, 2, 1, 3, 4)[seq, at]
    st.out.copy_(o.reshape(st.n_rows, nq * dim))
    return st.out


def _plain_pages(st):
    src, dst = st.pairs[:, 0].long(), st.pairs[:, 1].long()
    st.pool[:, dst] = st.pool[:, src]
    if st.case.get("remap"):
        st.table.copy_(st.map[st.table.long()])
        return {"pool": st.pool, "table": st.table}
    return {"pool": st.pool}


# ---------------------------------------------------------------- one pass

def run(st):
    case, kind = st.case, st.case["kind"]
    nq, nkv, dim = HEADS[case["heads"]]
    if not own:
        return {"store": _plain_store, "attn": _plain_attn, "pages": _plain_pages}[kind](st)
    if kind == "store":
        st.kv.store_dev(1, st.batch, st.k.data_ptr(), st.v.data_ptr(), q_ptr=st.q.data_ptr(), n_heads=nq,
                        q_norm_ptr=st.qn.data_ptr(), k_norm_ptr=st.kn.data_ptr(), eps=EPS, rope_base=ROPE_BASE,
                        q_out_ptr=st.out.data_ptr())
        return {"q": st.out, "pool": st.pool}
    if kind == "attn":
        st.kv.attn_dev(0, st.batch, st.q.data_ptr(), nq, st.out.data_ptr(), scale=1.0 / math.sqrt(dim),
                       window=case["window"], sinks=case["sinks"])
        return st.out
    st.kv.copy_pages_dev(st.pairs.data_ptr(), case["seqs"])
    if case.get("remap"):
        _ctx().kv_remap_dev(st.table.data_ptr(), st.table.numel(), st.map.data_ptr(), case["pool"])
        return {"pool": st.pool, "table": st.table}
    return {"pool": st.pool}


# ---------------------------------------------------------------- work

def _seen(p, window, sinks):
    """How many positions a row at position p sees."""
    if p < 0:
        return 0
    if not window or p < window:
        return p + 1
    return window + min(sinks, p - window + 1)


def work(case):
    nq, nkv, dim = HEADS[case["heads"]]
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "pages":
        page = case["layers"] * 2 * nkv * dim * case["page"] * size
        return {"bytes": 2.0 * case["seqs"] * page + (2 * 256 * 64 * 4 if case.get("remap") else 0), "flops": 0}
    lens, news = _lens(case)
    rows = sum(k for l, k in zip(lens, news) if l)
    if case["kind"] == "store":
        return {"bytes": rows * dim * (4.0 * (2 * nq + 2 * nkv) + 2.0 * nkv * size), "flops": 0}
    w, s = case["window"], case["sinks"]
    flops = touched = 0
    for l, k in zip(lens, news):
        if not l:
            continue
        flops += sum(_seen(p, w, s) for p in range(l - k, l)) * 4.0 * nq * dim
        low = max(0, l - k - w + 1) if w else 0
        touched += l - low + min(low, s)
    return {"bytes": touched * 2.0 * nkv * dim * size + 2.0 * rows * nq * dim * 4, "flops": flops}


# ---------------------------------------------------------------- the values in 64 bits

def _exact_store(st):
    """Row by row from the definition; the pool's other values as they are."""
    case = st.case
    nq, nkv, dim = HEADS[case["heads"]]
    ps, u, half = case["page"], _unit(case["type"]), dim // 2
    lens, news = _lens(case)
    seq = torch.tensor([b for b, k in enumerate(news) for _ in range(k)], device=st.q.device)
    pos = torch.tensor([l - k + i for l, k in zip(lens, news) for i in range(k)], device=st.q.device)
    inv = torch.tensor([1.0 / ROPE_BASE ** (i / half) for i in range(half)], dtype=torch.float64, device=st.q.device)

    def turned(x, w, heads):
        x = x.double().reshape(-1, heads, dim)
        x = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / dim + EPS) ** 0.5 * w.double()
        z = torch.complex(x[..., :half], x[..., half:])
        z = z * torch.polar(torch.ones_like(inv), pos[:, None].double() * inv)[:, None]
        return torch.cat([z.real, z.imag], -1)

    ok = pos >= 0
    q = torch.where(ok[:, None], turned(st.q, st.qn, nq).reshape(-1, nq * dim), 0.0)
    pool = st.pool.double().reshape(-1)
    block = nkv * ps * dim
    page = st.table[seq, pos.clamp(min=0) // ps].long()
    base = ((st.pool.shape[1] + page) * 2 * block)[:, None, None] + torch.arange(nkv, device=q.device)[:, None] * (ps * dim)
    d, slot = torch.arange(dim, device=q.device), (pos % ps)[:, None, None]
    pool[(base + ((d // u) * ps + slot) * u + d % u)[ok]] = turned(st.k, st.kn, nkv)[ok]
    pool[(base + block + ((slot // u) * dim + d) * u + slot % u)[ok]] = st.v.double().reshape(-1, nkv, dim)[ok]
    return {"q": q, "pool": pool.view(st.pool.shape)}


def _exact_attn(st):
    """Sequence by sequence and head by head."""
    case = st.case
    nq, nkv, dim = HEADS[case["heads"]]
    ps, u, grp = case["page"], _unit(case["type"]), nq // nkv
    lens, news = _lens(case)
    dev = st.q.device
    flat, block = st.pool.view(-1), nkv * ps * dim
    out = torch.zeros((st.n_rows, nq, dim), dtype=torch.float64, device=dev)
    q = st.q.view(-1, nq, dim)
    d, row = torch.arange(dim, device=dev), 0
    for b, (l, k) in enumerate(zip(lens, news)):
        if l:
            s = torch.arange(l, device=dev)
            slot = (s % ps)[:, None]
            base = st.table[b, s // ps].long()[:, None] * (2 * block)
            p = torch.arange(l - k, l, device=dev)[:, None]
            hide = s > p
            if case["window"]:
                hide |= (s <= p - case["window"]) & (s >= case["sinks"])
            for h in range(nkv):
                at = base + h * ps * dim
                key = flat[at + ((d // u) * ps + slot) * u + d % u].double()
                val = flat[at + block + ((slot // u) * dim + d) * u + slot % u].double()
                for g in range(h * grp, (h + 1) * grp):
                    score = (q[row:row + k, g].double() @ key.T.contiguous()) / dim ** 0.5
                    out[row:row + k, g] = torch.softmax(score.masked_fill(hide, float("-inf")), -1) @ val
        row += k
    return out.view(st.n_rows, -1)


def _exact_pages(st):
    """Every page from where it comes."""
    comes = list(range(st.case["pool"]))
    for src, dst in st.pairs.tolist():
        comes[dst] = src
    out = {"pool": st.pool.double().index_select(1, torch.tensor(comes, device=st.pool.device))}
    if st.case.get("remap"):
        goes = dict(st.pairs.tolist())
        out["table"] = torch.tensor([[goes.get(p, p) for p in row] for row in st.table.tolist()], dtype=torch.int32)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"store": _exact_store, "attn": _exact_attn, "pages": _exact_pages}[case["kind"]](st)

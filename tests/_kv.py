"""Paged key/value caches for the tests: pools filled place by place from the
documented layout, and attention and the stored rows in binary64."""
import numpy as np

F32, F16, BF16 = 0, 1, 30
NAMES = {"f32": F32, "f16": F16, "bf16": BF16}
EPS_HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # half a step, relative


def unit(typ):
    return 4 if typ == F32 else 8


def to_bits(x, typ):
    """fp32 values (already of the type) as the pool's raw values."""
    x = np.asarray(x, np.float32)
    if typ == F32:
        return x
    if typ == F16:
        return x.astype(np.float16).view(np.uint16)
    return (x.view(np.uint32) >> 16).astype(np.uint16)


def from_bits(b, typ):
    if typ == F32:
        return b.astype(np.float64)
    if typ == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(x, typ):
    """fp32 values rounded (bf16: cut) to the cache's type."""
    x = np.asarray(x, np.float32)
    if typ == F32:
        return x
    if typ == F16:
        return x.astype(np.float16).astype(np.float32)
    return (x.view(np.uint32) & 0xffff0000).view(np.float32)


class Pool:
    """[layer][page][K, V][head][page_size * head_dim] raw values on the host."""

    def __init__(self, layers, pages, ps, nkv, dim, typ, fill=0.0):
        self.layers, self.pages, self.ps, self.nkv, self.dim, self.typ = layers, pages, ps, nkv, dim, typ
        one = to_bits(np.array([fill], np.float32), typ)
        self.raw = np.full((layers, pages, 2, nkv, ps * dim), one[0], one.dtype)

    def _at(self, kv, slot):
        u, d = unit(self.typ), np.arange(self.dim)
        if kv == 0:
            return ((d // u) * self.ps + slot) * u + d % u
        return ((slot // u) * self.dim + d) * u + slot % u

    def put(self, layer, page, slot, k, v):
        """k, v [nkv, dim]"""
        self.raw[layer, page, 0][:, self._at(0, slot)] = to_bits(k, self.typ)
        self.raw[layer, page, 1][:, self._at(1, slot)] = to_bits(v, self.typ)

    def get(self, layer, page, slot):
        return (from_bits(self.raw[layer, page, 0][:, self._at(0, slot)], self.typ),
                from_bits(self.raw[layer, page, 1][:, self._at(1, slot)], self.typ))


def seen(p, s, window, sinks):
    """Whether a row at position p sees the positions s."""
    ok = s <= p
    if window:
        ok = ok & ((s > p - window) | (s < sinks))
    return ok


def attention(q, k, v, pos, scale, window, sinks, known=None):
    """q [n, nq, dim] of rows at positions pos, k, v [L, nkv, dim], in binary64:
    (out, bound): bound is what fp32 sums of exact products may be off by.

    A score is scale times a sum of D products, off by about sqrt(D) roundings
    of 2^-24 of the sum of their magnitudes (twice that for the factors 1 +
    2^-22 of fp16's two planes); the exponential, the sum of probabilities,
    the sum over values and the division add no more than 32 roundings; each
    moves the output by its share of sum p |v|."""
    n, nq, dim = q.shape
    nkv = k.shape[1]
    g = nq // nkv
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, bound = np.zeros((n, nq, dim)), np.zeros((n, nq, dim))
    s = np.arange(k.shape[0])
    for i in range(n):
        ok = seen(pos[i], s, window, sinks)
        if known is not None:
            ok = ok & known
        at = s[ok]
        if not at.size:
            continue
        for h in range(nq):
            kk, vv = k[at, h // g], v[at, h // g]
            sc = kk @ q[i, h] * scale
            e = np.exp(sc - sc.max())
            e /= e.sum()
            out[i, h] = e @ vv
            mag = np.abs(kk) @ np.abs(q[i, h]) * abs(scale)
            bound[i, h] = 2.0 ** -24 * (4.0 * np.sqrt(dim) * mag.max() + 32.0) * (e @ np.abs(vv))
    return out, bound


def norm_rope(x, w, pos, eps, base):
    """x [n, heads, dim] in binary64 (roundings to fp32 ahead of RoPE left out)."""
    x = np.asarray(x, np.float64)
    n, _, dim = x.shape
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if base:
        h = dim // 2
        th = np.asarray(pos, np.float64)[:, None] * (1.0 / base ** (np.arange(h) / h))
        c, s = np.cos(th)[:, None], np.sin(th)[:, None]
        a, b = x[..., :h], x[..., h:]
        x = np.concatenate([a * c - b * s, a * s + b * c], -1)
    return x

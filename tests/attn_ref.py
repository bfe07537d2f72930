"""Plain 64-bit forms of the attention operators and the inputs of their tests."""
from __future__ import annotations

import numpy as np

HALF16 = 2.0 ** -11       # half a step of fp16, relative
TINY16 = 2.0 ** -25       # half a step of fp16's subnormals
U32 = 2.0 ** -24          # half a step of fp32, relative


def visible(p: int, length: int, window: int, sinks: int) -> np.ndarray:
    """the keys that position p sees of a sequence of `length`"""
    j = np.arange(max(length, 0))
    m = j <= p
    if window:
        m &= (j > p - window) | (j < sinks)
    return j[m]


def norm_rope(x, gamma, inv_freq, pos, style, eps=1e-6):
    """x [M, H, D] float64 -> (result, bound of the fp32 and fp16 roundings)"""
    y = x.astype(np.float64)
    D = y.shape[-1]
    if gamma is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    z = y.copy()
    mag = np.abs(y)
    if inv_freq is not None and len(inv_freq):
        t = pos.astype(np.float64)[:, None] * np.asarray(inv_freq, np.float64)
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        n = len(inv_freq)
        a, b = (slice(0, n), slice(n, 2 * n)) if style == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., a] * s + y[..., b] * c
        mag[..., a] = mag[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    # fp32: the sum of D squares (D/8 + 8 adds: D rounds at most), the root, three products, the sine
    # and cosine (2 pi of half a step of the fraction of a turn, and 2 steps of their own): 24 + D
    # half steps of the pair's magnitudes; then one rounding to fp16
    return z, HALF16 * np.abs(z) + (24 + D) * U32 * mag + TINY16


def attention(q, k, v, seen, scale):
    """one head: q [D], k / v [n, D] (the keys seen) -> (result [D], bound) in 64 bits.
    The bound: the result's rounding to fp16; the weights' rounding to fp16 (half a step each); the
    error of a score (D products in fp32, each at most one step off, the product with the scale and
    the exponential: 16 more) in the weight and in the sum of the weights; and the fp32 sums over the
    keys, 16 keys in one instruction and one rounding (a step) for each."""
    D = q.shape[0]
    if len(seen) == 0:
        return np.zeros(D), np.zeros(D)
    e = k @ q * scale
    w = np.exp(e - e.max())
    w /= w.sum()
    o = w @ v
    W = w @ np.abs(v)
    delta = 2 * U32 * ((D + 16) * scale * (np.abs(k) @ np.abs(q)).max() + 16)
    n = len(seen)
    return o, HALF16 * np.abs(o) + W * (HALF16 + 2 * delta + 2 * U32 * (n / 16 + 32)) + TINY16


def bases(D, rot, base):
    return [base ** (-2.0 * j / rot) for j in range(rot // 2)]


class Paged:
    """A cache of random pages on the host: k, v fp16 [pages, K, page, D], table int32 [S, stride]."""

    def __init__(self, rng, lens, K, page, D, extra_pages=2, stride=None, fill=np.nan):
        self.page, self.K, self.D, self.lens = page, K, D, list(lens)
        need = [max(0, -(-n // page)) for n in lens]
        self.stride = stride or max(1, max(need))
        total = sum(need) + extra_pages
        order = rng.permutation(total).astype(np.int32)
        self.table = np.full((len(lens), self.stride), -7, np.int32)
        self.k = np.full((total, K, page, D), fill, np.float16)
        self.v = np.full((total, K, page, D), fill, np.float16)
        self.keys, self.values = [], []
        at = 0
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            n = max(n, 0)
            kk = rng.standard_normal((n, K, D)).astype(np.float16)
            vv = rng.standard_normal((n, K, D)).astype(np.float16)
            self.keys.append(kk)
            self.values.append(vv)
            for j in range(n):
                self.k[self.table[s, j // page], :, j % page] = kk[j]
                self.v[self.table[s, j // page], :, j % page] = vv[j]

    def forget(self, s, lo, sinks, value=np.nan):
        """poison positions [sinks, lo) of sequence s, drop the pages that hold nothing else"""
        for j in range(min(sinks, lo), lo):
            self.k[self.table[s, j // self.page], :, j % self.page] = value
            self.v[self.table[s, j // self.page], :, j % self.page] = value
        for p in range(lo // self.page):
            if p * self.page >= sinks:
                self.table[s, p] = 1 << 30


def expect(paged, q, rows, window, sinks, scale=None, heads=None):
    """rows: list of (row, sequence, position, length) -> (values, bounds) [len(rows), heads, D]"""
    heads = heads or q.shape[1]
    G = heads // paged.K
    scale = scale or paged.D ** -0.5
    out, tol = np.zeros((len(rows), heads, paged.D)), np.zeros((len(rows), heads, paged.D))
    for i, (r, s, p, n) in enumerate(rows):
        j = visible(p, n, window, sinks)
        k = paged.keys[s][j].astype(np.float64)
        v = paged.values[s][j].astype(np.float64)
        for h in range(heads):
            out[i, h], tol[i, h] = attention(q[r, h].astype(np.float64), k[:, h // G], v[:, h // G], j, scale)
    return out, tol

"""Norm and rotation, the append to the paged cache, decode and prefill attention on the GPU, against
plain 64-bit forms with bounds counted from the roundings (attn_ref)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import attn_ref as R
import npu880_mtk_npu_llm_runtime_b200 as kq

pytestmark = pytest.mark.gpu

SENTINEL = 7.5
SHAPE = -3


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def wide(rows, values, pad=16):
    """[rows, values] device view into rows that are `pad` values further apart, filled with a sentinel"""
    import torch
    t = torch.full((rows, values + pad), SENTINEL, dtype=torch.float16, device="cuda")
    return t, t[:, :values]


def close(got, want, tol, what=""):
    got = got.astype(np.float64)
    assert np.isfinite(got).all(), what
    off = np.abs(got - want) - tol
    assert off.max(initial=-1.0) <= 0, (what, "worst", off.max(), "at", np.unravel_index(off.argmax(), off.shape))


def cache_of(p: R.Paged):
    return kq.KvCache(dev(p.k), dev(p.v), dev(p.table))


# ------------------------------------------------------------------ norm and rotation

@pytest.mark.parametrize("D, H, K, rot, style", [
    (128, 32, 8, 128, "half"), (128, 32, 8, 128, "adjacent"), (64, 14, 2, 64, "half"), (64, 3, 1, 16, "adjacent"),
    (256, 16, 4, 64, "half"), (256, 5, 5, 256, "half"), (256, 16, 1, 48, "adjacent"), (128, 7, 3, 0, "half"), (128, 256, 256, 32, "half"),
])
@pytest.mark.parametrize("M", [1, 3, 130])
def test_norm_rope(kqctx, D, H, K, rot, style, M):
    rng = np.random.default_rng(D + H + rot + M)
    base = 1e6
    x = (rng.standard_normal((M, H + K, D)) * np.exp(rng.uniform(-3, 3, (M, H + K, 1)))).astype(np.float16)
    x[:, :, D // 3] *= 8
    x[M // 2, 0] = 0                                    # a zero head: eps alone under the root
    gamma = (1 + 0.2 * rng.standard_normal(D)).astype(np.float16)
    pos = rng.integers(0, 1 << 20, M).astype(np.int32)
    pos[0] = 0
    f = R.bases(D, rot, base)
    qkv = dev(x.reshape(M, -1))                         # q and k side by side in one buffer
    q, k = qkv[:, :H * D], qkv[:, H * D:]
    qb, qo = wide(M, H * D)
    kb, ko = wide(M, K * D, 8)
    rope = kq.Rope(rot, base=base, style=style) if rot else None
    kqctx.qk_norm_rope_async(rope, dev(pos) if rot else None, kq.Heads(q, H, gamma=dev(gamma), out=qo), kq.Heads(k, K, out=ko))
    kqctx.synchronize()
    for got, want, buf, n in ((qo, R.norm_rope(x[:, :H], gamma, f, pos, style), qb, H * D),
                              (ko, R.norm_rope(x[:, H:], None, f, pos, style), kb, K * D)):
        close(got.cpu().numpy().reshape(M, -1, D), *want)
        assert (buf[:, n:] == SENTINEL).all()
    assert np.array_equal(qkv.cpu().numpy().reshape(x.shape).view(np.uint16), x.view(np.uint16))
    # in place, and each side alone: the same bits
    a = qkv.clone()
    kqctx.qk_norm_rope_async(rope, dev(pos), kq.Heads(a[:, :H * D], H, gamma=dev(gamma), out=a[:, :H * D]), None)
    kqctx.qk_norm_rope_async(rope, dev(pos), None, kq.Heads(a[:, H * D:], K, out=a[:, H * D:]))
    kqctx.synchronize()
    assert (a[:, :H * D] == qo).all() and (a[:, H * D:] == ko).all()


def test_norm_rope_special_values(kqctx):
    """heads of fp16's largest and smallest values; infinities and NaN stay in their heads"""
    D = 128
    x = np.zeros((1, 6, D), np.float16)
    x[0, 0] = 65504
    x[0, 1] = 2.0 ** -24
    x[0, 2, 5] = np.inf
    x[0, 3, 9] = np.nan
    x[0, 4] = np.linspace(-1, 1, D)
    gamma = np.ones(D, np.float16)
    out = dev(np.zeros((1, 6 * D), np.float16))
    kqctx.qk_norm_rope_async(kq.Rope(D), dev(np.array([77], np.int32)), kq.Heads(dev(x.reshape(1, -1)), 6, gamma=dev(gamma), out=out))
    kqctx.synchronize()
    got = out.cpu().numpy().reshape(6, D)
    want, tol = R.norm_rope(x[:, [0, 1, 4, 5]], gamma, R.bases(D, D, 1e4), np.array([77]), "half")
    close(got[[0, 1, 4, 5]][None], want, tol)
    assert np.isnan(got[2, 5]) and np.isnan(got[3]).all()


def test_norm_rope_no_rows_and_refusals(kqctx):
    import torch
    e = torch.empty((0, 256), dtype=torch.float16, device="cuda")
    kqctx.qk_norm_rope_async(None, None, kq.Heads(e, 2, out=e))
    x = torch.zeros((2, 256), dtype=torch.float16, device="cuda")
    h = kq.Heads(x, 2, out=x)
    with pytest.raises(kq.KQError):
        kqctx.qk_norm_rope_async(kq.Rope(128), None, h)                       # no positions
    with pytest.raises(kq.KQError):
        kqctx.qk_norm_rope_async(None, None, h, eps=-1.0)
    with pytest.raises(kq.KQError):
        kqctx.qk_norm_rope_async(None, None, h, eps=float("nan"))
    with pytest.raises(kq.KQError):
        kqctx.qk_norm_rope_async(None, None, kq.Heads(x, 2))                  # no out
    with pytest.raises(kq.KQError):
        kqctx.qk_norm_rope_async(kq.Rope(256), torch.zeros(2, dtype=torch.int32, device="cuda"), h)
    y = torch.zeros((2, 260), dtype=torch.float16, device="cuda")
    for bad in (y[:, :256], y[:, 4:]):                                        # stride, alignment
        with pytest.raises(kq.KQError):
            kqctx.qk_norm_rope_async(None, None, kq.Heads(bad, 2, out=x))
    with pytest.raises(ValueError):
        kq.Heads(x.float(), 2)
    with pytest.raises(ValueError):
        kq.Heads(x.cpu(), 2)
    with pytest.raises(ValueError):
        kq.Heads(x, 3)
    with pytest.raises(ValueError):
        kq.Heads(x.t(), 2)
    kqctx.synchronize()


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("D, H, K, page, rot", [(128, 32, 8, 16, 128), (64, 14, 2, 32, 32), (256, 16, 4, 256, 64), (128, 4, 1, 64, 0)])
@pytest.mark.parametrize("with_q", [True, False])
def test_append(kqctx, D, H, K, page, rot, with_q):
    """rows of several sequences in mixed order with padding rows: the right slots, and only those"""
    rng = np.random.default_rng(D + page)
    lens = [page + 3, 5, 2 * page, 1]
    p = R.Paged(rng, lens, K, page, D, stride=4)
    rows = [(s, j) for s, n in enumerate(lens) for j in range(n) if rng.random() < 0.3 or j == n - 1] + [(-1, 0), (-5, 1 << 29)]
    rng.shuffle(rows)
    M = len(rows)
    seq, pos = (np.array(v, np.int32) for v in zip(*rows))
    x = rng.standard_normal((M, H + 2 * K, D)).astype(np.float16)
    gq, gk = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float16) for _ in range(2))
    f = R.bases(D, rot, 1e4)
    cache = cache_of(p)
    qkv = dev(x.reshape(M, -1))
    _, qo = wide(M, H * D)
    k = kq.Heads(qkv[:, H * D:(H + K) * D], K, gamma=dev(gk))
    v = kq.Heads(qkv[:, (H + K) * D:], K)
    q = kq.Heads(qkv[:, :H * D], H, gamma=dev(gq), out=qo) if with_q else None
    kqctx.kv_append_async(cache, kq.Rope(rot) if rot else None, dev(seq), dev(pos), k, v, q=q)
    kqctx.synchronize()
    live = seq >= 0
    kw, kt = R.norm_rope(x[:, H:H + K], gk, f, pos, "half")
    qw, qt = R.norm_rope(x[:, :H], gq, f, pos, "half")
    gotk, gotv = cache.k.cpu().numpy(), cache.v.cpu().numpy()
    wantk, wantv = p.k.copy(), p.v.copy()
    for i in np.flatnonzero(live):
        at = (p.table[seq[i], pos[i] // page], slice(None), pos[i] % page)
        close(gotk[at], kw[i], kt[i], i)
        wantk[at] = gotk[at]
        wantv[at] = x[i, H + K:]
    assert np.array_equal(gotk.view(np.uint16), wantk.view(np.uint16))    # nothing else was written
    assert np.array_equal(gotv.view(np.uint16), wantv.view(np.uint16))
    if with_q:
        got = qo.cpu().numpy().reshape(M, H, D)
        close(got[live], qw[live], qt[live])
        assert (got[~live] == SENTINEL).all()                             # padding rows as they were


def test_append_outside_the_cache_is_reported_and_not_written(kqctx):
    rng = np.random.default_rng(1)
    D, K, page = 64, 2, 16
    p = R.Paged(rng, [20, 20, 20], K, page, D, stride=3)
    p.table[1, 0] = p.k.shape[0]          # one past the last page
    p.table[2, 1] = -1
    bad = [(3, 0), (0, 48), (0, -1), (1, 2), (2, 17), (2 ** 31 - 1, 0), (0, 2 ** 31 - 1), (0, 47)]
    rows = bad + [(0, 7)]
    seq, pos = (np.array(v, np.int32) for v in zip(*rows))
    x = rng.standard_normal((len(rows), 2 * K * D)).astype(np.float16)
    cache = cache_of(p)
    h = dev(x)
    kqctx.kv_append_async(cache, kq.Rope(D), dev(seq), dev(pos), kq.Heads(h[:, :K * D], K), kq.Heads(h[:, K * D:], K))
    with pytest.raises(kq.KQError) as e:
        kqctx.synchronize()
    assert e.value.status == SHAPE
    got = cache.v.cpu().numpy()
    want = p.v.copy()
    want[p.table[0, 0], :, 7] = x[-1, K * D:].reshape(K, D)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    kqctx.kv_append_async(cache, None, dev(seq[-1:]), dev(pos[-1:]), kq.Heads(h[-1:, :K * D], K), kq.Heads(h[-1:, K * D:], K))
    kqctx.synchronize()                   # the context stays usable


# ------------------------------------------------------------------ decode

DECODE = [
    # D, heads, kv_heads, page, lengths, window, sinks
    (128, 32, 8, 16, [1, 2, 15, 16, 17, 33, 0, 100], 0, 0),
    (128, 8, 8, 64, [700], 0, 0),
    (128, 16, 1, 16, [5, 0, 0, 1300], 0, 0),
    (128, 12, 1, 32, [77], 0, 0),
    (64, 16, 2, 32, [64, 63, 65, 1], 0, 0),
    (64, 14, 2, 256, [300, 5], 0, 0),
    (256, 16, 4, 128, [129, 1, 600], 0, 0),
    (256, 16, 1, 16, [40], 0, 0),
    (128, 32, 8, 16, [1, 40, 200, 999], 64, 4),
    (128, 9, 3, 16, [1, 40, 200, 999], 50, 0),
    (64, 8, 2, 16, [1, 40, 200, 999], 1, 1),
    (256, 8, 2, 64, [1, 40, 200, 999], 100, 300),
    (128, 24, 8, 16, list(range(0, 70)), 0, 0),
]


@pytest.mark.parametrize("D, H, K, page, lens, window, sinks", DECODE)
def test_decode(kqctx, D, H, K, page, lens, window, sinks):
    rng = np.random.default_rng(len(lens) + D + H + window)
    p = R.Paged(rng, lens, K, page, D)
    if window:
        for s, n in enumerate(lens):
            p.forget(s, max(0, n - window), sinks)
    S = len(lens)
    q = (1.5 * rng.standard_normal((S, H, D))).astype(np.float16)
    qb, qv = wide(S, H * D)
    qv.copy_(dev(q.reshape(S, -1)))
    ob, ov = wide(S, H * D, 24)
    a = kq.Attention(cache_of(p), qv, ov, dev(np.array(lens, np.int32)), window=window, sinks=sinks)
    kqctx.attn_decode_async(a)
    kqctx.synchronize()
    want, tol = R.expect(p, q, [(s, s, n - 1, n) for s, n in enumerate(lens)], window, sinks)
    close(ov.cpu().numpy().reshape(S, H, D), want, tol)
    assert (ob[:, H * D:] == SENTINEL).all()
    first = ov.clone()
    for _ in range(3):
        kqctx.attn_decode_async(a)
    kqctx.synchronize()
    assert (ov == first).all()            # the same order of sums every time


@pytest.mark.parametrize("D, G", [(128, 4), (64, 8), (256, 4), (128, 16)])
def test_decode_long(kqctx, D, G):
    """one sequence over many CTAs, and a long one among short ones"""
    rng = np.random.default_rng(G)
    for lens in ([20011], [3, 9001, 17]):
        p = R.Paged(rng, lens, 1, 64, D)
        q = rng.standard_normal((len(lens), G, D)).astype(np.float16)
        out = dev(np.zeros_like(q))
        a = kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32)), scale=0.3)
        kqctx.attn_decode_async(a)
        kqctx.synchronize()
        want, tol = R.expect(p, q, [(s, s, n - 1, n) for s, n in enumerate(lens)], 0, 0, scale=float(np.float32(0.3)))
        close(out.cpu().numpy(), want, tol)


def test_decode_many_sequences(kqctx):
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, 40, 4096)]
    p = R.Paged(rng, lens, 1, 16, 64)
    q = rng.standard_normal((4096, 2, 64)).astype(np.float16)
    out = dev(np.full_like(q, SENTINEL))
    kqctx.attn_decode_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32))))
    kqctx.synchronize()
    want, tol = R.expect(p, q, [(s, s, n - 1, n) for s, n in enumerate(lens)], 0, 0)
    close(out.cpu().numpy(), want, tol)


def test_decode_large_scores(kqctx):
    """scores far apart and of both signs: the running maximum moves at every tile, later or earlier"""
    rng = np.random.default_rng(9)
    D, n = 128, 900
    p = R.Paged(rng, [n, n], 2, 16, D)
    ramp = np.linspace(-4, 4, n)
    for s, r in ((0, ramp), (1, ramp[::-1])):
        p.keys[s][:, :, 0] = (64 * r[:, None]).astype(np.float16)
        for j in range(n):
            p.k[p.table[s, j // 16], :, j % 16] = p.keys[s][j]
    q = rng.standard_normal((2, 4, D)).astype(np.float16)
    q[:, :, 0] = np.array([30, -30, 3, 0])[None]
    out = dev(np.zeros_like(q))
    kqctx.attn_decode_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array([n, n], np.int32))))
    kqctx.synchronize()
    want, tol = R.expect(p, q, [(s, s, n - 1, n) for s in range(2)], 0, 0)
    close(out.cpu().numpy(), want, tol)


def test_decode_nonfinite(kqctx):
    """what a row sees reaches it as in the formula; what it does not see has no effect"""
    rng = np.random.default_rng(4)
    D = 128
    lens = [40, 40, 40, 40]
    p = R.Paged(rng, lens, 1, 16, D, fill=np.inf)
    p.v[p.table[0, 1], 0, 3, 5] = np.inf          # a value that sequence 0 sees
    p.v[p.table[1, 0], 0, 3, 6] = np.nan
    p.k[p.table[2, 2], 0, 7, 0] = np.nan          # a NaN score
    q = np.abs(rng.standard_normal((4, 1, D))).astype(np.float16)
    p.k[p.table[3, 0], 0, 2, :] = -np.inf         # a score of -inf: weight 0
    p.keys[3] = np.delete(p.keys[3], 2, 0)
    p.values[3] = np.delete(p.values[3], 2, 0)
    out = dev(np.zeros_like(q))
    kqctx.attn_decode_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32))))
    kqctx.synchronize()
    got = out.cpu().numpy()[:, 0]
    assert np.isinf(got[0, 5]) and np.isfinite(np.delete(got[0], 5)).all()
    assert np.isnan(got[1, 6]) and np.isfinite(np.delete(got[1], 6)).all()
    assert np.isnan(got[2]).all()
    want, tol = R.expect(p, q, [(3, 3, 38, 39)], 0, 0)
    close(got[3][None, None], want, tol)


def test_decode_bad_pages_and_lengths(kqctx):
    rng = np.random.default_rng(6)
    D, page = 128, 16
    lens = [40, 40, 40, 40]
    p = R.Paged(rng, lens, 2, page, D, stride=3)
    p.table[0, 1] = p.k.shape[0]                  # positions 16..31 of sequence 0 are masked
    q = rng.standard_normal((4, 4, D)).astype(np.float16)
    out = dev(np.zeros_like(q))
    given = np.array([40, -3, 1000, 40], np.int32)
    a = kq.Attention(cache_of(p), dev(q), out, dev(given))
    kqctx.attn_decode_async(a)
    with pytest.raises(kq.KQError) as e:
        kqctx.synchronize()
    assert e.value.status == SHAPE
    got = out.cpu().numpy()
    keep = np.r_[0:16, 32:40]
    p.keys[0], p.values[0] = p.keys[0][keep], p.values[0][keep]
    want, tol = R.expect(p, q, [(0, 0, 23, 24), (3, 3, 39, 40)], 0, 0)
    close(got[[0, 3]], want, tol)
    assert (got[1] == 0).all()                    # a negative length counts as 0
    good = np.array([0, 40, 40, 0], np.int32)
    kqctx.attn_decode_async(kq.Attention(a.cache, dev(q), out, dev(good)))
    kqctx.synchronize()                           # the context stays usable
    got = out.cpu().numpy()
    want, tol = R.expect(p, q, [(1, 1, 39, 40), (2, 2, 39, 40)], 0, 0)
    close(got[1:3], want, tol)
    assert (got[[0, 3]] == 0).all()


# ------------------------------------------------------------------ prefill

PREFILL = [
    # D, heads, kv_heads, page, (rows, length) per sequence, window, sinks
    (128, 32, 8, 16, [(1, 1), (2, 2), (17, 17), (0, 9), (64, 64)], 0, 0),
    (128, 8, 8, 64, [(300, 300)], 0, 0),
    (128, 4, 1, 16, [(129, 700), (1, 513), (70, 70)], 0, 0),
    (128, 3, 1, 32, [(100, 260)], 0, 0),
    (128, 16, 1, 128, [(33, 150), (5, 5)], 0, 0),
    (64, 14, 2, 256, [(90, 400), (3, 3)], 0, 0),
    (64, 2, 1, 16, [(257, 257)], 0, 0),
    (256, 16, 4, 16, [(40, 40), (9, 200)], 0, 0),
    (256, 5, 5, 64, [(130, 131)], 0, 0),
    (128, 8, 2, 16, [(100, 300), (20, 20), (64, 500)], 64, 4),
    (128, 8, 2, 16, [(200, 200)], 1, 0),
    (64, 8, 2, 16, [(100, 900)], 50, 130),
    (256, 8, 2, 32, [(70, 400), (1, 399)], 100, 5),
    (128, 4, 4, 16, [(10, 4), (5, 0), (8, 8)], 0, 0),        # more rows than keys: the first rows see nothing
]


@pytest.mark.parametrize("D, H, K, page, seqs, window, sinks", PREFILL)
def test_prefill(kqctx, D, H, K, page, seqs, window, sinks):
    rng = np.random.default_rng(len(seqs) + D + H + window)
    lens = [b for _, b in seqs]
    p = R.Paged(rng, lens, K, page, D)
    if window:
        for s, (a, b) in enumerate(seqs):
            p.forget(s, max(0, b - a + 1 - window), sinks)
    start = np.cumsum([2] + [a for a, _ in seqs]).astype(np.int32)      # two rows before the first sequence
    M = int(start[-1]) + 3                                              # three behind the last
    q = (1.5 * rng.standard_normal((M, H, D))).astype(np.float16)
    _, qv = wide(M, H * D)
    qv.copy_(dev(q.reshape(M, -1)))
    ob, ov = wide(M, H * D, 24)
    a = kq.Attention(cache_of(p), qv, ov, dev(np.array(lens, np.int32)), q_start=dev(start), window=window, sinks=sinks)
    kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    rows = [(start[s] + i, s, b - n + i, b) for s, (n, b) in enumerate(seqs) for i in range(n)]
    want, tol = R.expect(p, q, rows, window, sinks)
    got = ov.cpu().numpy().reshape(M, H, D)
    close(got[[r[0] for r in rows]], want, tol)
    rest = np.setdiff1d(np.arange(M), [r[0] for r in rows])
    assert (got[rest] == SENTINEL).all() and (ob[:, H * D:] == SENTINEL).all()
    first = ov.clone()
    for _ in range(3):
        kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    assert (ov == first).all()


def test_prefill_rows_equal_decode(kqctx):
    """the last row of each sequence sees what decode sees"""
    rng = np.random.default_rng(3)
    seqs = [(5, 200), (1, 77), (130, 130)]
    p = R.Paged(rng, [b for _, b in seqs], 2, 16, 128)
    start = np.cumsum([0] + [a for a, _ in seqs]).astype(np.int32)
    q = rng.standard_normal((int(start[-1]), 8, 128)).astype(np.float16)
    cache, n = cache_of(p), dev(np.array([b for _, b in seqs], np.int32))
    o1, o2 = dev(np.zeros_like(q)), dev(np.zeros_like(q[:3]))
    kqctx.attn_prefill_async(kq.Attention(cache, dev(q), o1, n, q_start=dev(start)))
    kqctx.attn_decode_async(kq.Attention(cache, dev(q[start[1:] - 1]), o2, n))
    kqctx.synchronize()
    want, tol = R.expect(p, q, [(start[s + 1] - 1, s, b - 1, b) for s, (_, b) in enumerate(seqs)], 0, 0)
    close(o1.cpu().numpy()[start[1:] - 1], want, tol)
    close(o2.cpu().numpy(), want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_nonfinite_in_later_keys(kqctx, D):
    """infinities and NaN of a later token have no effect on the rows before it"""
    rng = np.random.default_rng(D)
    n = 150
    p = R.Paged(rng, [n], 1, 16, D)
    for j, kv, value in ((100, p.v, np.inf), (120, p.v, np.nan), (140, p.k, np.nan)):
        kv[p.table[0, j // 16], 0, j % 16, 3] = value
    q = rng.standard_normal((n, 2, D)).astype(np.float16)
    out = dev(np.zeros_like(q))
    kqctx.attn_prefill_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array([n], np.int32)), q_start=dev(np.array([0, n], np.int32))))
    kqctx.synchronize()
    got = out.cpu().numpy()
    want, tol = R.expect(p, q, [(i, 0, i, n) for i in range(100)], 0, 0)
    close(got[:100], want, tol)
    assert np.isinf(got[100:120, :, 3]).all() and np.isfinite(np.delete(got[100:120], 3, 2)).all()
    assert np.isnan(got[120:140, :, 3]).all() and np.isfinite(np.delete(got[120:140], 3, 2)).all()
    assert np.isnan(got[140:]).all()


def test_prefill_bad_tables(kqctx):
    """row ranges outside M, a missing page, lengths past the table: reported, the rest computed"""
    rng = np.random.default_rng(8)
    D = 128
    p = R.Paged(rng, [50, 50, 50], 1, 16, D, stride=4)
    p.table[1, 1] = -9                             # positions 16..31 of sequence 1 are masked
    q = rng.standard_normal((60, 2, D)).astype(np.float16)
    out = dev(np.full_like(q, SENTINEL))
    cache, dq = cache_of(p), dev(q)

    def call(start, lens):
        out.fill_(SENTINEL)
        kqctx.attn_prefill_async(kq.Attention(cache, dq, out, dev(np.array(lens, np.int32)), q_start=dev(np.array(start, np.int32))))
        with pytest.raises(kq.KQError) as e:
            kqctx.synchronize()
        assert e.value.status == SHAPE
        return out.cpu().numpy()

    got = call([0, 20, 40, 60], [50, 50, 50])
    want, tol = R.expect(p, q, [(r, 0, 30 + r, 50) for r in range(20)] + [(r, 2, r - 10, 50) for r in range(40, 60)], 0, 0)
    close(got[np.r_[0:20, 40:60]], want, tol)
    keep = np.r_[0:16, 32:50]
    k1, v1 = p.keys[1], p.values[1]
    p.keys[1], p.values[1] = k1[keep], v1[keep]
    want, tol = R.expect(p, q, [(r, 1, r - 20 + 30 - 16, 34) for r in range(22, 40)], 0, 0)
    close(got[22:40], want, tol)
    p.table[1, 1] = p.table[0, 0]
    cache = cache_of(p)
    for start, rows in (([0, 20, 61, 61], range(0)), ([-1, 20, 40, 60], range(40, 60)), ([5, 3, 40, 60], range(40, 60))):
        got = call(start, [50, 50, 50])
        r2 = [(r, 2, r - 10, 50) for r in rows]
        want, tol = R.expect(p, q, r2, 0, 0) if r2 else (np.zeros((0, 2, D)),) * 2
        close(got[list(rows)], want, tol)
    got = call([0, 20, 40, 60], [50, 50, 65])      # 64 positions are reached
    want, tol = R.expect(p, q, [(r, 0, 30 + r, 50) for r in range(20)], 0, 0)
    close(got[:20], want, tol)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("graph", [False, True])
def test_append_then_attend(kqctx, graph):
    """a prompt appended and attended, then tokens one by one (append, decode), eagerly or as one captured
    graph replayed with new positions: against the formulas over the whole sequences"""
    import torch
    rng = np.random.default_rng(5)
    D, H, K, page, window, sinks = 128, 8, 2, 16, 48, 4
    prompt, steps = [37, 0, 90], 5
    S, total = 3, [n + steps for n in prompt]
    stride = 8
    gq, gk = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float16) for _ in range(2))
    f = R.bases(D, D, 1e5)
    x = [rng.standard_normal((n, H + 2 * K, D)).astype(np.float16) for n in total]
    table = dev(rng.permutation(S * stride + 1)[:S * stride].reshape(S, stride).astype(np.int32))
    ck = torch.full((S * stride + 1, K, page, D), float("nan"), dtype=torch.float16, device="cuda")
    cv = torch.full_like(ck, float("nan"))
    cache, rope = kq.KvCache(ck, cv, table), kq.Rope(D, base=1e5)
    ctx = kq.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        def layer(rows):
            return (kq.Heads(rows[:, H * D:(H + K) * D], K, gamma=dgk), kq.Heads(rows[:, (H + K) * D:], K),
                    kq.Heads(rows[:, :H * D], H, gamma=dgq, out=rows[:, :H * D]))

        dgq, dgk = dev(gq), dev(gk)
        M = sum(prompt)
        rows = dev(np.concatenate([x[s][:n] for s, n in enumerate(prompt)]).reshape(M, -1))
        seq = dev(np.repeat(np.arange(S), prompt).astype(np.int32))
        pos = dev(np.concatenate([np.arange(n) for n in prompt]).astype(np.int32))
        start = dev(np.cumsum([0] + prompt).astype(np.int32))
        kv_len = dev(np.array(prompt, np.int32))
        out = torch.zeros((M, H * D), dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        k, v, q = layer(rows)
        ctx.kv_append_async(cache, rope, seq, pos, k, v, q=q)
        ctx.attn_prefill_async(kq.Attention(cache, rows[:, :H * D], out, kv_len, q_start=start, window=window, sinks=sinks))
        ctx.synchronize()
        got = [out.cpu().numpy().reshape(M, H, D)[a:a + n] for a, n in zip(np.cumsum([0] + prompt), prompt)]

        # decode: the same buffers every step
        rows = torch.zeros((S, (H + 2 * K) * D), dtype=torch.float16, device="cuda")
        seq, pos = dev(np.arange(S, dtype=np.int32)), dev(np.zeros(S, np.int32))
        out = torch.zeros((S, H * D), dtype=torch.float16, device="cuda")
        k, v, q = layer(rows)
        attn = kq.Attention(cache, rows[:, :H * D], out, kv_len, window=window, sinks=sinks)

        def step():
            ctx.kv_append_async(cache, rope, seq, pos, k, v, q=q)
            ctx.attn_decode_async(attn)

        g = None
        for i in range(steps):
            rows.copy_(dev(np.stack([x[s][n + i] for s, n in enumerate(prompt)]).reshape(S, -1)))
            pos.copy_(dev(np.array([n + i for n in prompt], np.int32)))
            kv_len.copy_(dev(np.array([n + i + 1 for n in prompt], np.int32)))
            torch.cuda.synchronize()
            if graph and i == 1:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    step()
            if g is not None:
                with torch.cuda.stream(stream):
                    g.replay()
            else:
                step()
            ctx.synchronize()
            o = out.cpu().numpy().reshape(S, 1, H, D)
            got = [np.concatenate([a, o[s]]) for s, a in enumerate(got)]
        del g
    finally:
        torch.cuda.synchronize()
        ctx.close()
    # the cache holds fp16 keys: take them from it (checked against the formula first)
    hk, hv, ht = ck.cpu().numpy(), cv.cpu().numpy(), table.cpu().numpy()
    p = R.Paged(rng, [0] * S, K, page, D)
    for s, n in enumerate(total):
        j = np.arange(n)
        p.keys[s], p.values[s] = hk[ht[s, j // page], :, j % page], hv[ht[s, j // page], :, j % page]
        close(p.keys[s], *R.norm_rope(x[s][:, H:H + K], gk, f, j, "half"))
        assert np.array_equal(p.values[s], x[s][:, H + K:])
        qw, qt = R.norm_rope(x[s][:, :H], gq, f, j, "half")
        # the queries were rounded to fp16 too: half a step of each value moves a score by at most
        # qt . |k| scale, and a weight (and the sum of weights) by its exponential
        want, tol = R.expect(p, qw, [(i, s, i, n) for i in range(n)], window, sinks, heads=H)
        for i in range(n):
            js = R.visible(i, n, window, sinks)
            for h in range(H):
                kk, vv = (a[s][js][:, h // (H // K)].astype(np.float64) for a in (p.keys, p.values))
                move = (np.abs(kk) @ qt[i, h]).max() * D ** -0.5
                tol[i, h] += np.expm1(2 * move) * np.abs(vv).max(0)
        close(got[s], want, tol, s)


def test_attention_refusals(kqctx):
    import torch
    rng = np.random.default_rng(0)
    cache = cache_of(R.Paged(rng, [5, 5], 2, 16, 64))
    q = torch.zeros((2, 4 * 64), dtype=torch.float16, device="cuda")
    n = dev(np.array([5, 5], np.int32))
    ok = kq.Attention(cache, q, torch.empty_like(q), n)
    for change in (dict(M=1), dict(heads=3), dict(q=q.data_ptr() + 2), dict(q_stride=252), dict(window=-1), dict(sinks=1), dict(scale=-1.0)):
        keep = {f: getattr(ok.struct, f) for f in change}
        for f, v in change.items():
            setattr(ok.struct, f, v)
        with pytest.raises(kq.KQError):
            kqctx.attn_decode_async(ok)
        for f, v in keep.items():
            setattr(ok.struct, f, v)
    with pytest.raises(kq.KQError):
        kqctx.attn_prefill_async(ok)                                          # no q_start
    kqctx.attn_decode_async(ok)
    with pytest.raises(ValueError):
        kq.Attention(cache, q, q[:1], n)
    with pytest.raises(ValueError):
        kq.Attention(cache, q, q, n.long())
    with pytest.raises(ValueError):
        kq.KvCache(cache.k, cache.v[:1], cache.page_table)
    with pytest.raises(ValueError):
        kq.KvCache(cache.k.transpose(1, 2), cache.v.transpose(1, 2), cache.page_table)
    kqctx.synchronize()


def test_empty_prefill(kqctx):
    import torch
    rng = np.random.default_rng(0)
    cache = cache_of(R.Paged(rng, [5], 2, 16, 64))
    q = torch.empty((0, 4 * 64), dtype=torch.float16, device="cuda")
    z = dev(np.zeros(2, np.int32))
    kqctx.attn_prefill_async(kq.Attention(cache, q, torch.empty_like(q), z[:1], q_start=z))
    kqctx.synchronize()


def test_prefill_wait_that_runs_out(kqctx):
    """a wait inside the kernel that nothing completes ends with KQ_ERR_TIMEOUT, and the context stays usable"""
    rng = np.random.default_rng(0)
    D, n = 128, 300
    p = R.Paged(rng, [n], 2, 16, D)
    q = rng.standard_normal((n, 4, D)).astype(np.float16)
    out = dev(np.zeros_like(q))
    ctx = kq.Context(0)
    try:
        a = kq.Attention(cache_of(p), dev(q), out, dev(np.array([n], np.int32)), q_start=dev(np.array([0, n], np.int32)))
        ctx.set_option("timeout_ms", 20)
        ctx.set_option("inject_timeout", 1)
        ctx.attn_prefill_async(a)
        with pytest.raises(kq.KQError) as e:
            ctx.synchronize()
        assert e.value.status == -7
        ctx.set_option("inject_timeout", 0)
        ctx.set_option("timeout_ms", 1000)
        ctx.attn_prefill_async(a)
        ctx.synchronize()
        want, tol = R.expect(p, q, [(i, 0, i, n) for i in range(n)], 0, 0)
        close(out.cpu().numpy(), want, tol)
    finally:
        ctx.close()


@pytest.mark.parametrize("D, H, K, seqs, window", [
    (128, 8, 2, [(20, 6000)], 0), (64, 4, 4, [(70, 5000), (3, 40)], 0), (256, 8, 2, [(9, 3000), (40, 40)], 0),
    (128, 4, 1, [(150, 9000)], 0), (128, 4, 1, [(150, 9000), (1, 8000)], 5000), (256, 2, 1, [(200, 4000)], 0), (64, 16, 1, [(30, 7001)], 6000),
])
def test_prefill_long_cache(kqctx, D, H, K, seqs, window):
    """few rows over long caches: the keys of an item are split over CTAs and joined"""
    rng = np.random.default_rng(D + H)
    p = R.Paged(rng, [b for _, b in seqs], K, 32, D)
    start = np.cumsum([0] + [a for a, _ in seqs]).astype(np.int32)
    q = (1.5 * rng.standard_normal((int(start[-1]), H, D))).astype(np.float16)
    out = dev(np.full_like(q, SENTINEL))
    a = kq.Attention(cache_of(p), dev(q), out, dev(np.array([b for _, b in seqs], np.int32)), q_start=dev(start), window=window,
                     sinks=7 if window else 0)
    kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    rows = [(start[s] + i, s, b - n + i, b) for s, (n, b) in enumerate(seqs) for i in range(n)]
    rows = [rows[i] for i in sorted({0, 1, len(rows) - 1, len(rows) - 2, *rng.integers(0, len(rows), 25).tolist()})]
    want, tol = R.expect(p, q, rows, window, 7 if window else 0)
    close(out.cpu().numpy()[[r[0] for r in rows]], want, tol)
    first = out.clone()
    for _ in range(3):
        kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    assert (out == first).all()


@pytest.mark.parametrize("where", ["value", "key", "query"])
def test_prefill_nonfinite_early(kqctx, where):
    """a value that almost every row sees: their rows hold it as in the formula, in reasonable time"""
    rng = np.random.default_rng(12)
    D, n = 128, 1500
    p = R.Paged(rng, [n], 2, 16, D)
    q = rng.standard_normal((n, 4, D)).astype(np.float16)
    if where == "value":
        p.v[p.table[0, 0], 1, 5, 3] = np.inf
    elif where == "key":
        p.k[p.table[0, 0], 1, 5, 3] = np.nan
    else:
        q[5:, 2:, 3] = np.nan
    out = dev(np.zeros_like(q))
    kqctx.attn_prefill_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array([n], np.int32)), q_start=dev(np.array([0, n], np.int32))))
    kqctx.synchronize()
    got = out.cpu().numpy()
    rows = [0, 3, 4, 5, 6, 127, 128, 700, n - 1]
    want, tol = R.expect(p, q, [(i, 0, i, n) for i in rows], 0, 0)
    close(got[rows][:, :2], want[:, :2], tol[:, :2])               # the other key head
    close(got[:5], *R.expect(p, q, [(i, 0, i, n) for i in range(5)], 0, 0))
    if where == "value":
        assert not np.isfinite(got[5:, 2:, 3]).any()
        keep = np.delete(np.arange(D), 3)
        close(got[rows][:, 2:][..., keep], want[:, 2:][..., keep], tol[:, 2:][..., keep])
    else:
        assert np.isnan(got[5:, 2:]).all()


def test_many_sequences_prefill(kqctx):
    rng = np.random.default_rng(13)
    for D, count in ((64, 4096), (128, 1000), (256, 4096)):
        lens = [int(x) for x in rng.integers(0, 30, count)]
        rows = [int(rng.integers(0, 2)) if count == 4096 else int(rng.integers(0, 9)) for _ in lens]
        p = R.Paged(rng, lens, 1, 16, D)
        start = np.cumsum([0] + rows).astype(np.int32)
        M = int(start[-1])
        assert M <= 4096
        q = rng.standard_normal((M, 2, D)).astype(np.float16)
        out = dev(np.full_like(q, SENTINEL))
        kqctx.attn_prefill_async(kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32)), q_start=dev(start)))
        kqctx.synchronize()
        want, tol = R.expect(p, q, [(start[s] + i, s, lens[s] - rows[s] + i, lens[s]) for s in range(count) for i in range(rows[s])], 0, 0)
        close(out.cpu().numpy(), want, tol, D)


def test_offsets_past_32_bits(kqctx):
    """pages at the far end of a cache of more than 2^32 values"""
    import torch
    rng = np.random.default_rng(14)
    D, K, page, n, pages = 128, 8, 256, 600, 16500
    assert (pages - 4) * K * page * D > 2 ** 32
    p = R.Paged(rng, [0], K, page, D)
    p.keys[0], p.values[0] = (rng.standard_normal((n, K, D)).astype(np.float16) for _ in range(2))
    table = np.array([[pages - 2, pages - 4, pages - 1]], np.int32)
    ck, cv = (torch.empty((pages, K, page, D), dtype=torch.float16, device="cuda") for _ in range(2))
    cache = kq.KvCache(ck, cv, dev(table))
    h = dev(np.concatenate([p.keys[0].reshape(n, -1), p.values[0].reshape(n, -1)], 1))
    seq, pos = dev(np.zeros(n, np.int32)), dev(np.arange(n, dtype=np.int32))
    kqctx.kv_append_async(cache, None, seq, pos, kq.Heads(h[:, :K * D], K), kq.Heads(h[:, K * D:], K))
    q = rng.standard_normal((3, 16, D)).astype(np.float16)
    lens = dev(np.array([n], np.int32))
    o1, o2 = dev(np.zeros_like(q)), dev(np.zeros_like(q[:1]))
    kqctx.attn_prefill_async(kq.Attention(cache, dev(q), o1, lens, q_start=dev(np.array([0, 3], np.int32))))
    kqctx.attn_decode_async(kq.Attention(cache, dev(q[2:]), o2, lens))
    kqctx.synchronize()
    want, tol = R.expect(p, q, [(i, 0, n - 3 + i, n) for i in range(3)], 0, 0)
    close(o1.cpu().numpy(), want, tol)
    close(o2.cpu().numpy(), want[2:], tol[2:])
    del ck, cv, cache


def test_two_contexts_at_once(kqctx):
    """two contexts on two streams, their kernels in flight together"""
    import torch
    rng = np.random.default_rng(15)
    D, n = 128, 700
    work = []
    for i in range(2):
        ctx, stream = kq.Context(0), torch.cuda.Stream()
        ctx.set_stream(stream.cuda_stream)
        p = R.Paged(rng, [n, 3000], 2, 16, D)
        q = rng.standard_normal((n + 2, 8, D)).astype(np.float16)
        o1, o2 = dev(np.zeros_like(q)), dev(np.zeros_like(q[:2]))
        lens = dev(np.array([n, 3000], np.int32))
        cache = cache_of(p)
        work.append((ctx, p, q, o1, o2, kq.Attention(cache, dev(q), o1, lens, q_start=dev(np.array([0, n, n + 2], np.int32))),
                     kq.Attention(cache, dev(q[n:]), o2, lens), stream))
    torch.cuda.synchronize()
    for _ in range(10):
        for w in work:
            w[0].attn_prefill_async(w[5])
            w[0].attn_decode_async(w[6])
    for ctx, p, q, o1, o2, _, _, _ in work:
        ctx.synchronize()
        rows = [(0, 0, 0, n), (350, 0, 350, n), (n - 1, 0, n - 1, n), (n, 1, 2998, 3000), (n + 1, 1, 2999, 3000)]
        want, tol = R.expect(p, q, rows, 0, 0)
        close(o1.cpu().numpy()[[r[0] for r in rows]], want, tol)
        want, tol = R.expect(p, q, [(n, 0, n - 1, n), (n + 1, 1, 2999, 3000)], 0, 0)
        close(o2.cpu().numpy(), want, tol)
        ctx.close()


def test_rows_at_any_16_bytes(kqctx):
    """q and out as views that begin 16 bytes into their rows, rows a multiple of 8 values apart"""
    import torch
    rng = np.random.default_rng(16)
    for D, H, K in ((64, 6, 2), (128, 4, 4), (256, 3, 1)):
        lens = [70, 33]
        p = R.Paged(rng, lens, K, 16, D)
        q = rng.standard_normal((40, H, D)).astype(np.float16)
        width = H * D + 24
        qb, ob = (torch.full((40, width), SENTINEL, dtype=torch.float16, device="cuda") for _ in range(2))
        qv, ov = qb[:, 8:8 + H * D], ob[:, 16:16 + H * D]
        qv.copy_(dev(q.reshape(40, -1)))
        n = dev(np.array(lens, np.int32))
        a = kq.Attention(cache_of(p), qv, ov, n, q_start=dev(np.array([0, 30, 40], np.int32)), heads=H)
        kqctx.attn_prefill_async(a)
        kqctx.synchronize()
        want, tol = R.expect(p, q, [(i, 0, 40 + i, 70) for i in range(30)] + [(30 + i, 1, 23 + i, 33) for i in range(10)], 0, 0)
        close(ov.cpu().numpy().reshape(40, H, D), want, tol)
        kqctx.attn_decode_async(kq.Attention(a.cache, qv[:2], ov[:2], n, heads=H))
        kqctx.synchronize()
        want, tol = R.expect(p, q, [(0, 0, 69, 70), (1, 1, 32, 33)], 0, 0)
        close(ov[:2].cpu().numpy().reshape(2, H, D), want, tol)
        assert (ob[:, :16] == SENTINEL).all() and (ob[:, 16 + H * D:] == SENTINEL).all()


def test_prefill_in_a_graph(kqctx):
    """a captured prompt call replayed with other row ranges and lengths: whole items, then items that are split"""
    import torch
    rng = np.random.default_rng(17)
    D, H, K, M, stride = 128, 4, 2, 200, 300
    ctx, stream = kq.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        lens = [4600, 500]
        p = R.Paged(rng, lens, K, 16, D, stride=stride)
        q = rng.standard_normal((M, H, D)).astype(np.float16)
        out = dev(np.zeros_like(q))
        start, n = dev(np.zeros(3, np.int32)), dev(np.zeros(2, np.int32))
        a = kq.Attention(cache_of(p), dev(q), out, n, q_start=start)
        torch.cuda.synchronize()
        ctx.attn_prefill_async(a)                                  # sizes the scratch: nothing to do yet
        ctx.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ctx.attn_prefill_async(a)
        for s, b in (([0, 100, 200], [100, 300]), ([0, 7, 9], [4600, 500]), ([0, 0, 150], [0, 500]), ([5, 60, 60], [4100, 0])):
            out.fill_(SENTINEL)
            start.copy_(dev(np.array(s, np.int32)))
            n.copy_(dev(np.array(b, np.int32)))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
                g.replay()
            ctx.synchronize()
            rows = [(s[i] + j, i, b[i] - (s[i + 1] - s[i]) + j, b[i]) for i in range(2) for j in range(s[i + 1] - s[i])]
            got = out.cpu().numpy()
            rest = np.setdiff1d(np.arange(M), [r[0] for r in rows])
            assert (got[rest] == SENTINEL).all()
            pick = rows[:: max(1, len(rows) // 20)]
            want, tol = R.expect(p, q, pick, 0, 0)
            close(got[[r[0] for r in pick]], want, tol, (s, b))
        del g
    finally:
        torch.cuda.synchronize()
        ctx.close()


def test_capture_between_a_timeout_and_the_next_call(kqctx):
    """a graph captured after a call that stopped early has only recorded the clearing of the arrival counts: an
    eager call before its first replay clears them itself, and the replay is right too"""
    import torch
    rng = np.random.default_rng(18)
    D, H, K, n, new = 128, 8, 2, 6000, 20
    ctx, stream = kq.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        p = R.Paged(rng, [n], K, 16, D)
        q = rng.standard_normal((new, H, D)).astype(np.float16)
        out = dev(np.zeros_like(q))
        a = kq.Attention(cache_of(p), dev(q), out, dev(np.array([n], np.int32)), q_start=dev(np.array([0, new], np.int32)))
        torch.cuda.synchronize()
        ctx.set_option("timeout_ms", 20)
        ctx.set_option("inject_timeout", 1)
        ctx.attn_prefill_async(a)
        with pytest.raises(kq.KQError) as e:
            ctx.synchronize()
        assert e.value.status == -7
        ctx.set_option("inject_timeout", 0)
        ctx.set_option("timeout_ms", 1000)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ctx.attn_prefill_async(a)
        want, tol = R.expect(p, q, [(i, 0, n - new + i, n) for i in range(new)], 0, 0)
        for call in (lambda: ctx.attn_prefill_async(a), g.replay, g.replay):
            out.fill_(SENTINEL)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                call()
            ctx.synchronize()
            close(out.cpu().numpy(), want, tol)
        del g, call
    finally:
        torch.cuda.synchronize()
        ctx.close()


@pytest.mark.parametrize("D, G, K, lens, page", [
    (128, 16, 1, [14368], 32), (128, 16, 1, [70001, 9], 64), (256, 8, 1, [30011], 16), (256, 16, 1, [25000], 64), (64, 16, 1, [50007], 64),
    (64, 1, 1, [90001], 64), (128, 12, 2, [33333], 128), (256, 2, 1, [61000], 256),
])
def test_decode_few_items_of_many_parts(kqctx, D, G, K, lens, page):
    """so few items that nearly every CTA has a part of one: parts joined in two steps, the same way every time"""
    import torch
    rng = np.random.default_rng(D + G)
    p = R.Paged(rng, lens, K, page, D)
    q = rng.standard_normal((len(lens), G * K, D)).astype(np.float16)
    out = dev(np.zeros_like(q))
    a = kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32)))
    kqctx.attn_decode_async(a)
    kqctx.synchronize()
    first = out.cpu().numpy()
    want, tol = R.expect(p, q, [(s, s, n - 1, n) for s, n in enumerate(lens)], 0, 0)
    close(first, want, tol)
    for _ in range(4):
        out.fill_(SENTINEL)
        torch.cuda.synchronize()
        kqctx.attn_decode_async(a)
        kqctx.synchronize()
        assert (out.cpu().numpy() == first).all()


@pytest.mark.parametrize("D, H, K, seqs, window", [
    (128, 4, 1, [(60, 20000)], 0), (64, 16, 1, [(16, 26000)], 0), (256, 8, 1, [(32, 9000)], 0), (128, 16, 2, [(5, 21000), (30, 12000)], 0),
    (128, 4, 1, [(64, 40001)], 30000),
])
def test_prefill_many_parts(kqctx, D, H, K, seqs, window):
    """few rows over long caches: items in so many parts that they are joined in two steps, the same way every time"""
    import torch
    rng = np.random.default_rng(D + H)
    lens = [n for _, n in seqs]
    p = R.Paged(rng, lens, K, 64, D)
    starts = np.cumsum([0] + [r for r, _ in seqs]).astype(np.int32)
    q = rng.standard_normal((starts[-1], H, D)).astype(np.float16)
    out = dev(np.zeros_like(q))
    a = kq.Attention(cache_of(p), dev(q), out, dev(np.array(lens, np.int32)), q_start=dev(starts), window=window)
    kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    first = out.cpu().numpy()
    rows = [(int(starts[s]) + i, s, n - r + i, n) for s, (r, n) in enumerate(seqs) for i in range(r)]
    pick = rows[:: max(1, len(rows) // 12)]
    want, tol = R.expect(p, q, pick, window, 0)
    close(first[[r[0] for r in pick]], want, tol)
    for _ in range(4):
        out.fill_(SENTINEL)
        torch.cuda.synchronize()
        kqctx.attn_prefill_async(a)
        kqctx.synchronize()
        assert (out.cpu().numpy() == first).all()


@pytest.mark.parametrize("prefill", [False, True])
def test_special_values_in_many_parts(kqctx, prefill):
    """items joined in two steps: a missing page is masked and reported, -inf scores weigh nothing, a NaN score
    and an infinite value reach the rows that see them"""
    rng = np.random.default_rng(19)
    D, G, n, new, page = 128, 16, 30000, 10 if prefill else 1, 64
    for what in ("page", "-inf", "all -inf", "nan", "inf"):
        p = R.Paged(rng, [n], 1, page, D)
        q = np.abs(rng.standard_normal((new, G, D))).astype(np.float16)
        keep = np.arange(n)
        if what == "page":
            p.table[0, 201] = p.k.shape[0] + 5
            keep = np.r_[0:201 * page, 202 * page:n]
        elif what == "-inf":                              # a whole part's scores, and more
            for i in range(100, 140):
                p.k[p.table[0, i], 0] = -np.inf
            keep = np.r_[0:100 * page, 140 * page:n]
        elif what == "all -inf":
            p.k[:] = -np.inf
        elif what == "nan":
            p.k[p.table[0, 77], 0, 5, 9] = np.nan
        else:
            p.v[p.table[0, 300], 0, 5, 9] = np.inf
        p.keys[0], p.values[0] = p.keys[0][keep], p.values[0][keep]
        out = dev(np.full_like(q, SENTINEL))
        kv_len, start = dev(np.array([n], np.int32)), dev(np.array([0, new], np.int32))
        if prefill:
            kqctx.attn_prefill_async(kq.Attention(cache_of(p), dev(q), out, kv_len, q_start=start))
        else:
            kqctx.attn_decode_async(kq.Attention(cache_of(p), dev(q), out, kv_len))
        if what == "page":
            with pytest.raises(kq.KQError) as e:
                kqctx.synchronize()
            assert e.value.status == SHAPE
        else:
            kqctx.synchronize()
        got = out.cpu().numpy()
        if what in ("nan", "all -inf"):
            assert np.isnan(got).all()
            continue
        m = len(keep)
        want, tol = R.expect(p, q, [(i, 0, m - new + i, m) for i in range(new)], 0, 0)
        cols = np.arange(D)
        if what == "inf":
            assert np.isinf(got[..., 9]).all()
            cols = np.delete(cols, 9)
        close(got[..., cols], want[..., cols], tol[..., cols], what)

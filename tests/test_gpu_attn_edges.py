"""Calls of the attention operators that their documentation allows and that are easy to get wrong, on the GPU,
against the plain 64-bit forms (attn_ref)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import attn_ref as R
import npu880_mtk_npu_llm_runtime_b200 as kq
from npu880_mtk_npu_llm_runtime_b200 import synth
from test_gpu_attn import SENTINEL, SHAPE, cache_of, close, dev
from test_gpu_attn_block import HIDDEN, Block

pytestmark = pytest.mark.gpu


def i32(*v):
    return dev(np.array(v, np.int32))


@pytest.mark.parametrize("D, H, starts", [(64, 16, "alternating"), (128, 2, "falling"), (256, 16, "alternating")])
def test_prefill_row_ranges_that_overlap(kqctx, D, H, starts):
    """q_start that falls and rises again: a range in front of an earlier one's end has no rows and is reported,
    the first sequence's rows are computed, nothing outside the tables is touched"""
    rng = np.random.default_rng(D)
    n, S, M = 40, 4096, 4096
    if starts == "falling":
        S, M = 3, 30
    p = R.Paged(rng, [n], 1, 16, D)
    p.table = np.repeat(p.table, S, 0)                    # every sequence has the same pages
    q = rng.standard_normal((M, H, D)).astype(np.float16)
    start = [0, 20, 10, 30] if starts == "falling" else [0, M] * (S // 2) + [0]
    out = dev(np.full_like(q, SENTINEL))
    a = kq.Attention(cache_of(p), dev(q), out, dev(np.full(S, n, np.int32)), q_start=i32(*start))
    kqctx.attn_prefill_async(a)
    with pytest.raises(kq.KQError) as e:
        kqctx.synchronize()
    assert e.value.status == SHAPE
    got, rows = out.cpu().numpy(), start[1]
    seeing = [(r, 0, n - rows + r, n) for r in range(max(0, rows - n), rows)]
    want, tol = R.expect(p, q, seeing, 0, 0)
    close(got[[r[0] for r in seeing]], want, tol)
    assert (got[:max(0, rows - n)] == 0).all()            # rows in front of the first key
    assert (got[rows:] == SENTINEL).all()
    a = kq.Attention(a.cache, dev(q), out, a.keep[2], q_start=dev(np.r_[0, np.full(S, rows)].astype(np.int32)))
    kqctx.attn_prefill_async(a)
    kqctx.synchronize()                                   # the context stays usable
    assert (out.cpu().numpy() == got).all()


@pytest.mark.parametrize("D, G, scale, terms", [(64, 2, 0.0, 64), (128, 4, 0.0, 128), (256, 2, 0.0, 256), (128, 4, 0.0, 1), (128, 16, 1e24, 1), (64, 1, 1e24, 64)])
@pytest.mark.parametrize("seqs", [[(70, 70), (3, 200)], [(300, 300)], [(9, 9000)]])
def test_very_large_scores(kqctx, D, G, scale, terms, seqs):
    """scores of up to 2^32 and more whose maxima stand far above the rest: the weights are 1 and 0, so the result is
    the value of the key with the largest score.  (Equal products make a score: fp32's roundings are far below the
    steps between scores.)  The weight of the maximum need not be a power of two (the reference m may be a little off it) and so has a rounding to fp16 that
    the sum of the weights has not, and the result has one: half a step each, and a few of fp32's."""
    rng = np.random.default_rng(D + G)
    lens = [n for _, n in seqs]
    p = R.Paged(rng, lens, 1, 16, D)
    starts = np.cumsum([0] + [r for r, _ in seqs]).astype(np.int32)
    q = np.zeros((starts[-1], G, D), np.float16)
    q[:, :, :terms] = rng.choice([-60000, -3000, 3000, 60000], q.shape[:2])[..., None]
    for s, n in enumerate(lens):
        p.keys[s][:] = 0
        p.keys[s][:, 0, :terms] = (rng.permutation(n) * (8 if n > 4000 else 32) - 32 * (n // 8))[:, None]
        for j in range(n):
            p.k[p.table[s, j // 16], :, j % 16] = p.keys[s][j]
    assert len(np.unique(p.keys[0][:, 0, 0])) == lens[0] or lens[0] > 4000
    kv_len = dev(np.array(lens, np.int32))
    o1, o2 = dev(np.full_like(q, SENTINEL)), dev(np.full_like(q[:len(lens)], SENTINEL))
    cache = cache_of(p)
    prompt = kq.Attention(cache, dev(q), o1, kv_len, q_start=dev(starts), scale=scale)   # (lives until they ended)
    token = kq.Attention(cache, dev(q[starts[1:] - 1]), o2, kv_len, scale=scale)
    kqctx.attn_prefill_async(prompt)
    kqctx.attn_decode_async(token)
    kqctx.synchronize()
    got, last = o1.cpu().numpy(), o2.cpu().numpy()
    checked = 0

    def close_to(x, v):
        v = v.astype(np.float64)
        return (np.abs(x.astype(np.float64) - v) <= np.abs(v) * (2 * R.HALF16 + 16 * R.U32) + R.TINY16).all()

    for s, (r, n) in enumerate(seqs):
        for i in range(r):
            e = p.keys[s][:n - r + i + 1, 0, 0].astype(np.float64)
            for g in range(G):
                score = e * float(q[starts[s] + i, g, 0])
                at = np.flatnonzero(score == score.max())
                if len(at) > 1:                           # (fp16 holds no 9,000 such numbers: a tie tells nothing)
                    continue
                checked += 1
                assert close_to(got[starts[s] + i, g], p.values[s][at[0], 0]), (s, i, g)
                if i == r - 1:
                    assert close_to(last[s, g], p.values[s][at[0], 0]), (s, g)
    assert checked > 4


@pytest.mark.parametrize("D, G", [(64, 2), (128, 4), (256, 1), (128, 16)])
@pytest.mark.parametrize("seqs", [[(90, 90), (2, 300)], [(300, 300)], [(9, 9000)]])
def test_means_of_the_largest_values(kqctx, D, G, seqs):
    """a weighted mean of 65504s is 65504: not an infinity, although every weight but one is rounded up by most of
    half a step (they are 0.5 (1 + 1.2 2^-11) of the largest)"""
    rng = np.random.default_rng(D + G)
    lens = [n for _, n in seqs]
    p = R.Paged(rng, lens, 1, 32, D)
    starts = np.cumsum([0] + [r for r, _ in seqs]).astype(np.int32)
    score = np.log(0.5 * (1 + 1.2 * 2.0 ** -11))
    coarse = np.float16(score)
    fine = np.float16((score - float(coarse)) * 1024)
    q = np.zeros((starts[-1], G, D), np.float16)
    q[:, :, 0], q[:, :, 1] = 1, 2.0 ** -10
    for s, n in enumerate(lens):
        p.keys[s][:] = 0
        p.keys[s][1:, 0, 0], p.keys[s][1:, 0, 1] = coarse, fine
        p.values[s][:, :, ::2], p.values[s][:, :, 1::2] = 65504, -65504
        for j in range(n):
            p.k[p.table[s, j // 32], :, j % 32] = p.keys[s][j]
            p.v[p.table[s, j // 32], :, j % 32] = p.values[s][j]
    cache, kv_len = cache_of(p), dev(np.array(lens, np.int32))
    o1, o2 = dev(np.full_like(q, SENTINEL)), dev(np.full_like(q[:len(lens)], SENTINEL))
    prompt = kq.Attention(cache, dev(q), o1, kv_len, q_start=dev(starts), scale=1.0)
    token = kq.Attention(cache, dev(q[starts[1:] - 1]), o2, kv_len, scale=1.0)
    kqctx.attn_prefill_async(prompt)
    kqctx.attn_decode_async(token)
    kqctx.synchronize()
    rows = [(starts[s] + i, s, n - r + i, n) for s, (r, n) in enumerate(seqs) for i in {0, r // 2, r - 1}]
    want, tol = R.expect(p, q, rows, 0, 0, scale=1.0)
    close(o1.cpu().numpy()[[r[0] for r in rows]], want, tol)
    want, tol = R.expect(p, q, [(starts[s + 1] - 1, s, n - 1, n) for s, n in enumerate(lens)], 0, 0, scale=1.0)
    close(o2.cpu().numpy(), want, tol)


@pytest.mark.parametrize("D, G", [(64, 2), (128, 4), (256, 1), (128, 16)])
@pytest.mark.parametrize("n, new", [(40, 40), (300, 3), (9000, 9)])
@pytest.mark.parametrize("gap", [30, 45, 140, 300, 900])
def test_infinite_values_under_vanishing_weights(kqctx, D, G, n, new, gap):
    """a weight of 2^-gap of the largest is no zero: an infinite value under it is infinite, before the largest
    score and behind it, one of each sign is NaN; under a score of -inf it is NaN, as 0 times infinity"""
    rng = np.random.default_rng(D + G + n)
    p = R.Paged(rng, [n], 1, 16, D)
    q = np.zeros((new, G, D), np.float16)
    q[:, :, 0] = 1
    top = min(n - new, n // 2)                             # every row sees the largest score (row 0 of a prompt: only that)
    places = [(0, 1, np.inf), (min(top + 1, n - 1), 2, -np.inf), (n - 1, 3, np.inf), (0, 4, np.inf), (n - 1, 4, -np.inf)]
    p.keys[0][:, 0] = 0
    p.keys[0][:, 0, 0] = -gap * np.log(2)
    p.keys[0][top, 0, 0] = 0
    zero = n // 3 if n // 3 not in (0, top, top + 1, n - 1) else n // 3 + 2
    p.keys[0][zero, 0, 0] = -np.inf
    p.values[0][zero, 0, 5] = np.inf
    for j, d, x in places:
        p.values[0][j, 0, d] = x
    for j in range(n):
        p.k[p.table[0, j // 16], :, j % 16] = p.keys[0][j]
        p.v[p.table[0, j // 16], :, j % 16] = p.values[0][j]
    cache, kv_len = cache_of(p), i32(n)
    o1, o2 = dev(np.full_like(q, SENTINEL)), dev(np.full_like(q[:1], SENTINEL))
    prompt = kq.Attention(cache, dev(q), o1, kv_len, q_start=i32(0, new), scale=1.0)
    token = kq.Attention(cache, dev(q[:1]), o2, kv_len, scale=1.0)
    kqctx.attn_prefill_async(prompt)
    kqctx.attn_decode_async(token)
    kqctx.synchronize()
    for got, i in [(o1.cpu().numpy()[i], i) for i in sorted({0, new // 2, new - 1})] + [(o2.cpu().numpy()[0], new - 1)]:
        seen = n - new + i + 1
        e = p.keys[0][:seen, 0, 0].astype(np.float64)
        with np.errstate(invalid="ignore"):
            w = np.exp(e - e.max())
            want = (w[:, None] * p.values[0][:seen, 0].astype(np.float64)).sum(0) / w.sum()
        odd = ~np.isfinite(want)
        assert odd[1] and (i < new - 1 or odd[[1, 2, 3, 4, 5]].all())
        for g in range(G):
            assert np.array_equal(got[g][odd].astype(np.float64), want[odd], equal_nan=True), (i, got[g][:6], want[:6])
            # the rest: bounded as any row's, the weights' 16 bits and the few below them (2^-29 of the largest)
            W = (w[:, None] * np.abs(p.values[0][:seen, 0][:, ~odd].astype(np.float64))).sum(0) / w.sum()
            off = np.abs(got[g][~odd].astype(np.float64) - want[~odd])
            assert (off <= R.HALF16 * (np.abs(want[~odd]) + W) + 2 * R.U32 * (seen + 64) * W + seen * 2.0 ** -29 * 8 + R.TINY16).all()


@pytest.mark.parametrize("prefill", [True, False])
def test_many_small_weights(kqctx, prefill):
    """a million keys of weight 2^-30.3 behind the first: each weight is off by half a step of fp16 or 2^-32 of the
    largest (decode: 2^-40), and so is the mean of values of one size, times their number.  As many sequences as
    SMs, on the same two pages, so that no item is split and its largest weight is everywhere the same."""
    import torch
    D, n, S, page = 64, 1 << 20, torch.cuda.get_device_properties(0).multi_processor_count, 256
    table = np.zeros((S, n // page), np.int32)
    table[:, 0] = 1
    k, v = np.zeros((2, 1, page, D), np.float16), np.ones((2, 1, page, D), np.float16)
    k[:, :, :, 0] = -30.3 * np.log(2)
    k[1, 0, 0] = 0
    v[1, 0, 0] = 0
    cache = kq.KvCache(dev(k), dev(v), dev(table))
    q = np.zeros((S, 1, D), np.float16)
    q[:, :, 0] = 1
    out = dev(np.full_like(q, SENTINEL))
    a = kq.Attention(cache, dev(q), out, dev(np.full(S, n, np.int32)), q_start=dev(np.arange(S + 1, dtype=np.int32)) if prefill else None,
                     scale=1.0)
    (kqctx.attn_prefill_async if prefill else kqctx.attn_decode_async)(a)
    kqctx.synchronize()
    w = np.exp(float(k[0, 0, 0, 0])) * (n - 1)
    want = w / (1 + w)
    # fp32: the score's product and the exponential (8 half steps), sums of n / 16 terms that grow evenly
    tol = want * (2 * R.HALF16 + U32_SUM) + n * 2.0 ** (-32 if prefill else -40)
    off = np.abs(out.cpu().numpy().astype(np.float64) - want)
    assert off.max() <= tol, (off.max(), tol, want)


U32_SUM = (8 + (1 << 16)) * 2 * R.U32                      # a rounding (a step) for every 16 of the million keys


def test_one_long_sequence_among_many_short_ones(kqctx):
    """hundreds of one-token sequences and one of 131,072 keys: the long one's keys are spread over the GPU, so that
    the batch takes no longer than its parts apart (a CTA that took a whole head of it took 11 times as long)"""
    import torch
    rng = np.random.default_rng(21)
    D, H, K, page, long, short = 128, 32, 8, 64, 131072, 100
    lens = [long] + [short] * 600
    need = [-(-n // page) for n in lens]
    table = np.zeros((len(lens), max(need)), np.int32)
    at = np.cumsum([0] + need)
    for s, n in enumerate(need):
        table[s, :n] = np.arange(at[s], at[s] + n)
    k, v = (torch.empty((at[-1], K, page, D), dtype=torch.float16, device="cuda").normal_() for _ in range(2))
    q = dev(rng.standard_normal((len(lens), H, D)).astype(np.float16))
    out = torch.full_like(q, SENTINEL)

    def call(pick):
        a = kq.Attention(kq.KvCache(k, v, dev(table[pick])), q[pick[0]:pick[-1] + 1], out[pick[0]:pick[-1] + 1],
                         dev(np.array(lens, np.int32)[pick]), q_start=dev(np.arange(len(pick) + 1, dtype=np.int32)))
        torch.cuda.synchronize()
        best, stream = 1e9, torch.cuda.ExternalStream(kqctx.stream)
        for _ in range(5):
            e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            e[0].record(stream)
            for _ in range(4):
                kqctx.attn_prefill_async(a)
            e[1].record(stream)
            kqctx.synchronize()
            best = min(best, e[0].elapsed_time(e[1]))
        return best

    alone = call(np.arange(1)) + call(np.arange(1, len(lens)))
    together = call(np.arange(len(lens)))
    assert together < 3 * alone, (together, alone)
    got = out.cpu().numpy()
    p = R.Paged(rng, [0] * len(lens), K, page, D)
    rows = [0, 1, 77, 600]
    for s in rows:
        t = table[s, :need[s]]
        p.keys[s], p.values[s] = (x[torch.from_numpy(t).long().cuda()].permute(0, 2, 1, 3).reshape(-1, K, D)[:lens[s]].cpu().numpy() for x in (k, v))
    want, tol = R.expect(p, q.cpu().numpy(), [(s, s, lens[s] - 1, lens[s]) for s in rows], 0, 0)
    close(got[rows], want, tol)


@pytest.mark.parametrize("D, H, K, n, new", [(128, 8, 2, 20000, 20), (64, 16, 1, 26000, 16), (256, 4, 1, 9000, 9)])
def test_counts_left_behind_by_a_call_that_stopped_early(kqctx, D, H, K, n, new):
    """every other CTA stops early, so the rest have counted arrivals at shared items that never get complete: the
    next call clears them, of either kind, and so does one after a capture that only recorded the clearing"""
    import torch
    rng = np.random.default_rng(D)
    ctx, stream = kq.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    p = R.Paged(rng, [n], K, 64, D)
    q = rng.standard_normal((new, H, D)).astype(np.float16)
    out, o1, cache, kv_len = dev(np.zeros_like(q)), dev(np.zeros_like(q[:1])), cache_of(p), i32(n)
    prompt = kq.Attention(cache, dev(q), out, kv_len, q_start=i32(0, new))
    token = kq.Attention(cache, dev(q[-1:]), o1, kv_len)
    want, tol = R.expect(p, q, [(i, 0, n - new + i, n) for i in range(new)], 0, 0)
    other = dev((2 * p.v.astype(np.float32)).astype(np.float16))      # parts of other values lie in the scratch
    before = kq.Attention(kq.KvCache(cache.k, other, cache.page_table), prompt.keep[0], out, kv_len, q_start=prompt.keep[3])

    def stop():
        ctx.attn_prefill_async(before)
        ctx.set_option("timeout_ms", 20)
        ctx.set_option("inject_timeout", 2)
        ctx.attn_prefill_async(prompt)
        with pytest.raises(kq.KQError) as e:
            ctx.synchronize()
        assert e.value.status == -7
        ctx.set_option("inject_timeout", 0)
        ctx.set_option("timeout_ms", 1000)

    def check(call, prefill=True):
        for t in (out, o1):
            t.fill_(SENTINEL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            call()
        ctx.synchronize()
        if prefill:
            close(out.cpu().numpy(), want, tol)
        else:
            close(o1.cpu().numpy(), want[-1:], tol[-1:])

    torch.cuda.synchronize()
    try:
        ctx.attn_prefill_async(prompt)
        stop()
        for _ in range(2):
            check(lambda: ctx.attn_prefill_async(prompt))
        stop()
        for _ in range(2):
            check(lambda: ctx.attn_decode_async(token), prefill=False)
        check(lambda: ctx.attn_prefill_async(prompt))
        stop()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            ctx.attn_prefill_async(prompt)
        for call in (lambda: ctx.attn_prefill_async(prompt), g.replay, g.replay):
            check(call)
        del g, call
        with pytest.raises(kq.KQError):
            ctx.set_option("inject_timeout", 3)
    finally:
        torch.cuda.synchronize()
        ctx.close()


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_block_refused_for_want_of_scratch_has_done_nothing(kqctx, prefill):
    """the block's first call of a context in a capture, where an FFN block has left all scratch but attention's: it is
    refused, and what the graph holds writes neither the cache nor the output"""
    import torch
    ctx, stream = kq.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    ctx.set_option("gemv_split", 0)
    b, ffn = Block(ctx, (12, 14, 12, 12)), 2048
    x = torch.randn((3, HIDDEN), device="cuda").half()
    out = torch.full_like(x, SENTINEL)
    w = [ctx.upload(synth.gen_weights(12, r, c, 50 + i), 12, r, c) for i, (r, c) in enumerate([(ffn, HIDDEN)] * 2 + [(HIDDEN, ffn)])]
    seq, pos, lens, start = i32(0, 1, 2), i32(4, 5, 6), i32(5, 6, 7), i32(0, 1, 2, 3)
    ctx.run_ffn_async(*w, 3, x, b.dg[0], torch.empty_like(x))
    ctx.synchronize()
    b.ck.fill_(SENTINEL)
    b.cv.fill_(SENTINEL)
    torch.cuda.synchronize()
    try:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            with pytest.raises(kq.KQError):
                ctx.run_attn_async(b.layer, seq, pos, lens, x, out, q_start=start if prefill else None)
        with torch.cuda.stream(stream):
            g.replay()
        ctx.synchronize()
        assert (b.ck == SENTINEL).all() and (b.cv == SENTINEL).all() and (out == SENTINEL).all()
        del g
        ctx.run_attn_async(b.layer, seq, pos, lens, x, out, q_start=start if prefill else None)   # eagerly it runs
        ctx.synchronize()
        want, _ = b.steps(ctx, seq, pos, lens, x, start if prefill else None)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        g = torch.cuda.CUDAGraph()                          # and then in a graph
        with torch.cuda.graph(g, stream=stream):
            ctx.run_attn_async(b.layer, seq, pos, lens, x, out, q_start=start if prefill else None)
        out.fill_(SENTINEL)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        ctx.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        del g
    finally:
        torch.cuda.synchronize()
        b.free()
        for t in w:
            t.free()
        ctx.close()


@pytest.mark.parametrize("D, pad", [(64, 0), (128, 8), (256, 16)])
def test_rows_stored_twice(kqctx, D, pad):
    """rows that are computed again (an infinity in one of every row's values, and rows that see nothing) are stored
    over their plain results by other threads: the second result is the one that stays, every time"""
    import torch
    rng = np.random.default_rng(D + pad)
    n, H = 200, 4
    p = R.Paged(rng, [n, 5], 2, 16, D)
    p.values[0][0, :, 7] = np.inf
    p.v[p.table[0, 0], :, 0, 7] = np.inf
    rows = n + 40                                          # sequence 1: 35 rows in front of its first key
    q = rng.standard_normal((rows, H, D)).astype(np.float16)
    buf = torch.full((rows, H * D + pad), SENTINEL, dtype=torch.float16, device="cuda")
    out = buf[:, :H * D]
    a = kq.Attention(cache_of(p), dev(q.reshape(rows, -1)), out, i32(n, 5), q_start=i32(0, n, rows), heads=H)
    torch.cuda.synchronize()
    kqctx.attn_prefill_async(a)
    kqctx.synchronize()
    first = out.cpu().numpy()
    got, keep = first.reshape(rows, H, D), np.delete(np.arange(D), 7)
    p.values[0][0, :, 7] = 0
    want, tol = R.expect(p, q, [(i, 0, i, n) for i in range(n)] + [(n + i, 1, i - 35, 5) for i in range(40)], 0, 0)
    close(got[..., keep], want[..., keep], tol[..., keep])
    assert np.isposinf(got[:n, :, 7]).all() and (got[n:n + 35] == 0).all()
    for _ in range(30):
        buf.fill_(SENTINEL)
        torch.cuda.synchronize()
        kqctx.attn_prefill_async(a)
        kqctx.synchronize()
        assert np.array_equal(out.cpu().numpy().view(np.uint16), first.view(np.uint16))


def test_outputs_that_lie_over_inputs_are_refused(kqctx):
    import torch
    D, H, K, M = 64, 4, 2, 6
    rng = np.random.default_rng(3)
    p = R.Paged(rng, [5] * M, K, 16, D)
    cache = cache_of(p)
    rows = torch.randn((M + 1, (H + 2 * K) * D), device="cuda").half()
    q, k, v = rows[:M, :H * D], rows[:M, H * D:(H + K) * D], rows[:M, (H + K) * D:]
    free = torch.empty((M, H * D), dtype=torch.float16, device="cuda")
    lens, seq, pos, rope = i32(*[5] * M), i32(*range(M)), i32(*[4] * M), kq.Rope(D)
    pages = cache.k.view(-1)
    over_cache = pages[:M * H * D].view(M, H * D)
    for out in (rows[1:, :H * D], rows[:M, 8:H * D + 8], over_cache):
        with pytest.raises(kq.KQError):
            kqctx.attn_decode_async(kq.Attention(cache, q, out, lens))
        with pytest.raises(kq.KQError):
            kqctx.kv_append_async(cache, rope, seq, pos, kq.Heads(k, K), kq.Heads(v, K), q=kq.Heads(q, H, out=out))
    for bad_q in (kq.Heads(q, H, out=rows[:M, K * D:(H + K) * D]), kq.Heads(q, H, out=free)):
        with pytest.raises(kq.KQError):
            kqctx.qk_norm_rope_async(rope, pos, bad_q, kq.Heads(k, K, out=free[:, :K * D]))
    with pytest.raises(kq.KQError):
        kqctx.kv_append_async(kq.KvCache(cache.k, cache.k, cache.page_table), rope, seq, pos, kq.Heads(k, K), kq.Heads(v, K))
    kqctx.synchronize()
    # in place and between the other rows of the buffer it runs: out over k and v once they are in the cache
    kqctx.kv_append_async(cache, rope, seq, pos, kq.Heads(k, K), kq.Heads(v, K), q=kq.Heads(q, H, out=q))
    kqctx.synchronize()
    hq = q.cpu().numpy().reshape(M, H, D)
    a = kq.Attention(cache, q, rows[:M, H * D:], lens)
    kqctx.attn_decode_async(a)
    kqctx.synchronize()
    at = p.table[np.arange(M), 0]
    for s in range(M):
        p.keys[s], p.values[s] = (t.cpu().numpy()[at[s], :, :5].transpose(1, 0, 2) for t in (cache.k, cache.v))
    want, tol = R.expect(p, hq, [(s, s, 4, 5) for s in range(M)], 0, 0)
    close(rows[:M, H * D:].cpu().numpy().reshape(M, H, D), want, tol)


def test_numbers_that_do_not_fit_are_refused(kqctx):
    """2^32 as a window is not 0, nor 1e-50 as a scale the default"""
    import torch
    cache = cache_of(R.Paged(np.random.default_rng(0), [5, 5], 2, 16, 64))
    q = torch.zeros((2, 256), dtype=torch.float16, device="cuda")
    lens = i32(5, 5)
    for bad in (dict(window=2 ** 32), dict(window=2 ** 31), dict(window=4, sinks=2 ** 32), dict(scale=1e-50)):
        with pytest.raises(ValueError):
            kq.Attention(cache, q, torch.empty_like(q), lens, **bad)
    b = Block(kqctx)
    for bad in (dict(window=2 ** 32), dict(window=4, sinks=-2 ** 32 - 1), dict(scale=-1e-50)):
        with pytest.raises(ValueError):
            kq.AttnLayer(*b.w, b.dg[0], b.cache, **bad)
    with pytest.raises(ValueError):                          # (rows that a stride of 0 makes)
        kq.Heads(q[:1].expand(2 ** 32, 256), 2)
    a = kq.Attention(cache, q, torch.empty_like(q), lens, window=2 ** 31 - 1, sinks=2 ** 31 - 1, scale=1e-40)
    kqctx.attn_decode_async(a)
    kqctx.synchronize()
    b.free()


@pytest.mark.parametrize("what", ["products", "attention"])
def test_clearing_that_a_capture_only_records(kqctx, what):
    """after a call that stopped early every capture clears the arrival counts, until an eager call has done so"""
    import torch
    ctx, stream = kq.Context(0), torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    rows, K, n = 300, 4096, 300
    w = ctx.upload(synth.gen_weights(12, rows, K, seed=5), 12, rows, K)
    x, y = torch.randn((2, K), device="cuda").half(), torch.zeros((2, rows), dtype=torch.float16, device="cuda")
    p = R.Paged(np.random.default_rng(1), [n], 2, 16, 128)
    q = torch.randn((n, 4 * 128), device="cuda").half()
    a = kq.Attention(cache_of(p), q, torch.empty_like(q), i32(n), q_start=i32(0, n))

    def call():
        if what == "products":
            ctx.gemm_multi_async(x, 2, K, [dict(w=w, dst=y)])
        else:
            ctx.attn_prefill_async(a)

    def clears():
        """whether a capture of the call holds a memset"""
        g = torch.cuda.CUDAGraph(keep_graph=True)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            call()
        graph, n, cu = C.c_void_p(g.raw_cuda_graph()), C.c_size_t(), C.CDLL("libcuda.so.1")
        assert cu.cuGraphGetNodes(graph, None, C.byref(n)) == 0 and n.value > 0
        nodes, kind = (C.c_void_p * n.value)(), C.c_int()
        assert cu.cuGraphGetNodes(graph, nodes, C.byref(n)) == 0
        kinds = []
        for node in nodes:
            assert cu.cuGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
            kinds.append(kind.value)
        return 2 in kinds                                  # CU_GRAPH_NODE_TYPE_MEMSET

    try:
        torch.cuda.synchronize()
        call()
        ctx.synchronize()
        assert not clears()
        ctx.set_option("timeout_ms", 20)
        ctx.set_option("inject_timeout", 1)
        call()
        with pytest.raises(kq.KQError) as e:
            ctx.synchronize()
        assert e.value.status == -7
        ctx.set_option("inject_timeout", 0)
        ctx.set_option("timeout_ms", 1000)
        assert clears() and clears()
        call()
        ctx.synchronize()
        assert not clears()
    finally:
        torch.cuda.synchronize()
        w.free()
        ctx.close()

"""The attention block of a layer (kq_run_attn_async): bit for bit the calls it stands for, on prompts,
single tokens and captured graphs, and against the oracle's products and the formulas."""
from __future__ import annotations

import numpy as np
import pytest

import attn_ref as R
import npu880_mtk_npu_llm_runtime_b200 as kq
from npu880_mtk_npu_llm_runtime_b200 import synth

pytestmark = pytest.mark.gpu

HIDDEN, H, K, D, PAGE = 512, 8, 2, 64, 16


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Block:
    def __init__(self, ctx, types=(12, 14, 8, 12), n_seqs=3, stride=16, window=0, sinks=0, norms=True, seed=3):
        import torch
        self.types = types
        rows = (H * D, K * D, K * D, HIDDEN)
        cols = (HIDDEN, HIDDEN, HIDDEN, H * D)
        self.host = [synth.gen_weights(t, r, c, seed + i) for i, (t, r, c) in enumerate(zip(types, rows, cols))]
        self.w = [ctx.upload(b, t, r, c) for b, t, r, c in zip(self.host, types, rows, cols)]
        rng = np.random.default_rng(seed)
        g = [(0.1 * (1 + 0.2 * rng.standard_normal(n))).astype(np.float16) for n in (HIDDEN, D, D)]
        g[1:] = [(10 * x).astype(np.float16) for x in g[1:]]
        self.gamma = g
        self.dg = [dev(x) for x in g]
        pages = n_seqs * stride + 1
        table = rng.permutation(pages)[:n_seqs * stride].reshape(n_seqs, stride).astype(np.int32)
        self.ck = torch.full((pages, K, PAGE, D), float("nan"), dtype=torch.float16, device="cuda")
        self.cv = torch.full_like(self.ck, float("nan"))
        self.cache = kq.KvCache(self.ck, self.cv, dev(table))
        self.rope = kq.Rope(D, base=1e5)
        self.norms = norms
        self.window, self.sinks = window, sinks
        self.layer = kq.AttnLayer(*self.w, self.dg[0], self.cache, rope=self.rope, q_gamma=self.dg[1] if norms else None,
                                  k_gamma=self.dg[2] if norms else None, window=window, sinks=sinks)

    def steps(self, ctx, seq, pos, kv_len, x, q_start=None):
        """the calls that the block stands for"""
        import torch
        M = x.shape[0]
        f16 = dict(dtype=torch.float16, device="cuda")
        xn, qkv = torch.zeros(M, HIDDEN, **f16), torch.zeros(M, (H + 2 * K) * D, **f16)
        att, out = torch.zeros(M, H * D, **f16), torch.zeros(M, HIDDEN, **f16)
        q8 = torch.zeros(kq.q8k_bytes(M, HIDDEN), dtype=torch.uint8, device="cuda")
        q80 = torch.zeros(kq.q8_0_bytes(M, HIDDEN), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        ctx.rmsnorm_q8k_async(x, self.dg[0], xn, M, HIDDEN, q8)
        ctx.quantize_q8_0_async(xn, M, HIDDEN, q80)
        q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + K) * D], qkv[:, (H + K) * D:]
        ctx.gemm_multi_q8_async(q8, q80, M, HIDDEN, [dict(w=w, dst=t, dst_stride=qkv.shape[1]) for w, t in zip(self.w, (q, k, v))])
        gq, gk = (self.dg[1], self.dg[2]) if self.norms else (None, None)
        ctx.kv_append_async(self.cache, self.rope, seq, pos, kq.Heads(k, K, gamma=gk), kq.Heads(v, K), q=kq.Heads(q, H, gamma=gq, out=q))
        a = kq.Attention(self.cache, q, att, kv_len, q_start=q_start, window=self.window, sinks=self.sinks)
        (ctx.attn_prefill_async if q_start is not None else ctx.attn_decode_async)(a)
        ctx.gemm_multi_async(att, M, H * D, [dict(w=self.w[3], dst=out, residual=x)])
        ctx.synchronize()
        return out, att

    def free(self):
        for w in self.w:
            w.free()


@pytest.mark.parametrize("types", [(12, 14, 8, 12), (13, 13, 13, 14), (8, 8, 12, 8)])
@pytest.mark.parametrize("window, sinks, norms", [(0, 0, True), (20, 3, False)])
def test_block_equals_its_calls(kqctx, types, window, sinks, norms):
    import torch
    rng = np.random.default_rng(1)
    b = Block(kqctx, types, window=window, sinks=sinks, norms=norms)
    n = [40, 0, 77]
    start = np.cumsum([0] + n)
    M = int(start[-1]) + 2                                   # two rows of no sequence
    seq = dev(np.r_[np.repeat(np.arange(3), n), -1, -1].astype(np.int32))
    pos = dev(np.r_[np.arange(40), np.arange(77), 0, 0].astype(np.int32))
    x = dev(rng.standard_normal((M, HIDDEN)).astype(np.float16))
    out = torch.zeros_like(x)
    lens, q_start = dev(np.array(n, np.int32)), dev(start.astype(np.int32))
    torch.cuda.synchronize()
    kqctx.run_attn_async(b.layer, seq, pos, lens, x, out, q_start=q_start)
    kqctx.synchronize()
    want, _ = b.steps(kqctx, seq, pos, lens, x, q_start)
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    assert torch.equal(out[-2:], x[-2:])                     # as they went in
    for step in range(3):                                    # single tokens, one sequence not yet begun
        lens = dev(np.array([40 + step + 1, 0, 77 + step + 1], np.int32))
        seq = dev(np.array([0, -1, 2], np.int32))
        pos = dev(np.array([40 + step, 0, 77 + step], np.int32))
        x = dev(rng.standard_normal((3, HIDDEN)).astype(np.float16))
        out = torch.zeros_like(x)
        torch.cuda.synchronize()
        kqctx.run_attn_async(b.layer, seq, pos, lens, x, out)
        kqctx.synchronize()
        want, att = b.steps(kqctx, seq, pos, lens, x)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        assert torch.isfinite(out).all() and (att[1] == 0).all() and torch.equal(out[1], x[1])
    b.free()


def test_block_against_the_oracle(kqctx, oracle):
    """one prompt: the oracle's bit-exact norm and products around the attention formulas in 64 bits.  The
    attention's output enters the last product rounded, so that the product is checked on the attention
    that the device computed, and the attention against the formulas."""
    rng = np.random.default_rng(2)
    b = Block(kqctx, (12, 14, 12, 12), n_seqs=1)
    n = 60
    x = rng.standard_normal((n, HIDDEN)).astype(np.float16)
    seq, pos = dev(np.zeros(n, np.int32)), dev(np.arange(n, dtype=np.int32))
    lens, q_start = dev(np.array([n], np.int32)), dev(np.array([0, n], np.int32))
    import torch
    out = torch.zeros((n, HIDDEN), dtype=torch.float16, device="cuda")
    dx = dev(x)
    torch.cuda.synchronize()
    kqctx.run_attn_async(b.layer, seq, pos, lens, dx, out, q_start=q_start)
    kqctx.synchronize()
    _, att = b.steps(kqctx, seq, pos, lens, dx, q_start)
    att = att.cpu().numpy()
    xn, _ = oracle.rmsnorm(x, b.gamma[0])
    q, k, v = (oracle.epilogue_f16(oracle.gemm(t, w, HIDDEN, oracle.act_for(t, xn))) for t, w in zip(b.types[:3], b.host[:3]))
    f = R.bases(D, D, 1e5)
    kk, kt = R.norm_rope(k.reshape(n, K, D), b.gamma[2], f, np.arange(n), "half")
    table, ck, cv = (t.cpu().numpy() for t in (b.cache.page_table, b.ck, b.cv))
    j = np.arange(n)
    gk, gv = ck[table[0, j // PAGE], :, j % PAGE], cv[table[0, j // PAGE], :, j % PAGE]
    assert (np.abs(gk - kk) <= kt).all()
    assert np.array_equal(gv.reshape(n, -1).view(np.uint16), v.view(np.uint16))
    qq, qt = R.norm_rope(q.reshape(n, H, D), b.gamma[1], f, np.arange(n), "half")
    p = R.Paged(rng, [0], K, PAGE, D)
    p.keys[0], p.values[0] = gk, gv
    want, tol = R.expect(p, qq, [(i, 0, i, n) for i in range(n)], 0, 0, heads=H)
    for i in range(n):                                       # the queries' own rounding moves the weights
        for h in range(H):
            move = (np.abs(gk[:i + 1, h // (H // K)].astype(np.float64)) @ qt[i, h]).max() * D ** -0.5
            tol[i, h] += np.expm1(2 * move) * np.abs(gv[:i + 1, h // (H // K)].astype(np.float64)).max(0)
    assert (np.abs(att.reshape(n, H, D) - want) <= tol).all()
    ref = oracle.epilogue_f16(oracle.gemm(b.types[3], b.host[3], H * D, oracle.act_for(b.types[3], att)), x)
    assert np.array_equal(out.cpu().numpy().view(np.uint16), ref.view(np.uint16))
    b.free()


def test_block_as_one_graph(kqctx):
    """a decode step captured once and replayed with new rows, positions and lengths"""
    import torch
    rng = np.random.default_rng(7)
    ctx = kq.Context(0)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    b = Block(ctx, (12, 14, 12, 12))
    try:
        seq = dev(np.arange(3, dtype=np.int32))
        pos, lens = dev(np.zeros(3, np.int32)), dev(np.zeros(3, np.int32))
        x = torch.zeros((3, HIDDEN), dtype=torch.float16, device="cuda")
        out, g = torch.zeros_like(x), None
        for i in range(5):
            p = np.array([i, 3 * i, 40 + i], np.int32)
            x.copy_(dev(rng.standard_normal((3, HIDDEN)).astype(np.float16)))
            pos.copy_(dev(p))
            lens.copy_(dev(p + 1))
            if i == 0:                                      # every earlier position gets finite keys
                b.ck.normal_()
                b.cv.normal_()
            torch.cuda.synchronize()
            if i == 1:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=stream):
                    ctx.run_attn_async(b.layer, seq, pos, lens, x, out)
            if g is None:
                ctx.run_attn_async(b.layer, seq, pos, lens, x, out)
            else:
                with torch.cuda.stream(stream):
                    g.replay()
            ctx.synchronize()
            want, _ = b.steps(ctx, seq, pos, lens, x)
            assert torch.equal(out.view(torch.int16), want.view(torch.int16)), i
        del g
    finally:
        torch.cuda.synchronize()
        b.free()
        ctx.close()


def test_block_refusals(kqctx):
    import torch
    b = Block(kqctx)
    x = torch.zeros((3, HIDDEN), dtype=torch.float16, device="cuda")
    i3 = dev(np.zeros(3, np.int32))
    with pytest.raises(ValueError):
        kqctx.run_attn_async(b.layer, i3[:2], i3, i3, x, x)
    with pytest.raises(ValueError):
        kqctx.run_attn_async(b.layer, i3, i3, i3, x[:, :256], x)
    with pytest.raises(kq.KQError):                          # decode takes a row per sequence
        kqctx.run_attn_async(b.layer, i3[:2], i3[:2], i3, x[:2], x[:2])
    bad = kq.AttnLayer(b.w[0], b.w[2], b.w[1], b.w[0], b.dg[0], b.cache)
    with pytest.raises(kq.KQError):                          # o is not [hidden][heads * D]
        bad.struct.o = b.w[1].handle
        kqctx.run_attn_async(bad, i3, i3, i3, x, torch.empty_like(x))
    for y in (x, x.bfloat16()):                              # in place; another type
        with pytest.raises((kq.KQError, ValueError)):
            kqctx.run_attn_async(b.layer, i3, i3, i3, y, y)
    both = torch.zeros((4, HIDDEN), dtype=torch.float16, device="cuda")
    with pytest.raises(kq.KQError):                          # x_out lies over a part of x_in
        kqctx.run_attn_async(b.layer, i3, i3, i3, both[:3], both[1:])
    for field, value in (("window", -1), ("sinks", 2), ("eps", -1.0), ("gamma", None), ("heads", 7), ("cache", None), ("q", None)):
        keep = getattr(b.layer.struct, field)
        setattr(b.layer.struct, field, value)
        with pytest.raises(kq.KQError):
            kqctx.run_attn_async(b.layer, i3, i3, i3, x, torch.empty_like(x))
        setattr(b.layer.struct, field, keep)
    kqctx.synchronize()
    b.free()
    with pytest.raises(ValueError):                          # the layer's weights are gone
        kqctx.run_attn_async(b.layer, i3, i3, i3, x, torch.empty_like(x))

"""The attention operators of the library as they are measured: cases, inputs, plain forms.

Four operators stand between the q/k/v products and the o product of a decoder layer:

  norm_rope  per-head RMS norm of queries and keys and the rotary rotation, one pass
  append     keys and values of new tokens into a paged cache, keys normed and rotated on the way
             (and the queries of the same rows normed and rotated)
  decode     attention of one new token per sequence over the paged cache
  prefill    attention of ragged prompt rows over the paged cache: causal, optionally a sliding
             window with the first tokens kept visible

`run` computes an operator in elementary torch operations (own = False) or through the library's
entry points (own = True).  The cache is fp16 [pages][kv heads][page size][head dim], the table
[sequences][pages of a sequence]; activations are fp16 rows of heads side by side.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
DEV = "cuda"


# ------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoded token of one sequence, 32 query and 8 key heads of 128: pure latency
        dict(name="norm_rope_1", op="norm_rope", M=1, heads=32, kv_heads=8, D=128, rot=128, style="half", base=1e6,
             q_norm=True, k_norm=True, packed=True, far=4096),
        # the largest number of rows of a call, as in the prefill of a long prompt
        dict(name="norm_rope_4096", op="norm_rope", M=4096, heads=32, kv_heads=8, D=128, rot=128, style="half",
             base=1e6, q_norm=True, k_norm=True, packed=False, far=32768),
        # odd row count, heads of 256 of which 64 values turn, adjacent pairs, far positions, q/k/v side by side
        dict(name="norm_rope_partial_1001", op="norm_rope", M=1001, heads=16, kv_heads=4, D=256, rot=64,
             style="adjacent", base=1e7, q_norm=True, k_norm=False, packed=True, far=1000000),
        # a decode step of 64 sequences: one token each, at far positions
        dict(name="append_64_tokens", op="append", S=64, n_max=1, n_min=1, heads=32, kv_heads=8, D=128, rot=128,
             style="half", base=1e6, k_norm=True, page=16, far=32000, lens=1),
        # the rows of one 2,048-token prompt
        dict(name="append_2048_prompt", op="append", S=1, n_max=2048, n_min=2048, heads=32, kv_heads=8, D=128,
             rot=128, style="half", base=1e6, k_norm=True, page=64, far=0, lens=2),
        # one user, a short conversation: latency
        dict(name="decode_1x1000", op="decode", S=1, len_min=1000, len_max=1000, heads=32, kv_heads=8, D=128, page=16,
             window=0, sinks=0, lens=3),
        # 64 sequences of very different lengths, the batched decode
        dict(name="decode_64_ragged", op="decode", S=64, len_min=1, len_max=8192, heads=32, kv_heads=8, D=128, page=16,
             window=0, sinks=0, lens=4),
        # few sequences, very long contexts: the work is split over the length
        dict(name="decode_4x131072", op="decode", S=4, len_min=131001, len_max=131072, heads=32, kv_heads=8, D=128,
             page=64, window=0, sinks=0, lens=5),
        # many sequences that keep a window and the first tokens
        dict(name="decode_128_window", op="decode", S=128, len_min=100, len_max=32768, heads=16, kv_heads=2, D=64,
             page=32, window=1024, sinks=4, lens=6),
        # one 2,048-token prompt
        dict(name="prefill_2048", op="prefill", S=1, n_min=2048, n_max=2048, past_max=0, heads=32, kv_heads=8, D=128,
             page=64, window=0, sinks=0, lens=7),
        # a 512-token chunk at the end of a long context
        dict(name="prefill_512_at_32768", op="prefill", S=1, n_min=512, n_max=512, past_min=32256, past_max=32256,
             heads=32, kv_heads=8, D=128, page=16, window=0, sinks=0, lens=8),
        # ragged sequences with a window and first tokens, heads of 256
        dict(name="prefill_ragged_window", op="prefill", S=13, n_min=1, n_max=600, past_max=900, heads=16, kv_heads=4,
             D=256, page=32, window=512, sinks=4, lens=9),
    ]


HEADS = [(32, 8, 128), (32, 8, 128), (16, 4, 256), (16, 2, 64), (24, 8, 128), (8, 8, 64), (14, 2, 64), (16, 1, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "decode", "decode", "prefill", "prefill"])
    heads, kv_heads, D = rng.choice(HEADS)
    head = dict(heads=heads, kv_heads=kv_heads, D=D)
    turn = dict(rot=rng.choice([D, D, D // 2, D // 4]), style=rng.choice(["half", "half", "adjacent"]),
                base=rng.choice([1e4, 5e5, 1e6, 1e7]))
    lens = rng.randrange(1 << 20)
    if op == "norm_rope":
        return dict(op=op, M=_log(rng, 1, 4096), **head, **turn, q_norm=rng.random() < 0.8, k_norm=rng.random() < 0.8,
                    packed=rng.random() < 0.5, far=_log(rng, 64, 1000000))
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if op == "append":
        S = _log(rng, 1, 256)
        n_max = _log(rng, 1, max(1, 4096 // S))
        return dict(op=op, S=S, n_min=_log(rng, 1, n_max), n_max=n_max, **head, **turn, k_norm=rng.random() < 0.8,
                    page=page, far=_log(rng, 64, 200000), lens=lens)
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randrange(1, 100)]) if window else 0
    if op == "decode":
        S = _log(rng, 1, 256)
        longest = max(1, int(1.8e9 // (S * kv_heads * D * 4)))
        len_max = _log(rng, 1, min(131072, longest))
        return dict(op=op, S=S, len_min=_log(rng, 1, len_max), len_max=len_max, **head, page=page, window=window,
                    sinks=sinks, lens=lens)
    S = _log(rng, 1, 32)
    n_max = _log(rng, 1, 4096 // S)
    room = int(2.5e8 // (S * heads * n_max))  # padded scores of the plain form
    past_max = _log(rng, 1, max(1, min(32768, room - n_max)))
    return dict(op=op, S=S, n_min=_log(rng, 1, n_max), n_max=n_max, past_max=past_max, **head, page=page,
                window=window, sinks=sinks, lens=lens)


def _spread(rng, lo, hi, n):
    """n lengths between lo and hi, both ends among them where there is room"""
    v = [_log(rng, max(1, lo), max(1, hi)) for _ in range(n)]
    if n > 1:
        v[0], v[1] = max(1, hi), max(1, lo)
    elif n == 1:
        v[0] = max(1, hi)
    rng.shuffle(v)
    return v


def _lengths(case):
    """per sequence: new rows n and length with them"""
    rng = random.Random(case["lens"])
    S = case["S"]
    if case["op"] == "decode":
        return [1] * S, _spread(rng, case["len_min"], case["len_max"], S)
    n = _spread(rng, case["n_min"], case["n_max"], S)
    if case["op"] == "append":
        return n, [x + rng.randrange(case["far"] + 1) for x in n]
    lo, hi = case.get("past_min", 0), case["past_max"]
    return n, [x + (0 if hi == 0 else hi if S == 1 else rng.randrange(lo, hi + 1)) for x in n]


def _visible(case, p):
    """number of keys that position p sees"""
    w, s = case["window"], case["sinks"]
    if not w or p + 1 <= w:
        return p + 1
    return w + min(s, p + 1 - w)


def work(case):
    H, K, D = case["heads"], case["kv_heads"], case["D"]
    if case["op"] == "norm_rope":
        return {"bytes": case["M"] * ((H + K) * D * 4 + 4), "flops": case["M"] * (H + K) * D * 8}
    n, length = _lengths(case)
    if case["op"] == "append":
        rows = sum(n)
        return {"bytes": rows * ((H + 2 * K) * D * 4 + 12), "flops": rows * (H + K) * D * 8}
    pairs = keys = 0
    for a, b in zip(n, length):
        pairs += sum(_visible(case, p) for p in range(b - a, b))
        first = b - a  # the oldest new row's position: keys from its window's start on are read
        lo = max(0, first - case["window"] + 1) if case["window"] else 0
        keys += b - lo + min(case["sinks"], lo)
    rows = sum(n)
    return {"bytes": rows * H * D * 4 + keys * K * D * 4 + len(n) * 4, "flops": 4 * pairs * H * D}


# ----------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).half()


def _gamma(g, D):
    return (1.0 + 0.2 * torch.randn(D, generator=g, device=DEV)).half()


def _rows(g, M, case, packed):
    """q, k, v rows as the q/k/v products leave them: side by side in one buffer, or apart"""
    H, K, D = case["heads"], case["kv_heads"], case["D"]
    # a few channels of a projection are much larger than the others
    wide = torch.ones(H + 2 * K, D, device=DEV)
    wide[:, D // 3] = 6.0
    x = (torch.randn(M, H + 2 * K, D, generator=g, device=DEV) * wide).half().view(M, (H + 2 * K) * D)
    q, k, v = x[:, :H * D], x[:, H * D:(H + K) * D], x[:, (H + K) * D:]
    return (q, k, v) if packed else (q.contiguous(), k.contiguous(), v.contiguous())


def _cache(g, case, length, first):
    """pages in random order; the pages of a sequence before position first[s] (and past its end)
    are not there, except those of its first tokens"""
    page, K, D, S = case["page"], case["kv_heads"], case["D"], len(length)
    stride = max(1, max(-(-n // page) for n in length))
    sinks = case.get("sinks", 0)
    live = [[p for p in range(-(-n // page)) if (p + 1) * page > lo or p * page < sinks] for n, lo in zip(length, first)]
    total = sum(len(x) for x in live) + 3
    order = torch.randperm(total, generator=g, device=DEV).int()
    rows, cols = [], []
    for s, x in enumerate(live):
        rows += [s] * len(x)
        cols += x
    table = torch.full((S, stride), -1, dtype=torch.int32, device=DEV)
    at = torch.tensor([rows, cols], device=DEV)
    table[at[0], at[1]] = order[:len(rows)]
    k = torch.empty(total, K, page, D, dtype=torch.float16, device=DEV).normal_(generator=g)
    v = torch.empty(total, K, page, D, dtype=torch.float16, device=DEV).normal_(generator=g)
    return k, v, table


_library = {}


def _own(state, case):
    """what a program that uses the library keeps: a context for each stream, here of the stream on which
    the inputs are made, and the descriptions of its buffers"""
    import npu880_mtk_npu_llm_runtime_b200 as kq
    torch.cuda.init()
    at = (torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    if at not in _library:
        _library[at] = kq.Context(at[0])
        _library[at].set_stream(at[1])
    state["ctx"] = _library[at]
    if "inv_freq" in state:
        state["rope"] = kq.Rope(case["rot"], base=case["base"], style=case["style"])
    if case["op"] != "norm_rope":
        state["cache"] = kq.KvCache(state["ck"], state["cv"], state["table"])
    if case["op"] == "norm_rope":
        state["hq"] = kq.Heads(state["q"], case["heads"], gamma=state["q_gamma"], out=state["q_out"])
        state["hk"] = kq.Heads(state["k"], case["kv_heads"], gamma=state["k_gamma"], out=state["k_out"])
    elif case["op"] == "append":
        state["hq"] = kq.Heads(state["q"], case["heads"], gamma=state["q_gamma"], out=state["q_out"])
        state["hk"] = kq.Heads(state["k"], case["kv_heads"], gamma=state["k_gamma"])
        state["hv"] = kq.Heads(state["v"], case["kv_heads"])
    else:
        state["attn"] = kq.Attention(state["cache"], state["q"], state["out"], state["kv_len"],
                                     q_start=state.get("q_start"), window=case["window"], sinks=case["sinks"])


def prepare(case, seed):
    g = _gen(seed)
    H, K, D = case["heads"], case["kv_heads"], case["D"]
    s = {"case": case}
    if case["op"] in ("norm_rope", "append"):
        j = torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
        s["inv_freq"] = case["base"] ** (-2.0 * j / case["rot"])
    if case["op"] == "norm_rope":
        M = case["M"]
        s["q"], s["k"], _ = _rows(g, M, case, case["packed"])
        s["pos"] = torch.randint(0, case["far"], (M,), generator=g, device=DEV, dtype=torch.int32)
        s["q_gamma"] = _gamma(g, D) if case["q_norm"] else None
        s["k_gamma"] = _gamma(g, D) if case["k_norm"] else None
        s["q_out"] = torch.zeros(M, H * D, dtype=torch.float16, device=DEV)
        s["k_out"] = torch.zeros(M, K * D, dtype=torch.float16, device=DEV)
    else:
        n, length = _lengths(case)
        S, M = len(n), sum(n)
        if case["op"] == "append":
            first = [b - a for a, b in zip(n, length)]
            s["ck"], s["cv"], s["table"] = _cache(g, case, length, first)
            s["q"], s["k"], s["v"] = _rows(g, M, case, True)
            cnt = torch.tensor(n, device=DEV)
            s["seq"] = torch.repeat_interleave(torch.arange(S, device=DEV), cnt).int()
            start = torch.cumsum(cnt, 0) - cnt
            s["pos"] = (torch.arange(M, device=DEV) - start[s["seq"].long()]
                        + torch.tensor(first, device=DEV)[s["seq"].long()]).int()
            s["q_gamma"] = s["k_gamma"] = None
            if case["k_norm"]:
                s["q_gamma"], s["k_gamma"] = _gamma(g, D), _gamma(g, D)
            s["q_out"] = torch.zeros(M, H * D, dtype=torch.float16, device=DEV)
        else:
            w = case["window"]
            first = [max(0, b - a - w + 1) if w else 0 for a, b in zip(n, length)]
            s["ck"], s["cv"], s["table"] = _cache(g, case, length, first)
            s["q"] = _randn(g, M, H * D, scale=1.5)
            s["out"] = torch.zeros(M, H * D, dtype=torch.float16, device=DEV)
            s["kv_len"] = torch.tensor(length, dtype=torch.int32, device=DEV)
            s["longest"] = max(length)
            if case["op"] == "prefill":
                s["q_start"] = torch.tensor([sum(n[:i]) for i in range(S + 1)], dtype=torch.int32, device=DEV)
                s["most"] = max(n)
    if own:
        _own(s, case)
    return s


# ------------------------------------------------------------------------------ plain forms

def _norm_rope(x, heads, D, gamma, inv_freq, pos, style):
    """[M, heads * D] fp16 -> the same, normed per head and turned, in 32 bits; angles in 64"""
    M = x.shape[0]
    y = x.reshape(M, heads, D).float()
    if gamma is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gamma.float()
    t = pos.double()[:, None] * inv_freq
    c, s = torch.cos(t).float()[:, None], torch.sin(t).float()[:, None]
    R = 2 * inv_freq.shape[0]
    if style == "half":
        a, b = y[..., :R // 2], y[..., R // 2:R]
        z = torch.cat([a * c - b * s, a * s + b * c, y[..., R:]], -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        z = torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), y[..., R:]], -1)
    return z.reshape(M, heads * D).half()


def _decode(st, case):
    H, K, D, page, w, sinks = (case[x] for x in ("heads", "kv_heads", "D", "page", "window", "sinks"))
    S = st["q"].shape[0]
    n = st["kv_len"].long()
    lo = (n - w).clamp(min=0) if w else torch.zeros_like(n)
    kept = torch.minimum(lo, torch.full_like(lo, sinks))
    most = min(st["longest"], w + sinks) if w else st["longest"]
    e = torch.arange(most, device=DEV)[None]
    key = torch.where(e < kept[:, None], e, e - kept[:, None] + lo[:, None])     # [S, most]
    seen = key < n[:, None]
    key = torch.where(seen, key, torch.zeros_like(key))
    pg = torch.gather(st["table"].long(), 1, key // page).clamp(min=0)
    k = st["ck"][pg, :, key % page].float()                                       # [S, most, K, D]
    q = st["q"].view(S, K, H // K, D).float() / math.sqrt(D)
    a = torch.matmul(q, k.permute(0, 2, 3, 1)).masked_fill(~seen[:, None, None], float("-inf"))
    del k
    a = torch.softmax(a, -1)
    v = st["cv"][pg, :, key % page].float()
    o = torch.matmul(a, v.permute(0, 2, 1, 3))
    return o.reshape(S, H * D).half()


def _prefill(st, case):
    H, K, D, page, w, sinks = (case[x] for x in ("heads", "kv_heads", "D", "page", "window", "sinks"))
    S, N, L = st["kv_len"].shape[0], st["most"], st["longest"]
    start, n = st["q_start"][:-1].long(), (st["q_start"][1:] - st["q_start"][:-1]).long()
    length = st["kv_len"].long()
    i = torch.arange(N, device=DEV)[None]
    there = i < n[:, None]                                                        # [S, N]
    row = torch.where(there, start[:, None] + i, torch.zeros_like(i))
    pos = (length - n)[:, None] + i
    j = torch.arange(L, device=DEV)
    key = torch.minimum(j[None], length[:, None] - 1)
    pg = torch.gather(st["table"].long(), 1, key // page).clamp(min=0)
    seen = j[None, None] <= pos[..., None]
    if w:
        seen &= (j[None, None] > pos[..., None] - w) | (j < sinks)
    k = st["ck"][pg, :, key % page].float().permute(0, 2, 3, 1)                   # [S, K, D, L]
    q = st["q"].view(-1, K, H // K, D)[row].float().permute(0, 2, 3, 1, 4)        # [S, K, G, N, D]
    a = torch.matmul(q.reshape(S, K, -1, D), k).view(S, K, H // K, N, L)
    del k
    a.mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], float("-inf"))
    a = torch.softmax(a, -1)
    v = st["cv"][pg, :, key % page].float().permute(0, 2, 1, 3)                   # [S, K, L, D]
    o = torch.matmul(a.view(S, K, -1, L), v).view(S, K, H // K, N, D).permute(0, 3, 1, 2, 4)
    out = st["out"]
    out[row[there]] = o.reshape(S, N, H * D)[there].half()
    return out


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        ctx = state["ctx"]
        if op == "norm_rope":
            ctx.qk_norm_rope_async(state["rope"], state["pos"], state["hq"], state["hk"], eps=EPS)
            return {"q": state["q_out"], "k": state["k_out"]}
        if op == "append":
            ctx.kv_append_async(state["cache"], state["rope"], state["seq"], state["pos"], state["hk"], state["hv"],
                                q=state["hq"], eps=EPS)
            return {"q": state["q_out"], "k": state["ck"], "v": state["cv"]}
        (ctx.attn_decode_async if op == "decode" else ctx.attn_prefill_async)(state["attn"])
        return {"out": state["out"]}
    H, K, D = case["heads"], case["kv_heads"], case["D"]
    if op == "decode":
        return {"out": _decode(state, case)}
    if op == "prefill":
        return {"out": _prefill(state, case)}
    turn = (state["inv_freq"], state["pos"], case["style"])
    q = _norm_rope(state["q"], H, D, state["q_gamma"], *turn)
    k = _norm_rope(state["k"], K, D, state["k_gamma"], *turn)
    if op == "norm_rope":
        return {"q": q, "k": k}
    pos = state["pos"].long()
    pg = state["table"].long()[state["seq"].long(), pos // case["page"]]
    state["ck"][pg, :, pos % case["page"]] = k.view(-1, K, D)
    state["cv"][pg, :, pos % case["page"]] = state["v"].reshape(-1, K, D)
    return {"q": q, "k": state["ck"], "v": state["cv"]}


# ---------------------------------------------------------------------------- in 64 bits

def _turned(x, heads, D, gamma, base, rot, style, pos):
    """the definition, value by value of a pair, in 64 bits"""
    y = x.double().unflatten(-1, (heads, D)).clone()
    if gamma is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + EPS) * gamma.double()
    z = y.clone()
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if style == "half" else (2 * j, 2 * j + 1)
        t = pos.double() / base ** (2.0 * j / rot)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        z[..., a] = y[..., a] * c - y[..., b] * s
        z[..., b] = y[..., b] * c + y[..., a] * s
    return z.flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    H, K, D = case["heads"], case["kv_heads"], case["D"]
    if case["op"] in ("norm_rope", "append"):
        turn = (case["base"], case["rot"], case["style"], st["pos"])
        q = _turned(st["q"], H, D, st["q_gamma"], *turn)
        k = _turned(st["k"], K, D, st["k_gamma"], *turn)
        if case["op"] == "norm_rope":
            return {"q": q, "k": k}
        ck, cv = st["ck"].double(), st["cv"].double()
        page = case["page"]
        for s, p, kr, vr in zip(st["seq"].tolist(), st["pos"].tolist(), k, st["v"].double()):
            at = int(st["table"][s, p // page])
            ck[at, :, p % page] = kr.view(K, D)
            cv[at, :, p % page] = vr.view(K, D)
        return {"q": q, "k": ck, "v": cv}
    n, length = _lengths(case)
    out = torch.zeros(sum(n), H, D, dtype=torch.float64, device=DEV)
    r = 0
    for s, (a, b) in enumerate(zip(n, length)):
        p = torch.arange(b - a, b, device=DEV)
        j = torch.arange(b, device=DEV)
        seen = j[None] <= p[:, None]
        if case["window"]:
            seen &= (p[:, None] - j[None] < case["window"]) | (j[None] < case["sinks"])
        used = seen.any(0).nonzero()[:, 0]      # keys that some row sees; the other pages may be gone
        at = st["table"][s].long()[used // case["page"]]
        for h in range(H):
            kk = st["ck"][at, h // (H // K), used % case["page"]].double()
            vv = st["cv"][at, h // (H // K), used % case["page"]].double()
            e = st["q"][r:r + a, h * D:(h + 1) * D].double() @ kk.T / math.sqrt(D)
            e = torch.where(seen[:, used], e, float("-inf"))
            e = torch.exp(e - e.max(-1, keepdim=True).values)
            out[r:r + a, h] = (e / e.sum(-1, keepdim=True)) @ vv
        r += a
    return {"out": out.view(-1, H * D)}

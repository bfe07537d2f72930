"""Calls of the attention operators that their documentation allows and that are easy to get wrong, on the GPU,
against the plain 64-bit forms (attn_ref)."""
from __future__ import annotations

import numpy as np
import pytest

import attn_ref as R
import npu880_mtk_npu_llm_runtime_b200 as kq
from test_gpu_attn import SENTINEL, SHAPE, cache_of, close, dev

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

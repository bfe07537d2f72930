"""Calls of the attention operators at the edge of what their documentation allows, on the host: row ranges,
overlapping buffers, numbers that do not fit."""
from __future__ import annotations

import ctypes as C
import random
import subprocess

import pytest

from conftest import ROOT

import npu880_mtk_npu_llm_runtime_b200 as kq
from npu880_mtk_npu_llm_runtime_b200 import build as kqbuild
from test_attn_host import INVALID, attn_struct, cache_struct, heads_struct

SOURCE = r'''
#include "npu880_mtk_npu_llm_runtime_b200/csrc/kq_kv.h"
using namespace kq;
extern "C" {
int rows(int start, int end, int M, int *begin) { bool b = false; KvRows r = kv_rows(start, end, M, b); *begin = r.begin; return r.n; }
int rows_behind(int start, int end, int M, int limit, int *begin, int *bad) {
    bool b = false; KvRows r = kv_rows_behind(start, end, M, limit, b); *begin = r.begin; *bad = b; return r.n; }
int c_attn(const kq_kv_cache *c, const kq_attn *a, int prefill) { const char *w; return check_attn(c, a, prefill != 0, &w); }
int overlap(size_t a, size_t as, size_t aw, int an, size_t b, size_t bs, size_t bw, int bn) {
    return rows_overlap(Rows{(void *)a, as, aw, an}, Rows{(void *)b, bs, bw, bn});
}
int heads_apart(const kq_kv_cache *c, int dim, int M, const kq_heads *q, const kq_heads *k, const kq_heads *v) {
    const char *w; return check_heads_apart(c, dim, M, q, k, v, &w);
}
int attn_apart(const kq_kv_cache *c, const kq_attn *a) { const char *w; return check_attn_apart(c, a, &w); }
}
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "kv.cc").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", ROOT, "-o", str(d / "kv.so"),
                           str(d / "kv.cc")])
    L = C.CDLL(str(d / "kv.so"))
    L.overlap.argtypes = [C.c_size_t, C.c_size_t, C.c_size_t, C.c_int] * 2
    return L


def ranges(host, q_start, M):
    """the ranges that a prefill call takes, as its plan makes them"""
    begin, bad = C.c_int(), C.c_int()
    limit, out, wrong = 0, [], False
    for a, b in zip(q_start, q_start[1:]):
        n = host.rows_behind(a, b, M, limit, C.byref(begin), C.byref(bad))
        out.append((begin.value, n))
        wrong |= bool(bad.value)
        n = host.rows(a, b, M, C.byref(begin))
        limit = max(limit, begin.value + n)
    return out, wrong


def test_row_ranges_never_overlap(host):
    """whatever q_start holds: the ranges are disjoint, so all of them have M rows at most and the row tiles
    (one a sequence more than the rows fill) fit the tables sized for that"""
    rng = random.Random(1)
    M = 4096
    cases = [[0, M] * 2048 + [0], [M, 0] * 2048 + [M], [0, 20, 10, 30], [0, 9999, 5, 10], [-1, 5, 3, 7]]
    cases += [[rng.randrange(-5, M + 5) for _ in range(rng.randrange(2, 200))] for _ in range(300)]
    for q_start in cases:
        got, wrong = ranges(host, q_start, M)
        used = sorted((b, n) for b, n in got if n)
        assert all(b + n <= b2 for (b, n), (b2, _) in zip(used, used[1:])), q_start
        assert sum(n for _, n in got) <= M and all(0 <= b and b + n <= M for b, n in got)
        assert wrong == (q_start != sorted(q_start) or q_start[0] < 0 or q_start[-1] > M)
    # ranges in order are taken as they are
    for _ in range(100):
        q_start = sorted(rng.randrange(M + 1) for _ in range(rng.randrange(2, 100)))
        got, wrong = ranges(host, q_start, M)
        assert not wrong and got == [(a, b - a) for a, b in zip(q_start, q_start[1:])]
    assert ranges(host, [0, 20, 10, 30], 30)[0] == [(0, 20), (0, 0), (0, 0)]
    assert ranges(host, [5, 3, 10, 12], 30)[0] == [(0, 0), (3, 7), (10, 2)]


@pytest.mark.parametrize("scale, status", [(0.0, 0), (-0.0, 0), (1e-40, 0), (1e24, 0), (1.1e24, INVALID), (1e30, INVALID)])
def test_scales(host, scale, status):
    """the largest scale keeps every finite score below fp32's largest number: 256 * 65504^2 * 1e24 / ln 2"""
    assert 256 * 65504.0 ** 2 * 1e24 * 1.4427 < 3.4e38
    for prefill in (0, 1):
        assert host.c_attn(C.byref(cache_struct()), C.byref(attn_struct(scale=scale)), prefill) == status


def test_rows_that_share_bytes(host):
    """against the sets of bytes themselves"""
    rng = random.Random(5)
    seen = set()
    for _ in range(6000):
        sets, args = [], []
        same = rng.choice([0, rng.randrange(1, 40)])
        for _ in range(2):
            width = rng.randrange(1, 12)
            n = rng.randrange(0, 7)
            stride = max(width, same or rng.randrange(1, 40))
            at = rng.randrange(1, 200)
            sets.append({at + i * stride + j for i in range(n) for j in range(width)})
            args += [at, stride, width, n]
        want = bool(sets[0] & sets[1])
        assert host.overlap(*args) == want, args
        seen.add((want, args[1] == args[5]))
    assert len(seen) == 4
    # many rows of large strides
    far = 1 << 39
    assert not host.overlap(1 << 20, far, 8192, 4096, (1 << 20) + 8192, far, 8192, 4096)
    assert host.overlap(1 << 20, far, 8192, 4096, (1 << 20) + 4095 * far + 8191, far, 8192, 4096)
    assert not host.overlap(1 << 20, far, 8192, 4096, (1 << 20) + 4095 * far + 8192, far, 8192, 4096)


def test_outputs_over_inputs(host):
    """q, k and v side by side in one buffer, in place or to another one; not over each other, nor over the pages"""
    M, D, base = 100, 64, 1 << 24
    row = (8 + 2 + 2) * D                                  # q of 8 heads, k and v of 2
    q_at, k_at, v_at = (base + 2 * D * h for h in (0, 8, 10))
    pages = dict(k=1 << 30, v=1 << 31, n_pages=1000, page_size=16, kv_heads=2, head_dim=D)
    size = 1000 * 16 * 2 * D * 2

    def call(cache=None, M=M, q_out=q_at, q_out_stride=row, **kw):
        c = cache_struct(**dict(pages, **(cache or {})))
        q = heads_struct(8, **dict(dict(in_=q_at, in_stride=row, out=q_out, out_stride=q_out_stride), **kw))
        k, v = (heads_struct(2, in_=a, in_stride=row) for a in (k_at, v_at))
        return host.heads_apart(C.byref(c), D, M, C.byref(q), C.byref(k), C.byref(v))

    assert call() == 0                                     # in place, between the rows of k and v
    assert call(q_out=1 << 28, q_out_stride=8 * D) == 0
    assert call(q_out=q_at - 2 * 8 * D) == INVALID         # the row before: over k and v of it
    assert call(q_out=q_at + 2 * D) == INVALID             # a head further on
    assert call(q_out_stride=row + 8) == INVALID           # in place with another stride
    assert call(M=1, q_out_stride=row + 8) == 0            # (of one row it does not matter)
    assert call(q_out=q_at + 2 * row * M) == 0
    assert call(q_out=q_at + 2 * row * (M - 1)) == INVALID
    assert call(cache=dict(v=(1 << 30) + size - 16)) == INVALID
    assert call(cache=dict(v=(1 << 30) + size)) == 0
    assert call(cache=dict(k=base - size + 16)) == INVALID
    assert call(cache=dict(v=base + 2 * row * M - 16)) == INVALID
    assert call(q_out=(1 << 30) + size - 16, q_out_stride=8 * D) == INVALID

    def turn(k_out, q_out=1 << 28):                        # without a cache: two outputs
        q = heads_struct(8, in_=q_at, in_stride=row, out=q_out, out_stride=8 * D)
        k = heads_struct(2, in_=k_at, in_stride=row, out=k_out, out_stride=8 * D)
        return host.heads_apart(None, D, M, C.byref(q), C.byref(k), None)

    assert turn(1 << 29) == 0 and turn((1 << 28) + 8 * D * 2 * M) == 0
    assert turn((1 << 28) + 16) == INVALID and turn(q_at) == INVALID and turn(1 << 29, q_out=k_at) == INVALID

    def attend(out, stride, cache=pages):
        c = cache_struct(**cache)
        a = attn_struct(q=q_at, q_stride=row, out=out, out_stride=stride, heads=8, M=M)
        return host.attn_apart(C.byref(c), C.byref(a))

    assert attend(1 << 28, 8 * D) == 0 and attend(k_at + 2 * 4 * D, 2 * row) == INVALID
    assert attend(q_at, row) == INVALID and attend(q_at + 16, 8 * D) == INVALID
    assert attend((1 << 30) - 2 * 8 * D * M, 8 * D) == 0 and attend((1 << 30) - 2 * 8 * D * M + 16, 8 * D) == INVALID
    assert attend((1 << 31) + size, 8 * D) == 0 and attend((1 << 31) + size - 16, 8 * D) == INVALID


def test_numbers_of_32_bits():
    kqbuild.build()
    for rot in (2 ** 32 + 64, 2 ** 32, -2 ** 32 + 16):
        with pytest.raises(ValueError):
            kq.Rope(rot)
    assert kq._int32(2 ** 31 - 1, "x") == 2 ** 31 - 1 and kq._int32(-2 ** 31, "x") == -2 ** 31
    for v in (2 ** 31, -2 ** 31 - 1, 2 ** 64):
        with pytest.raises(ValueError):
            kq._int32(v, "x")
    assert kq._scale(0) == 0 and kq._scale(1e-40) == 1e-40
    for v in (1e-50, -1e-60):
        with pytest.raises(ValueError):
            kq._scale(v)

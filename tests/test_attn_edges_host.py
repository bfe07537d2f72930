"""Calls of the attention operators at the edge of what their documentation allows, on the host: row ranges,
overlapping buffers, numbers that do not fit."""
from __future__ import annotations

import ctypes as C
import random
import subprocess

import pytest

from conftest import ROOT
from test_attn_host import INVALID, attn_struct, cache_struct

SOURCE = r'''
#include "npu880_mtk_npu_llm_runtime_b200/csrc/kq_kv.h"
using namespace kq;
extern "C" {
int rows(int start, int end, int M, int *begin) { bool b = false; KvRows r = kv_rows(start, end, M, b); *begin = r.begin; return r.n; }
int rows_behind(int start, int end, int M, int limit, int *begin, int *bad) {
    bool b = false; KvRows r = kv_rows_behind(start, end, M, limit, b); *begin = r.begin; *bad = b; return r.n; }
int c_attn(const kq_kv_cache *c, const kq_attn *a, int prefill) { const char *w; return check_attn(c, a, prefill != 0, &w); }
}
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "kv.cc").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", ROOT, "-o", str(d / "kv.so"),
                           str(d / "kv.cc")])
    return C.CDLL(str(d / "kv.so"))


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

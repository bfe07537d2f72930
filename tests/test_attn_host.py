"""The paged cache's index arithmetic and the refusals of the attention calls, compiled for the host."""
from __future__ import annotations

import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

import attn_ref
from conftest import ROOT

import npu880_mtk_npu_llm_runtime_b200 as kq
from npu880_mtk_npu_llm_runtime_b200 import build as kqbuild

SOURCE = r'''
#include "npu880_mtk_npu_llm_runtime_b200/csrc/kq_kv.h"
using namespace kq;
extern "C" {
void span(int p, int len, int window, int sinks, int *o) { KvSpan s = kv_span(p, len, window, sinks); o[0] = s.kept; o[1] = s.lo; o[2] = s.hi; }
int sees(int p, int len, int window, int sinks, int j) { return kv_sees(kv_span(p, len, window, sinks), j); }
int count(int p, int len, int window, int sinks) { return kv_count(kv_span(p, len, window, sinks)); }
int nth(int p, int len, int window, int sinks, int e) { return kv_nth(kv_span(p, len, window, sinks), e); }
int blocks(int kept, int lo, int hi, int B, int *o) { KvBlocks b = kv_blocks(kept, lo, hi, B); for (int i = 0; i < b.count; ++i) o[i] = kv_block(b, i); return b.count; }
long long begin_of(long long total, int parts, int c) { return Shares(total, parts).begin(c); }
int part(long long total, int parts, long long u) { return Shares(total, parts).of(u); }
long long row(int n_pages, int shift, int heads, int dim, int page, int head, int slot) {
    KvView v{}; v.n_pages = n_pages; v.page_shift = shift; v.kv_heads = heads; v.head_dim = dim; return kv_row(v, page, head, slot); }
int length(int stride, int shift, int len, int *bad) { KvView v{}; v.table_stride = stride; v.page_shift = shift; bool b = false; int r = kv_length(v, len, b); *bad = b; return r; }
int rows(int start, int end, int M, int *begin, int *bad) { bool b = false; KvRows r = kv_rows(start, end, M, b); *begin = r.begin; *bad = b; return r.n; }
int page_ok(int n_pages, int page) { KvView v{}; v.n_pages = n_pages; return kv_page_ok(v, page); }
int c_cache(const kq_kv_cache *c) { const char *w; return check_cache(c, &w); }
int c_attn(const kq_kv_cache *c, const kq_attn *a, int prefill) { const char *w; return check_attn(c, a, prefill != 0, &w); }
int c_append(const kq_kv_cache *c, const kq_rope *r, int M, const int *seq, const int *pos, const kq_heads *q, const kq_heads *k, const kq_heads *v) {
    const char *w; return check_append(c, r, M, seq, pos, q, k, v, &w); }
int c_heads(const kq_heads *h, int dim, int to) { const char *w; return check_heads(h, dim, to, &w); }
int c_rope(const kq_rope *r, int dim) { const char *w; return check_rope(r, dim, &w); }
}
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv")
    (d / "kv.cc").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", ROOT, "-o", str(d / "kv.so"),
                           str(d / "kv.cc")])
    L = C.CDLL(str(d / "kv.so"))
    L.begin_of.restype = C.c_longlong
    L.begin_of.argtypes = [C.c_longlong, C.c_int, C.c_int]
    L.part.argtypes = [C.c_longlong, C.c_int, C.c_longlong]
    L.row.restype = C.c_longlong
    for f in ("c_cache", "c_attn", "c_append", "c_heads", "c_rope"):
        getattr(L, f).argtypes = None
    return L


def test_visible_keys(host):
    """span, count and enumeration against the definition, windows and first tokens of every relation"""
    for length in (0, 1, 2, 5, 17, 40):
        for p in range(-2, length):
            for window in (0, 1, 2, 5, 16, 100):
                for sinks in (0,) if window == 0 else (0, 1, 4, 18, 200):
                    want = attn_ref.visible(p, length, window, sinks).tolist()
                    n = host.count(p, length, window, sinks)
                    got = [host.nth(p, length, window, sinks, e) for e in range(n)]
                    assert got == want, (length, p, window, sinks)
                    assert [j for j in range(length + 2) if host.sees(p, length, window, sinks, j)] == want


def test_far_positions(host):
    o = (C.c_int * 3)()
    host.span(2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 7, o)
    assert list(o) == [0, 0, 2 ** 30]
    host.span(2 ** 30 - 1, 2 ** 30, 4096, 7, o)
    assert list(o) == [7, 2 ** 30 - 4096, 2 ** 30]
    # a cache of more than 2^31 values, and of more than 2^32
    assert host.row(400000, 4, 8, 128, 399999, 7, 15) == ((399999 * 8 + 7) * 16 + 15) * 128 > 2 ** 32


@pytest.mark.parametrize("B", [16, 64, 128])
def test_blocks_cover_the_visible_keys_once(host, B):
    rng = random.Random(B)
    o = (C.c_int * 4096)()
    for _ in range(2000):
        hi = rng.choice([0, 1, B - 1, B, B + 1, rng.randrange(3000)])
        lo = rng.randrange(hi + 1)
        kept = rng.choice([0, min(4, lo), rng.randrange(lo + 1)])
        n = host.blocks(kept, lo, hi, B, o)
        got = list(o[:n])
        assert got == sorted(set(got))
        need = {j // B for j in range(hi) if j >= lo or j < kept}
        assert need <= set(got)
        assert all(0 <= b * B < max(hi, 1) for b in got)
        assert set(got) - need <= {lo // B}      # an empty span may keep its first block


def test_parts_are_even_and_found_again(host):
    rng = random.Random(3)
    for _ in range(300):
        total, parts = rng.choice([1, 7, rng.randrange(1, 5000), 2 ** 40 + 13]), rng.choice([1, 2, 148, 296, 1000])
        edges = [host.begin_of(total, parts, c) for c in range(parts + 1)]
        assert edges[0] == 0 and edges[-1] == total
        sizes = [b - a for a, b in zip(edges, edges[1:])]
        assert max(sizes) - min(sizes) <= 1
        for u in {0, total - 1, total // 2, rng.randrange(total)}:
            c = host.part(total, parts, u)
            assert edges[c] <= u < edges[c + 1]


def test_lengths_rows_and_pages_are_held(host):
    bad = C.c_int()
    for length, want, flag in [(0, 0, 0), (-1, 0, 1), (160, 160, 0), (161, 160, 1), (-2 ** 31, 0, 1), (2 ** 31 - 1, 160, 1)]:
        assert (host.length(10, 4, length, C.byref(bad)), bad.value) == (want, flag)
    begin = C.c_int()
    for start, end, want in [(0, 0, (0, 0, 0)), (3, 7, (4, 3, 0)), (7, 3, (0, 0, 1)), (-1, 4, (0, 0, 1)), (5, 11, (0, 0, 1)),
                             (10, 10, (0, 10, 0))]:
        n = host.rows(start, end, 10, C.byref(begin), C.byref(bad))
        assert (n, begin.value, bad.value) == want
    assert [host.page_ok(5, p) for p in (-1, 0, 4, 5, -2 ** 31, 2 ** 31 - 1)] == [0, 1, 1, 0, 0, 0]


def cache_struct(**kw):
    s = kq.KvCacheStruct(k=256, v=512, page_table=1024, n_pages=4, page_size=16, kv_heads=2, head_dim=64, n_seqs=3, table_stride=2)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def attn_struct(**kw):
    s = kq.AttnStruct(q=256, q_stride=512, out=512, out_stride=512, heads=8, M=3, kv_len=64, q_start=64)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def heads_struct(heads=2, **kw):
    s = kq.HeadsStruct(in_=256, in_stride=512, out=None, out_stride=0, heads=heads, gamma=None)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


INVALID, SHAPE = -1, -3


@pytest.mark.parametrize("change, status", [
    (dict(), 0), (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(page_table=None), INVALID), (dict(k=8), INVALID),
    (dict(v=513), INVALID), (dict(page_table=2), INVALID), (dict(head_dim=96), SHAPE), (dict(head_dim=0), SHAPE),
    (dict(page_size=8), SHAPE), (dict(page_size=512), SHAPE), (dict(page_size=48), SHAPE), (dict(page_size=-16), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(kv_heads=257), SHAPE), (dict(n_pages=0), SHAPE), (dict(n_seqs=0), SHAPE),
    (dict(n_seqs=4097), SHAPE), (dict(table_stride=0), SHAPE), (dict(table_stride=2 ** 27), SHAPE), (dict(table_stride=2 ** 26), 0),
    (dict(table_stride=2 ** 26, n_seqs=16), 0), (dict(table_stride=2 ** 26, n_seqs=17), SHAPE),
])
def test_cache_refusals(host, change, status):
    assert host.c_cache(C.byref(cache_struct(**change))) == status


def test_null_structs(host):
    a, c, h = attn_struct(), cache_struct(), heads_struct()
    assert host.c_cache(None) == INVALID
    assert host.c_attn(None, C.byref(a), 0) == INVALID
    assert host.c_attn(C.byref(c), None, 0) == INVALID
    assert host.c_heads(None, 64, 0) == INVALID
    assert host.c_rope(None, 64) == 0
    for k, v in ((None, h), (h, None)):
        assert host.c_append(C.byref(c), None, 1, C.c_void_p(64), C.c_void_p(64), None, k and C.byref(k), v and C.byref(v)) == INVALID


@pytest.mark.parametrize("change, decode, prefill", [
    (dict(), 0, 0), (dict(q=None), INVALID, INVALID), (dict(out=None), INVALID, INVALID), (dict(kv_len=None), INVALID, INVALID),
    (dict(q_start=None), 0, INVALID), (dict(M=2), SHAPE, 0), (dict(M=0), SHAPE, 0), (dict(M=-1), SHAPE, SHAPE),
    (dict(M=4097), SHAPE, SHAPE), (dict(heads=7), SHAPE, SHAPE), (dict(heads=0), SHAPE, SHAPE), (dict(heads=34, q_stride=4096, out_stride=4096), SHAPE, SHAPE),
    (dict(heads=32, q_stride=2048, out_stride=2048), 0, 0), (dict(q_stride=504), INVALID, INVALID), (dict(q_stride=516), INVALID, INVALID),
    (dict(out_stride=8), INVALID, INVALID), (dict(q=8), INVALID, INVALID), (dict(out=520), INVALID, INVALID), (dict(window=-1), INVALID, INVALID),
    (dict(sinks=4), INVALID, INVALID), (dict(window=8, sinks=-1), INVALID, INVALID), (dict(window=8, sinks=4), 0, 0),
    (dict(scale=-1.0), INVALID, INVALID), (dict(scale=float("nan")), INVALID, INVALID), (dict(scale=float("inf")), INVALID, INVALID),
    (dict(scale=0.125), 0, 0), (dict(kv_len=66), INVALID, INVALID), (dict(q_start=65), 0, INVALID), (dict(out=256), INVALID, INVALID),
])
def test_attention_refusals(host, change, decode, prefill):
    c, a = cache_struct(), attn_struct(**change)
    assert host.c_attn(C.byref(c), C.byref(a), 0) == decode
    assert host.c_attn(C.byref(c), C.byref(a), 1) == prefill


@pytest.mark.parametrize("change, status", [
    (dict(), 0), (dict(M=-1), SHAPE), (dict(M=4097), SHAPE), (dict(M=0), 0), (dict(seq=None), INVALID), (dict(pos=None), INVALID),
    (dict(seq=66), INVALID), (dict(pos=65), INVALID),
    (dict(k=heads_struct(3)), SHAPE), (dict(v=heads_struct(1)), SHAPE), (dict(k=heads_struct(out=512, out_stride=512)), INVALID),
    (dict(v=heads_struct(gamma=64)), INVALID), (dict(k=heads_struct(gamma=64)), 0), (dict(k=heads_struct(gamma=72)), INVALID),
    (dict(k=heads_struct(in_=None)), INVALID), (dict(k=heads_struct(in_=260)), INVALID), (dict(k=heads_struct(in_stride=120)), INVALID),
    (dict(q=heads_struct(8)), INVALID), (dict(q=heads_struct(8, out=512, out_stride=512)), 0), (dict(q=heads_struct(0, out=512, out_stride=512)), SHAPE),
    (dict(q=heads_struct(257, in_stride=1 << 15, out=512, out_stride=1 << 15)), SHAPE),
])
def test_append_refusals(host, change, status):
    c = cache_struct()
    a = dict(M=1, seq=64, pos=64, q=None, k=heads_struct(), v=heads_struct())
    a.update(change)
    ref = lambda x: x and C.byref(x)  # noqa: E731
    assert host.c_append(C.byref(c), None, a["M"], C.c_void_p(a["seq"]), C.c_void_p(a["pos"]), ref(a["q"]), ref(a["k"]),
                         ref(a["v"])) == status


@pytest.mark.parametrize("rot, style, status", [(0, 0, 0), (16, 0, 0), (64, 1, 0), (80, 0, SHAPE), (8, 0, SHAPE), (-16, 0, SHAPE),
                                                (64, 2, INVALID), (64, -1, INVALID)])
def test_rope_refusals(host, rot, style, status):
    assert host.c_rope(C.byref(kq.RopeStruct(rot_dim=rot, style=style)), 64) == status


def test_rope_init():
    kqbuild.build()
    lib = kq.load_library()
    r = kq.Rope(64, base=1e6, style="adjacent")
    assert (r.struct.rot_dim, r.struct.style) == (64, 1)
    assert np.allclose(r.struct.inv_freq[:32], [1e6 ** (-2 * j / 64) for j in range(32)], rtol=1e-14)
    assert r.struct.inv_freq[32] == 0.0
    assert kq.Rope(32, inv_freq=[0.5] * 16).struct.inv_freq[15] == 0.5
    for bad in (dict(rot_dim=24), dict(rot_dim=-16), dict(rot_dim=272), dict(rot_dim=64, base=0.0), dict(rot_dim=64, base=float("nan")),
                dict(rot_dim=64, base=float("inf"))):
        with pytest.raises(kq.KQError):
            kq.Rope(**bad)
    assert lib.kq_rope_init(None, 64, 0, 1e4) == INVALID
    assert lib.kq_rope_init(C.addressof(r.struct), 64, 2, 1e4) == INVALID


def test_no_context_is_refused():
    lib = kq.load_library()
    c, a, h = cache_struct(), attn_struct(), heads_struct()
    assert lib.kq_attn_decode_async(None, C.addressof(c), C.addressof(a)) == INVALID
    assert lib.kq_attn_prefill_async(None, C.addressof(c), C.addressof(a)) == INVALID
    assert lib.kq_qk_norm_rope_async(None, None, 64, 1, None, None, None, 0.0) == INVALID
    assert lib.kq_kv_append_async(None, C.addressof(c), None, 1, 64, 64, None, C.addressof(h), C.addressof(h), 0.0) == INVALID


def test_structs_have_the_header_layout(tmp_path):
    """the ctypes mirrors of the attention structs against the C compiler's offsets"""
    mirrors = {"kq_rope": kq.RopeStruct, "kq_kv_cache": kq.KvCacheStruct, "kq_heads": kq.HeadsStruct, "kq_attn": kq.AttnStruct,
               "kq_attn_layer": kq.AttnLayerStruct}
    src = "#include <stddef.h>\n#include <stdio.h>\n#include \"kq.h\"\nint main(void) {\n"
    for name, S in mirrors.items():
        for f, _ in S._fields_:
            src += f'printf("%zu ", offsetof({name}, {f.rstrip("_")}));\n'
        src += f'printf("%zu\\n", sizeof({name}));\n'
    (tmp_path / "l.c").write_text(src + "return 0; }\n")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")])
    lines = subprocess.check_output([str(tmp_path / "l")]).decode().splitlines()
    for line, S in zip(lines, mirrors.values()):
        assert [int(v) for v in line.split()] == [getattr(S, f).offset for f, _ in S._fields_] + [C.sizeof(S)]

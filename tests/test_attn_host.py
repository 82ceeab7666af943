"""CPU checks of the attention half: the kernels' index helpers (compiled for the host), the
refusals of the C ABI and of the operators, output shapes, and the plain forms that the GPU tests
use."""
from __future__ import annotations

import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

import attn_ref as R
from conftest import PKG_DIR

SRC = r'''
#include "%s/csrc/paged.cuh"
using namespace pmoe;
extern "C" int h_page_of(const int* table, long stride, int max_pages, int shift, int n_pages, int b, int j) {
  PagedKV kv{};
  kv.table = table; kv.table_stride = stride; kv.max_pages = max_pages; kv.page_shift = shift;
  kv.n_pages = n_pages;
  return page_of(kv, b, j);
}
extern "C" int h_len(int len, int max_pages, int shift, int* over) {
  bool o; int r = kv_len_of(len, max_pages, shift, &o); *over = o; return r;
}
extern "C" void h_visible(int p, int w, int s, int* lo, int* sink) { visible_keys(p, w, s, lo, sink); }
'''


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    from paris_moe_b200 import build
    d = tmp_path_factory.mktemp("host")
    (d / "h.cu").write_text(SRC % PKG_DIR)
    so = d / "h.so"
    subprocess.check_call([build.nvcc_path(), "-std=c++17", *build.ARCH, "-shared", "-Xcompiler",
                           "-fPIC", "--expt-relaxed-constexpr", str(d / "h.cu"), "-o", str(so)])
    return ctypes.CDLL(str(so))


@pytest.fixture(scope="module")
def lib():
    from paris_moe_b200 import build, _lib
    build.build()
    return _lib.load()


def ints(v):
    return (ctypes.c_int * len(v))(*v)


def test_page_lookup_never_leaves_the_table_or_the_pool(host):
    n_pages, shift, width = 9, 4, 3
    table = [3, -1, 9, 0, 8, -2147483648, 2147483647, 5, 5]
    for b in range(3):
        for j in [-1, -16, 0, 15, 16, 31, 32, 47, 48, 1 << 30, (1 << 31) - 1]:
            got = host.h_page_of(ints(table), ctypes.c_long(width), width, shift, n_pages, b, j)
            i = j >> 4
            want = table[b * width + i] if 0 <= i < width else -1
            assert got == (want if 0 <= want < n_pages else -1)


def test_lengths_beyond_the_table_are_cut_and_reported(host):
    over = ctypes.c_int()
    for n, want, o in [(-5, 0, 0), (0, 0, 0), (48, 48, 0), (49, 48, 1), (2 ** 31 - 1, 48, 1)]:
        assert host.h_len(n, 3, 4, ctypes.byref(over)) == want and over.value == o


def test_visible_keys(host):
    lo, sink = ctypes.c_int(), ctypes.c_int()
    for p in (0, 1, 5, 17, 100):
        for w in (0, 1, 4, 18, 1000, 2 ** 31 - 1):
            for s in (0, 1, 7, 200):
                host.h_visible(p, w, s, ctypes.byref(lo), ctypes.byref(sink))
                got = [j for j in range(p + 1) if j < sink.value or j >= lo.value]
                assert got == torch.nonzero(R.visible(p, p + 1, w, s))[:, 0].tolist()
                assert sink.value <= lo.value or sink.value == 0


# ---- refusals: before any pointer or device use -------------------------------------------

P = ctypes.c_void_p
A = P(0x10000)    # aligned, never dereferenced: the checks fail first


def decode(lib, q=A, st=256, sh=256, B=2, Hq=4, Hkv=2, D=128, k=A, v=A, ks=4096, vs=4096, n=8,
           ps=16, table=A, ts=4, mp=4, lens=A, window=0, sinks=0, out=A, ws=A, nb=1 << 30):
    return lib.pmoe_attn_decode(q, st, sh, B, Hq, Hkv, D, k, v, ks, vs, n, ps, table, ts, mp, lens,
                                1.0, window, sinks, out, ws, nb, None)


def prefill(lib, q=A, st=256, sh=256, T=5, Hq=4, Hkv=2, D=128, ps=16, cu=A, B=2, window=0, sinks=0,
            mp=4, out=A):
    return lib.pmoe_attn_prefill(q, st, sh, T, Hq, Hkv, D, A, A, 1 << 20, 1 << 20, 8, ps, A, 4, mp,
                                 A, cu, B, 1.0, window, sinks, out, A, 1 << 30, None)


def rope(lib, T=2, B=2, D=128, rot=32, axes=3, sec=(6, 5, 5), st=256, cu=None, pos=A, q=A, ps=16,
         pos_stride=2):
    s = ints(list(sec)) if sec is not None else None
    return lib.pmoe_rope_append(q, st, 128, A, st, 128, A, st, 128, T, 4, 2, D, pos, pos_stride,
                                axes, s, 0, A, rot, None, None, 1e-6, 1.0, A, A, 4096, 4096, 8, ps,
                                A, 4, 4, A, cu, B, A, None)


@pytest.mark.parametrize("bad,status", [
    (dict(B=-1), -1), (dict(Hq=5), -1), (dict(Hkv=0), -1), (dict(D=96), -5), (dict(ps=24), -5),
    (dict(ps=8), -5), (dict(ks=100), -1), (dict(ks=4100), -2), (dict(st=12), -2),
    (dict(sh=-8), -2), (dict(st=0), -2), (dict(window=-1), -1), (dict(sinks=-1), -1), (dict(ts=3), -1),
    (dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1), (dict(table=None), -1),
    (dict(q=P(0x10008)), -2), (dict(k=P(0x10002)), -2), (dict(lens=P(0x10001)), -2),
    (dict(Hq=2 * 129), -5), (dict(mp=1 << 28, ts=1 << 28), -5), (dict(n=-1), -1)])
def test_decode_refuses(lib, bad, status):
    assert decode(lib, **bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(T=-1), -1), (dict(cu=None), -1), (dict(B=0), -1), (dict(D=32), -5), (dict(ps=0), -5),
    (dict(window=-3), -1), (dict(sinks=-1), -1), (dict(st=4), -2), (dict(out=None), -1),
    (dict(cu=P(0x10002)), -2), (dict(T=1 << 30), -5)])
def test_prefill_refuses(lib, bad, status):
    assert prefill(lib, **bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(T=3), -1), (dict(axes=0), -1), (dict(axes=5), -1), (dict(sec=None), -1),
    (dict(sec=(6, 5, 4)), -1), (dict(sec=(-1, 9, 8)), -1), (dict(rot=144, sec=(72, 0, 0)), -1),
    (dict(rot=24, sec=(12, 0, 0)), -5), (dict(st=20), -2), (dict(pos=None), -1),
    (dict(pos=P(0x10004)), -2), (dict(pos_stride=1), -1), (dict(q=P(0x10001)), -2), (dict(ps=1), -5)])
def test_rope_refuses(lib, bad, status):
    assert rope(lib, **bad) == status


def test_empty_calls_are_no_ops(lib):
    assert decode(lib, B=0) == 0 and prefill(lib, T=0) == 0 and rope(lib, T=0, B=0) == 0
    assert lib.pmoe_pages_grow(A, 8, 16, A, 4, 4, 3, A, A, A, 0, A, A, 1 << 20, None) == 0
    assert lib.pmoe_pages_fork(A, 8, 4, 16, 64, A, A, 4, 4, 3, A, A, A, A, 0, A, A, 1 << 20, None) == 0
    assert lib.pmoe_pages_free(A, 8, 16, A, 4, 4, 3, A, A, 0, 0, 0, None) == 0


def test_page_operations_refuse(lib):
    grow = lambda n_pages=8, ps=16, ts=4, mp=4, S=3, n=2, slots=A, ws=A, nb=1 << 20: \
        lib.pmoe_pages_grow(A, n_pages, ps, A, ts, mp, S, A, slots, A, n, A, ws, nb, None)  # noqa: E731
    assert grow(ps=20) == -5 and grow(ts=3) == -1 and grow(n=-1) == -1 and grow(S=-1) == -1
    assert grow(slots=None) == -1 and grow(ws=None) == -3 and grow(nb=16) == -3
    assert grow(slots=P(0x10001)) == -2 and grow(n_pages=-1) == -1
    fork = lambda chunks=4, D=64, n=2, pages=A, src=A, nb=1 << 20: \
        lib.pmoe_pages_fork(pages, 8, chunks, 16, D, A, A, 4, 4, 3, A, src, A, A, n, A, A, nb, None)  # noqa: E731
    assert fork(chunks=0) == -1 and fork(D=12) == -5 and fork(pages=None) == -1
    assert fork(src=None) == -1 and fork(nb=8) == -3 and fork(pages=P(0x10008)) == -2
    assert lib.pmoe_pages_free(A, 8, 16, A, 4, 4, 3, A, A, 2, -1, 0, None) == -1
    assert lib.pmoe_pages_free(A, 8, 16, A, 4, 4, 3, A, A, 2, 1, -1, None) == -1
    assert lib.pmoe_pages_free(A, 8, 16, A, 4, 4, 3, None, A, 2, 0, 0, None) == -1
    comp = lambda live=A, remap=A, nb=1 << 20: \
        lib.pmoe_pages_compact(A, 8, 4, 16, 64, A, A, 4, 4, 3, live, remap, A, nb, None)  # noqa: E731
    assert comp(live=None) == -1 and comp(remap=None) == -1 and comp(nb=0) == -3
    n = ctypes.c_size_t()
    assert lib.pmoe_pages_workspace(3, 2, 8, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.pmoe_pages_workspace(-1, 2, 8, ctypes.byref(n)) == -1


def test_meta_shapes_and_no_cpu_path():
    from paris_moe_b200 import ops
    m = dict(device="meta", dtype=torch.bfloat16)
    i = dict(device="meta", dtype=torch.int32)
    q, kv = torch.empty(5, 4, 64, **m), torch.empty(9, 2, 16, 64, **m)
    t, n, cu = torch.empty(2, 3, **i), torch.empty(2, **i), torch.empty(3, **i)
    assert ops.attn_decode(q, kv, kv, t, n, 1.0).shape == q.shape
    assert ops.attn_prefill(q, kv, kv, t, n, cu, 1.0, 8, 2).shape == q.shape
    pages, refs = torch.empty(9, 1, 2, 2, 16, 64, **m), torch.empty(9, **i)
    assert ops.pages_grow(refs, t, n, n, n, 16).shape == (2,)
    assert ops.pages_fork(pages, refs, t, n, n, n, n).shape == (2,)
    live, remap = ops.pages_compact(pages, refs, t)
    assert live.shape == (1,) and remap.shape == (9,)
    c = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.attn_decode(c, c[:, None], c[:, None], z[:, None], z, 1.0)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.pages_free(z, z[:, None], z, z, 16)


def test_cache_sizes_are_checked():
    from paris_moe_b200 import PagedKVCache
    for bad in (dict(page_size=24), dict(head_dim=96), dict(n_pages=0), dict(max_len=0)):
        kw = dict(n_pages=4, page_size=16, layers=1, kv_heads=1, head_dim=64, max_seqs=2,
                  max_len=40, device="cpu") | bad
        with pytest.raises(ValueError):
            PagedKVCache(**kw)
    c = PagedKVCache(4, 16, 3, 2, 64, 2, 40, device="cpu")
    assert c.tables.shape == (2, 3) and c.k(1).shape == (4, 2, 16, 64)
    assert c.v(2).data_ptr() - c.k(2).data_ptr() == 2 * 16 * 64 * 2


# ---- the plain forms themselves -----------------------------------------------------------


def test_plain_attention_agrees_with_softmax_over_a_mask():
    g = torch.Generator().manual_seed(0)
    D, ps, n = 64, 16, 37
    pages = torch.randn(4, 1, 2, 1, ps, D, generator=g).to(R.BF16)
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32), torch.tensor([n])
    q = torch.randn(5, 2, D, generator=g).to(R.BF16)
    cu = torch.tensor([0, 5])
    for window, sinks in ((0, 0), (9, 0), (9, 3), (1, 0), (64, 5)):
        out, _ = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], table, lens, cu, 0.1, window, sinks)
        k = pages[[2, 0, 3], 0, 0, 0].reshape(-1, D)[:n].double()
        v = pages[[2, 0, 3], 0, 1, 0].reshape(-1, D)[:n].double()
        for t in range(5):
            bias = torch.where(R.visible(n - 5 + t, n, window, sinks), 0.0, -math.inf)
            want = torch.softmax(q[t].double() @ k.T * 0.1 + bias, -1) @ v
            assert torch.allclose(out[t], want, atol=1e-12)


def test_plain_rope_turns_pairs():
    x = torch.randn(3, 2, 64).double()
    pos = torch.tensor([[0, 1, 50], [0, 7, 2]])
    f = torch.tensor([1.0, 0.5, 0.25, 0.125, 0.1, 0.01, 0.02, 0.03])
    y, _ = R.rope(x, pos, f, [5, 3], True)
    assert torch.equal(y[0], x[0]) and torch.equal(y[..., 16:], x[..., 16:])
    assert torch.allclose(y.pow(2).sum(-1), x.pow(2).sum(-1))
    assert [R.axis_of(i, 3, [4, 2, 2], True) for i in range(8)] == [0, 1, 2, 0, 1, 2, 0, 0]
    assert [R.axis_of(i, 2, [5, 3], False) for i in range(8)] == [0] * 5 + [1] * 3


def test_plain_page_bookkeeping_keeps_its_invariants():
    rng = random.Random(1)
    c = R.Cache(20, 16, 6, 5)
    for _ in range(400):
        op = rng.randrange(5)
        n = rng.randrange(4)
        slots = [rng.randrange(-1, 7) for _ in range(n)]
        if op == 0:
            c.grow(slots, [rng.randrange(-1, 40) for _ in slots])
        elif op == 1:
            c.fork(slots, [rng.randrange(-1, 7) for _ in slots], [rng.randrange(60) for _ in slots])
        elif op == 2:
            c.free(slots)
        elif op == 3:
            c.free(slots, 17, rng.randrange(20))
        else:
            c.compact()
        held = [p for row in c.tables for p in row if p >= 0]
        assert [held.count(p) for p in range(20)] == c.refs
        for n, row in zip(c.lens, c.tables):
            assert all(p < 0 for p in row[-(-n // 16):])
            assert n % 16 == 0 or c.refs[row[n // 16]] == 1     # a partly filled page has one owner

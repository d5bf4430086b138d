"""Refusals of the paged-cache and logit-adjustment entry points: bad arguments raise before anything is launched (no
GPU needed), and the 64-bit oracle against small hand-made cases."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import paged as opaged


@pytest.fixture(scope="module")
def L():
    from ai_b200 import build, _lib
    build.build()
    return _lib.lib()


def kv(**kw):
    from ai_b200._lib import PagedKv
    a = dict(k=1 << 20, v=1 << 21, page_stride=4096, head_stride=2048, row_stride=128, pages=4, page=16, KV=2, HD=128)
    a.update(kw)
    return PagedKv(*(a[n] for n, _ in PagedKv._fields_))


A = C.c_void_p(1 << 20)  # stands for a device pointer: never read by a refused call


def append(L, c=None, **kw):
    a = dict(table=A, ld=4, width=4, pos=A, cu=None, B=2, T=2, H=4, q=A, k=A, v=A, q_out=A, dtype=0)
    a.update(kw)
    return L.aib_paged_append(C.byref(c or kv()), a["table"], a["ld"], a["width"], a["pos"], a["cu"], a["B"], a["T"],
                              a["H"], a["q"], 512, 128, a["k"], 256, 128, a["v"], 256, 128, a["q_out"], 512, 128,
                              a["dtype"], None, None, None, 1e-6, None)


def attn(L, c=None, **kw):
    a = dict(table=A, ld=4, width=4, pos=A, B=2, H=4, q=A, q_ld=512, out=A, out_ld=512, dtype=0, lse=None, window=0,
             scale=0.1, ws=A, n=1 << 40)
    a.update(kw)
    return L.aib_paged_attn(C.byref(c or kv()), a["table"], a["ld"], a["width"], a["pos"], a["B"], a["H"], a["q"],
                            a["q_ld"], a["out"], a["out_ld"], a["dtype"], a["lse"], a["window"], a["scale"], a["ws"],
                            a["n"], None)


BAD_CACHE = [(dict(k=None), -1), (dict(v=None), -1), (dict(pages=0), -1), (dict(KV=0), -1), (dict(HD=96), -4),
             (dict(page=0), -1), (dict(page=24), -1), (dict(k=(1 << 20) + 8), -1), (dict(row_stride=132), -1),
             (dict(page_stride=-4096), -1), (dict(head_stride=64), -1), (dict(row_stride=0), -1)]


@pytest.mark.parametrize("bad,code", BAD_CACHE)
def test_bad_caches_are_refused(L, bad, code):
    assert append(L, kv(**bad)) == code and L.aib_last_error().startswith(b"aib_paged_append")
    assert attn(L, kv(**bad)) == code and L.aib_last_error().startswith(b"aib_paged_attn")


@pytest.mark.parametrize("bad", [dict(table=None), dict(pos=None), dict(k=None), dict(v=None), dict(B=0), dict(T=0),
                                 dict(T=3), dict(width=0), dict(dtype=2), dict(H=-1), dict(H=0), dict(q=None),
                                 dict(q_out=None), dict(k=C.c_void_p((1 << 20) + 2))])
def test_append_refusals(L, bad):
    assert append(L, **bad) == -1 and L.aib_last_error().startswith(b"aib_paged_append")


@pytest.mark.parametrize("bad,code", [(dict(table=None), -1), (dict(pos=None), -1), (dict(q=None), -1),
                                      (dict(out=None), -1), (dict(B=0), -1), (dict(B=4097), -4), (dict(H=3), -1),
                                      (dict(H=0), -1), (dict(window=-1), -1), (dict(dtype=3), -1), (dict(width=0), -1),
                                      (dict(ws=None), -3), (dict(n=1), -3), (dict(width=1 << 27), -4),
                                      (dict(width=1 << 26, B=4096, ld=1 << 26), -4)])
def test_attention_refusals(L, bad, code):
    assert attn(L, **bad) == code and L.aib_last_error().startswith(b"aib_paged_attn")


@pytest.mark.parametrize("bad,code", [
    (dict(x=None), -1), (dict(out=None), -1), (dict(B=0), -1), (dict(V=0), -1), (dict(dtype=2), -1),
    (dict(out_ld=9), -1), (dict(n_prior=1), -1), (dict(n_bias=1), -1), (dict(n_prior=-1), -1), (dict(ld=-1), -1),
    (dict(prior=A, n_prior=32768), -4), (dict(ids=A, bias=A, n_bias=1025), -4), (dict(x=C.c_void_p((1 << 20) + 2)), -1)])
def test_adjust_refusals(L, bad, code):
    a = dict(x=A, ld=10, out=A, out_ld=10, dtype=0, B=2, V=10, prior=None, n_prior=0, ids=None, bias=None, n_bias=0)
    a.update(bad)
    rc = L.aib_adjust_logits(a["x"], a["ld"], a["out"], a["out_ld"], a["dtype"], a["B"], a["V"], a["prior"], 0,
                             a["n_prior"], None, None, None, a["ids"], 0, a["bias"], 0, a["n_bias"], None, 0, None)
    assert rc == code and L.aib_last_error().startswith(b"aib_adjust_logits")


def test_workspace_query(L):
    assert L.aib_paged_attn_workspace(1, 8, 2, 128) > 0
    for bad in ((0, 8, 2, 128), (1, 7, 2, 128), (1, 8, 2, 96), (1, 0, 2, 128)):
        assert L.aib_paged_attn_workspace(*bad) == 0


def test_python_wrappers_refuse_cpu_tensors():
    from ai_b200 import paged, sampler
    with pytest.raises(ValueError):
        paged.Cache(torch.zeros(2, 2, 16, 64).bfloat16(), torch.zeros(2, 2, 16, 64).bfloat16())
    with pytest.raises(ValueError):
        sampler.adjust(torch.zeros(2, 10))


# ----------------------------------------------------------------------------------------------- oracle
def test_oracle_append_and_attention_by_hand():
    kc, vc = np.zeros((3, 1, 2, 4)), np.zeros((3, 1, 2, 4))
    table = np.array([[2, 0], [1, -1]])
    k = np.arange(12, dtype=float).reshape(3, 1, 4) / 8
    q, at = opaged.append(kc, vc, table, [1, 1], [0, 2, 3], None, k, k + 1, None, None, None, 0.0)
    assert q is None and at == [(2, 1), (0, 0), (1, 1)]
    assert (kc[2, 0, 1] == k[0, 0]).all() and (vc[0, 0, 0] == k[1, 0] + 1).all()
    x = np.array([[[1.0, 0, 0, 0]], [[0, 1.0, 0, 0]]])
    out, lse, _, _ = opaged.attention(x, kc, vc, table, [2, 2], 2, 1.0)
    s = np.array([kc[2, 0, 1, 0], kc[0, 0, 0, 0]])  # sequence 0, the last two positions
    w = np.exp(s) / np.exp(s).sum()
    np.testing.assert_allclose(out[0, 0], w[0] * vc[2, 0, 1] + w[1] * vc[0, 0, 0])
    np.testing.assert_allclose(lse[0, 0], np.log(np.exp(s).sum()))
    np.testing.assert_allclose(out[1, 0], vc[1, 0, 1])  # position 2 is on a page outside the pool
    # rotation keeps lengths and turns by the angle; norm gives unit mean square times the weight
    v = np.array([3.0, 0, 4.0, 0])
    r = opaged.norm_rope(v, None, np.array([0.5, 1.0]), 3, 0.0)
    np.testing.assert_allclose(np.hypot(r[0], r[2]), 5.0)
    np.testing.assert_allclose(np.arctan2(r[2], r[0]) - np.arctan2(4.0, 3.0), 1.5)
    np.testing.assert_allclose((opaged.norm_rope(v, np.full(4, 2.0), None, 0, 0.0) ** 2).mean(), 4.0)


def test_oracle_adjust_by_hand():
    mask = np.array([0b01111], np.uint32).view(np.int32)
    x, _ = opaged.adjust([2.0, -2.0, 1.0, 0.0, 9.0], [0, 1, 1, -1, 7], 2.0, 0.5, 0.25, [2, 2, 9], [1.0, 3.0, 5.0], mask)
    np.testing.assert_array_equal(x, [2.0 / 2 - 0.75, -4.0 - 1.0, 5.0, 0.0, -np.inf])


# ------------------------------------------------------------------------------------------------ pages
def test_pages_are_handed_out_and_come_back():
    from ai_b200 import paged
    p = paged.Pages(6, 3, 4, 16, "cpu")
    p.grow(0, 17)
    p.grow(2, 48)
    p.grow(0, 32)  # fits what it has
    held = p.table.tolist()
    assert [sum(x >= 0 for x in r) for r in held] == [2, 0, 3]
    used = [x for r in held for x in r if x >= 0]
    assert len(set(used)) == 5 and len(p.left) == 1
    with pytest.raises(ValueError):
        p.grow(1, 33)  # more than are free: nothing is taken
    assert len(p.left) == 1 and p.table[1].tolist() == [-1] * 4
    with pytest.raises(ValueError):
        p.grow(0, 65)  # wider than the table
    p.free(2)
    p.grow(1, 64)
    assert sum(x >= 0 for x in p.table[1].tolist()) == 4 and not p.left
    assert p.table[2].tolist() == [-1] * 4
    assert not set(p.table[1].tolist()) & set(p.table[0, :2].tolist())
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            paged.Pages(*bad, "cpu")

"""C entry points of the paged cache and the logit adjustment: which overlaps, alignments and sizes they refuse. The
addresses are made up. A refused call reads nothing; one that would be accepted is only made where there is no GPU, so that
its launch fails before it can reach one."""
import ctypes as C

import numpy as np
import pytest
import torch

EINVAL, ECUDA, EWORKSPACE, ENOTSUP = -1, -2, -3, -4


@pytest.fixture(scope="module")
def L():
    from ai_b200 import build, _lib
    build.build()
    return _lib.lib()


@pytest.fixture
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("an accepted call would be launched")


def at(element, size=4):
    """Address of an element of one buffer."""
    return C.c_void_p((1 << 20) + element * size)


def adjust(L, x, ld, out, out_ld, B, V, dtype=0, **kw):
    a = dict(prior=None, n_prior=0, rep=None, ids=None, bias=None, n_bias=0, mask=None)
    a.update(kw)
    return L.aib_adjust_logits(x, ld, out, out_ld, dtype, B, V, a["prior"], 0, a["n_prior"], a["rep"], None, None, a["ids"],
                               0, a["bias"], 0, a["n_bias"], a["mask"], 0, None)


# ---------------------------------------------------------------------------------------------- adjust
@pytest.mark.parametrize("x,ld,out,out_ld,B,V", [
    (0, 10, 0, 12, 2, 10),     # the same start, rows further apart
    (0, 12, 0, 10, 2, 10),
    (0, 0, 0, 10, 2, 10),      # one row for all, written as the first
    (0, 10, 5, 10, 1, 10),     # half a row on
    (0, 20, 19, 20, 3, 10),    # interleaved, one element too many on either side
    (0, 20, 9, 20, 3, 10),
    (0, 20, 29, 20, 1, 30),
    (100, 40, 5, 40, 3, 35),   # its last row is elements 85 .. 119
    (100, 7, 0, 40, 4, 5),     # rows of two distances that meet somewhere
])
def test_adjust_refuses_an_out_that_shares_memory_with_the_logits(L, x, ld, out, out_ld, B, V):
    assert adjust(L, at(x), ld, at(out), out_ld, B, V) == EINVAL
    assert L.aib_last_error().startswith(b"aib_adjust_logits")


def test_adjust_takes_rows_that_interleave_apart(L, no_gpu):
    for x, ld, out, out_ld, B, V in ((0, 20, 10, 20, 3, 10), (10, 20, 0, 20, 3, 10), (0, 10, 0, 10, 4, 10),
                                     (0, 10, 0, 12, 1, 10), (0, 0, 10, 10, 4, 10),
                                     (0, 10, 40, 10, 4, 10), (5, 30, 12, 20, 2, 3)):
        assert adjust(L, at(x), ld, at(out), out_ld, B, V) == ECUDA, (x, ld, out, out_ld, B, V)


def test_adjust_overlap_is_exact(L, no_gpu):
    """Random rows against the sets of their elements."""
    r = np.random.default_rng(1)
    seen = [0, 0]
    for _ in range(3000):
        B, V = int(r.integers(1, 5)), int(r.integers(1, 7))
        ld, out_ld = int(r.integers(0, 16)), int(r.integers(V, 16))
        x, out = (int(v) for v in r.integers(0, 40, 2))
        a = {x + b * ld + i for b in range(B) for i in range(V)}
        z = {out + b * out_ld + i for b in range(B) for i in range(V)}
        same = x == out and (B == 1 or ld == out_ld)
        bad = bool(a & z) and not same
        seen[bad] += 1
        assert adjust(L, at(x), ld, at(out), out_ld, B, V) == (EINVAL if bad else ECUDA), (x, ld, out, out_ld, B, V)
    assert min(seen) > 500


# --------------------------------------------------------------------------------------- paged attention
def kv(**kw):
    from ai_b200._lib import PagedKv
    a = dict(k=1 << 30, v=1 << 31, page_stride=4096, head_stride=2048, row_stride=128, pages=4, page=16, KV=2, HD=128)
    a.update(kw)
    return PagedKv(*(a[n] for n, _ in PagedKv._fields_))


A = C.c_void_p(1 << 26)


def attend(L, c=None, **kw):
    a = dict(table=A, ld=4, width=4, pos=A, B=2, H=4, q=at(0), q_ld=512, out=at(1024), out_ld=512, dtype=0, lse=None,
             window=0, ws=None, n=0)
    a.update(kw)
    return L.aib_paged_attn(C.byref(c or kv()), a["table"], a["ld"], a["width"], a["pos"], a["B"], a["H"], a["q"],
                            a["q_ld"], a["out"], a["out_ld"], a["dtype"], a["lse"], a["window"], 0.1, a["ws"], a["n"], None)


def append(L, c=None, **kw):
    a = dict(table=A, ld=4, width=4, pos=A, cu=None, B=2, T=2, H=4, q=at(0), q_s=(512, 128), k=at(10000), k_s=(256, 128),
             v=at(20000), v_s=(256, 128), q_out=at(30000), qo_s=(512, 128), dtype=0, qn=None, kn=None, inv=None)
    a.update(kw)
    return L.aib_paged_append(C.byref(c or kv()), a["table"], a["ld"], a["width"], a["pos"], a["cu"], a["B"], a["T"],
                              a["H"], a["q"], *a["q_s"], a["k"], *a["k_s"], a["v"], *a["v_s"], a["q_out"], *a["qo_s"],
                              a["dtype"], a["qn"], a["kn"], a["inv"], 1e-6, None)


def off(n):
    return C.c_void_p((1 << 26) + n)


# ------------------------------------------------------------------------------------------- alignment
@pytest.mark.parametrize("bad", [dict(table=off(2)), dict(pos=off(4)), dict(q=off(2)), dict(out=off(3)), dict(lse=off(2)),
                                 dict(dtype=1, q=off(1)), dict(dtype=1, out=off(1))])
def test_attention_refuses_addresses_off_their_elements(L, bad):
    assert attend(L, **bad) == EINVAL and L.aib_last_error().startswith(b"aib_paged_attn")


@pytest.mark.parametrize("bad", [dict(table=off(2)), dict(pos=off(4)), dict(cu=off(1)), dict(inv=off(2)), dict(qn=off(1)),
                                 dict(kn=off(1)), dict(v=off(2)), dict(dtype=1, q_out=off(1))])
def test_append_refuses_addresses_off_their_elements(L, bad):
    assert append(L, **bad) == EINVAL and L.aib_last_error().startswith(b"aib_paged_append")


@pytest.mark.parametrize("bad", [dict(prior=off(2), n_prior=3), dict(rep=off(1)), dict(ids=off(2), bias=A, n_bias=3),
                                 dict(ids=A, bias=off(2), n_bias=3), dict(mask=off(2))])
def test_adjust_refuses_addresses_off_their_elements(L, bad):
    assert adjust(L, at(0), 10, at(100), 10, 2, 10, **bad) == EINVAL
    assert L.aib_last_error().startswith(b"aib_adjust_logits")

"""C entry points of the paged cache and the logit adjustment: which overlaps, alignments and sizes they refuse. The
addresses are made up. A refused call reads nothing; one that would be accepted is only made where there is no GPU, so that
its launch fails before it can reach one."""
import ctypes as C

import numpy as np
import pytest
import torch

EINVAL, ECUDA = -1, -2


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
    for _ in range(400):
        B, V = int(r.integers(1, 5)), int(r.integers(1, 7))
        ld, out_ld = int(r.integers(0, 16)), int(r.integers(V, 16))
        x, out = (int(v) for v in r.integers(0, 40, 2))
        a = {x + b * ld + i for b in range(B) for i in range(V)}
        z = {out + b * out_ld + i for b in range(B) for i in range(V)}
        same = x == out and (B == 1 or ld == out_ld)
        bad = bool(a & z) and not same
        seen[bad] += 1
        assert adjust(L, at(x), ld, at(out), out_ld, B, V) == (EINVAL if bad else ECUDA), (x, ld, out, out_ld, B, V)
    assert min(seen) > 60


# --------------------------------------------------------------------------------------- paged attention
def kv(**kw):
    from ai_b200._lib import PagedKv
    a = dict(k=1 << 30, v=1 << 31, page_stride=4096, head_stride=2048, row_stride=128, pages=4, page=16, KV=2, HD=128)
    a.update(kw)
    return PagedKv(*(a[n] for n, _ in PagedKv._fields_))


A = C.c_void_p(1 << 26)


def attend(L, c=None, **kw):
    a = dict(table=A, ld=4, width=4, pos=A, B=2, H=4, q=at(0), q_ld=512, out=at(1024), out_ld=512, dtype=0, lse=None,
             window=0, ws=C.c_void_p(1 << 27), n=1 << 30)
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


# -------------------------------------------------------------------------------------------- overlaps
@pytest.mark.parametrize("bad", [
    dict(q_out=at(0), qo_s=(1024, 128)), dict(q_out=at(0), qo_s=(512, 256)),  # q with other strides
    dict(q_out=at(128)),                                   # a head further
    dict(q_out=at(10000)), dict(q_out=at(20000 + 511)),    # k, the last element of v
    dict(q=at(0), q_s=(1024, 128), k=at(512), k_s=(1024, 128), v=at(768), v_s=(1024, 128), q_out=at(400), qo_s=(1024, 128)),
    dict(qo_s=(128, 128)), dict(qo_s=(0, 128)), dict(qo_s=(512, 0)), dict(qo_s=(512, 64)),  # its own rows meet
    dict(q_s=(128, 256), q_out=at(128), qo_s=(256, 256), k=at(5000)),
])
def test_append_refuses_a_q_out_that_shares_memory(L, bad):
    assert append(L, **bad) == EINVAL and L.aib_last_error().startswith(b"aib_paged_append")


def test_append_takes_cuts_of_one_buffer(L, no_gpu):
    fused = dict(q=at(0), q_s=(1024, 128), k=at(512), k_s=(1024, 128), v=at(768), v_s=(1024, 128), T=2)
    assert append(L, **fused) == ECUDA
    assert append(L, **fused, q_out=at(0), qo_s=(1024, 128)) == ECUDA  # in place, k and v between its rows
    wide = {k: (s[0] + 512, s[1]) if k.endswith("_s") else s for k, s in fused.items()}
    assert append(L, **wide, q_out=at(1024), qo_s=(1536, 128)) == ECUDA
    # heads apart, tokens between them: [heads, T, HD]
    assert append(L, q=at(0), q_s=(128, 256), q_out=at(1024), qo_s=(128, 256), k=at(2048), k_s=(128, 256), v=at(2560),
                  v_s=(128, 256)) == ECUDA
    assert append(L, q=at(0), q_s=(128, 512), q_out=at(256), qo_s=(128, 512), k=at(4096)) == ECUDA


def test_append_overlap_is_exact(L, no_gpu):
    """Random strides against the sets of their elements (64 wide heads, two sequences' tokens)."""
    r = np.random.default_rng(2)
    seen = [0, 0]
    c = kv(HD=64, KV=1, head_stride=64, row_stride=64, page_stride=1024)

    def rows(base, ts, hs, T, H):
        return [base + t * ts + h * hs + i for t in range(T) for h in range(H) for i in range(64)]

    for _ in range(600):
        T, H = int(r.integers(1, 5)), int(r.integers(1, 4))
        ts, hs = (int(v) * 16 for v in r.permutation(r.integers(1, 24, 2)))
        big, small = max(ts, hs), min(ts, hs)
        n_small = H if small == hs else T
        if small < 64 or big < (n_small - 1) * small + 64:
            continue  # (rows of q_out that meet are refused anyway; what may interleave more finely is not looked at)
        if r.random() < 0.5:
            qts, qhs = ts, hs
        else:
            qts, qhs = (int(v) * 16 for v in r.integers(0, 24, 2))
        q, qo = (int(v) * 16 for v in r.integers(0, 60, 2))
        same = q == qo and (T == 1 or ts == qts) and (H == 1 or hs == qhs)
        bad = not same and bool(set(rows(q, qts, qhs, T, H)) & set(rows(qo, ts, hs, T, H)))
        seen[bad] += 1
        cu = C.c_void_p(1 << 26)
        got = append(L, c, q=at(q), q_s=(qts, qhs), q_out=at(qo), qo_s=(ts, hs), T=T, B=1, cu=cu, H=H, k_s=(64, 64),
                     v_s=(64, 64))
        assert got == (EINVAL if bad else ECUDA), (T, H, q, qts, qhs, qo, ts, hs)
    assert min(seen) > 60


@pytest.mark.parametrize("bad", [dict(out=at(0)), dict(out=at(511)), dict(out=at(512), out_ld=1024, q_ld=512),
                                 dict(out=at(256), out_ld=1024, q_ld=1024), dict(out_ld=511), dict(out_ld=0),
                                 dict(lse=at(1024)), dict(lse=at(0)), dict(lse=at(1024 + 1023))])
def test_attention_refuses_outputs_that_share_memory(L, bad):
    assert attend(L, **bad) == EINVAL and L.aib_last_error().startswith(b"aib_paged_attn")


def test_attention_takes_rows_that_interleave_apart(L, no_gpu):
    for ok in (dict(), dict(out=at(512), out_ld=1024, q_ld=1024), dict(q=at(512), q_ld=1030, out=at(0), out_ld=1030),
               dict(lse=at(2048)), dict(q_ld=0, out=at(512)), dict(lse=at(512), q_ld=1024, out=at(4096))):
        assert attend(L, **ok) == ECUDA, ok


# ------------------------------------------------------------------------------------------------ pools
OVERLAPS = [dict(page_stride=2048, head_stride=2048),                      # a page's second head is the next page's first
            dict(page_stride=128, head_stride=2048, row_stride=128),
            dict(page_stride=4096, head_stride=128, row_stride=128),        # heads among the rows
            dict(page_stride=4096, head_stride=2048 - 128, row_stride=128), # the last row is the next head's first
            dict(page_stride=4096 - 8, head_stride=2048, row_stride=128),
            dict(page_stride=2048, head_stride=128, row_stride=256, pages=2, page=16)]
APART = [dict(), dict(head_stride=128, row_stride=256), dict(page_stride=8192, head_stride=128, row_stride=512),
         dict(page_stride=128, head_stride=512 * 16, row_stride=512), dict(KV=1, head_stride=8, page_stride=2048),
         dict(pages=1, page_stride=0), dict(page=1, row_stride=0, head_stride=128, page_stride=256),
         dict(page_stride=2 ** 61, head_stride=2048)]


@pytest.mark.parametrize("bad", OVERLAPS)
def test_pools_whose_rows_overlap_are_refused(L, bad):
    assert append(L, kv(**bad)) == EINVAL and attend(L, kv(**bad)) == EINVAL
    assert b"overlap" in L.aib_last_error()


def test_pools_of_every_order_are_taken(L, no_gpu):
    for ok in APART:
        assert append(L, kv(**ok)) == ECUDA, ok

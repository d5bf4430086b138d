"""Paged cache and logit adjustment at the edges of what their documentation allows."""

import numpy as np
import pytest
import torch

from oracle import paged as opaged

pytestmark = pytest.mark.gpu
E32, EBF = 2.0 ** -24, 2.0 ** -8  # half a step relative to the value
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def mod(cuda_dev):
    from ai_b200 import build, _lib, paged, sampler
    build.build()
    _lib.status(clear=True)
    return paged, sampler, _lib


def f64(t):
    return t.detach().double().cpu().numpy()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(*rows, dtype=torch.int32):
    return torch.tensor(rows if len(rows) > 1 else rows[0], dtype=dtype, device="cuda")


# ---------------------------------------------------------------------------------------------- adjust
@pytest.mark.parametrize("dtype", list(DT))
def test_adjust_rows_that_interleave_in_one_buffer(mod, dtype):
    """Logits and out as two cuts of the same rows, either first, share no memory: the same numbers as with an out of its
    own, and nothing between them is touched."""
    _, sampler, lib = mod
    g = gen(1)
    for V, gap in ((40, 0), (1003, 5)):
        buf = torch.randn(5, 2 * V + gap, generator=g, device="cuda").to(DT[dtype])
        prior, one = torch.randint(0, V, (5, 30), generator=g, device="cuda", dtype=torch.int32), torch.ones(5, device="cuda")
        for x, out in ((buf[:, :V], buf[:, V + gap:]), (buf[:, V + gap:], buf[:, :V])):
            before = buf.clone()
            want = sampler.adjust(x, out=torch.empty(5, V, dtype=buf.dtype, device="cuda"), prior=prior, presence=one)
            sampler.adjust(x, out=out, prior=prior, presence=one)
            assert torch.equal(out, want)
            out.copy_(before[:, V + gap:] if out.data_ptr() != buf.data_ptr() else before[:, :V])
            assert torch.equal(buf, before)
    assert lib.status() == 0


# ---------------------------------------------------------------------------------------------- append
def test_append_positions_at_the_end_of_64_bits(mod):
    """A first position so far out that its tokens' positions leave 64 bits lies past the table, as all far ones do."""
    paged, _, lib = mod
    g = gen(2)
    k0, v0 = (torch.randn(6, 2, 8, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    for first in (2 ** 63 - 1, 2 ** 63 - 2, 2 ** 62, 2 ** 31, 16):
        c = paged.Cache(k0.clone(), v0.clone())
        table = ints([0, 1], [2, 3])
        k, v = (torch.randn(7, 2, 64, generator=g, device="cuda") for _ in range(2))
        paged.append(c, table, ints([first, 5], dtype=torch.int64), k, v, cu=ints([0, 4, 7]))
        assert lib.status() == 104
        want_k, want_v = k0.clone(), v0.clone()
        for t in range(3):  # the neighbour's rows are written, and nothing else
            page, row = 2 + (5 + t) // 8, (5 + t) % 8
            want_k[page, :, row], want_v[page, :, row] = k[4 + t].bfloat16(), v[4 + t].bfloat16()
        assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v), first


def test_outputs_that_share_memory_are_refused(mod):
    """By the wrappers too, before anything is launched; cuts of one fused row stay allowed."""
    paged, _, lib = mod
    g = gen(3)
    c = paged.Cache(*(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    table, pos = ints([0, 1], [2, 3]), ints([3, 17], dtype=torch.int64)
    rows = torch.randn(2, 8, 64, generator=g, device="cuda")
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    square = torch.randn(4, 4, 64, generator=g, device="cuda")
    before = rows.clone()
    for bad in (dict(q_out=rows[:, 1:5]), dict(q_out=rows[:, 3:7]), dict(q_out=torch.zeros(1, 4, 64, device="cuda").expand(2, 4, 64)),
                dict(q=square[:2], q_out=square[:, :2].transpose(0, 1))):
        with pytest.raises(ValueError):
            paged.append(c, table, pos, k, v, **{"q": q, **bad})
    q2 = torch.randn(2, 4, 64, generator=g, device="cuda")
    for bad in (dict(out=q2), dict(out=torch.empty(2, 4, 64, device="cuda"), lse=q2.view(-1)[:8].view(2, 4))):
        with pytest.raises(ValueError):
            paged.attention(q2, c, table, pos, **bad)
    assert torch.equal(rows, before) and not c.k.any() and not c.v.any()
    want = paged.append(c, table, pos, k, v, q=q, q_out=torch.empty(2, 4, 64, device="cuda"), qn=torch.ones(64, device="cuda").bfloat16())
    paged.append(c, table, pos, k, v, q=q, q_out=q, qn=torch.ones(64, device="cuda").bfloat16())
    assert torch.equal(rows[:, :4], want) and torch.equal(rows[:, 4:], before[:, 4:])
    assert lib.status() == 0


# ------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("page,HD", [(16, 64), (1, 128), (2, 128)])
def test_attention_windows_beyond_the_cache(mod, page, HD):
    """Windows as large as their type allows are no windows; those up to the length cut where they should."""
    paged, _, lib = mod
    g = gen(4)
    pos, pages = [70, 3, -1, 511], 600 // page + 8
    c = paged.Cache(*(torch.randn(pages, 2, page, HD, generator=g, device="cuda").bfloat16() for _ in range(2)))
    table = torch.randperm(pages, generator=g, device="cuda")[:512 // page].to(torch.int32).expand(4, -1).contiguous()
    q, p = torch.randn(4, 6, HD, generator=g, device="cuda"), torch.tensor(pos, device="cuda")
    full = paged.attention(q, c, table, p)
    for window in (512, 513, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 63 - 33, 2 ** 63 - 32, 2 ** 63 - 1, 2 ** 64 + 5):
        assert torch.equal(paged.attention(q, c, table, p, window=window), full), window
    ref, lse, mag, dot = opaged.attention(f64(q), f64(c.k), f64(c.v), table.cpu().numpy(), pos, 71, HD ** -0.5)
    got = f64(paged.attention(q, c, table, p, window=71))
    # a score: HD + 8 roundings of sum |q||k| and 4 of its own, twice (numerator and sum); 71 + 64 of the sums, twice
    shift = (HD + 8) * E32 * dot + 4 * E32 * np.abs(np.where(np.isinf(lse), 0, lse))
    assert (np.abs(got - ref) <= (2 * shift[..., None] + 2 * (71 + 64) * E32) * mag + E32 * np.abs(ref)).all()
    assert lib.status() == 0


@pytest.mark.parametrize("dtype", list(DT))
def test_append_without_rotation_keeps_neighbours_of_infinities(mod, dtype):
    """Without rotation no element of a row enters another: rows are copied as they are, whatever they hold. With a
    norm an infinite element leaves zeros beside itself."""
    paged, _, lib = mod
    for HD in (64, 128):
        g = gen(5)
        c = paged.Cache(*(torch.zeros(3, 2, 8, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
        k, v, q = (torch.randn(5, n, HD, generator=g, device="cuda").to(DT[dtype]) for n in (2, 2, 3))
        k[1, 0, 3], k[2, 1, HD // 2 + 5], k[3, 0, 9] = float("inf"), float("-inf"), float("nan")
        k[4, 1, 0], k[4, 1, HD // 2] = -0.0, 0.0
        q[0, 2, HD - 1], q[4, 0, 0], v[2, 0, 1] = float("inf"), float("nan"), float("inf")
        q_out = torch.empty_like(q)
        paged.append(c, ints([[2, 0]]), ints([6], dtype=torch.int64), k, v, cu=ints([0, 5]), q=q, q_out=q_out)
        at = [(2, 6), (2, 7), (0, 0), (0, 1), (0, 2)]
        bits = lambda t: t.view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)  # noqa: E731
        for t, (i, r) in enumerate(at):
            for got, want in ((c.k[i, :, r], k[t].bfloat16()), (c.v[i, :, r], v[t].bfloat16()), (q_out[t], q[t])):
                nan = want.isnan()
                assert torch.equal(got.isnan(), nan) and torch.equal(bits(got)[~nan], bits(want)[~nan])
        w = torch.ones(HD, device="cuda").bfloat16()
        paged.append(c, ints([[2, 0]]), ints([6], dtype=torch.int64), k, v, cu=ints([0, 5]), kn=w)
        got = c.k[2, 0, 7]  # token 1, head 0
        assert got[3].isnan() and not got[:3].any() and not got[4:].any()
    assert lib.status() == 0


def attend_with_lse(paged, q, c, table, pos, **kw):
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    return paged.attention(q, c, table, ints(pos, dtype=torch.int64), lse=lse, **kw), lse


@pytest.mark.parametrize("HD", [64, 128])
def test_attention_scores_that_are_all_minus_infinity(mod, HD):
    """No weight is left, so the output is NaN and the log of the sum -inf; rows with a finite score among them count
    alone; a row that attends nothing keeps zeros."""
    paged, _, lib = mod
    g = gen(6)
    pos, page, pages = [0, 45, 2999, 2999, 700, -1], 16, 480
    k, v = (torch.randn(pages, 2, page, HD, generator=g, device="cuda").bfloat16() for _ in range(2))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(6, 188, dtype=torch.int32, device="cuda")
    n = [-(-(p + 1) // page) for p in pos]
    for b in range(5):
        table[b, :n[b]] = order[sum(n[:b]):sum(n[:b + 1])]
    q = torch.randn(6, 6, HD, generator=g, device="cuda").bfloat16()
    q[:, :, 2] = 1.0
    for b in (0, 1, 2):  # every key of these
        k[table[b, :n[b]].long(), :, :, 2] = -float("inf")
    k[table[3, :90].long(), :, :, 2] = -float("inf")  # rows 0 .. 1439 of this one
    k[table[4, 40].long(), :, 4:9, 2] = -float("inf")
    c = paged.Cache(k, v)
    out, lse = attend_with_lse(paged, q, c, table, pos)
    assert out[:3].isnan().all() and (lse[:3] == -float("inf")).all()
    assert not out[5].any() and (lse[5] == -float("inf")).all()
    with np.errstate(invalid="ignore"):
        ref, rl, mag, _ = opaged.attention(f64(q), f64(k), f64(v), table.cpu().numpy(), [-1, -1, -1, 2999, 700, -1], 0,
                                           HD ** -0.5)
    # scores: |q||k| <= sqrt(3 HD) * sqrt(2 HD) and the scale give below 3 sqrt(HD) in size, HD + 8 roundings of it
    tol = 2 * (HD + 8) * E32 * 3 * HD ** 0.5 + 2 * (3000 + 64) * E32 + 2 * 2.0 ** -16
    assert (np.abs(f64(out) - ref)[3:5] <= tol * mag[3:5] + EBF * np.abs(ref[3:5])).all()
    assert np.abs(f64(lse)[3:5] - rl[3:5]).max() <= tol + 4 * E32 * 12
    # a window that holds no finite score, and one that does
    out, lse = attend_with_lse(paged, q[3:4], c, table[3:4], [1439], window=300)
    assert out.isnan().all() and (lse == -float("inf")).all()
    out, _ = attend_with_lse(paged, q[3:4], c, table[3:4], [1440], window=300)
    torch.testing.assert_close(out[0].float(), v[table[3, 90].long(), :, 0].repeat_interleave(3, 0).float(), rtol=2 * EBF, atol=0)
    assert lib.status() == 0


@pytest.mark.parametrize("HD", [64, 128])
def test_attention_fp32_queries_at_the_end_of_their_range(mod, HD):
    """fp32 queries above the largest bf16 number (3.39e38): the scores are those of the definition. Infinite ones make
    their heads NaN and no others."""
    paged, _, lib = mod
    g = gen(7)
    pos, page = [40, 700, 5], 16
    k = torch.randn(64, 2, page, HD, generator=g, device="cuda")
    k[..., 1] *= 1e-38 / HD ** 0.5  # what meets the large element
    k[..., 4] = k[..., 4].abs() + 0.25
    c = paged.Cache(k.bfloat16(), torch.randn(64, 2, page, HD, generator=g, device="cuda").bfloat16())
    table = torch.randperm(64, generator=g, device="cuda")[:44].to(torch.int32).expand(3, -1).contiguous()
    top = torch.finfo(torch.float32).max
    q = torch.randn(3, 4, HD, generator=g, device="cuda")
    q[0, :, 1] = torch.tensor([top, -top, 3.3953e38, 3.3895e38], device="cuda")
    q[1, :, 1] = torch.tensor([3.4e38, -3.392e38, 3.2e38, -top], device="cuda")
    out, lse = attend_with_lse(paged, q, c, table, pos)
    ref, rl, mag, dot = opaged.attention(f64(q), f64(c.k), f64(c.v), table.cpu().numpy(), pos, 0, HD ** -0.5)
    shift = (HD + 8) * E32 * dot + 4 * E32 * np.abs(rl)
    assert (np.abs(f64(out) - ref) <= (2 * shift[..., None] + 2 * (701 + 64) * E32) * mag + E32 * np.abs(ref)).all()
    assert (np.abs(f64(lse) - rl) <= shift + (701 + 64) * E32 + 4 * E32 * (1 + np.abs(rl))).all()
    q[:, 1, 4] = -float("inf")
    q[:, 2, 4] = float("inf")
    out, lse = attend_with_lse(paged, q, c, table, pos)
    assert out[:, 1:3].isnan().all() and not torch.isfinite(lse[:, 1:3]).any()
    assert torch.isfinite(out[:, [0, 3]]).all() and torch.isfinite(lse[:, [0, 3]]).all()
    assert lib.status() == 0


# ------------------------------------------------------------------------------------------- the step
def test_unused_rows_stay_unused_as_the_batch_advances(mod):
    """A negative position marks an unused row: a step leaves its position, its id and its ring alone."""
    _, _, lib = mod
    from ai_b200._lib import ptr, stream_ptr
    for B in (3, 16, 70):
        pos = torch.arange(B, device="cuda") * 3
        pos[1::3] = -1
        pos[2::5] = -2 ** 62
        ids, out_ids = torch.arange(B, device="cuda") + 100, torch.arange(B, device="cuda") + 500
        ring = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
        used = pos >= 0
        want_pos, want_ids, want_ring = torch.where(used, pos + 2, pos), torch.where(used, out_ids, ids), ring.clone()
        for b in torch.nonzero(used).flatten().tolist():
            for s in (1, 2):
                want_ring[b, (pos[b].item() + s) % 8] = 500 + b
        for r in (ring, None):
            p, i = pos.clone(), ids.clone()
            for _ in range(2):
                lib.call("aib_batch_advance_prior", ptr(p), ptr(i), ptr(out_ids), B, ptr(r), 8 if r is not None else 0,
                         8 if r is not None else 0, stream_ptr())
            assert torch.equal(p, want_pos) and torch.equal(i, want_ids)
        assert torch.equal(ring, want_ring)
        p, i = pos.clone(), ids.clone()
        lib.call("aib_batch_advance", ptr(p), ptr(i), ptr(out_ids), B, stream_ptr())  # this one knows no unused rows
        assert torch.equal(p, pos + 1) and torch.equal(i, out_ids)
    assert lib.status() == 0


def test_a_captured_step_with_unused_rows(mod):
    """Append, attention and advance replayed: the unused row writes to no page, its table's entries notwithstanding."""
    paged, _, lib = mod
    from ai_b200._lib import ptr, stream_ptr
    g = gen(8)
    c = paged.Cache(*(torch.zeros(6, 1, 8, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    table = ints([0, 1], [2, 3], [4, 5])
    pos, ids, out_ids = ints([3, -1, 6], dtype=torch.int64), ints([0, 0, 0], dtype=torch.int64), ints([7, 8, 9], dtype=torch.int64)
    ring, ws = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), paged.workspace(3, 2, c)
    q, k, v = (torch.randn(3, n, 64, generator=g, device="cuda") for n in (2, 1, 1))
    out = torch.full((3, 2, 64), 5.0, device="cuda")

    def step():
        paged.append(c, table, pos, k, v)
        paged.attention(q, c, table, pos, out=out, ws=ws)
        lib.call("aib_batch_advance_prior", ptr(pos), ptr(ids), ptr(out_ids), 3, ptr(ring), 4, 4, stream_ptr())

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        graph.replay()
    assert pos.tolist() == [8, -1, 11] and ids.tolist() == [7, 0, 9] and ring[1].tolist() == [-1] * 4
    assert not c.k[2:4].any() and not c.v[2:4].any() and not out[1].any()
    want = k.bfloat16()
    for b, first in ((0, 3), (2, 6)):
        for p in range(first, first + 5):
            assert torch.equal(c.k[table[b, p // 8].item(), :, p % 8], want[b])
    assert lib.status() == 0

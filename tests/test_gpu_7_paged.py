"""Paged cache (append, attention) and logit adjustment against 64-bit definitions.

Tolerances count roundings (half a step relative to the value: fp32 2^-24, bf16 2^-8):
  append: norm and rotation take fewer than 32 fp32 roundings of numbers no larger than the pair's length, the sum of
    HD squares enters with half its relative error (HD / 2 at most); the cache adds one bf16 rounding.
  attention: a score carries (HD + 8) roundings of sum |q||k| and 4 of itself, which shifts its weight by that much
    relative (twice: numerator and sum); sums over n weights carry at most n + 64 roundings of sum p|v| and as many of
    the sum of p. With bf16 rows the weights are held in two bf16 parts (2^-16) and the output is rounded once.
  adjust: fewer than 8 + (biases of the id) roundings of the terms' magnitudes; bf16 output rounded once.
"""

import numpy as np
import pytest
import torch

from oracle import paged as opaged

pytestmark = pytest.mark.gpu
E32, EBF = 2.0 ** -24, 2.0 ** -8
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


def make_cache(paged, pages, KV, page, HD, g, order="heads", fill=None):
    """Pool of one layer; order 'rows': the heads of a row are neighbours; 'fused': k and v interleaved by page."""
    if order == "heads":
        k, v = (torch.randn(pages, KV, page, HD, generator=g, device="cuda").bfloat16() for _ in range(2))
    elif order == "rows":
        k, v = (torch.randn(pages, page, KV, HD, generator=g, device="cuda").bfloat16().transpose(1, 2)
                for _ in range(2))
    else:
        kv = torch.randn(pages, 2, KV, page, HD, generator=g, device="cuda").bfloat16()
        k, v = kv[:, 0], kv[:, 1]
    if fill is not None:
        k.fill_(fill)
        v.fill_(fill)
    return paged.Cache(k, v)


def make_table(lens, page, pages, g, width=None):
    """Random distinct pages for every sequence; entries past a sequence's need are out of the pool's range."""
    need = [-(-max(n, 0) // page) for n in lens]
    width = width or max(max(need), 1)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(lens), width), 1 << 30, dtype=torch.int32, device="cuda")
    k = 0
    for b, n in enumerate(need):
        t[b, :n] = order[k:k + n]
        k += n
    assert k <= pages
    return t


def inv_of(HD, theta=1e6):
    return 1.0 / (theta ** (torch.arange(0, HD, 2, dtype=torch.float32, device="cuda") / HD))


# ---------------------------------------------------------------------------------------------- append
APPEND = [  # new tokens of each sequence, first positions, H, KV, HD, page, order
    ([1], [0], 4, 2, 128, 16, "heads"),
    ([1, 1, 1], [5, -1, 1000], 32, 8, 128, 64, "fused"),
    ([3, 0, 17, 1], [0, 7, 15, 100003], 14, 2, 64, 16, "rows"),
    ([40, 33], [1, 62], 3, 1, 128, 1, "heads"),
    ([70, 5], [250, 2 ** 20 + 1], 8, 8, 64, 256, "heads"),
    ([0, 0, 9], [3, 4, 5], 16, 1, 128, 8, "rows"),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (False, False), (True, False)])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(mod, case, norm, rope, dtype):
    paged, _, lib = mod
    new, pos, H, KV, HD, page, order = APPEND[case]
    g = gen(case)
    base = [max(0, p) // page for p in pos]  # pages before the first written one are not needed
    lens = [max(0, p) % page + n for p, n in zip(pos, new)]
    pages = sum(-(-n // page) for n in lens) + 2
    c = make_cache(paged, pages, KV, page, HD, g, order)
    part = make_table(lens, page, pages, g)
    table = torch.full((len(new), max(base) + part.shape[1]), -7, dtype=torch.int32, device="cuda")
    for b, s in enumerate(base):
        table[b, s:s + part.shape[1]] = part[b]
    T, pad = sum(new), 2
    qkv = (torch.randn(T + pad, (H + 2 * KV) * HD, generator=g, device="cuda") * 3).to(DT[dtype])
    q, k, v = (t.view(T + pad, -1, HD) for t in qkv.split([H * HD, KV * HD, KV * HD], 1))
    cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32, device="cuda")
    qn, kn = ((1 + 0.2 * torch.randn(2, HD, generator=g, device="cuda")).bfloat16() if norm else (None, None))
    inv = inv_of(HD) if rope else None
    q_out = torch.full((T + pad, H, HD), 77.0, dtype=DT[dtype], device="cuda")
    k0, v0 = f64(c.k), f64(c.v)
    paged.append(c, table, torch.tensor(pos, device="cuda"), k, v, cu=cu, q=q, q_out=q_out, qn=qn, kn=kn, inv=inv,
                 eps=1e-6)
    opt = lambda t: None if t is None else f64(t)  # noqa: E731
    rq, at = opaged.append(k0, v0, table.cpu().numpy(), pos, cu.tolist(), f64(q), f64(k), f64(v), opt(qn), opt(kn),
                           opt(inv), 1e-6)
    rel = (32 + HD / 2) * E32
    half = HD // 2

    def check(got, want, last):
        size = np.sqrt(want ** 2 + np.roll(want, half, -1) ** 2)  # the pair's length
        bad = np.abs(got - want) > rel * size + last * (np.abs(want) + rel * size)
        assert not bad.any(), np.abs(got - want).max()

    wrote = ~np.isnan(rq[:, 0, 0])
    assert (f64(q_out)[~wrote] == 77.0).all()
    check(f64(q_out)[wrote], rq[wrote], EBF if dtype == "bf16" else E32)
    i, r = [a for a, _ in at], [a for _, a in at]
    if at:
        check(f64(c.k)[i, :, r], k0[i, :, r], EBF)
        np.testing.assert_array_equal(f64(c.v)[i, :, r], f64(v.bfloat16())[wrote])
    left = np.ones((pages, page), bool)
    left[i, r] = False
    for got, want in ((c.k, k0), (c.v, v0)):  # every other row as it was
        np.testing.assert_array_equal(f64(got).transpose(0, 2, 1, 3)[left], want.transpose(0, 2, 1, 3)[left])
    assert lib.status() == 0


def test_append_in_place_and_without_q(mod):
    paged, _, lib = mod
    g = gen(1)
    c, d = (make_cache(paged, 4, 2, 16, 128, gen(2)) for _ in range(2))
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([17, 3], device="cuda")
    q, k, v = (torch.randn(2, n, 128, generator=g, device="cuda") for n in (6, 2, 2))
    q_out = torch.empty_like(q)
    paged.append(c, table, pos, k, v, q=q, q_out=q_out, inv=inv_of(128))
    paged.append(d, table, pos, k, v, inv=inv_of(128))
    assert torch.equal(c.k, d.k) and torch.equal(c.v, d.v)
    paged.append(d, table, pos, k, v, q=q, q_out=q, inv=inv_of(128))
    assert torch.equal(q, q_out) and lib.status() == 0


def test_append_odd_strides(mod):
    """Rows whose strides and start allow no paired access."""
    paged, _, lib = mod
    g = gen(4)
    for dt in DT.values():
        c, d = (make_cache(paged, 4, 2, 16, 128, gen(2)) for _ in range(2))
        table = torch.tensor([[3, 1]], dtype=torch.int32, device="cuda")
        pos, cu = torch.tensor([9], device="cuda"), torch.tensor([0, 5], dtype=torch.int32, device="cuda")
        wide = torch.randn(5, 7, 129, generator=g, device="cuda").to(dt)
        q, k, v = wide[:, 0:3, 1:], wide[:, 3:5, 1:], wide[:, 5:7, 1:]
        out, odd = torch.empty(5, 3, 128, dtype=dt, device="cuda"), torch.empty(5, 3, 131, dtype=dt, device="cuda")
        paged.append(c, table, pos, k.contiguous(), v.contiguous(), cu=cu, q=q.contiguous(), q_out=out,
                     inv=inv_of(128))
        paged.append(d, table, pos, k, v, cu=cu, q=q, q_out=odd[..., 3:], inv=inv_of(128))
        assert torch.equal(c.k, d.k) and torch.equal(c.v, d.v) and torch.equal(out, odd[..., 3:])
    assert lib.status() == 0


def test_append_bad_pages_and_positions(mod):
    """Rows past the table and page ids outside the pool are left out, recorded, and harm no neighbour."""
    paged, _, lib = mod
    g = gen(5)
    c = make_cache(paged, 3, 1, 8, 64, g)
    k0 = c.k.clone()
    k, v = torch.ones(3, 1, 64, device="cuda"), torch.ones(3, 1, 64, device="cuda")
    for bad, code in ((-1, 107), (3, 107), (2 ** 31 - 1, 107)):
        table = torch.tensor([[0], [bad], [2]], dtype=torch.int32, device="cuda")
        paged.append(c, table, torch.tensor([1, 2, 3], device="cuda"), k, v)
        assert lib.status() == code
    paged.append(c, torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda"),
                 torch.tensor([1, 8, 3], device="cuda"), k, v)
    assert lib.status() == 104
    k0[0, 0, 1] = 1
    k0[2, 0, 3] = 1
    assert torch.equal(c.k, k0)


# ------------------------------------------------------------------------------------------- attention
def run_attention(paged, c, q, table, pos, window, scale=None, ws=None, lse=True):
    out = torch.full_like(q, float("nan"))
    z = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None
    paged.attention(q, c, table, torch.as_tensor(pos, device="cuda"), out=out, scale=scale, window=window, lse=z, ws=ws)
    return out, z


def check_attention(c, q, table, pos, window, scale, out, lse, kv=None):
    HD = q.shape[2]
    kd, vd = kv or (f64(c.k), f64(c.v))
    ref, rl, mag, dot = opaged.attention(f64(q), kd, vd, table.cpu().numpy(), pos, window, scale)
    n = max(1, max(pos) + 1 if not window else min(window, max(pos) + 1))
    bf = q.dtype == torch.bfloat16
    shift = (HD + 8) * E32 * dot + 4 * E32 * np.abs(np.where(np.isinf(rl), 0, rl))  # error of a score
    tol = (2 * shift[..., None] + 2 * (n + 64) * E32 + (2 * 2.0 ** -16 if bf else 0)) * mag
    tol += (EBF if bf else E32) * np.abs(ref) + 1e-30
    bad = ~(np.abs(f64(out) - ref) <= tol)
    assert not bad.any(), (np.abs(f64(out) - ref).max(), tol.min())
    if lse is not None:
        got = f64(lse)
        np.testing.assert_array_equal(np.isinf(got), np.isinf(rl))
        ok = ~np.isinf(rl)
        lt = shift + (n + 64) * E32 + 4 * E32 * (1 + np.abs(np.where(ok, rl, 0))) + (2.0 ** -16 if bf else 0)
        assert (np.abs(got - np.where(ok, rl, 0))[ok] <= lt[ok]).all()


ATTENTION = [  # positions, H, KV, HD, page, window, order
    ([0], 4, 2, 128, 16, 0, "heads"),
    ([0, -1, 1, 15, 16, 17, 31, 32], 32, 8, 128, 16, 0, "heads"),
    ([516], 32, 8, 128, 64, 0, "fused"),
    ([5000, 3, 700, -1, 2047], 32, 8, 128, 64, 0, "rows"),
    ([100, 1000, 33], 14, 2, 64, 32, 0, "heads"),
    ([100, 1000, 33], 14, 2, 64, 32, 40, "rows"),
    ([300, 2, 7], 5, 5, 64, 1, 0, "heads"),
    ([300, 900], 16, 1, 128, 8, 0, "rows"),
    ([300, 901], 9, 1, 128, 8, 1, "heads"),
    ([2000], 40, 2, 64, 256, 333, "fused"),
    ([20000], 8, 8, 128, 128, 0, "heads"),
    ([64 * i + i % 3 - 1 for i in range(70)], 6, 2, 128, 16, 0, "heads"),
    ([(37 * i) % 90 for i in range(300)], 4, 4, 64, 8, 20, "heads"),
    ([-1, -1], 4, 2, 128, 16, 0, "heads"),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention(mod, case, dtype):
    paged, _, lib = mod
    pos, H, KV, HD, page, window, order = ATTENTION[case]
    g = gen(100 + case)
    pages = sum(-(-(p + 1) // page) for p in pos) + 2
    c = make_cache(paged, pages, KV, page, HD, g, order)
    table = make_table([p + 1 for p in pos], page, pages, g)
    q = (torch.randn(len(pos), H, HD, generator=g, device="cuda") * 2).to(DT[dtype])
    out, lse = run_attention(paged, c, q, table, pos, window)
    check_attention(c, q, table, pos, window, HD ** -0.5, out, lse)
    again, _ = run_attention(paged, c, q, table, pos, window)
    assert torch.equal(out, again)  # the same sums in the same order
    assert lib.status() == 0


def test_attention_garbage_outside_the_attended_rows(mod):
    """NaN and infinities in rows past the new token, before the window, and in pages of other sequences."""
    paged, _, lib = mod
    for HD, dtype in ((128, "f32"), (64, "bf16")):
        g = gen(7)
        pos, page, window = [0, 45, 130, 31, -1], 16, 50
        c = make_cache(paged, 30, 2, page, HD, g)
        table = make_table([p + 1 for p in pos], page, 30, g)
        kd, vd = f64(c.k), f64(c.v)
        mark = torch.zeros(30, page, dtype=torch.bool, device="cuda")
        for b, p in enumerate(pos):
            for j in range(max(0, p + 1 - window), p + 1):
                mark[table[b, j // page].long(), j % page] = True
        junk = ~mark[:, None, :, None].expand_as(c.k)
        c.k.masked_fill_(junk, float("nan"))
        c.v.masked_fill_(junk, float("inf"))
        q = torch.randn(5, 6, HD, generator=g, device="cuda").to(DT[dtype])
        out, lse = run_attention(paged, c, q, table, pos, window)
        check_attention(c, q, table, pos, window, HD ** -0.5, out, lse, (kd, vd))
    assert lib.status() == 0


def test_attention_nan_queries_and_keys(mod):
    """A NaN query head gives NaN there and nowhere else; a NaN key gives NaN to its group."""
    paged, _, lib = mod
    for HD, dtype in ((128, "f32"), (64, "bf16")):
        g = gen(27)
        pos = [0, 40, 900]
        c = make_cache(paged, 70, 2, 16, HD, g)
        table = make_table([p + 1 for p in pos], 16, 70, g)
        q = torch.randn(3, 8, HD, generator=g, device="cuda").to(DT[dtype])
        q[:, 1, 3] = float("nan")
        out, lse = run_attention(paged, c, q, table, pos, 0)
        assert out[:, 1].isnan().all() and lse[:, 1].isnan().all()
        keep = [0, 2, 3, 4, 5, 6, 7]
        assert not out[:, keep].isnan().any()
        c.k[table[2, 30].long(), 1, 5, 7] = float("nan")
        out, lse = run_attention(paged, c, q, table, pos, 0)
        assert out[2, 4:].isnan().all() and lse[2, 4:].isnan().all() and not out[2, [0, 2, 3]].isnan().any()
        assert not out[:2, keep].isnan().any()
    assert lib.status() == 0


def test_attention_bad_pages_and_positions(mod):
    """Rows on pages outside the pool, or past the table, are left out and recorded."""
    paged, _, lib = mod
    g = gen(8)
    c = make_cache(paged, 12, 2, 8, 64, g)
    table = make_table([30, 40, 9], 8, 12, g)
    table[0, 1], table[1, 0], table[2, 0], table[2, 1] = -1, 12, 2 ** 31 - 1, -2 ** 31
    q = torch.randn(3, 4, 64, generator=g, device="cuda")
    pos = [29, 39, 8]
    out, lse = run_attention(paged, c, q, table, pos, 0)
    check_attention(c, q, table, pos, 0, 64 ** -0.5, out, lse)
    assert lib.status() == 107
    table = make_table([24, 40], 8, 12, g)
    pos = [10 ** 12, 39]
    table[0, 3:] = table[0, :2]
    out, lse = run_attention(paged, c, q[:2], table, pos, 0)
    check_attention(c, q[:2], table, [39, 39], 0, 64 ** -0.5, out, lse)
    assert lib.status() == 104


def test_attention_scales_and_large_scores(mod):
    paged, _, lib = mod
    g = gen(9)
    c = make_cache(paged, 40, 2, 16, 128, g)
    table = make_table([333, 300], 16, 40, g)
    q = torch.randn(2, 4, 128, generator=g, device="cuda")
    for scale in (1.0, 0.0, -0.3, 4.0):
        out, lse = run_attention(paged, c, q, table, [332, 299], 0, scale=scale)
        check_attention(c, q, table, [332, 299], 0, scale, out, lse)
    assert lib.status() == 0


def test_attention_far_offsets(mod):
    """Cache rows more than 2^31 elements (and 2^32 bytes) into the pool."""
    paged, _, lib = mod
    g = gen(10)
    pages, KV, page, HD = 34000, 4, 64, 128  # k and v fused: 2.2e9 elements
    pool = torch.zeros(pages, 2, KV, page, HD, dtype=torch.bfloat16, device="cuda")
    pos = [900]
    ids = torch.tensor([[33999, 3, 32800, 17000] + list(range(33900, 33911))], dtype=torch.int32, device="cuda")
    for i in ids[0].tolist():
        pool[i].normal_(generator=g)
    assert pool.numel() > 2 ** 31
    c = paged.Cache(pool[:, 0], pool[:, 1])
    k, v = (torch.randn(1, KV, HD, generator=g, device="cuda") for _ in range(2))
    paged.append(c, ids, torch.tensor(pos, device="cuda"), k, v)
    assert torch.equal(pool[ids[0, 900 // 64].item(), 0, :, 900 % 64], k[0].bfloat16())
    q = torch.randn(1, 8, HD, generator=g, device="cuda")
    out, lse = run_attention(paged, c, q, ids, pos, 0)
    at = ids[0].long()
    small = torch.arange(at.numel(), dtype=torch.int32, device="cuda")[None]
    check_attention(None, q, small, pos, 0, HD ** -0.5, out, lse, (f64(pool[at, 0]), f64(pool[at, 1])))
    assert lib.status() == 0


def test_attention_workspace_survives_other_shapes(mod):
    """One workspace over calls of different batches and lengths in one stream, then the first call again."""
    paged, _, lib = mod
    g = gen(11)
    c = make_cache(paged, 600, 2, 16, 128, g)
    ws = paged.workspace(300, 16, c)
    first = None
    for pos, H in (([4000], 4), ([(31 * i) % 30 for i in range(300)], 16), ([8000, 100], 2), ([4000], 4)):
        table = make_table([p + 1 for p in pos], 16, 600, gen(12))
        q = torch.randn(len(pos), H, 128, generator=gen(13), device="cuda")
        out, lse = run_attention(paged, c, q, table, pos, 0, ws=ws)
        check_attention(c, q, table, pos, 0, 128 ** -0.5, out, lse)
        first = out if first is None else first
    assert torch.equal(first, out) and lib.status() == 0


def test_step_captured_on_another_stream(mod):
    """Append, attention and adjustment captured as one step on a side stream and replayed as the sequences grow,
    against the same calls made one by one."""
    paged, sampler, lib = mod
    B, H, KV, HD, page, V, steps = 3, 8, 2, 64, 16, 500, 40
    g = gen(14)
    caches = [make_cache(paged, 40, KV, page, HD, gen(15)) for _ in range(2)]
    start = [0, 14, 130]
    table = make_table([p + steps + 1 for p in start], page, 40, g)
    qkv = torch.randn(steps, B, H + 2 * KV, HD, generator=g, device="cuda")
    logits = torch.randn(B, V, generator=g, device="cuda")
    prior = torch.randint(0, V, (B, 50), generator=g, device="cuda", dtype=torch.int32)
    rep = torch.full((B,), 1.3, device="cuda")

    def step(c, rows, pos, q_out, out, adj, ws):
        paged.append(c, table, pos, rows[:, H:H + KV], rows[:, H + KV:], q=rows[:, :H], q_out=q_out, inv=inv_of(HD))
        paged.attention(q_out, c, table, pos, out=out, ws=ws)
        sampler.adjust(logits, out=adj, prior=prior, repetition=rep)
        pos += 1

    want = []
    pos = torch.tensor(start, device="cuda")
    for s in range(steps):
        q_out, out, adj = torch.empty(B, H, HD, device="cuda"), torch.empty(B, H, HD, device="cuda"), logits.clone()
        step(caches[0], qkv[s], pos, q_out, out, adj, None)
        want.append((out, adj))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        rows, pos = torch.zeros_like(qkv[0]), torch.full((B,), -1, device="cuda")
        q_out, out, adj = torch.empty(B, H, HD, device="cuda"), torch.empty(B, H, HD, device="cuda"), logits.clone()
        ws = paged.workspace(B, H, caches[1])
        step(caches[1], rows, pos, q_out, out, adj, ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(caches[1], rows, pos, q_out, out, adj, ws)
        pos.copy_(torch.tensor(start))
        for s in range(steps):
            rows.copy_(qkv[s])
            graph.replay()
            assert torch.equal(out, want[s][0]) and torch.equal(adj, want[s][1]), s
    side.synchronize()
    assert torch.equal(caches[0].k, caches[1].k) and lib.status() == 0


def test_attention_wait_runs_out_reports_status_and_recovers(mod):
    """Copies that never come: every wait gives up, the status says so, and the context stays usable."""
    paged, _, lib = mod
    g = gen(21)
    pos, page = [700, 5, 90], 16
    c = make_cache(paged, 60, 2, page, 128, g)
    table = make_table([p + 1 for p in pos], page, 60, g)
    q = torch.randn(3, 8, 128, generator=g, device="cuda")
    ws = paged.workspace(3, 8, c)
    lib.call("aib_debug_knob", 1, 4096)
    lib.call("aib_debug_knob", 2, 1)
    try:
        run_attention(paged, c, q, table, pos, 0, ws=ws)
        torch.cuda.synchronize()
        st = lib.status(clear=True)
    finally:
        lib.call("aib_debug_knob", 2, 0)
        lib.call("aib_debug_knob", 1, 0)
    assert st == 101
    ws.zero_()
    out, lse = run_attention(paged, c, q, table, pos, 0, ws=ws)
    check_attention(c, q, table, pos, 0, 128 ** -0.5, out, lse)
    assert lib.status() == 0


@pytest.mark.parametrize("HD,dtype", [(128, "f32"), (64, "bf16")])
def test_attention_batches_of_every_size(mod, HD, dtype):
    """From one row to the largest batch, with rows of one token, unused rows and a shared table row."""
    paged, _, lib = mod
    g = gen(22)
    page, KV, H = 4, 1, 2
    c = make_cache(paged, 512, KV, page, HD, g)
    for B in (1, 2, 257, 4096):
        r = np.random.default_rng(B)
        pos = [int(p) for p in r.choice([-1, 0, 1, 3, 4, 30, 31, 32, 33, 70], B)]
        table = torch.randint(0, 512, (1, 18), generator=g, device="cuda", dtype=torch.int32).expand(B, 18)
        q = torch.randn(B, H, HD, generator=g, device="cuda").to(DT[dtype])
        out, lse = run_attention(paged, c, q, table, pos, 0)
        check_attention(c, q, table, pos, 0, HD ** -0.5, out, lse)
    assert lib.status() == 0


def test_attention_rows_apart_and_odd(mod):
    """q and out as cuts of wider rows, on addresses that allow no wide access; what lies between stays."""
    paged, _, lib = mod
    g = gen(23)
    pos, H, HD, page = [40, 300], 6, 64, 32
    c = make_cache(paged, 16, 2, page, HD, g, "rows")
    table = make_table([p + 1 for p in pos], page, 16, g)
    for dt in DT.values():
        wide = torch.randn(2, H * HD + 11, generator=g, device="cuda").to(dt)
        res = torch.full((2, H * HD + 7), 9.0, device="cuda", dtype=dt)
        q, out = wide[:, 3:3 + H * HD].view(2, H, HD), res[:, 5:5 + H * HD].view(2, H, HD)
        paged.attention(q, c, table, torch.tensor(pos, device="cuda"), out=out)
        check_attention(c, q.contiguous(), table, pos, 0, HD ** -0.5, out, None)
        assert (res[:, :5] == 9).all() and (res[:, 5 + H * HD:] == 9).all()
    assert lib.status() == 0


def test_graphs_that_share_a_workspace(mod):
    """Two captured calls with one workspace, replayed in turn in one stream, and an eager call between."""
    paged, _, lib = mod
    g = gen(24)
    c = make_cache(paged, 400, 2, 16, 128, g)
    ws = paged.workspace(8, 8, c)
    made = []
    for pos in ([3000], [700, 20, 1500]):
        table = make_table([p + 1 for p in pos], 16, 400, g)
        q = torch.randn(len(pos), 8, 128, generator=g, device="cuda")
        p = torch.tensor(pos, device="cuda")
        want = paged.attention(q, c, table, p, ws=ws).clone()
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.attention(q, c, table, p, out=out, ws=ws)
        made.append((graph, out, want, (q, c, table, p)))
    for _ in range(3):
        for graph, out, want, args in made:
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
            assert torch.equal(paged.attention(*args, ws=ws), want)
    assert lib.status() == 0


def test_calls_on_two_streams(mod):
    """Calls that overlap on the GPU, each with its own workspace, and one without a workspace of its own."""
    paged, sampler, lib = mod
    g = gen(25)
    c = make_cache(paged, 900, 2, 16, 128, g)
    jobs = []
    for pos in ([5000, 4], [2000, 2500, 300]):
        table = make_table([p + 1 for p in pos], 16, 900, g)
        q = torch.randn(len(pos), 8, 128, generator=g, device="cuda")
        p = torch.tensor(pos, device="cuda")
        x = torch.randn(len(pos), 50257, generator=g, device="cuda")
        prior = torch.randint(0, 500, (len(pos), 300), generator=g, device="cuda", dtype=torch.int32)
        rep = torch.full((len(pos),), 1.2, device="cuda")
        jobs.append((torch.cuda.Stream(), paged.workspace(len(pos), 8, c), (q, c, table, p), (x, prior, rep),
                     paged.attention(q, c, table, p), sampler.adjust(x.clone(), prior=prior, repetition=rep)))
    torch.cuda.synchronize()
    got = []
    for i in range(30):
        for stream, ws, args, (x, prior, rep), _, _ in jobs:
            with torch.cuda.stream(stream):
                got.append((paged.attention(*args, ws=ws if i % 3 else None),
                            sampler.adjust(x, out=torch.empty_like(x), prior=prior, repetition=rep)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, jobs[i % 2][4]) and torch.equal(b, jobs[i % 2][5])
    assert lib.status() == 0


def test_python_refusals(mod):
    """Shapes, types, strides and devices that do not fit raise ValueError before anything is launched."""
    paged, sampler, lib = mod
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    b, i32, i64 = torch.bfloat16, torch.int32, torch.int64
    kv = lambda *s: (z(*s, dtype=b), z(*s, dtype=b))  # noqa: E731
    for k, v in (kv(2, 2, 16, 96), kv(2, 2, 12, 64), (z(2, 2, 16, 64), z(2, 2, 16, 64)),
                 (kv(2, 2, 16, 64)[0], kv(2, 2, 8, 64)[0]), (kv(2, 2, 16, 65)[0][..., 1:],) * 2,
                 (kv(2, 2, 16, 128)[0][..., ::2],) * 2, (kv(1, 1, 16, 64)[0].expand(2, 2, 16, 64),) * 2,
                 (kv(2, 2, 16, 64)[0], kv(2, 2, 16, 64)[0].cpu())):
        with pytest.raises(ValueError):
            paged.Cache(k, v)
    c = paged.Cache(*kv(4, 2, 16, 64))
    t, p, k = z(3, 2, dtype=i32), z(3, dtype=i64), z(3, 2, 64)
    good = dict(cache=c, table=t, pos=p, k=k, v=k, q=z(3, 4, 64), q_out=z(3, 4, 64))
    for bad in (dict(table=z(2, 2, dtype=i32)), dict(table=z(3, 2, dtype=i64)), dict(table=t.cpu()),
                dict(table=z(3, 4, dtype=i32)[:, ::2]), dict(pos=z(3)), dict(pos=z(6, dtype=i64)[::2]), dict(pos=p.cpu()),
                dict(k=k.half()), dict(k=k.to(b)), dict(k=z(3, 2, 128)[..., ::2]), dict(v=z(3, 1, 64)),
                dict(q=z(3, 4, 128)), dict(q=z(3, 256)), dict(q_out=z(3, 256)), dict(q_out=None), dict(q_out=z(3, 4, 64).to(b)), dict(q=z(3, 4, 64).cpu()),
                dict(cu=z(3, dtype=i32)), dict(cu=z(4, dtype=i64)), dict(inv=z(64)), dict(inv=z(32).to(b)),
                dict(qn=z(64)), dict(kn=z(32, dtype=b)), dict(k=z(2, 2, 64), v=z(2, 2, 64), q=None, q_out=None)):
        with pytest.raises(ValueError):
            paged.append(**{**good, **bad})
    good = dict(q=z(3, 4, 64), cache=c, table=t, pos=p)
    for bad in (dict(q=z(3, 3, 64)), dict(q=z(2, 4, 64)), dict(q=z(3, 4, 64).half()), dict(q=z(3, 4, 64).cpu()),
                dict(q=z(3, 4, 128)), dict(q=z(3, 8, 64)[:, ::2]), dict(out=z(3, 4, 64).to(b)), dict(out=z(3, 2, 64)),
                dict(out=z(1, 4, 64).expand(3, 4, 64)), dict(lse=z(3)), dict(lse=z(4, 3).t()), dict(window=-1),
                dict(ws=z(1 << 20)), dict(ws=z(1, dtype=torch.uint8).cpu())):
        with pytest.raises(ValueError):
            paged.attention(**{**good, **bad})
    with pytest.raises(RuntimeError):
        paged.attention(**good, ws=z(64, dtype=torch.uint8))
    x, W = z(3, 70), z(3, 3, dtype=i32)
    wide = z(3, 80)
    for bad in (dict(logits=x[0]), dict(logits=x.half()), dict(logits=x.double()), dict(logits=z(3, 140)[:, ::2]),
                dict(out=z(3, 71)), dict(out=x.to(b)), dict(logits=wide[:, :70], out=wide[:, 10:]),
                dict(out=z(1, 70).expand(3, 70)), dict(prior=z(2, 5, dtype=i32)), dict(prior=z(3, 5, dtype=i64)),
                dict(prior=z(3, 5, dtype=i32).cpu()), dict(mask=z(3, 2, dtype=i32)), dict(mask=z(3, 6, dtype=i32)[:, ::2]),
                dict(bias_ids=W), dict(bias=z(3, 3)), dict(bias_ids=W, bias=z(3, 4)), dict(repetition=z(2)),
                dict(presence=z(3).double()), dict(frequency=z(6)[::2])):
        with pytest.raises(ValueError):
            sampler.adjust(**{"logits": x, **bad})
    with pytest.raises(RuntimeError):
        sampler.adjust(x, prior=z(3, 32768, dtype=i32), repetition=z(3))
    with pytest.raises(RuntimeError):
        sampler.adjust(x, bias_ids=z(3, 1025, dtype=i32), bias=z(3, 1025))
    # nothing to do: no tokens, no rows
    assert paged.append(c, z(0, 1, dtype=i32), z(0, dtype=i64), z(0, 2, 64), z(0, 2, 64)) is None
    assert paged.attention(z(0, 4, 64), c, z(0, 1, dtype=i32), z(0, dtype=i64)).shape == (0, 4, 64)
    assert sampler.adjust(z(0, 70)).shape == (0, 70) and sampler.adjust(z(3, 0)).shape == (3, 0)
    assert lib.status() == 0


# ---------------------------------------------------------------------------------------------- adjust
ADJUST = [  # B, V, prior ids, biases, mask, logits row stride beyond V, out row stride beyond V
    (1, 1, 0, 0, False, 0, 0),
    (1, 1, 3, 2, True, 0, 0),
    (3, 31, 5, 0, True, 1, 3),
    (2, 1000, 4096, 300, True, 0, 0),
    (5, 4099, 1, 1, False, 0, 5),
    (2, 50257, 600, 64, True, 0, 0),
    (2, 151936, 5000, 1024, True, 64, 0),
    (1, 9000, 32767, 7, False, 0, 0),
    (17, 8192, 0, 33, False, 0, 0),
    (4, 40000, 100, 0, False, 3, 3),
    (300, 77, 9, 4, True, 0, 0),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(ADJUST)))
def test_adjust(mod, case, dtype, inplace):
    _, sampler, lib = mod
    B, V, P, nb, masked, ex, ey = ADJUST[case]
    g = gen(200 + case)
    x = (torch.randn(B, V + ex, generator=g, device="cuda") * 5).to(DT[dtype])[:, :V]
    y = x if inplace else torch.full((B, V + ey), 55.0, dtype=DT[dtype], device="cuda")[:, :V]
    rnd = lambda n, lo, hi: torch.randint(lo, hi, (B, n), generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    prior = torch.minimum(rnd(P, -3, V + 3), rnd(P, 0, 40) * 11) if P else None  # many repeats
    ids = torch.minimum(rnd(nb, -2, V + 2), rnd(nb, 0, V + 2)) if nb else None
    if nb > 5:
        ids[:, 3], ids[:, 5] = ids[:, 1], ids[:, 1]  # one id three times
    bias = torch.randn(B, nb, generator=g, device="cuda") * 4 if nb else None
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device="cuda").to(torch.int32) \
        if masked else None
    if masked:
        mask[0] = 0  # a row whose mask leaves nothing
        x.masked_fill_(torch.rand(B, V, generator=g, device="cuda") < 0.01, float("-inf"))
    rep, pres, freq = (torch.rand(3, B, generator=g, device="cuda") + torch.tensor([[0.6], [-0.5], [-0.3]],
                                                                                  device="cuda"))
    rep[0], pres[0], freq[0] = 1.0, 0.0, 0.0  # a row with neutral penalties
    want, tol = np.zeros((B, V)), np.zeros((B, V))
    c = lambda t, b: None if t is None else t[b].cpu().numpy()  # noqa: E731
    for b in range(B):
        want[b], mag = opaged.adjust(f64(x[b]), c(prior, b), float(rep[b]), float(pres[b]), float(freq[b]), c(ids, b),
                                     c(bias, b), c(mask, b))
        tol[b] = (8 + nb) * E32 * np.where(np.isfinite(mag), mag, 0)
    got = sampler.adjust(x, out=None if inplace else y, prior=prior, repetition=rep, presence=pres, frequency=freq,
                         bias_ids=ids, bias=bias, mask=mask)
    assert got is y
    got = f64(got)
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    d = np.abs(got - np.where(inf, 0, want))[~inf]
    tol = (tol + (EBF if dtype == "bf16" else E32) * (np.abs(np.where(inf, 0, want)) + tol))[~inf]
    assert (d <= tol).all(), d.max()
    if not inplace and ey:
        assert (y._base[:, V:] == 55).all()
    assert lib.status() == 0


def test_adjust_matches_the_sampler(mod):
    """Greedy ids of adjusted logits are those of the sampler's own penalties and mask."""
    _, sampler, lib = mod
    g = gen(3)
    B, V = 8, 151936
    x = torch.randn(B, V, generator=g, device="cuda")
    prior = x.topk(200, 1).indices.to(torch.int32)
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, V // 32), generator=g, device="cuda").to(torch.int32)
    full = lambda a: torch.full((B,), a, device="cuda")  # noqa: E731
    want = sampler.sample(x, prior=prior, mask=mask, repetition_penalty=1.7, presence_penalty=0.4,
                          frequency_penalty=0.2)
    y = sampler.adjust(x, out=torch.empty_like(x), prior=prior, repetition=full(1.7), presence=full(0.4),
                       frequency=full(0.2), mask=mask)
    assert sampler.sample(y) == want and lib.status() == 0


def test_adjust_nan_and_shared_rows(mod):
    """NaN in masked places is masked, elsewhere it stays; one prior, bias and mask row for the whole batch."""
    _, sampler, lib = mod
    g = gen(5)
    x = torch.randn(6, 777, generator=g, device="cuda")
    x[:, ::7] = float("nan")
    mask = torch.randint(-2 ** 31, 2 ** 31, (1, 25), generator=g, device="cuda").to(torch.int32)
    prior = torch.tensor([[1, 2, 2, 9]], dtype=torch.int32, device="cuda")
    ids = torch.tensor([[2, 3, 2]], dtype=torch.int32, device="cuda")
    bias = torch.tensor([[0.5, 1.0, 0.25]], device="cuda")
    one = torch.ones(6, device="cuda")
    many = lambda t: t.repeat(6, 1)  # noqa: E731
    few = lambda t: t.expand(6, -1)  # noqa: E731
    a, b = (sampler.adjust(x, out=torch.empty_like(x), prior=f(prior), presence=one, bias_ids=f(ids), bias=f(bias),
                           mask=f(mask)) for f in (many, few))
    assert torch.equal(a.nan_to_num(5.0, 6.0, 7.0), b.nan_to_num(5.0, 6.0, 7.0))
    j = torch.arange(777, device="cuda")
    ok = (mask[0][j // 32] >> (j % 32).int()) & 1 != 0
    assert (a[:, ~ok] == float("-inf")).all() and torch.equal(a[:, ok].isnan(), x[:, ok].isnan())
    assert lib.status() == 0

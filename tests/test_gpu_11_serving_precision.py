"""What the paged attention says of its precision with fp32 rows, and the adjustment's variant for many rows.

Attention: products and sums as accurate as fp32. In the root mean square over the outputs, relative to theirs, that is
  (8 + 4 rms|s|) 2^-24, s the scores in nats:
a weight carries about 8 roundings of its own (exponential, two scalings, its parts, the sums over rows and states) and its
score about 4 of the score's size. Weights held in two bf16 parts instead of three give 2.0e-6 to 2.6e-6 at scores of 0.1 and
1, above it; queries in two parts 2.5e-6 at scores of 1 and 2.9e-6 to 8.5e-6 at 5, above it; a single accumulator over all
rows gave 3.9e-6 at 131072 rows.
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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("size", [0.1, 1.0, 5.0])  # of the scores
@pytest.mark.parametrize("n", [500, 5000, 131072])
@pytest.mark.parametrize("HD", [64, 128])
def test_attention_fp32_precision(mod, HD, n, size):
    paged, _, lib = mod
    g = gen(n + HD)
    KV, G, page = 2, 4, 64
    pages = -(-n // page)
    k, v = (torch.randn(pages, KV, page, HD, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    q = torch.randn(1, KV * G, HD, generator=g, device="cuda") * size
    lse = torch.empty(1, KV * G, device="cuda")
    out = paged.attention(q, paged.Cache(k, v), table, torch.tensor([n - 1], device="cuda"), lse=lse)
    kd, vd = (t[table[0].long()].transpose(0, 1).reshape(KV, -1, HD)[:, :n].double() for t in (k, v))
    s = q.double().view(KV, G, HD) @ kd.transpose(1, 2) * HD ** -0.5
    ref = (torch.softmax(s, -1) @ vd).view(1, KV * G, HD)
    rl = torch.logsumexp(s, -1).view(1, -1)
    rms = lambda t: t.square().mean().sqrt().item()  # noqa: E731
    err, tol = rms(out.double() - ref) / rms(ref), (8 + 4 * rms(s)) * E32
    print(f"HD {HD} n {n} scores {size}: {err:.2e} of {tol:.2e}")
    assert err <= tol
    # the log of the sum: its own few roundings (in base 2) and a largest score's
    assert (lse.double() - rl).abs().max().item() <= (8 + 8 * rl.abs().max().item() + 8 * s.abs().max().item()) * E32
    assert lib.status() == 0


# More CTAs than four an SM (148 of them): slices of the largest size, so that a thread's loads go round twice, and lists
# that take several rounds of 256 threads.
MANY = [("f32", 70, 100003, 1500, 700), ("bf16", 100, 100003, 1500, 700), ("f32", 256, 20011, 1100, 513),
        ("bf16", 600, 4099, 5, 3), ("f32", 80, 65537, 0, 0)]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_adjust_of_many_rows(mod, case, inplace):
    _, sampler, lib = mod
    dtype, B, V, P, nb = MANY[case]
    g = gen(case)
    x = (torch.randn(B, V, generator=g, device="cuda") * 5).to(DT[dtype])
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device="cuda").to(torch.int32)
    rnd = lambda n, lo, hi: torch.randint(lo, hi, (B, n), generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    prior = torch.where(rnd(P, 0, 2) > 0, rnd(P, -3, V + 3), rnd(P, 0, 300) * (V // 300)) if P else None  # many repeats
    ids = torch.where(rnd(nb, 0, 2) > 0, rnd(nb, -2, V + 2), rnd(nb, 0, 300) * (V // 300)) if nb else None
    bias = torch.randn(B, nb, generator=g, device="cuda") * 4 if nb else None
    rep, pres, freq = torch.rand(3, B, generator=g, device="cuda") + torch.tensor([[0.6], [-0.5], [-0.3]], device="cuda")
    want, tol = np.zeros((B, V)), np.zeros((B, V))
    host = lambda t, b: None if t is None else t[b].cpu().numpy()  # noqa: E731
    xd = x.double().cpu().numpy()
    for b in range(B):
        want[b], mag = opaged.adjust(xd[b], host(prior, b), float(rep[b]), float(pres[b]), float(freq[b]), host(ids, b),
                                     host(bias, b), host(mask, b))
        tol[b] = (8 + nb) * E32 * mag
    y = x if inplace else torch.full_like(x, 55.0)
    sampler.adjust(x, out=None if inplace else y, prior=prior, repetition=rep, presence=pres, frequency=freq, bias_ids=ids,
                   bias=bias, mask=mask)
    got, inf = y.double().cpu().numpy(), np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])
    tol = (tol + (EBF if dtype == "bf16" else E32) * (np.abs(np.where(inf, 0, want)) + tol))[~inf]
    assert (np.abs(got[~inf] - want[~inf]) <= tol).all()
    assert lib.status() == 0

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

"""The engine's paged batches after device failures, beside the engine's own sequence, and as their pools change."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["tiny", "small-1k"])
def eng(request, cuda_dev):
    from ai_b200 import build, _lib
    from ai_b200.engine import Engine
    from ai_b200.model import CONFIGS, RandomWeights
    build.build()
    _lib.status(clear=True)
    cfg = CONFIGS[request.param]
    e = Engine(cfg, maxt=128, weights=RandomWeights(cfg, seed=11, norm_noise=0.1, std=0.05), log=None)
    yield e
    assert _lib.status() == 0


def prompts_of(eng, lens, seed=12):
    g = np.random.default_rng(seed)
    return [[int(t) for t in g.integers(0, eng.V, n)] for n in lens]


def test_counts_left_in_the_workspace_do_not_reach_the_next_batch(eng):
    """A wait that runs out may leave the joins' counters above zero."""
    prompts = prompts_of(eng, (90, 33, 70))
    want = eng.generate_batch(prompts, max_new=20)
    assert eng.generate_batch(prompts, max_new=20, page=16) == want
    eng._pbt.ws[:1024].view(torch.int32).fill_(1)
    assert eng.generate_batch(prompts, max_new=20, page=16) == want


def test_device_failures_of_a_paged_batch_are_raised(eng):
    """Copies that never come, and a page outside the pool; the next batch is right again."""
    from ai_b200 import _lib
    prompts = prompts_of(eng, (40, 9))
    want = eng.generate_batch(prompts, max_new=6, page=16)
    _lib.call("aib_debug_knob", 1, 4096)
    _lib.call("aib_debug_knob", 2, 1)
    try:
        with pytest.raises(RuntimeError, match="101"):
            eng.generate_batch(prompts, max_new=3, page=16)
    finally:
        _lib.call("aib_debug_knob", 2, 0)
        _lib.call("aib_debug_knob", 1, 0)
    assert _lib.status() == 0  # it has been raised
    assert eng.generate_batch(prompts, max_new=6, page=16) == want

    def spoil(out):  # between two steps
        if len(out[0]) == 2:
            eng._pbt.pages.table[1, 0] = eng._pbt.pages.total
        return torch.full((1, (eng.V + 31) // 32), -1, dtype=torch.int32)

    with pytest.raises(RuntimeError, match="107"):
        eng.generate_batch(prompts, max_new=5, page=16, mask=spoil)
    assert eng.generate_batch(prompts, max_new=6, page=16) == want and _lib.status() == 0


def test_a_failure_of_an_earlier_call_is_left_to_its_owner(eng):
    from ai_b200 import _lib, paged
    prompts = prompts_of(eng, (40, 9))
    want = eng.generate_batch(prompts, max_new=6, page=16)
    c = paged.Cache(*(torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    row = torch.zeros(1, 1, 64, device="cuda")
    paged.append(c, torch.full((1, 1), 9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"),
                 row, row)
    assert eng.generate_batch(prompts, max_new=6, page=16) == want
    assert _lib.status() == 107


def test_the_engines_own_sequence_survives_a_paged_batch(eng):
    """Prompts of a paged batch run in the engine's cache; what was in it is put back, also when the batch fails."""
    text, tail = prompts_of(eng, (40, 7), seed=5)
    first = eng.process(text, 0)
    kept = eng.kv[:, :, :, :40].clone()
    want = eng.process(tail, 40)
    assert torch.equal(eng.kv[:, :, :, :40], kept)
    for lens in ((60, 3), (5, 9)):  # longer and shorter than the sequence
        assert eng.process(text, 0) == first
        prompts = prompts_of(eng, lens)
        alone = eng.generate_batch(prompts, max_new=4)
        assert eng.generate_batch(prompts, max_new=4, page=8) == alone
        assert eng.ctx == text and torch.equal(eng.kv[:, :, :, :40], kept)
        with pytest.raises(ValueError):
            eng.generate_batch(prompts, max_new=4, page=8, mask=lambda out: torch.zeros(1, 1))
        with pytest.raises(ZeroDivisionError):
            eng.generate_batch(prompts, max_new=4, page=8,
                               mask=lambda out: 1 // 0 if len(out[0]) else torch.full((1, (eng.V + 31) // 32), -1,
                                                                                      dtype=torch.int32))
        assert eng.process(tail, 40) == want


def test_pages_hold_the_rows_that_are_written_and_no_more(eng):
    """The last token drawn gets no row: a prompt that fills its pages, or the context, leaves room for one draw."""
    for lens, max_new, page, pages in (((16, 32), 1, 16, 3), ((13, 5), 4, 8, 3), ((128,), 0, 16, 8), ((127, 9), 1, 32, 5)):
        prompts = prompts_of(eng, lens)
        want = eng.generate_batch(prompts, max_new=max_new)
        assert eng.generate_batch(prompts, max_new=max_new, page=page, pages=pages) == want
        if pages > len(lens):
            with pytest.raises(ValueError):
                eng.generate_batch(prompts, max_new=max_new, page=page, pages=pages - 1)


def test_the_samplers_notice_is_no_failure_of_a_batch(eng):
    """A draw beyond the sampler's candidates (status 105) is noted, not raised, and hides no failure after it."""
    from ai_b200 import _lib, sampler
    prompts = prompts_of(eng, (40, 9))
    want = eng.generate_batch(prompts, max_new=6, page=16)
    flat = torch.zeros(1, 151936, device="cuda")
    free = torch.full((1, (eng.V + 31) // 32), -1, dtype=torch.int32)

    def noticed(out):
        sampler.sample(flat, temperature=1.0, us=[0.999])
        return free

    assert eng.generate_batch(prompts, max_new=6, page=16, mask=noticed) == want
    assert _lib.status(clear=False) == 105  # left for whoever asks
    assert eng.generate_batch(prompts, max_new=6, page=16) == want

    def spoil(out):
        noticed(out)
        if len(out[0]) == 2:
            eng._pbt.pages.table[1, 0] = -5
        return free

    with pytest.raises(RuntimeError, match="107"):
        eng.generate_batch(prompts, max_new=5, page=16, mask=spoil)
    assert _lib.status() == 0
    sampler.sample(flat, temperature=1.0, us=[0.999])
    assert _lib.status() == 105

"""The engine's batches over a paged cache and with per-request penalties, biases and masks, against the contiguous
batch and against single sequences."""
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
    cfg = CONFIGS[request.param]
    e = Engine(cfg, maxt=128, weights=RandomWeights(cfg, seed=11, norm_noise=0.1, std=0.05), log=None)
    yield e
    assert _lib.status() == 0


def prompts_of(eng, lens, seed=12):
    g = np.random.default_rng(seed)
    return [[int(t) for t in g.integers(0, eng.V, n)] for n in lens]


@pytest.mark.parametrize("page", [1, 8, 64])
def test_paged_batch_equals_contiguous_batch(eng, page):
    for lens, seed in (((5, 20, 33), 12), ((40, 1, 16), 13), ((8, 7, 64), 14)):  # the pool is used again
        prompts = prompts_of(eng, lens, seed)
        want = eng.generate_batch(prompts, max_new=20)
        assert eng.generate_batch(prompts, max_new=20, page=page, pages=3 * 128 // page) == want
    assert len(eng._pbt.pages.left) == 3 * 128 // page  # every page came back


def test_paged_batch_sampled_and_sized_to_need(eng):
    prompts = prompts_of(eng, (30, 4))
    want = eng.generate_batch(prompts, max_new=12, temperature=0.8, top_p=0.95, seed=3)
    got = eng.generate_batch(prompts, max_new=12, temperature=0.8, top_p=0.95, seed=3, page=16)
    assert got == want
    assert eng._pbt.pages.total == 3 + 1
    cached = list(eng.generate(prompts[0], max_new=6))  # the engine's own sequence is still right afterwards
    eng.generate_batch(prompts, max_new=3, page=16)
    assert list(eng.generate(prompts[0], max_new=6)) == cached


@pytest.mark.parametrize("page", [None, 16])
def test_penalties_of_every_prompt(eng, page):
    prompts = prompts_of(eng, (5, 20, 33))
    prompts[1] = prompts[1][:4] * 5
    pen = [dict(repetition_penalty=1.4), dict(presence_penalty=0.7, frequency_penalty=0.3), dict()]
    alone = [list(eng.generate(p, max_new=14, **kw)) for p, kw in zip(prompts, pen)]
    got = eng.generate_batch(prompts, max_new=14, page=page, repetition_penalty=[1.4, 1.0, 1.0],
                             presence_penalty=[0, 0.7, 0], frequency_penalty=[0, 0.3, 0])
    assert got == alone
    assert eng.generate_batch(prompts, max_new=14, page=page) != alone  # and nothing of it stays behind


def test_biases_and_masks(eng):
    prompts = prompts_of(eng, (6, 18))
    plain = eng.generate_batch(prompts, max_new=8, page=16)
    got = eng.generate_batch(prompts, max_new=8, page=16, logit_bias=[{17: 1e4, 5: -3.0}, None])
    assert got == [[17] * 8, plain[1]]
    W = (eng.V + 31) // 32

    def only(*ids):
        m = np.zeros((2, W), np.uint32)
        for b, i in enumerate(ids):
            m[b, i // 32] |= np.uint32(1 << (i % 32))
        return torch.from_numpy(m.view(np.int32))

    assert eng.generate_batch(prompts, max_new=3, mask=only(eng.V - 1, 31)) == [[eng.V - 1] * 3, [31] * 3]
    seen = []

    def grammar(out):
        seen.append([len(o) for o in out])
        n = len(out[0])
        return only(10 + n, 40 + n)

    got = eng.generate_batch(prompts, max_new=4, page=16, temperature=0.9, seed=1, mask=grammar)
    assert got == [[10, 11, 12, 13], [40, 41, 42, 43]]
    assert seen == [[i, i] for i in range(4)]
    ban = torch.full((1, W), -1, dtype=torch.int32)  # one row for all: everything but the tokens of the plain run
    for t in set(sum(plain, [])):
        ban[0, t // 32] &= ~(1 << (t % 32)) if t % 32 != 31 else 0x7FFFFFFF
    got = eng.generate_batch(prompts, max_new=8, mask=ban)
    assert not set(sum(got, [])) & set(sum(plain, []))


def test_refusals(eng):
    prompts = prompts_of(eng, (6, 18))
    W = (eng.V + 31) // 32
    for kw in (dict(page=12), dict(page=0), dict(pages=4), dict(page=16, pages=2), dict(repetition_penalty=[1.0]),
               dict(repetition_penalty=0.0), dict(logit_bias=[{}]), dict(logit_bias=[{eng.V: 1.0}, None]),
               dict(logit_bias=[{-1: 1.0}, None]), dict(mask=torch.zeros(2, W + 1, dtype=torch.int32)),
               dict(mask=torch.zeros(2, W))):
        with pytest.raises(ValueError):
            eng.generate_batch(prompts, max_new=3, **kw)
    with pytest.raises(ValueError):
        eng.generate_batch(prompts, max_new=3, page=16, mask=lambda out: torch.zeros(1, 1, dtype=torch.int32))
    assert len(eng._pbt.pages.left) == eng._pbt.pages.total  # a refused mask gives the pages back

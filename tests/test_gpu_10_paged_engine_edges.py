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

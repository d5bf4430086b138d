"""Calls of the paged cache and the logit adjustment that must be refused before anything is launched, and what the
wrappers hand on, on tensors that only say that they are on a GPU."""
import pytest
import torch


class OnGpu(torch.Tensor):
    """A CPU tensor that reports device cuda:0 (its memory is never touched: nothing is launched)."""
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 0))

    def get_device(self):
        return 0


def on_gpu(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


@pytest.fixture
def launched(monkeypatch):
    """Records the C calls instead of making them."""
    from ai_b200 import _lib
    calls = []

    class Device:
        def __init__(self, index):
            pass

        def __enter__(self):
            return 0

        def __exit__(self, *exc):
            return False

    monkeypatch.setattr(_lib, "on_device", Device)
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append((name, args)))
    return calls


# ---------------------------------------------------------------------------------------------- adjust
def test_adjust_refuses_rows_of_one_repeated_element(launched):
    """A row expanded from one element has a column stride of 0, whatever the other tensor's is."""
    from ai_b200 import sampler
    one, x = on_gpu(1, 1), on_gpu(1, 70)
    for kw in (dict(logits=x, out=one.expand(1, 70)), dict(logits=one.expand(1, 70), out=x),
               dict(logits=on_gpu(3, 1).expand(3, 70), out=on_gpu(3, 70)), dict(logits=one.expand(1, 70))):
        with pytest.raises(ValueError):
            sampler.adjust(**kw)
    assert not launched
    sampler.adjust(x)
    sampler.adjust(on_gpu(1, 70).expand(3, 70), out=on_gpu(3, 70))  # one row for all is read, not written
    assert len(launched) == 2


# ------------------------------------------------------------------------------------------- attention
def fake_cache(paged, KV=2, page=16, HD=64):
    return paged.Cache(*(on_gpu(4, KV, page, HD, dtype=torch.bfloat16) for _ in range(2)))


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 63 - 32, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 5, 10 ** 30])
def test_attention_hands_on_windows_of_any_size(launched, window):
    """A window beyond 64 bits reaches every row; its lower bits alone would be another window."""
    from ai_b200 import paged
    q = on_gpu(1, 4, 64)
    paged.attention(q, fake_cache(paged), on_gpu(1, 4, dtype=torch.int32), on_gpu(1, dtype=torch.int64), out=on_gpu(1, 4, 64),
                    window=window, ws=on_gpu(1 << 12, dtype=torch.uint8))
    (name, args), = launched
    assert name == "aib_paged_attn" and args[13] == min(window, 2 ** 63 - 1)


# --------------------------------------------------------------------------------------- engine's pools
def test_a_pool_is_freed_before_the_next_one_is_made(monkeypatch):
    """A pool may take most of the memory: there are never two."""
    import weakref
    from ai_b200 import engine
    alive = weakref.WeakSet()

    class Pool:
        def __init__(self, eng, B, page, pages):
            assert not alive, "the old pool is still there"
            alive.add(self)
            self.B, self.page, self.pages = B, page, type("Pages", (), {"total": pages})()

    monkeypatch.setattr(engine, "PagedBatch", Pool)
    eng = engine.Engine.__new__(engine.Engine)
    for B, page, pages, rows in ((2, 16, None, [17, 5]), (2, 16, None, [40, 5]), (3, 16, 9, [16, 16, 16]), (3, 8, None, [8] * 3)):
        bt = eng._paged_batch(B, page, pages, rows)
        assert bt.B == B and bt.page == page
        del bt
    same = eng._paged_batch(3, 8, None, [8, 8, 1])
    assert eng._paged_batch(3, 8, None, [1, 1, 1]) is same


def test_a_cache_of_rows_that_overlap_is_refused():
    from ai_b200 import paged
    pool = on_gpu(1 << 16, dtype=torch.bfloat16)
    for size, stride in (((4, 2, 16, 64), (1024, 1024, 64, 1)), ((4, 2, 16, 64), (2048, 64, 64, 1)),
                         ((4, 2, 16, 64), (64, 1024, 64, 1)), ((2, 2, 16, 128), (4096 - 8, 2048, 128, 1))):
        with pytest.raises(ValueError):
            paged.Cache(*(pool.as_strided(size, stride),) * 2)
    for size, stride in (((4, 2, 16, 64), (2048, 1024, 64, 1)), ((4, 2, 16, 64), (2048, 64, 128, 1)),
                         ((4, 2, 16, 64), (64, 4096, 256, 1)), ((1, 2, 16, 64), (0, 1024, 64, 1)),
                         ((4, 1, 1, 64), (64, 0, 0, 1))):
        paged.Cache(*(pool.as_strided(size, stride),) * 2)


# --------------------------------------------------------------------------------------- current device
@pytest.mark.parametrize("current,tensors", [(0, 0), (0, 3), (5, 2)])
def test_calls_run_on_the_device_of_their_tensors(monkeypatch, current, tensors):
    """The device of the tensors is made current for a call, with its own stream, and the old one again afterwards, also
    when the call is refused."""
    from ai_b200 import _lib
    state = [current]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 1000 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: state.__setitem__(0, i))
    with _lib.on_device(tensors) as stream:
        assert state[0] == tensors and stream == 1000 + tensors
    assert state[0] == current
    with pytest.raises(ValueError):
        with _lib.on_device(tensors):
            raise ValueError
    assert state[0] == current

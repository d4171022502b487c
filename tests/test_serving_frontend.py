"""KVCache, DecoderBlock.decode, token_logprobs and TokenLoss check their
arguments before any device call.  CPU only: tensors are metadata without buffers."""

import numpy as np
import pytest

import ember_amd as em
from ember_amd import _core, loss
from ember_amd.loss import TokenLoss
from ember_amd.tensor import Tensor


def fake(shape):
    return Tensor._from_core(None, shape)


class _Buffer:
    """A stand-in for a device buffer, as the cache's own bookkeeping sees one."""

    def __init__(self, size):
        self.size = size


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(_core, "_Tensor", _Buffer)
    return em.KVCache(2, 3, 64, tokens=40, page_size=16, pages=4)


def test_names():
    for name in ("_kv_cache_write", "_kv_cache_read", "_kv_cache_attention", "_token_logprobs", "_token_logprobs_bwd"):
        assert callable(getattr(_core, name)) and name in _core.__all__
    assert {"KVCache", "token_logprobs"} <= set(em.__all__)


@pytest.mark.parametrize("change", [
    dict(head_dim=16), dict(head_dim=96), dict(page_size=8), dict(page_size=24), dict(page_size=1 << 17), dict(sequences=0),
    dict(sequences=65536), dict(heads=0), dict(tokens=0), dict(tokens=2 ** 31), dict(pages=0), dict(pages=2 ** 31),
])
def test_cache_sizes(change):
    with pytest.raises(ValueError):
        em.KVCache(**{**dict(sequences=2, heads=3, head_dim=64, tokens=40), **change})


def test_cache_arguments(cache):
    good = fake((2, 5, 3, 64))
    with pytest.raises(TypeError):
        cache.write(good, np.zeros((2, 5, 3, 64)))
    for shape in ((2, 5, 3, 32), (3, 5, 3, 64), (2, 5, 2, 64), (2, 5, 192)):
        with pytest.raises(ValueError):
            cache.write(fake(shape), fake(shape))
    with pytest.raises(ValueError):
        cache.write(good, fake((2, 4, 3, 64)))
    for count in ([5], [5, 6], [-1, 2], [1.0, 2.0], "ab", [[1, 2]]):
        with pytest.raises(ValueError):
            cache.write(good, good, count=count)
    with pytest.raises(ValueError, match="room"):
        cache.write(fake((2, 41, 3, 64)), fake((2, 41, 3, 64)))
    with pytest.raises(ValueError, match="pages"):
        cache.write(fake((2, 33, 3, 64)), fake((2, 33, 3, 64)))
    with pytest.raises(RuntimeError):
        cache.attention(fake((2, 5, 3, 64)))
    for sequence in (-1, 2):
        with pytest.raises(ValueError):
            cache.reset(sequence)
    assert cache.lengths == [0, 0] and len(cache._free) == 4


def test_a_failed_write_changes_nothing(cache, monkeypatch):
    calls = []

    def failing(*args):
        calls.append(args)
        raise RuntimeError("no device")

    monkeypatch.setattr(_core, "_from_numpy", lambda a: _Buffer(a.size))
    monkeypatch.setattr(_core, "_kv_cache_write", failing)
    x = fake((2, 20, 3, 64))
    free = list(cache._free)
    with pytest.raises(RuntimeError, match="no device"):
        cache.write(x, x)
    assert calls and cache.lengths == [0, 0] and cache._free == free and (cache._table == -1).all()


def test_bookkeeping(cache, monkeypatch):
    monkeypatch.setattr(_core, "_from_numpy", lambda a: _Buffer(a.size))
    monkeypatch.setattr(_core, "_kv_cache_write", lambda *args: None)
    cache.write(fake((2, 16, 3, 64)), fake((2, 16, 3, 64)), count=[16, 1])
    assert cache.lengths == [16, 1] and len(cache._free) == 2
    cache.write(fake((2, 1, 3, 64)), fake((2, 1, 3, 64)))
    assert cache.lengths == [17, 2] and len(cache._free) == 1
    pages = cache._table[cache._table >= 0]
    assert len(set(pages.tolist())) == len(pages) == 3
    for T, H in ((2, 3), (1, 4)):
        with pytest.raises(ValueError):
            cache.attention(fake((2, T, H, 64)))
    cache.reset(0)
    assert cache.lengths == [0, 2] and sorted([*cache._free, *pages[pages == cache._table[1, 0]].tolist()]) == [0, 1, 2, 3]


def test_decode_arguments(cache, monkeypatch):
    from ember_amd import nn
    monkeypatch.setattr(nn.DecoderBlock, "reset", lambda self: None)
    block = nn.DecoderBlock(192, 3)
    for x in (fake((5, 192)), fake((4, 128)), fake((2, 2, 192))):
        with pytest.raises(ValueError):
            block.decode(x, cache)
    with pytest.raises(ValueError):
        nn.DecoderBlock(128, 2).decode(fake((2, 128)), cache)
    with pytest.raises(ValueError):
        nn.DecoderBlock(192, 3, causal=False).decode(fake((2, 192)), cache)


@pytest.mark.parametrize("tokens, top", [
    (np.zeros(3, int), 0), (np.zeros((4, 1), int), 0), (np.zeros(4), 0), ([0.0] * 4, 0), (np.zeros(4, int), -1), (np.zeros(4, int), 65),
    (np.zeros(4, int), 11), (None, 0),
])
def test_token_arguments(tokens, top):
    with pytest.raises(ValueError):
        em.token_logprobs(fake((4, 10)), tokens, top)


def test_token_types():
    with pytest.raises(TypeError):
        em.token_logprobs(np.zeros((4, 10)), np.zeros(4, int))
    with pytest.raises(TypeError):
        TokenLoss()(np.zeros((4, 10)), np.zeros(4, int))
    with pytest.raises(ValueError):
        em.token_logprobs(fake((4, 0)), np.zeros(4, int))
    with pytest.raises(RuntimeError):
        TokenLoss().backward()


@pytest.mark.parametrize("kind", [np.uint8, np.uint16, np.uint32, np.uint64, np.int8, np.int16, np.int64])
def test_ids_out_of_range_are_padded_in_any_type(kind):
    ids = np.array([[0, 99], [100, np.iinfo(kind).max]], kind)
    assert loss._token_ids(fake((2, 2, 100)), ids).tolist() == [0, 99, -1, -1]


def test_binding_checks_sizes_before_device_work():
    with pytest.raises(TypeError):
        _core._kv_cache_read(None, 1, None, None)
    with pytest.raises(TypeError):
        _core._kv_cache_write((1, 2), None, 0, None, 0, 1, 1, 1, 1, None, None, None)
    with pytest.raises(TypeError):
        _core._token_logprobs(None, None, 1, 1, 0)
    with pytest.raises(TypeError):
        _core._token_logprobs_bwd(None, None, None, None, None, None, 1, 1)

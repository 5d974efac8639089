"""EncoderCache.extend and encoder_states without a GPU: arrays of a picture's rows that are smaller than what the library
reads of them, or of another shape, never reach it."""
import numpy as np
import pytest

import exn_hip as X


@pytest.fixture
def cache(monkeypatch):
    """A cache of two sequences whose calls are noted."""
    calls = []
    monkeypatch.setattr(X, "call", lambda name, *a: calls.append(name))
    c = X.EncoderCache.__new__(X.EncoderCache)
    c.e, c.h, c.seqs = None, None, 2
    return c, calls


def f(*shape):
    return np.zeros(shape, np.float32)


@pytest.mark.parametrize("merged,deep", [
    (f(3, 4095), None), (f(3, 4097), None), (f(3), None), (f(4096 * 3), None), (f(1, 3, 4096), None),
    (f(3, 4096), f(3, 4096)), (f(3, 4096), f(2, 3, 4096)), (f(3, 4096), f(3, 2, 4096)), (f(3, 4096), f(3, 3, 4095))])
def test_shapes_refused(cache, merged, deep):
    c, calls = cache
    with pytest.raises(X.ExnError) as e:
        c.extend({0: np.zeros(10, np.int32)}, picture=(0, 1, merged, deep))
    assert e.value.code == X.EINVAL and not calls
    with pytest.raises(X.ExnError) as e:
        X.encoder_states(c, np.zeros(10, np.int32), picture=(1, merged, deep))
    assert e.value.code == X.EINVAL and not calls


@pytest.mark.parametrize("seq,a0", [(-1, 0), (2, 0), (0, 0), (1, -1), (1, 8)])
def test_places_refused(cache, seq, a0):
    c, calls = cache
    with pytest.raises(X.ExnError) as e:
        c.extend({1: np.zeros(10, np.int32)}, picture=(seq, a0, f(3, 4096), None))
    assert e.value.code == X.EINVAL and not calls


def test_taken(cache):
    c, calls = cache
    for deep in (None, f(3, 3, 4096), [f(3, 4096)] * 3):
        X.encoder_states(c, np.zeros(10, np.int32), picture=(7, f(3, 4096), deep))
        c.extend({0: np.zeros(4, np.int32), 1: np.zeros(10, np.int32)}, picture=(1, 7, f(3, 4096), deep))
    assert calls == ["exn_enc_states", "exn_enc_cache_extend"] * 3

"""An EncoderCache that is dropped frees what it holds, once, so that its encoder can be destroyed;
after its context is closed it calls nothing.  Without a GPU: the library's calls are noted."""
import gc
import types

import pytest

import exn_hip as X


@pytest.fixture
def calls(monkeypatch):
    noted = []

    def call(name, *a):
        noted.append(name)
        if name == "exn_enc_cache_create":
            a[-1]._obj.value = 4096
    monkeypatch.setattr(X, "call", call)
    return noted


def encoder():
    return types.SimpleNamespace(h=1, ctx=types.SimpleNamespace(h=1))


def test_dropped(calls):
    c = X.EncoderCache(encoder(), 2, 100)
    del c
    gc.collect()
    assert calls == ["exn_enc_cache_create", "exn_enc_cache_destroy"]


def test_destroyed_then_dropped(calls):
    c = X.EncoderCache(encoder(), 2, 100)
    c.destroy()
    c.destroy()
    del c
    gc.collect()
    assert calls == ["exn_enc_cache_create", "exn_enc_cache_destroy"]


def test_dropped_after_its_context(calls):
    e = encoder()
    c = X.EncoderCache(e, 2, 100)
    e.ctx.h = None
    del c
    gc.collect()
    assert calls == ["exn_enc_cache_create"]


def test_not_made(calls, monkeypatch):
    def refuse(name, *a):
        calls.append(name)
        raise X.ExnError(X.EINVAL, "refused")
    monkeypatch.setattr(X, "call", refuse)
    with pytest.raises(X.ExnError):
        X.EncoderCache(encoder(), 0, 100)
    gc.collect()
    assert calls == ["exn_enc_cache_create"]

"""The encoder's kept prompts without a GPU: their pages and lengths through extends, forks and
resets, and after failures.  tests/host/encoder_cache_host.cpp stands in for the device and the
kernels (linked with this build's own api_encoder.o and api_prompts.o)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import exn_hip as X

HERE = os.path.dirname(os.path.abspath(__file__))
BUILD = os.path.join(HERE, "..", "ex-nihilo_amd", "_build")
OBJS = [os.path.join(BUILD, n) for n in ("api_encoder.o", "api_prompts.o")]
vp = ctypes.c_void_p
SEQS, TOKENS, COLS = 3, 256, 4


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not all(os.path.exists(o) for o in OBJS):
        pytest.skip("the library's objects are not here")
    d = tmp_path_factory.mktemp("encoder_cache_host")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "encoder_cache_host.cpp"), "-o", o], check=True)
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", "-o", so, o, *OBJS], check=True)
    lib = ctypes.CDLL(so)
    lib.eh_error.restype = ctypes.c_char_p
    lib.eh_ctx.restype = vp
    lib.eh_fail_new.argtypes = [ctypes.c_long]
    for n, (res, args) in X.SIGNATURES.items():
        if n.startswith(("exn_enc", "exn_seqs")):
            f = getattr(lib, n)
            f.restype, f.argtypes = res, args
    return lib


@pytest.fixture
def cache(L):
    e, c = vp(), vp()
    assert L.exn_enc_create(L.eh_ctx(), 1, 5e6, ctypes.byref(e)) == X.OK
    assert L.exn_enc_synth(e, 1, 100) == X.OK
    assert L.exn_enc_cache_create(e, SEQS, TOKENS, ctypes.byref(c)) == X.OK
    yield c
    assert L.exn_enc_destroy(e) == X.ESTATE     # its cache first
    assert L.exn_enc_cache_destroy(c) == X.OK
    assert L.exn_enc_destroy(e) == X.OK


def extend(L, c, new):
    n = sum(new)
    ids, lens, out = np.zeros(n, np.int32), np.asarray(new, np.int32), np.zeros((n, 4096), np.float32)
    return L.exn_enc_cache_extend(c, ids.ctypes.data_as(vp), lens.ctypes.data_as(vp), len(new), None, 0, 0, None, None,
                                  out.ctypes.data_as(vp))


def lens(L, c):
    a = np.zeros(SEQS, np.int32)
    assert L.exn_enc_cache_lens(c, a.ctypes.data_as(vp), SEQS) == X.OK
    return a.tolist()


def table(L):
    a = np.zeros(SEQS * COLS, np.int32)
    assert L.eh_table(a.ctypes.data_as(vp), a.size) == a.size
    return a.reshape(SEQS, COLS)


def fills(L, c):
    """Every page is there to be had: all sequences emptied, then filled to the end."""
    for i in range(SEQS):
        assert L.exn_enc_cache_reset(c, i) == X.OK
    assert extend(L, c, [TOKENS] * SEQS) == X.OK, L.eh_error()
    assert sorted(table(L).ravel()) == list(range(SEQS * COLS))
    assert extend(L, c, [0, 1, 0]) == X.EINVAL and lens(L, c) == [TOKENS] * SEQS


def test_pages_through_forks_and_resets(L, cache):
    assert extend(L, cache, [130, 0, 64]) == X.OK
    t = table(L)
    assert (t[0] >= 0).tolist() == [True, True, False, False] and (t[2] >= 0).tolist() == [True, False, False, False]
    assert L.exn_enc_cache_fork(cache, 0, 1) == X.OK and L.exn_enc_cache_fork(cache, 0, 2) == X.OK
    assert L.exn_enc_cache_fork(cache, 1, 1) == X.OK
    assert lens(L, cache) == [130, 130, 130]
    assert extend(L, cache, [0, 70, 100]) == X.OK
    u = table(L)
    assert (u[1:, :2] == t[0, :2]).all() and (u[0] == t[0]).all()      # the shared blocks
    assert u[1, 2] >= 0 and u[2, 2] >= 0 and u[1, 2] != u[2, 2]        # each its own from there
    assert L.exn_enc_cache_reset(cache, 0) == X.OK
    assert extend(L, cache, [64, 0, 0]) == X.OK
    v = table(L)
    assert v[0, 0] not in u[1] and v[0, 0] not in u[2] and (v[1:] == u[1:]).all()
    assert lens(L, cache) == [64, 200, 230]
    fills(L, cache)


def test_extend_where_memory_ends(L, cache):
    """Each host allocation of an extend fails in turn: a status, and a cache that is as it was or
    whose extended sequences are empty, with no page lost."""
    k, kept, emptied = 0, 0, 0
    while True:
        for i in range(SEQS):
            assert L.exn_enc_cache_reset(cache, i) == X.OK
        assert extend(L, cache, [70, 100, 0]) == X.OK
        L.eh_fail_new(k)
        r = extend(L, cache, [130, 0, 64])
        done = not L.eh_failed()
        L.eh_fail_new(-1)
        if done:
            assert r == X.OK
            break
        if r == X.OK:        # an allocation that has another way
            assert lens(L, cache) == [200, 100, 64]
        else:
            assert r == X.ENOMEM, (k, L.eh_error())
            assert lens(L, cache) in ([70, 100, 0], [0, 100, 0])
            kept += lens(L, cache)[0] == 70
            emptied += lens(L, cache)[0] == 0
        fills(L, cache)
        k += 1
    assert kept and emptied


def test_fork_whose_copy_fails(L, cache):
    """The sequence that was to be is empty, the other as it was."""
    for at in (0, 1):
        assert extend(L, cache, [70, 80, 0]) == X.OK
        L.eh_fail_copy(at)
        assert L.exn_enc_cache_fork(cache, 0, 1) == X.EHIP
        assert lens(L, cache) == [70, 0, 0]
        fills(L, cache)
        for i in range(SEQS):
            assert L.exn_enc_cache_reset(cache, i) == X.OK

"""A fork of a kept prompt, without a GPU: its copies are done when the call returns, one that fails
leaves the new sequence empty, and none is made in a capture.  tests/host/encoder_fork_host.cpp stands in
for the device (linked with this build's own api_encoder.o and api_prompts.o)."""
import ctypes
import os
import subprocess

import pytest

import exn_hip as X
from test_encoder_cache_host import HERE, OBJS, cache, extend, fills, lens  # noqa: F401

vp = ctypes.c_void_p


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not all(os.path.exists(o) for o in OBJS):
        pytest.skip("the library's objects are not here")
    d = tmp_path_factory.mktemp("encoder_fork_host")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "encoder_fork_host.cpp"), "-o", o], check=True)
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


def test_a_fork_is_whole_when_it_returns(L, cache):  # noqa: F811
    assert extend(L, cache, [70, 80, 0]) == X.OK
    assert L.exn_enc_cache_fork(cache, 0, 1) == X.OK
    assert L.ef_queued() == 0
    assert lens(L, cache) == [70, 70, 0]
    fills(L, cache)


def test_a_fork_whose_copies_fail_later(L, cache):  # noqa: F811
    assert extend(L, cache, [70, 80, 0]) == X.OK
    L.ef_fail_wait(1)
    r = L.exn_enc_cache_fork(cache, 0, 1)
    L.ef_fail_wait(0)
    assert r == X.EHIP and lens(L, cache) == [70, 0, 0]
    fills(L, cache)


def test_a_fork_in_a_capture_is_refused(L, cache):  # noqa: F811
    assert extend(L, cache, [70, 80, 0]) == X.OK
    L.ef_capturing(1)
    r = L.exn_enc_cache_fork(cache, 0, 1)
    L.ef_capturing(0)
    assert r == X.ESTATE and b"capture" in L.eh_error()
    assert L.ef_queued() == 0 and lens(L, cache) == [70, 80, 0]
    fills(L, cache)

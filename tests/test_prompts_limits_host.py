"""The largest plans and head counts that the prompt side's calls document, without a GPU: a launch counts
a grid axis' threads in 32 bits, and one of more workgroups than that holds is refused before it is
made.  tests/host/prompts_limits_host.cpp calls the launches (this build's own packed.o and kv8.o)."""
import ctypes
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
BUILD = os.path.join(HERE, "..", "ex-nihilo_amd", "_build")
OBJS = [os.path.join(BUILD, n) for n in ("packed.o", "kv8.o")]
N = 1 << 16


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not all(os.path.exists(o) for o in OBJS):
        pytest.skip("the library's objects are not here")
    if torch.cuda.device_count():
        pytest.skip("calls that are not refused are to find no device")
    d = tmp_path_factory.mktemp("prompts_limits")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "prompts_limits_host.cpp"), "-o", o], check=True)
    subprocess.run(["/opt/rocm/bin/hipcc", "-shared", "--offload-arch=gfx950", "-o", so, o, *OBJS], check=True)
    return ctypes.CDLL(so)


def test_packed(L):
    assert not L.pl_packed(N, 1024, 1024, 64) and not L.pl_packed(N, 256, 256, 64)
    assert L.pl_packed(N, 255, 255, 64) and L.pl_packed(N, 1024, 128, 64)


def test_append_and_read(L):
    for f in (L.pl_append, L.pl_read):
        assert not f(N, 1024) and not f(N, 256)
        assert f(N, 255) and f(N - 1, 256)


def test_attend(L):
    for longest, heads, kv, cols, ok in ((1, 1024, 1024, 8, False), (1, 256, 256, 8, False), (1, 255, 255, 8, True),
                                         (1, 1024, 64, 8, True), (40, 512, 512, 8, False), (40, 128, 128, 8, True)):
        assert bool(L.pl_attend(N, longest, heads, kv, cols)) == ok, (longest, heads, kv)

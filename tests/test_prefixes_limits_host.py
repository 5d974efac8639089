"""attend_shared's largest plans and its scratch, without a GPU: what no grid holds is refused before a launch, what only
the shared passes do not fit runs unshared, and the scratch is that of the passes that run.
tests/host/prefixes_limits_host.cpp calls the launches (this build's own kv8.o)."""
import ctypes
import os
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
OBJ = os.path.join(HERE, "..", "ex-nihilo_amd", "_build", "kv8.o")
N = 1 << 16


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not os.path.exists(OBJ):
        pytest.skip("the library's objects are not here")
    if torch.cuda.device_count():
        pytest.skip("calls that are not refused are to find no device")
    d = tmp_path_factory.mktemp("prefixes_limits")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "prefixes_limits_host.cpp"), "-o", o], check=True)
    subprocess.run(["/opt/rocm/bin/hipcc", "-shared", "--offload-arch=gfx950", "-o", so, o, OBJ], check=True)
    lib = ctypes.CDLL(so)
    lib.ps_part.restype = ctypes.c_int64
    return lib


def test_sizes(L):
    assert not L.ps_shared(N, 1024, 1024, 20) and not L.ps_shared(N, 256, 256, 20)
    # the sequences' own workgroups fit by themselves, with the prefix's they do not: unshared
    assert L.ps_shared(N, 255, 255, 20)
    assert L.ps_shared(N, 8, 8, 20) and L.ps_shared(2, 8, 8, 1 << 19) and L.ps_shared(300, 1024, 1, 40)


@pytest.mark.parametrize("n,longest,heads,kv,hd,blocks,cols,pays", [
    (8, 1, 32, 8, 128, 17, 20, True), (64, 1, 32, 8, 128, 128, 160, True), (4, 1, 16, 2, 64, 2000, 2003, True),
    (2, 1, 32, 8, 128, 400, 403, True), (8, 4, 32, 8, 128, 17, 20, True),
    (8, 1, 32, 8, 128, 16, 20, False),          # short prefixes
    (8, 1, 32, 8, 128, 17, 16, False),          # of which the table holds less
    (6, 1, 32, 8, 128, 17, 20, False),          # little to save
    (2, 1, 32, 8, 128, 300, 303, False),
    (64, 5, 32, 8, 128, 128, 160, True), (64, 2, 16, 1, 128, 128, 160, True), (20, 16, 32, 8, 128, 21, 30, True),
    (20, 64, 8, 8, 64, 21, 30, True),           # sequences of 17 to 64 rows a head
    (19, 5, 32, 8, 128, 21, 30, False),         # little to save
    (64, 17, 32, 8, 128, 128, 160, True), (64, 20, 32, 8, 128, 128, 160, True), (10, 40, 32, 8, 128, 100, 130, True),
    (64, 9, 16, 1, 128, 128, 160, True), (16, 160, 8, 8, 128, 100, 130, True),   # of more, in tiles that they do not fill
    (8, 40, 32, 8, 128, 100, 130, False),       # little to save
    (64, 21, 32, 8, 128, 128, 160, False), (64, 76, 32, 8, 128, 128, 160, False), (64, 32, 32, 8, 128, 128, 160, False),
    (64, 11, 16, 1, 128, 128, 160, False), (64, 32, 40, 8, 128, 128, 160, False),
])
def test_scratch_and_what_is_shared(L, n, longest, heads, kv, hd, blocks, cols, pays):
    alone = ctypes.c_int64()
    got = L.ps_part(n, longest, heads, kv, hd, blocks, cols, ctypes.byref(alone))
    if not pays:
        assert got == alone.value
        return
    assert got != alone.value
    # a whole number of splits of at most 64 each, of the prefix's rows and of the sequences', and the tiles' notes
    each = n * longest * heads * (hd + 2)
    tokens = 8
    while 2 * tokens * min(8, heads // kv) <= 64 and longest * min(16, heads // kv) > 16:
        tokens *= 2
    tiles = n * -(-longest // tokens)
    splits, left = divmod(got - 4 * tiles, each)
    assert left == 0 and 2 <= splits <= 128

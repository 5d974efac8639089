"""attend_shared's rules, without a GPU: into how many splits its passes go.  tests/host/prefixes_limits_host.cpp calls
them (this build's own kv8.o)."""
import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OBJ = os.path.join(HERE, "..", "ex-nihilo_amd", "_build", "kv8.o")


@pytest.fixture(scope="module")
def L(tmp_path_factory):
    if not os.path.exists(OBJ):
        pytest.skip("the library's objects are not here")
    d = tmp_path_factory.mktemp("prefixes_rules")
    o, so = str(d / "host.o"), str(d / "host.so")
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC", "-c",
                    os.path.join(HERE, "host", "prefixes_limits_host.cpp"), "-o", o], check=True)
    subprocess.run(["/opt/rocm/bin/hipcc", "-shared", "--offload-arch=gfx950", "-o", so, o, OBJ], check=True)
    lib = ctypes.CDLL(so)
    lib.ps_part.restype = ctypes.c_int64
    return lib


def part(L, n, longest, heads, kv, hd, blocks, cols):
    """The floats that a call of N sequences of LONGEST tokens after BLOCKS blocks has a use for, and kv8_attend's."""
    alone = ctypes.c_int64()
    return L.ps_part(n, longest, heads, kv, hd, blocks, cols, ctypes.byref(alone)), alone.value


@pytest.mark.parametrize("n,heads,kv,hd,blocks,cols,prefix,own", [
    # a split of 8 blocks for every workgroup that finds a place: 512 of 128-wide heads, 1024 of 64-wide
    (4, 16, 2, 64, 512, 516, 64, 64), (8, 32, 8, 128, 2047, 2062, 32, 8), (8, 32, 8, 128, 17, 20, 5, 3),
])
def test_own_blocks_are_split_by_the_whole_table(L, n, heads, kv, hd, blocks, cols, prefix, own):
    """A sequence whose table parts from its prefix has all its blocks to itself: as many splits as those need."""
    got, alone = part(L, n, 1, heads, kv, hd, blocks, cols)
    assert got != alone
    splits, left = divmod(got - 4 * n, n * heads * (hd + 2))
    assert left == 0 and splits == prefix + own

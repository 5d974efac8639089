"""attend_shared's rules, without a GPU: into how many splits its passes go, and where nothing is shared.  tests/host/prefixes_limits_host.cpp calls
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


@pytest.mark.parametrize("n,longest,heads,kv,hd,blocks,cols,shared", [
    # each side's time on the card (us), unshared and shared
    (32, 8, 32, 8, 128, 32, 36, False),      # 35.2, 37.8: a workgroup of kv8_attend for each sequence and head fits the chip
    (32, 32, 8, 8, 128, 32, 36, False),      # 34.9, 39.6
    (8, 32, 32, 32, 128, 32, 36, False),     # 35.1, 40.0
    (2, 1, 16, 1, 128, 512, 516, False),     # 24.0, 26.0: few workgroups for the prefix
    (4, 1, 16, 1, 128, 2000, 2004, False),   # 42.6, 55.5
    (3, 1, 16, 1, 64, 2000, 2004, False),    # 31.1, 42.1
    (4, 16, 4, 1, 128, 128, 132, False),     # 21.2, 26.2
    (16, 1, 32, 32, 128, 8, 12, False),      # 19.4, 22.4: a short prefix, 63 MB
    (64, 1, 32, 32, 128, 16, 20, True),      # 98.9, 41.9: 529 MB
    (64, 1, 32, 32, 128, 8, 12, True),       # 59.8, 40.4
    (256, 1, 32, 8, 128, 16, 20, True),      # 94.3, 47.2
    (256, 1, 32, 8, 128, 8, 12, True),       # 59.1, 45.4
    (2, 1, 32, 32, 128, 128, 132, True),     # 34.3, 25.2: many heads
    (4, 24, 32, 32, 128, 64, 68, True),      # 46.4, 34.5
    (16, 17, 32, 32, 128, 17, 21, True),     # 56.6, 35.9
    (16, 1, 16, 1, 128, 512, 516, True),     # 40.4, 34.7
    (4, 1, 16, 4, 64, 512, 516, True),       # 26.7, 17.7
    (8, 1, 8, 1, 64, 32, 36, True),          # 13.7, 12.7
    # more than 64 rows a head and sequence
    (2, 9, 8, 1, 128, 2000, 2004, False),    # 47.9, 73.4
    (2, 17, 16, 4, 64, 1000, 1004, False),   # 40.7, 52.3
    (32, 160, 32, 32, 128, 17, 23, False),   # 236.8, 268.4
    (16, 40, 32, 8, 128, 128, 132, True),    # 174, 125
    (10, 40, 32, 8, 128, 100, 104, True),
])
def test_the_faster_side_runs(L, n, longest, heads, kv, hd, blocks, cols, shared):
    got, alone = part(L, n, longest, heads, kv, hd, blocks, cols)
    assert (got != alone) == shared


def test_a_hint_past_the_table_saves_no_more_than_the_table(L):
    """A prefix said to be of a million blocks, in tables of 12: as one of 12."""
    assert part(L, 8, 1, 32, 8, 128, 1 << 20, 12) == part(L, 8, 1, 32, 8, 128, 12, 12)

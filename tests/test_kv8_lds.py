"""What the cache's attention kernels keep in LDS, from this build's own kv8.o (its code object's notes; no GPU needed):
kernels of a sequence's whole keys hold their stages, or a tail and the waves' sums, and nothing of the shared passes'."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OBJ = os.path.join(HERE, "..", "ex-nihilo_amd", "_build", "kv8.o")
LLVM = "/opt/rocm/llvm/bin"


def lds(tmp):
    fat, co = os.path.join(tmp, "fat.bin"), os.path.join(tmp, "kv8.co")
    subprocess.run([os.path.join(LLVM, "llvm-objcopy"), "--dump-section", ".hip_fatbin=" + fat, OBJ, os.devnull], check=True)
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o", "--input=" + fat,
                    "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--output=" + co], check=True)
    notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", co], check=True, capture_output=True,
                           text=True).stdout
    return {m.group(2): int(m.group(1))
            for m in re.finditer(r"\.group_segment_fixed_size:\s+(\d+).*?\.name:\s+(\S+)", notes, re.S)}


@pytest.mark.skipif(not os.path.exists(OBJ), reason="kv8.o not built (__graft_entry__.build())")
@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-readelf")), reason="no ROCm llvm-readelf")
def test_lds(tmp_path):
    size = lds(str(tmp_path))
    want = {}
    for bf in (0, 1):
        for hd in (64, 128):
            # two stages each of 64 keys' and values' 16 bits
            want["k_kv8_chunkILi%dELi%dEE" % (bf, hd)] = 4 * 64 * hd * 2
            for rt in (1, 2):
                # the tail's keys and values, four waves' sums (rows 4 floats further apart), references and weights, and weights of
                # 64 keys and 16 rows (17 apart)
                want["k_kv8_fewILi%dELi%dELi%dEE" % (bf, hd, rt)] = 2 * 64 * hd * 2 + 4 * (4 * 16 * (hd + 4) + 2 * 4 * 16 + 64 * 17)
    for part, bytes_ in want.items():
        names = [n for n in size if part in n]
        assert len(names) == 1 and size[names[0]] == bytes_, (part, names, [size[n] for n in names])

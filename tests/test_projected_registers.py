"""The compiled product kernels whose loads to LDS are written out: m0, which says where those write to, is theirs alone (the compiler is not told of it)."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from bmtk_amd import _lib

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-objdump")), reason="no llvm-objdump")
def test_m0_is_written_by_the_loads_alone(tmp_path):
    _lib.load()
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    objdump = os.path.join(LLVM, "llvm-objdump")
    subprocess.run([objdump, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    looked_at = 0
    for code in sorted(glob.glob(str(tmp_path / "lib.so.*gfx950"))):
        if b"product_kernel" not in open(code, "rb").read():
            continue
        text = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr", code], check=True, stdout=subprocess.PIPE, text=True).stdout
        for name, body in re.findall(r"^<(\w*product_kernel\w*)>:\n(.*?)(?=^<|\Z)", text, re.M | re.S):
            if not re.search(r"Li[24]E(Lb1ELb[01]|Lb0ELb1)E", name):
                continue
            lines = [line.split("//")[0].strip() for line in body.splitlines()]
            given = [k for k, line in enumerate(lines) if re.search(r"\bm0\b", line)]
            loads = [k for k, line in enumerate(lines) if line.startswith("buffer_load") and line.endswith(" lds")]
            assert given and [k + 2 for k in given] == loads, name
            assert all(re.match(r"s_mov_b32 m0, s\d+$", lines[k]) and lines[k + 1] == "s_nop 3" for k in given), name
            looked_at += 1
    assert looked_at == 18   # (two types of 16 bits and fp32, two sizes of tiles, dx to slabs, d_weight to slabs or to its place)

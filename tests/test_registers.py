"""Waves that kernels of the built library leave room for: their registers, where a few more would cost a wave a SIMD."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from ztensor_amd import build

LLVM = Path("/opt/rocm/llvm/bin")
# a part of the kernel's name, and waves a SIMD (512 registers, dealt out 8 at a time)
WAVES = [("attn_many_kernelIDF16_Li1E", 3), ("append_kernelIfLi4ELi4ENS_8RopeArgs", 7), ("append_kernelIDF16_Li4ELi8ENS_8RopeArgs", 7),
         ("append_kernelIDF16_Li4ELi8ENS_8NormArgs", 4), ("append_kernelIfLi4ELi4ENS_8NormArgs", 4)]


@pytest.fixture(scope="module")
def registers(tmp_path_factory):
    """{kernel: registers of a lane}, by the code objects' notes."""
    if not (LLVM / "llvm-readelf").exists() or not (LLVM / "llvm-objdump").exists():
        pytest.skip("no llvm-readelf")
    if not build.LIB.exists():
        build.build()
    path = tmp_path_factory.mktemp("lib")
    lib = shutil.copy(build.LIB, path / "lib.so")
    subprocess.run([LLVM / "llvm-objdump", "--offloading", lib], check=True, capture_output=True, cwd=path)
    found = {}
    for obj in path.glob(f"lib.so.*{build.ARCH}"):
        notes = subprocess.run([LLVM / "llvm-readelf", "--notes", obj], check=True, capture_output=True, text=True).stdout
        for kernel in notes.split("- .agpr_count:")[1:]:
            found[re.search(r"\.name:\s+(\S+)", kernel).group(1)] = int(re.search(r"\.vgpr_count:\s+(\d+)", kernel).group(1))
    return found


@pytest.mark.parametrize("name,waves", WAVES)
def test_waves(registers, name, waves):
    kernels = {k: n for k, n in registers.items() if name in k}
    assert kernels
    for k, n in kernels.items():
        assert 512 // (-(-n // 8) * 8) >= waves, (k, n)

"""Reports of given-up waits of the 8-bit products: one stream's question does not take another's answer (give_ups.h)."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "nvmai_b200" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_streams_owner_is_told_once(tmp_path):
    exe = tmp_path / "give_ups_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", str(ROOT / "tests" / "cpp" / "give_ups_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr


def test_the_count_never_goes_back():
    """the device adds to it, the host reads it: nothing clears what another stream has not read"""
    kernel, host = (CSRC / "int8_gemm.cuh").read_text(), (CSRC / "int8_matmul.cu").read_text()
    assert re.findall(r"\w+\(&g_int8_give_ups", kernel) == ["atomicAdd(&g_int8_give_ups"]
    assert re.findall(r"\w+\(&?\w*,? ?g_int8_give_ups", host) == ["cudaMemcpyFromSymbolAsync(&count, g_int8_give_ups"]

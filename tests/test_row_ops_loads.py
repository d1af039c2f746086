"""Read from the sources: the row operators' kernels start beside the kernel in front, which may still write what they read behind
their wait, so none of them uses the non-coherent load, whose memory nobody may write while its kernel lives."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "nvmai_b200" / "csrc"


@pytest.mark.parametrize("name", ["row_ops.cu", "row_elem.cuh", "int8_matmul.cu", "int8_stream.cuh", "int8_gemm.cuh"])
def test_no_non_coherent_loads(name):
    lines = [re.sub(r"//.*", "", line) for line in (CSRC / name).read_text().splitlines()]
    assert not [line for line in lines if re.search(r"ldg|\.nc\b|__restrict__", line)]

"""GPU tests of the row operators where their first tests do not reach: reports of given-up waits by stream, calls with nothing
to do, activations in their tails, tile plans of large products, second turns of persistent loops, offsets past 32 bits.

Tolerances as in test_gpu_row_ops.py: `U` = 2^-24 is half a step of fp32, `half_step(t)` the output type's."""

import pytest
import torch

import nvmai_b200 as nv
from nvmai_b200 import _lib
from nvmai_b200 import format as fmt
from test_gpu_row_ops import check_product, code_of, codes

pytestmark = pytest.mark.gpu


# ---- reports of given-up waits ------------------------------------------------------------------------------------

def test_a_report_reaches_every_streams_owner():
    """a product on one stream gives up: asking on another stream does not take the answer from the one it concerns"""
    from nvmai_b200.moe import debug_set_wait_limit
    from nvmai_b200.row_ops import debug_drop_int8_copy
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, one, two):
        with torch.cuda.stream(stream):
            check_product(300, 640, 130, fmt.ACT_NONE, stream=stream)
    rows, k, n = 300, 640, 130
    a, sa = codes(61, rows, k)
    b, sb = codes(62, n, k)
    y = torch.empty((rows, n), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    debug_set_wait_limit(2_000_000)
    try:
        debug_drop_int8_copy()
        nv.int8_matmul(a, b, sb, y, rows, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=b.shape[1], stream=two)
        torch.cuda.synchronize()
        told = {name: code_of(lambda: nv.int8_matmul_status(stream)) for name, stream in (("one", one), ("two", two), ("none", None))}
        assert told == {"one": _lib.ETIMEOUT, "two": _lib.ETIMEOUT, "none": _lib.ETIMEOUT}
        for stream in (one, two, None):                # once each, and the next product is right
            with torch.cuda.stream(stream):
                check_product(rows, k, n, fmt.ACT_SILU, stream=stream)
    finally:
        debug_set_wait_limit(0)
        for stream in (one, two, None):
            code_of(lambda: nv.int8_matmul_status(stream))

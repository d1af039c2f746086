"""GPU tests of the row operators where their first tests do not reach: reports of given-up waits by stream, calls with nothing
to do, activations in their tails, tile plans of large products, second turns of persistent loops, offsets past 32 bits.

Tolerances as in test_gpu_row_ops.py: `U` = 2^-24 is half a step of fp32, `half_step(t)` the output type's."""

import numpy as np
import pytest
import torch

import nvmai_b200 as nv
from nvmai_b200 import _lib
from nvmai_b200 import format as fmt
from test_gpu_row_ops import TYPES, U, check_product, code_of, codes, half_step

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


# ---- calls with nothing to do ------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows_elem", [fmt.ELEM_F16, fmt.ELEM_I8])
@pytest.mark.parametrize("sized", [False, True])
def test_sorting_no_tokens_writes_empty_experts(rows_elem, sized):
    """an empty chunk: tensors without elements have no address, buffers for the largest chunk have one"""
    d, e, n = 64, 8, 4 if sized else 0
    x = torch.empty((0, d), dtype=torch.float16, device="cuda")
    idx, position = torch.empty((0, 2), dtype=torch.int32, device="cuda"), torch.empty((n, 2), dtype=torch.int32, device="cuda")
    source, begin = torch.empty(2 * n, dtype=torch.int32, device="cuda"), torch.full((e + 1,), 5, dtype=torch.int32, device="cuda")
    int8 = rows_elem == fmt.ELEM_I8
    rows = torch.full((2 * n, d), 77, dtype=torch.int8 if int8 else torch.float16, device="cuda")
    scales = torch.full((2 * n,), 77.0, device="cuda") if int8 else None
    nv.sort_rows(idx, 0, 2, e, position, source, begin, x=x, d=d, rows=rows, rows_elem=rows_elem, row_scales=scales)
    assert begin.tolist() == [0] * (e + 1) and (rows == 77).all()


# ---- activations in their tails ----------------------------------------------------------------------------------

def tails(rows, first, scale, up, activation, out):
    """rows of one code 1: gate values are -(first + j) * scale exactly, for j = 0 .. 47, up values are `up`.  -> output, gates"""
    n, k = 48, 16
    a = torch.zeros((rows, k), dtype=torch.int8, device="cuda")
    a[:, 0] = 1
    b = torch.zeros((2 * n, k), dtype=torch.int8, device="cuda")
    b[:n, 0] = -(first + torch.arange(n, device="cuda")).to(torch.int8)
    b[n:, 0] = 1
    sb = torch.full((2 * n,), scale, device="cuda")
    sb[n:] = up
    t, elem = TYPES[out]
    y = torch.empty((rows, n), dtype=t, device="cuda")
    nv.int8_matmul(a, b, sb, y, rows, k, n, a_scales=torch.ones(rows, device="cuda"), activation=activation, out_elem=elem)
    return y, b[:n, 0].double()[None, :] * scale


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows", [1, 8, 40])
def test_silu_far_below_zero(rows, out):
    """e^-g leaves fp32 below -88.7 while the gate times a large up row does not: 2^-149 is the step of fp32 below 2^-126, which e^g
    is off by two of, and its product with g by half of one"""
    up = float(np.float32(1e30))
    y, g = tails(rows, 80, 1.0, up, fmt.ACT_SILU, out)
    want = g * torch.exp(g) / (1 + torch.exp(g)) * up
    tol = ((1 + g.abs()) * 3 + 11) * U * want.abs() * 1.01 + (2 * g.abs() + 1) * 2.0 ** -149 * up + half_step(TYPES[out][0], want) * 1.01
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows", [1, 8, 40])
@pytest.mark.parametrize("first", [0, 48, 80])
def test_gelu_far_below_zero(rows, out, first):
    """0.5 g (1 + tanh y) = g / (1 + e^-2y).  y: two constants, a cube of two steps, a fused step and a product are 6 roundings; with
    the argument's for exp2 8 |2 y| U of e^2y, and 12 U for exp, sum, quotient and products.  Below 2^-126 e^2y
    is off by two steps of 2^-149 and its product with g by half of one"""
    y, g = tails(rows, first, 0.125, 1.0, fmt.ACT_GELU_TANH, out)
    z = 2 * 0.7978845608028654 * (g + 0.044715 * g ** 3)
    want = g * torch.exp(z) / (1 + torch.exp(z))
    tol = (8 * z.abs() + 12) * U * want.abs() * 1.01 + (2 * g.abs() + 1) * 2.0 ** -149 + half_step(TYPES[out][0], want) * 1.01
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_gelu_of_large_gates(rows, out):
    """far above zero the gate itself (its product and the up row's: two roundings), far below it nothing"""
    up = float(np.float32(1e-30))
    for scale in (1e20, -1e20, 1e30, -1e30):
        y, g = tails(rows, 1, float(np.float32(scale)), up, fmt.ACT_GELU_TANH, out)
        want = g.clamp(min=0) * up
        assert ((y.double() - want).abs() <= 2 * U * want * 1.01 + half_step(TYPES[out][0], want) * 1.01).all()


@pytest.mark.parametrize("k,n", [(512, 136), (2048, 24), (700, 33)])
def test_gelu_has_the_same_bits_in_every_kernel(k, n):
    most = 200
    a, sa = codes(171, most, k)
    b, sb = codes(172, 2 * n, k)
    sb = sb * (0.5 / (k ** 0.5 * 74 * 74))
    for t, elem in TYPES.values():
        def run(rows, experts=1, begin=None):
            y = torch.empty((rows, n), dtype=t, device="cuda")
            nv.int8_matmul(a, b.repeat(experts, 1), sb.repeat(experts), y, rows, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=b.shape[1],
                           num_experts=experts, expert_begin=begin, activation=fmt.ACT_GELU_TANH, out_elem=elem)
            return y
        whole = run(most)
        for rows in (1, 7, 16, 31, 32, 33, 100):
            assert torch.equal(run(rows), whole[:rows]), rows
        begin = torch.tensor([0, 3, 3, 60, most], dtype=torch.int32, device="cuda")
        assert torch.equal(run(most, 4, begin), whole)

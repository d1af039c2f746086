"""GPU tests of the row operators where their first tests do not reach: reports of given-up waits by stream, calls with nothing
to do, activations in their tails, tile plans of large products, second turns of persistent loops, offsets past 32 bits.

Tolerances as in test_gpu_row_ops.py: `U` = 2^-24 is half a step of fp32, `half_step(t)` the output type's."""

import numpy as np
import pytest
import torch

import nvmai_b200 as nv
from nvmai_b200 import _lib
from nvmai_b200 import format as fmt
from test_gpu_row_ops import (TYPES, U, check_order, check_product, code_of, codes, codes64, half_step, plan, random_idx, randn,
                              spread)

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


# ---- plans that small calls do not take --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["even", "random", "behind"])
@pytest.mark.parametrize("rows,k,n,experts,activation,out", [
    (8192, 160, 1100, 64, fmt.ACT_SILU, "fp16"),         # tiles of 160 rows, one set of accumulators, an output above 16 MB
    (8192, 160, 1100, 64, fmt.ACT_GELU_TANH, "fp32"),
    (8000, 300, 1801, 64, fmt.ACT_NONE, "bf16"),
    (6144, 128, 1000, 64, fmt.ACT_SILU, "bf16"),         # 128 rows, two sets, below 16 MB
    (3000, 2048, 96, 4, fmt.ACT_NONE, "fp16"),           # by the model: few units
])
def test_wide_tiles_by_expert(rows, k, n, experts, activation, out, kind):
    check_product(rows, k, n, activation, out=out, experts=experts, begin=spread(rows + experts, rows, experts, kind))


@pytest.mark.parametrize("rows,k,n,activation", [(20000, 160, 500, fmt.ACT_NONE), (9000, 1024, 1000, fmt.ACT_SILU), (4096, 96, 130, fmt.ACT_GELU_TANH),
                                                 (30011, 48, 128, fmt.ACT_NONE), (16384, 160, 2048, fmt.ACT_NONE)])
def test_wide_tiles_of_one_matrix(rows, k, n, activation):
    check_product(rows, k, n, activation, out=("fp32", "fp16")[rows % 2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,d,drop,base,weights", [
    (1531, 8, 2048, 0.0, True, "fp16"), (1531, 8, 2044, 0.2, False, "fp32"), (4001, 3, 2048, 0.1, True, None), (1200, 11, 1030, 0.1, False, "bf16"),
    (9001, 1, 2048, 0.3, True, "fp32"),
    (5, 64, 37, 0.2, True, "fp32"), (3, 40, 1001, 0.0, False, "fp16"), (70, 33, 999, 0.5, True, None),     # 16-bit: odd rows, more than 32 slots
])
def test_sums_of_many_turns_and_slots(dtype, tokens, top_k, d, drop, base, weights):
    t, elem = TYPES[dtype]
    experts = max(64, top_k)
    idx = random_idx(tokens, top_k, experts, 17 + tokens, drop)
    position, _, begin = plan(idx, experts)
    kept, pos = int(begin[-1]), torch.from_numpy(position).to(torch.int32).cuda()
    rows, dy = randn(11, max(1, kept), d).to(t), randn(14, tokens, d).to(t)
    w = None if weights is None else randn(12, tokens, top_k).to(TYPES[weights][0])
    b = randn(13, tokens, d).to(t) if base else None
    y, kw = torch.empty((tokens, d), dtype=t, device="cuda"), dict(elem=elem, w_elem=TYPES[weights or "fp32"][1])
    nv.merge_rows(rows, kept, pos, tokens, top_k, d, y, w=w, base=b, **kw)
    drows, dw = torch.full_like(rows, 77), torch.full((tokens, top_k), 77.0, device="cuda")
    nv.merge_rows_grad(dy, rows, kept, pos, w, tokens, top_k, d, drows, dw, **kw)
    held = pos >= 0
    w64 = torch.where(held, 1.0 if w is None else w.double(), 0.0)
    want = torch.zeros((tokens, d), dtype=torch.float64, device="cuda") if b is None else b.double()
    size = want.abs()
    for s in range(top_k):
        v, g = rows[pos[:, s].clamp(min=0).long()].double(), dy.double()
        want, size = want + w64[:, s, None] * v, size + (w64[:, s, None] * v).abs()
        dot = torch.where(held[:, s, None], v * g, 0.0)
        assert ((dw[:, s].double() - dot.sum(1)).abs() <= d * U * dot.abs().sum(1) * 1.01 + 1e-40).all()
        at, grad = pos[held[:, s], s].long(), (w64[:, s, None] * g)[held[:, s]]
        assert ((drows[at].double() - grad).abs() <= U * grad.abs() * 1.01 + half_step(t, grad) * 1.01).all()
    assert ((y.double() - want).abs() <= (top_k + 1) * U * size * 1.01 + half_step(t, want) * 1.01).all()


# ---- offsets past 32 bits ------------------------------------------------------------------------------------------

FAR = 0x60000000                   # elements between rows: 3 GB of 16 bits, the third row starts past 2^32 bytes


def far(rows, fill=None):
    """rows [3][d] FAR elements apart, with 64 elements of 77 behind each -> the buffer and a view of the rows"""
    n, d = rows.shape
    flat = torch.empty((n - 1) * FAR + d + 64, dtype=rows.dtype, device="cuda")
    for r in range(n):
        flat[r * FAR:r * FAR + d] = rows[r] if fill is None else fill
        flat[r * FAR + d:r * FAR + d + 64] = 77
    return flat, lambda: torch.stack([flat[r * FAR:r * FAR + d] for r in range(n)]), \
        lambda: all((flat[r * FAR + d:r * FAR + d + 64] == 77).all() for r in range(n))


@pytest.mark.parametrize("d", [64, 63])
def test_sorted_and_summed_rows_past_32_bits(d):
    x = randn(21, 3, d).half()
    idx = torch.tensor([[2], [0], [1]], dtype=torch.int32, device="cuda")
    position, source, begin = torch.empty_like(idx), torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    src, _, _ = far(x)
    dst, rows, clean = far(x, fill=7)
    nv.sort_rows(idx, 3, 1, 3, position, source, begin, x=src, d=d, x_stride=FAR, rows=dst, rows_stride=FAR)
    check_order(idx, 3, position, source, begin)
    assert torch.equal(rows(), x[[1, 2, 0]]) and clean()
    # back again, into the first buffer: a sum of one row is the row, and its gradient is dy
    nv.merge_rows(dst, 3, position, 3, 1, d, src, rows_stride=FAR, y_stride=FAR, base=src, base_stride=FAR)
    back = torch.stack([src[r * FAR:r * FAR + d] for r in range(3)])
    assert torch.equal(back, (x.double() * 2).half())
    dw = torch.empty(3, 1, device="cuda")
    nv.merge_rows_grad(src, dst, 3, position, None, 3, 1, d, dst, dw, dy_stride=FAR, rows_stride=FAR, drows_stride=FAR)
    assert torch.equal(rows(), back[[1, 2, 0]]) and clean()
    terms = back.double() * x.double()
    assert ((dw[:, 0].double() - terms.sum(1)).abs() <= d * U * terms.abs().sum(1) * 1.01).all()
    del src, dst, rows, clean
    torch.cuda.empty_cache()


def test_codes_of_sorted_rows_past_32_bits():
    d, stride = 80, 0xC0000000
    x = randn(22, 3, d)
    idx = torch.tensor([[2], [0], [1]], dtype=torch.int32, device="cuda")
    position, source, begin = torch.empty_like(idx), torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
    q, s = torch.empty(2 * stride + d, dtype=torch.int8, device="cuda"), torch.empty(3, device="cuda")
    nv.sort_rows(idx, 3, 1, 3, position, source, begin, x=x, d=d, elem=fmt.ELEM_F32, rows=q, rows_elem=fmt.ELEM_I8, rows_stride=stride, row_scales=s)
    want, scale = codes64(x[[1, 2, 0]])
    for r in range(3):
        assert torch.equal(q[r * stride:r * stride + d].double(), want[r])
    assert torch.equal(s.double(), scale)
    del q
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [3, 40])
def test_products_of_matrices_and_outputs_past_32_bits(rows):
    """channels 2 GB apart, output rows 1 GB apart: the third channel and the fifth row start past 2^32 bytes"""
    k, n, far_b, far_out = 200, 4, 0x80000000, 0x20000000
    a, sa = codes(23, rows, k)
    b, sb = codes(24, n, k)
    sb = sb * (0.5 / (k ** 0.5 * 74 * 74))
    wide = torch.empty((n - 1) * far_b + b.shape[1], dtype=torch.int8, device="cuda")
    for c in range(n):
        wide[c * far_b:c * far_b + b.shape[1]] = b[c]
    out = torch.empty((rows - 1) * far_out + n, dtype=torch.float16, device="cuda")
    near = torch.empty((rows, n), dtype=torch.float16, device="cuda")
    nv.int8_matmul(a, wide, sb, out, rows, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=far_b, out_stride=far_out)
    nv.int8_matmul(a, b, sb, near, rows, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=b.shape[1])
    nv.int8_matmul_status()
    for r in range(rows):
        assert torch.equal(out[r * far_out:r * far_out + n], near[r])
    del wide, out
    torch.cuda.empty_cache()


def test_codes_of_four_billion_rows():
    """as many rows as the count's 32 bits hold: the last block's are not lost in a sum past them"""
    rows = 0xFFFFFFFF
    x = torch.zeros(rows, dtype=torch.float16, device="cuda")
    x[-3:], x[0] = torch.tensor([2.0, -127.0, 0.5]), 1.0
    q, s = torch.full((rows,), 77, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    nv.quantize_rows(x, rows, 1, q, s)
    want, scale = codes64(torch.stack([x[0], *x[-4:]])[:, None])
    at = torch.tensor([0, rows - 4, rows - 3, rows - 2, rows - 1], device="cuda")
    assert torch.equal(q[at].double(), want[:, 0]) and torch.equal(s[at].double(), scale)
    assert int(q.count_nonzero()) == 4
    del x, q, s
    torch.cuda.empty_cache()

"""GPU tests of the row operators against plain implementations in 64 bits: sorting by expert and back, the gradients,
8-bit codes of rows, products in 8-bit integers, and a whole block made of them.

Tolerances: `u` = 2^-24 is half a step of fp32, `half_step(t)` the output type's.  A sum of n fp32 products is off by at most
n u (1 + n u) times the sum of their magnitudes; rounding to the output adds half a step of the value."""

import numpy as np
import pytest
import torch

import gpu_util as gu
import nvmai_b200 as nv
from nvmai_b200 import NvmaiError, _lib
from nvmai_b200 import format as fmt

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp16": (torch.float16, fmt.ELEM_F16), "bf16": (torch.bfloat16, fmt.ELEM_BF16), "fp32": (torch.float32, fmt.ELEM_F32)}
NONE = -1                      # 0xFFFFFFFF as torch.int32 sees it


def code_of(call):
    """The error code of a call, 0 for none.  No exception outlives this: one that is kept holds its frames and their graphs
    and handles until a garbage collection, which may come inside another test's capture and end it."""
    try:
        call()
    except NvmaiError as e:
        return e.code
    return _lib.OK


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(seed, *shape):
    return torch.randn(shape, device="cuda", generator=gen(seed))


def strided(rows, pad, offset=0):
    """The same rows with `pad` elements between them, starting `offset` elements into a buffer; what is between them is 77."""
    n, d = rows.shape
    flat = torch.full((offset + n * (d + pad),), 77, dtype=rows.dtype, device="cuda")
    view = flat[offset:].view(n, d + pad)
    view[:, :d] = rows
    return flat[offset:], view


def half_step(t, value):
    """Half a step of type t at |value|, subnormals included."""
    f = torch.finfo(t)
    return torch.clamp(value.abs() * (f.eps / 2), min=f.smallest_normal * f.eps / 2)


def random_idx(tokens, top_k, num_experts, seed, drop=0.0, repeats=False):
    g = gen(seed)
    if repeats or top_k > num_experts:
        idx = torch.randint(0, num_experts, (tokens, top_k), device="cuda", generator=g)
    else:
        idx = torch.rand((tokens, num_experts), device="cuda", generator=g).topk(top_k, dim=1).indices
    if drop:
        gone = torch.rand((tokens, top_k), device="cuda", generator=g) < drop
        far = torch.where(torch.rand((tokens, top_k), device="cuda", generator=g) < 0.5, num_experts, NONE)
        idx = torch.where(gone, far, idx)
    return idx.to(torch.int32).contiguous()


def plan(idx, num_experts):
    """position, source, begin by counting, on the host"""
    flat = idx.cpu().numpy().view(np.uint32).reshape(-1)
    kept = np.nonzero(flat < num_experts)[0]
    order = kept[np.argsort(flat[kept], kind="stable")]
    position = np.full(flat.size, NONE, dtype=np.int64)
    position[order] = np.arange(order.size)
    source = np.full(flat.size, NONE, dtype=np.int64)
    source[:order.size] = order
    begin = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=num_experts)[:num_experts])])
    return position.reshape(idx.shape), source, begin


def codes64(x):
    """codes and scales by the definition: every step rounded to fp32 (double holds the products exactly)"""
    x = x.double()
    top = x.abs().max(dim=1).values
    bad, tiny = ~torch.isfinite(top), top < 2.0 ** -120
    inverse = (127.0 / torch.where(bad | tiny, 1.0, top)).float().double()
    q = torch.round((torch.nan_to_num(x, 0.0, 0.0, 0.0) * inverse[:, None]).float().double())
    q = torch.where((bad | tiny)[:, None], 0.0, q)
    scale = torch.where(bad, float("nan"), torch.where(tiny, 0.0, (top / 127.0).float().double()))
    return q, scale


def sort(idx, num_experts, x=None, rows_elem=None, x_pad=0, rows_pad=0, offset=0, stream=None):
    """-> position, source, begin, rows buffer (filled with 77 before), scales"""
    tokens, top_k = idx.shape
    pairs = tokens * top_k
    position = torch.full((tokens, top_k), 5, dtype=torch.int32, device="cuda")
    source = torch.full((pairs,), 5, dtype=torch.int32, device="cuda")
    begin = torch.full((num_experts + 1,), 5, dtype=torch.int32, device="cuda")
    work = torch.empty(max(16, nv.sort_rows_workspace(tokens, top_k, num_experts)), dtype=torch.uint8, device="cuda")
    kw, rows, scales = {}, None, None
    if x is not None:
        d = x.shape[1]
        elem = {v[0]: v[1] for v in TYPES.values()}[x.dtype]
        flat, _ = strided(x, x_pad, offset)
        int8 = rows_elem == fmt.ELEM_I8
        rows = torch.full((pairs, d + rows_pad), 77, dtype=torch.int8 if int8 else x.dtype, device="cuda")
        scales = torch.full((pairs,), 77.0, device="cuda") if int8 else None
        kw = dict(x=flat, d=d, elem=elem, rows=rows, rows_elem=rows_elem, x_stride=d + x_pad, rows_stride=d + rows_pad,
                  row_scales=scales)
    nv.sort_rows(idx, tokens, top_k, num_experts, position, source, begin, workspace=work, workspace_bytes=work.numel(),
                 stream=stream, **kw)
    return position, source, begin, rows, scales


def check_order(idx, num_experts, position, source, begin):
    want = plan(idx, num_experts)
    for got, w, what in zip((position, source, begin), want, ("position", "source", "begin")):
        assert np.array_equal(got.cpu().numpy().astype(np.int64), w), what
    return want


ORDERS = [  # tokens, top_k, experts, drop, repeats
    (1, 8, 256, 0.0, False), (1, 1, 1, 0.0, False), (2, 3, 5, 0.5, False), (3, 64, 7, 0.0, True), (13, 8, 256, 0.0, False),
    (147, 8, 64, 0.2, False), (149, 7, 1024, 0.0, True), (201, 8, 256, 1.0, False), (1000, 2, 3, 0.1, True),
    (1531, 8, 256, 0.3, False), (4096, 8, 256, 0.0, False), (4097, 1, 1, 0.0, True), (20011, 8, 256, 0.05, False),
    (70001, 5, 1000, 0.0, True),
]


@pytest.mark.parametrize("tokens,top_k,experts,drop,repeats", ORDERS)
def test_order_of_pairs(tokens, top_k, experts, drop, repeats):
    idx = random_idx(tokens, top_k, experts, 100 + tokens, drop, repeats)
    position, source, begin, _, _ = sort(idx, experts)
    check_order(idx, experts, position, source, begin)


def test_order_agrees_with_group_pairs():
    """the same order as the framework's own grouping, expert by expert"""
    tokens, k, e = 201, 8, 64
    idx = random_idx(tokens, k, e, 3)
    w = randn(4, tokens, k).half()
    moe = nv.MoE(nv.MoEConfig(d=64, f=64, shared_f=0, num_experts=e, top_k=k, max_tokens=tokens))
    pairs = gu.dev_empty(tokens * k * 4, "u32")
    off, cnt = gu.dev_empty(e, "u32"), gu.dev_empty(e, "u32")
    moe.group_pairs(idx, w, tokens, pairs, off, cnt)
    _, source, begin, _, _ = sort(idx, e)
    torch.cuda.synchronize()
    records = gu.from_dev(pairs, np.uint32).reshape(-1, 4)
    assert np.array_equal(records[:, 0] * k + records[:, 2], source.cpu().numpy().astype(np.uint32))
    assert np.array_equal(np.diff(begin.cpu().numpy()), gu.from_dev(cnt, np.uint32))


def test_no_tokens_leaves_empty_experts():
    begin = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    nv.sort_rows(None, 0, 2, 8, None, None, begin)
    assert begin.tolist() == [0] * 9


ROWS = [  # tokens, top_k, experts, d, x_pad, rows_pad, offset, drop
    (1, 8, 256, 2048, 0, 0, 0, 0.0), (5, 3, 4, 1, 0, 0, 0, 0.4), (7, 2, 9, 37, 0, 0, 1, 0.0), (33, 8, 16, 64, 8, 16, 8, 0.3),
    (150, 8, 256, 2048, 0, 0, 0, 0.5), (201, 5, 100, 999, 3, 2, 0, 0.1), (300, 1, 8, 520, 0, 8, 0, 0.0),
    (9001, 8, 64, 40, 0, 0, 0, 0.2), (6000, 3, 200, 33, 0, 0, 0, 0.0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,experts,d,x_pad,rows_pad,offset,drop", ROWS)
def test_rows_go_to_their_experts(dtype, tokens, top_k, experts, d, x_pad, rows_pad, offset, drop):
    t, elem = TYPES[dtype]
    idx = random_idx(tokens, top_k, experts, 7 + tokens, drop)
    x = randn(8, tokens, d).to(t)
    x.view(-1)[0] = float("nan")                       # bits are copied, whatever they are
    position, source, begin, rows, _ = sort(idx, experts, x, elem, x_pad, rows_pad, offset)
    _, src, bounds = check_order(idx, experts, position, source, begin)
    kept = int(bounds[-1])
    raw = torch.int16 if t.itemsize == 2 else torch.int32
    want = x.view(raw)[torch.from_numpy(src[:kept] // top_k).cuda()]
    assert torch.equal(rows[:kept, :d].contiguous().view(raw), want)
    assert (rows[kept:] == 77).all() and (rows[:, d:] == 77).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,experts,d,x_pad,rows_pad,offset,drop", ROWS)
def test_rows_as_codes(dtype, tokens, top_k, experts, d, x_pad, rows_pad, offset, drop):
    t, _ = TYPES[dtype]
    idx = random_idx(tokens, top_k, experts, 7 + tokens, drop)
    x = randn(9, tokens, d).to(t)
    position, source, begin, rows, scales = sort(idx, experts, x, fmt.ELEM_I8, x_pad, rows_pad, offset)
    _, src, bounds = check_order(idx, experts, position, source, begin)
    kept = int(bounds[-1])
    q, s = codes64(x)
    at = torch.from_numpy(src[:kept] // top_k).cuda()
    assert torch.equal(rows[:kept, :d].double(), q[at])
    assert torch.equal(scales[:kept].double(), s[at])
    assert (rows[kept:] == 77).all() and (rows[:, d:] == 77).all() and (scales[kept:] == 77).all()


# ---- back to the tokens, and the gradients ----------------------------------------------------------------

MERGES = [  # tokens, top_k, experts, d, pad, offset, drop, base, weights
    (1, 8, 256, 2048, 0, 0, 0.0, True, "fp16"), (3, 1, 4, 1, 0, 0, 0.3, False, "fp32"), (9, 8, 8, 37, 0, 1, 0.2, True, None),
    (64, 6, 32, 640, 8, 8, 0.5, True, "bf16"), (201, 8, 256, 2048, 0, 0, 0.0, False, "fp32"), (300, 3, 9, 77, 2, 0, 0.1, False, None),
    (5, 64, 80, 264, 0, 0, 0.0, False, "fp16"), (8, 4, 16, 96, 0, 0, 1.0, True, "fp16"), (8, 4, 16, 96, 0, 0, 1.0, False, "fp16"),
]


def merged(idx, experts, d, t, pad, offset, base, weights):
    """position, rows buffer and view, w, base; rows behind the kept ones hold NaN, and so do weights of what is not kept"""
    tokens, top_k = idx.shape
    position, _, begin = plan(idx, experts)
    kept = int(begin[-1])
    rows = torch.full((tokens * top_k, d), float("nan"), device="cuda")
    rows[:kept] = randn(11, tokens * top_k, d)[:kept]
    flat, view = strided(rows.to(t), pad, offset)
    w = None
    pos = torch.from_numpy(position).to(torch.int32).cuda()
    if weights:
        w = torch.where(pos >= 0, randn(12, tokens, top_k), float("nan")).to(TYPES[weights][0])
    return pos, kept, flat, view, w, (randn(13, tokens, d).to(t) if base else None)


def weight64(pos, w):
    one = torch.ones(pos.shape, dtype=torch.float64, device="cuda") if w is None else w.double()
    return torch.where(pos >= 0, one, 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,experts,d,pad,offset,drop,base,weights", MERGES)
def test_weighted_sum(dtype, tokens, top_k, experts, d, pad, offset, drop, base, weights):
    t, elem = TYPES[dtype]
    idx = random_idx(tokens, top_k, experts, 17 + tokens, drop)
    pos, kept, flat, view, w, b = merged(idx, experts, d, t, pad, offset, base, weights)
    y = torch.full((tokens, d + pad), 77, dtype=t, device="cuda")
    nv.merge_rows(flat, kept, pos, tokens, top_k, d, y, elem=elem, w=w, w_elem=TYPES[weights or "fp32"][1], base=b,
                  rows_stride=d + pad, y_stride=d + pad)
    w64 = weight64(pos, w)
    v = torch.nan_to_num(view[:, :d].double())[pos.clamp(min=0).long()]
    terms = w64[:, :, None] * v
    b64 = b.double() if base else torch.zeros((tokens, d), dtype=torch.float64, device="cuda")
    want, size = b64 + terms.sum(1), b64.abs() + terms.abs().sum(1)
    assert ((y[:, :d].double() - want).abs() <= (top_k + 1) * U * size * 1.01 + half_step(t, want) * 1.01).all()
    assert (y[:, d:] == 77).all()
    if base:                                           # in place gives the same bits
        again = b.clone()
        nv.merge_rows(flat, kept, pos, tokens, top_k, d, again, elem=elem, w=w, w_elem=TYPES[weights or "fp32"][1], base=again,
                      rows_stride=d + pad)
        assert torch.equal(again, y[:, :d])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,experts,d,pad,offset,drop,base,weights", MERGES)
def test_gradients_of_the_weighted_sum(dtype, tokens, top_k, experts, d, pad, offset, drop, base, weights):
    t, elem = TYPES[dtype]
    idx = random_idx(tokens, top_k, experts, 17 + tokens, drop)
    pos, kept, flat, view, w, _ = merged(idx, experts, d, t, pad, offset, False, weights)
    dy = randn(14, tokens, d).to(t)
    drows = torch.full((tokens * top_k, d + pad), 77, dtype=t, device="cuda")
    dw = torch.full((tokens, top_k), 77.0, device="cuda")
    kw = dict(elem=elem, w_elem=TYPES[weights or "fp32"][1], rows_stride=d + pad, drows_stride=d + pad)
    nv.merge_rows_grad(dy, flat, kept, pos, w, tokens, top_k, d, drows, dw, **kw)
    held = pos >= 0
    w64 = weight64(pos, w)
    v = torch.nan_to_num(view[:, :d].double())[pos.clamp(min=0).long()]
    terms = torch.where(held[:, :, None], v * dy.double()[:, None, :], 0.0)
    assert ((dw.double() - terms.sum(2)).abs() <= d * U * terms.abs().sum(2) * 1.01 + 1e-40).all()
    want = (w64[:, :, None] * dy.double()[:, None, :])[held]
    got = drows[pos[held].long(), :d].double()
    assert ((got - want).abs() <= U * want.abs() * 1.01 + half_step(t, want) * 1.01).all()
    assert (drows[kept:] == 77).all() and (drows[:, d:] == 77).all()
    # each alone, and the rows' gradient over the rows themselves
    dw2 = torch.zeros_like(dw)
    nv.merge_rows_grad(dy, flat, kept, pos, w, tokens, top_k, d, None, dw2, **kw)
    assert torch.equal(dw, dw2)
    only = torch.full_like(drows, 77)
    nv.merge_rows_grad(dy, None, kept, pos, w, tokens, top_k, d, only, None, **kw)
    assert torch.equal(only, drows)
    over = view.clone()
    nv.merge_rows_grad(dy, over, kept, pos, w, tokens, top_k, d, over, dw2, **kw)
    assert torch.equal(dw, dw2) and torch.equal(over[:kept, :d], drows[:kept, :d])


def test_gradients_against_differences():
    """L = <g, merge(sort(x), w)> is linear in x and in w: a difference of 1 / 8 is exact in 64 bits and shows the gradient"""
    tokens, k, e, d = 6, 3, 5, 24
    idx = random_idx(tokens, k, e, 31, 0.2)
    x, w, g = randn(32, tokens, d), randn(33, tokens, k), randn(34, tokens, d)
    position, _, begin, rows, _ = sort(idx, e, x, fmt.ELEM_F32)
    kept = int(begin[-1])
    drows, dw, dx = torch.zeros_like(rows), torch.empty_like(w), torch.empty_like(x)
    nv.merge_rows_grad(g, rows, kept, position, w, tokens, k, d, drows, dw, elem=fmt.ELEM_F32, w_elem=fmt.ELEM_F32)
    nv.merge_rows(drows, kept, position, tokens, k, d, dx, elem=fmt.ELEM_F32)
    held = (position >= 0).double()

    def loss(x, w):
        return (g.double() * (w * held)[:, :, None].sum(1) * x).sum()

    x, w = x.double(), w.double()
    base = loss(x, w)
    for t in range(tokens):
        for i in range(0, d, 5):
            moved = x.clone()
            moved[t, i] += 0.125
            assert abs((loss(moved, w) - base) / 0.125 - dx[t, i].double()) <= 1e-5
        for s in range(k):
            moved = w.clone()
            moved[t, s] += 0.125
            assert abs((loss(x, moved) - base) / 0.125 - dw[t, s].double()) <= 1e-4


def test_positions_out_of_range_are_never_addresses():
    """positions at and far behind the last row count as not held, in all three directions"""
    tokens, k, d, n = 4, 2, 64, 5
    pos = torch.tensor([[0, 5], [4, 0x7FFFFFFF], [NONE, 1], [-2, 6]], dtype=torch.int32, device="cuda")
    rows, dy = randn(41, n, d), randn(42, tokens, d)
    y, drows, dw = torch.empty(tokens, d, device="cuda"), torch.full((n, d), 77.0, device="cuda"), torch.full((tokens, k), 77.0, device="cuda")
    nv.merge_rows(rows, n, pos, tokens, k, d, y, elem=fmt.ELEM_F32)
    nv.merge_rows_grad(dy, rows, n, pos, None, tokens, k, d, drows, dw, elem=fmt.ELEM_F32)
    assert torch.equal(y, torch.stack([rows[0], rows[4], rows[1], torch.zeros(d, device="cuda")]))
    assert torch.equal(drows[[0, 4, 1]], dy[:3]) and (drows[2:4] == 77).all()
    assert dw[0, 1] == 0 and dw[1, 1] == 0 and dw[2, 0] == 0 and (dw[3] == 0).all()


def test_a_row_named_twice():
    """forward every naming counts; the gradient's row is the product of one of the two"""
    tokens, k, d = 3, 2, 40
    pos = torch.tensor([[0, 0], [1, 0], [2, 1]], dtype=torch.int32, device="cuda")
    rows, dy = randn(45, 3, d), randn(46, tokens, d)
    y, drows, dw = torch.empty(tokens, d, device="cuda"), torch.empty(3, d, device="cuda"), torch.empty(tokens, k, device="cuda")
    nv.merge_rows(rows, 3, pos, tokens, k, d, y, elem=fmt.ELEM_F32)
    assert torch.equal(y, torch.stack([rows[0] + rows[0], rows[1] + rows[0], rows[2] + rows[1]]))
    nv.merge_rows_grad(dy, rows, 3, pos, None, tokens, k, d, drows, dw, elem=fmt.ELEM_F32)
    for r, names in enumerate(([0, 1], [1, 2], [2])):
        assert all(any(v == dy[t, i] for t in names) for i, v in enumerate(drows[r]))
    terms = rows[pos.long()].double() * dy.double()[:, None]
    assert ((dw.double() - terms.sum(2)).abs() <= d * U * terms.abs().sum(2) * 1.01).all()


@pytest.mark.parametrize("d", [64, 63])
def test_rows_between_kernels_of_other_streams(d):
    """two calls at once on two streams, each with buffers of its own, while the default stream is busy"""
    tokens, k, e = 257, 4, 16
    jobs = []
    for i in range(2):
        idx = random_idx(tokens, k, e, 300 + i, 0.1)
        x = randn(302 + i, tokens, d).half()
        bufs = dict(position=torch.empty_like(idx), source=torch.empty(tokens * k, dtype=torch.int32, device="cuda"),
                    begin=torch.empty(e + 1, dtype=torch.int32, device="cuda"), rows=torch.zeros(tokens * k, d, dtype=torch.float16, device="cuda"),
                    y=torch.empty(tokens, d, dtype=torch.float16, device="cuda"))
        jobs.append((idx, x, bufs, torch.cuda.Stream()))
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        busy = busy @ busy * 1e-3
        for idx, x, b, stream in jobs:
            nv.sort_rows(idx, tokens, k, e, b["position"], b["source"], b["begin"], x=x, d=d, rows=b["rows"], stream=stream)
            nv.merge_rows(b["rows"], tokens * k, b["position"], tokens, k, d, b["y"], stream=stream)
    torch.cuda.synchronize()
    for idx, x, b, _ in jobs:
        check_order(idx, e, b["position"], b["source"], b["begin"])
        held = (b["position"] >= 0).double().sum(1, keepdim=True)
        want = x.double() * held                       # the same row, as many times as it is held: exact in fp32, rounded once
        assert torch.equal(b["y"], want.half())


def test_rows_from_a_pointer_inside_a_buffer():
    """pieces of every width: the same rows from bases 16-, 4- and 2-byte aligned give the same bits"""
    tokens, k, e, d = 37, 3, 8, 120
    idx = random_idx(tokens, k, e, 310)
    x, w = randn(311, tokens, d).bfloat16(), randn(312, tokens, k)
    outs = []
    for offset in (0, 2, 1):
        position, _, begin, rows, _ = sort(idx, e, x, fmt.ELEM_BF16, offset=offset)
        flat, view = strided(rows, 0, offset)
        y = torch.empty(offset + tokens * d, dtype=torch.bfloat16, device="cuda")
        nv.merge_rows(flat, tokens * k, position, tokens, k, d, y[offset:], elem=fmt.ELEM_BF16, w=w, w_elem=fmt.ELEM_F32)
        q, s = torch.empty(tokens, d, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
        nv.quantize_rows(strided(x, 0, offset)[0], tokens, d, q, s, elem=fmt.ELEM_BF16)
        dr, dw = torch.empty(offset + tokens * k * d, dtype=torch.bfloat16, device="cuda"), torch.empty(tokens, k, device="cuda")
        nv.merge_rows_grad(strided(x, 0, offset)[0], flat, tokens * k, position, w, tokens, k, d, dr[offset:], dw, elem=fmt.ELEM_BF16,
                           w_elem=fmt.ELEM_F32)
        outs.append((rows, y[offset:].clone(), q, s, dr[offset:].clone()))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


# ---- 8-bit codes ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,pad,offset,q_pad", [(1, 1, 0, 0, 0), (3, 37, 0, 1, 3), (5, 64, 8, 8, 16), (201, 512, 0, 0, 0),
                                                     (17, 2048, 0, 0, 0), (9, 2049, 0, 0, 7), (4, 20000, 0, 0, 0), (2, 70000, 0, 1, 0)])
def test_codes_of_rows(dtype, rows, n, pad, offset, q_pad):
    t, elem = TYPES[dtype]
    x = randn(51, rows, n).to(t)
    flat, _ = strided(x, pad, offset)
    q = torch.full((rows, n + q_pad), 77, dtype=torch.int8, device="cuda")
    s = torch.full((rows,), 77.0, device="cuda")
    nv.quantize_rows(flat, rows, n, q, s, elem=elem, x_stride=n + pad, q_stride=n + q_pad)
    want, scale = codes64(x)
    assert torch.equal(q[:, :n].double(), want) and torch.equal(s.double(), scale)
    assert (q[:, n:] == 77).all()


def test_codes_of_special_rows():
    big, tiny = torch.finfo(torch.float32).max, 2.0 ** -120
    x = torch.zeros(9, 40, device="cuda")
    x[1, 3] = -0.0
    x[2, 5], x[2, 6] = float("inf"), 1.0
    x[3, 39] = float("nan")
    x[4, 0], x[4, 1], x[4, 2] = big, -big, big / 2
    x[5, 0] = tiny
    x[6, 0] = tiny * 0.99
    x[7, 0], x[7, 1], x[7, 2], x[7, 3] = 127.0, 0.5, 1.5, -2.5              # ties go to the even code
    x[8, 0], x[8, 1] = -float("inf"), float("nan")
    q = torch.full((9, 40), 77, dtype=torch.int8, device="cuda")
    s = torch.full((9,), 77.0, device="cuda")
    nv.quantize_rows(x, 9, 40, q, s, elem=fmt.ELEM_F32)
    want, scale = codes64(x)
    assert torch.equal(q.double(), want)
    assert torch.equal(torch.isnan(s), torch.tensor([0, 0, 1, 1, 0, 0, 0, 0, 1], device="cuda").bool())
    assert torch.equal(torch.nan_to_num(s.double()), torch.nan_to_num(scale))
    assert q[4, :3].tolist() == [127, -127, 64] and q[7, :4].tolist() == [127, 0, 2, -2] and q[5, 0] == 127 and q[6, 0] == 0


def test_rows_past_32_bits():
    """rows whose byte offsets pass 2^32: the last row is right and nothing else is written"""
    n, stride = 48, 0xC0000000                           # three rows 3 GB apart
    q = torch.full((2 * stride + n,), 77, dtype=torch.int8, device="cuda")
    s = torch.empty(3, device="cuda")
    x = randn(53, 3, n)
    nv.quantize_rows(x, 3, n, q, s, elem=fmt.ELEM_F32, q_stride=stride)
    want, _ = codes64(x)
    for r in range(3):
        assert torch.equal(q[r * stride:r * stride + n].double(), want[r])
    assert (q[stride + n:stride + 4096] == 77).all() and (q[:n + 4096][n:] == 77).all()


# ---- products --------------------------------------------------------------------------------------------------

def act64(v, activation):
    if activation == fmt.ACT_SILU:
        return v * torch.sigmoid(v)
    inner = (0.7978845608028654 * (v + 0.044715 * v ** 3)).clamp(-20, 20)
    return 0.5 * v * (1 + torch.tanh(inner))


def product64(a, sa, b, sb, n, activation, begin=None):
    """-> the product, how far fp32 steps may be from it before the output is rounded, rows that are somebody's"""
    rows = a.shape[0]
    v = torch.zeros((rows, b.shape[1]), dtype=torch.float64, device="cuda")
    own = torch.zeros(rows, dtype=torch.bool, device="cuda")
    ends = [0, rows] if begin is None else begin
    for e in range(len(ends) - 1):
        lo, hi = int(ends[e]), int(ends[e + 1])
        if hi > lo:
            v[lo:hi] = (a[lo:hi].double() @ b[e].double().T) * sa[lo:hi, None].double() * sb[e].double()
            own[lo:hi] = True
    if activation == fmt.ACT_NONE:
        return v, 3 * U * v.abs(), own            # the sum, the scales' product and their product are rounded once each
    g, up = v[:, :n], v[:, n:]
    y = act64(g, activation) * up
    if activation == fmt.ACT_SILU:
        # silu'(g) g = silu(g) (1 + g (1 - sigmoid(g))): a relative error grows by 1 + |g| at most.  3 steps of g, 7 of the
        # activation itself (exp 2 ulp = 4, sum, quotient, and one for the product), 3 of up, 1 of the last product
        return y, ((1 + g.abs()) * 3 + 11) * U * y.abs() * 1.01, own
    # tanh 2 ulp at 1 = 2 steps, its argument off by 9 steps times z (1 - tanh^2 z) <= 0.45, the sum 2; then 3 + 3 + 2 relative
    return y, (0.5 * g * up).abs() * 10 * U + 8 * U * y.abs() * 1.01, own


def codes(seed, rows, k, pad=0):
    """random codes with the extremes among them, rows a multiple of 16 bytes apart"""
    g = gen(seed)
    width = (k + 15) // 16 * 16 + pad
    q = torch.randint(-127, 128, (rows, width), device="cuda", generator=g, dtype=torch.int8)
    q[0, :k] = 127 if seed % 2 else -128
    return q, torch.rand(rows, device="cuda", generator=g) + 0.1


def check_product(rows, k, n, activation, out="fp16", a_type=None, experts=1, begin=None, a_pad=0, b_pad=0, out_pad=0, seed=61,
                  stream=None):
    gated = activation != fmt.ACT_NONE
    channels = 2 * n if gated else n
    b, sb = codes(seed, experts * channels, k, b_pad)
    sb = sb * (0.5 / (k ** 0.5 * 74 * (74 if a_type is None else 1)))              # products of some units
    t_out, out_elem = TYPES[out]
    kw = {}
    if a_type is None:
        a, sa = codes(seed + 1, rows, k, a_pad)
        qa, kw = a[:, :k], dict(a_scales=sa, a_stride=a.shape[1])
    else:
        x = randn(seed + 1, rows, k).to(TYPES[a_type][0])
        qa, sa = codes64(x)
        size = nv.int8_matmul_workspace(rows, k, TYPES[a_type][1])
        work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        flat, _ = strided(x, a_pad)
        a, kw = flat, dict(a_elem=TYPES[a_type][1], a_stride=k + a_pad, workspace=work, workspace_bytes=work.numel())
    dev_begin = None if begin is None else torch.tensor(begin, dtype=torch.int64, device="cuda").to(torch.int32)
    y = torch.full((rows, n + out_pad), 77, dtype=t_out, device="cuda")
    nv.int8_matmul(a, b, sb, y, rows, k, n, num_experts=experts, expert_begin=dev_begin, activation=activation, out_elem=out_elem,
                   b_stride=b.shape[1], out_stride=n + out_pad, stream=stream, **kw)
    nv.int8_matmul_status(stream)
    want, off, own = product64(qa, sa, b[:, :k].view(experts, channels, k), sb.view(experts, channels), n, activation, begin)
    over = want.abs() > torch.finfo(t_out).max * 0.999
    assert not over.any(), "the case leaves the output type"
    err = (y[own, :n].double() - want[own]).abs()
    tol = off[own] + half_step(t_out, want[own]) * 1.01
    assert (err <= tol).all(), f"worst {float((err / tol).max())} at {int((err / tol).argmax())}"
    assert (y[~own] == 77).all() and (y[:, n:] == 77).all()
    return y


DENSE = [  # rows, k, n
    (1, 1, 1), (1, 2048, 512), (2, 16, 8), (3, 100, 33), (7, 511, 130), (8, 512, 2048), (9, 2048, 96), (16, 128, 256), (17, 64, 31),
    (31, 300, 129), (32, 2048, 512), (33, 2047, 64), (64, 640, 1000), (100, 96, 257), (127, 2048, 128), (129, 128, 300),
    (201, 513, 511), (300, 4096, 200), (1000, 272, 384),
]


@pytest.mark.parametrize("rows,k,n", DENSE)
@pytest.mark.parametrize("activation", [fmt.ACT_NONE, fmt.ACT_SILU, fmt.ACT_GELU_TANH])
def test_product_with_one_matrix(rows, k, n, activation):
    check_product(rows, k, n, activation, out=("fp16", "bf16", "fp32")[(rows + activation) % 3])


@pytest.mark.parametrize("a_type", TYPES)
@pytest.mark.parametrize("rows,k,n,a_pad", [(1, 2048, 512, 0), (1, 37, 9, 0), (5, 512, 130, 8), (13, 513, 64, 1), (40, 2048, 256, 0), (201, 300, 100, 0)])
@pytest.mark.parametrize("activation", [fmt.ACT_NONE, fmt.ACT_SILU])
def test_product_quantises_its_rows(a_type, rows, k, n, a_pad, activation):
    check_product(rows, k, n, activation, out="fp32", a_type=a_type, a_pad=a_pad)


@pytest.mark.parametrize("a_pad,b_pad,out_pad", [(16, 0, 0), (0, 48, 0), (0, 0, 5), (32, 16, 1)])
@pytest.mark.parametrize("rows", [3, 20, 150])
def test_product_of_strided_rows(rows, a_pad, b_pad, out_pad):
    check_product(rows, 160, 72, fmt.ACT_NONE, a_pad=a_pad, b_pad=b_pad, out_pad=out_pad)
    check_product(rows, 150, 72, fmt.ACT_SILU, a_pad=a_pad, b_pad=b_pad, out_pad=out_pad)


def spread(seed, rows, experts, kind):
    """begin of `rows` rows over the experts"""
    r = np.random.default_rng(seed)
    if kind == "even":
        return np.linspace(0, rows, experts + 1).astype(np.int64).tolist()
    if kind == "one":
        at = int(r.integers(0, experts))
        return [0] * (at + 1) + [rows] * (experts - at)
    if kind == "behind":                               # rows in front of the first and behind the last expert are nobody's
        cuts = np.sort(r.integers(rows // 4, rows - rows // 4 + 1, experts + 1))
        return cuts.tolist()
    cuts = np.sort(r.integers(0, rows + 1, experts - 1))
    return [0, *cuts.tolist(), rows]


@pytest.mark.parametrize("kind", ["even", "random", "one", "behind"])
@pytest.mark.parametrize("rows,k,n,experts", [(8, 2048, 64, 256), (1, 64, 16, 4), (13, 200, 40, 5), (64, 512, 130, 256), (104, 2048, 48, 64),
                                              (300, 96, 64, 3), (700, 640, 100, 9), (2000, 128, 200, 31), (1608, 512, 256, 256)])
@pytest.mark.parametrize("activation", [fmt.ACT_NONE, fmt.ACT_SILU])
def test_product_by_expert(rows, k, n, experts, kind, activation):
    check_product(rows, k, n, activation, out=("fp16", "fp32")[rows % 2], experts=experts, begin=spread(rows + experts, rows, experts, kind))


@pytest.mark.parametrize("activation", [fmt.ACT_NONE, fmt.ACT_SILU])
@pytest.mark.parametrize("k,n", [(512, 136), (2048, 24), (700, 33)])
def test_a_rows_bits_do_not_depend_on_the_others(k, n, activation):
    """the kernels for few and for many rows give the same bits: every prefix of the rows has those of all of them"""
    most = 200
    gated = activation != fmt.ACT_NONE
    a, sa = codes(171, most, k)
    b, sb = codes(172, n * (2 if gated else 1), k)
    sb = sb * (0.5 / (k ** 0.5 * 74 * 74))
    for out in TYPES:
        t, elem = TYPES[out]
        y = {}
        for rows in (1, 7, 16, 31, 32, 33, 100, most):
            y[rows] = torch.empty((rows, n), dtype=t, device="cuda")
            nv.int8_matmul(a, b, sb, y[rows], rows, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=b.shape[1], activation=activation, out_elem=elem)
        for rows in y:
            assert torch.equal(y[rows], y[most][:rows]), rows
        begin = torch.tensor([0, 3, 3, 60, most], dtype=torch.int32, device="cuda")     # four experts with the same matrix
        z = torch.empty((most, n), dtype=t, device="cuda")
        nv.int8_matmul(a, b.repeat(4, 1), sb.repeat(4), z, most, k, n, a_scales=sa, a_stride=a.shape[1], b_stride=b.shape[1], num_experts=4,
                       expert_begin=begin, activation=activation, out_elem=elem)
        assert torch.equal(z, y[most])


@pytest.mark.parametrize("a_type", TYPES)
@pytest.mark.parametrize("rows,experts", [(8, 64), (200, 16), (900, 4)])
def test_product_by_expert_quantises_its_rows(a_type, rows, experts):
    check_product(rows, 530, 90, fmt.ACT_SILU, out="fp32", a_type=a_type, experts=experts, begin=spread(rows, rows, experts, "behind"))


def test_product_begins_that_lie():
    """begins behind the rows or out of order name no row outside; what they do name is some expert's product or left alone"""
    rows, k, n, experts = 40, 64, 16, 4
    a, sa = codes(70, rows, k)
    b, sb = codes(71, experts * n, k)
    for begin in ([0, 10, 20, 30, 1000000], [0, 50, 60, 70, 80], [-1, -1, -1, -1, -1], [0, 30, 10, 35, 40], [40, 30, 20, 10, 0]):
        y = torch.full((rows + 8, n), 77.0, device="cuda")
        nv.int8_matmul(a, b, sb, y, rows, k, n, a_scales=sa, num_experts=experts, out_elem=fmt.ELEM_F32,
                       expert_begin=torch.tensor(begin, device="cuda").to(torch.int32))
        nv.int8_matmul_status()
        assert (y[rows:] == 77).all()


def test_product_with_a_row_that_is_not_finite():
    rows, k, n = 6, 128, 24
    x = randn(81, rows, k)
    x[2, 7], x[4, 0] = float("inf"), float("nan")
    x[5] = 0
    b, sb = codes(82, n, k)
    work = torch.empty(nv.int8_matmul_workspace(rows, k, fmt.ELEM_F32), dtype=torch.uint8, device="cuda")
    y = torch.empty((rows, n), device="cuda")
    nv.int8_matmul(x, b, sb, y, rows, k, n, a_elem=fmt.ELEM_F32, out_elem=fmt.ELEM_F32, workspace=work, workspace_bytes=work.numel())
    assert torch.isnan(y[[2, 4]]).all() and torch.isfinite(y[[0, 1, 3, 5]]).all() and (y[5] == 0).all()


def test_largest_sum_is_exact():
    """the longest rows that are allowed, all codes at -128: the sum is 2^31 - 2^14 and does not wrap"""
    k = 131071
    for rows in (1, 40):
        a = torch.full((rows, k + 1), -128, dtype=torch.int8, device="cuda")
        b = torch.full((8, k + 1), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(max(rows, 8), device="cuda")
        y = torch.empty((rows, 8), device="cuda")
        nv.int8_matmul(a, b, one, y, rows, k, 8, a_stride=k + 1, b_stride=k + 1, a_scales=one, out_elem=fmt.ELEM_F32)
        nv.int8_matmul_status()
        assert (y == float(np.float32(16384 * k))).all()


# ---- together ----------------------------------------------------------------------------------------------------

class Block:
    """A block of experts in 8-bit codes made of the operators, weights from the framework's affine blobs."""

    def __init__(self, tokens, d, f, e, k, seed):
        from nvmai_b200 import synthetic
        self.host = synthetic.layer(seed, d=d, f=f, shared_f=0, num_experts=e, routed_bits=8, meta=fmt.META_BF16)
        self.size = tokens, d, f, e, k
        self.moe = nv.MoE(nv.MoEConfig(d=d, f=f, shared_f=0, num_experts=e, top_k=k, routed_bits=8, shared_bits=8,
                                       shared_gate_kind=fmt.GATE_NONE, max_tokens=tokens, out_dtype=fmt.OUT_FP32))
        self.layer = gu.DeviceLayer(self.host)
        self.layer.register(self.moe, 0)
        self.gate_up, self.gate_up_scales = self.weights(("gate", "up"), f, d)
        self.down, self.down_scales = self.weights(("down",), d, f)
        pairs, dev = tokens * k, dict(device="cuda")
        self.idx, self.w = torch.empty((tokens, k), dtype=torch.int32, **dev), torch.empty((tokens, k), dtype=torch.float16, **dev)
        self.position, self.source = torch.empty((tokens, k), dtype=torch.int32, **dev), torch.empty(pairs, dtype=torch.int32, **dev)
        self.begin = torch.empty(e + 1, dtype=torch.int32, **dev)
        self.rows, self.scales = torch.empty((pairs, d), dtype=torch.int8, **dev), torch.empty(pairs, **dev)
        self.acts, self.out = torch.empty((pairs, f), dtype=torch.float16, **dev), torch.empty((pairs, d), dtype=torch.float32, **dev)
        self.y = torch.empty((tokens, d), **dev)
        self.work = torch.empty(max(16, nv.sort_rows_workspace(tokens, k, e), nv.int8_matmul_workspace(pairs, f, fmt.ELEM_F16)),
                                dtype=torch.uint8, **dev)

    def weights(self, names, rows, n):
        e, off = self.size[3], self.host["offsets"]
        values = torch.empty((e, len(names), rows, n), device="cuda")
        blob = self.layer.experts.data_ptr()
        for x in range(e):
            for i, name in enumerate(names):
                w, s, b = (blob + x * self.host["stride"] + off[f"{name}_{p}"] for p in "wsb")
                nv.dequant(8, fmt.META_BF16, w, s, b, rows, n, values[x, i])
        q = torch.empty((e, len(names) * rows, n), dtype=torch.int8, device="cuda")
        s = torch.empty((e, len(names) * rows), device="cuda")
        nv.quantize_rows(values, e * len(names) * rows, n, q, s, elem=fmt.ELEM_F32)
        return q, s

    def run(self, x, stream=None):
        tokens, d, f, e, k = self.size
        work = dict(workspace=self.work, workspace_bytes=self.work.numel(), stream=stream)
        self.moe.encode_router(0, x, self.idx, self.w, tokens=tokens, stream=stream)
        nv.sort_rows(self.idx, tokens, k, e, self.position, self.source, self.begin, x=x, d=d, rows=self.rows, rows_elem=fmt.ELEM_I8,
                     row_scales=self.scales, **work)
        nv.int8_matmul(self.rows, self.gate_up, self.gate_up_scales, self.acts, tokens * k, d, f, a_scales=self.scales, num_experts=e,
                       expert_begin=self.begin, activation=fmt.ACT_SILU, **work)
        nv.int8_matmul(self.acts, self.down, self.down_scales, self.out, tokens * k, f, d, a_elem=fmt.ELEM_F16, num_experts=e,
                       expert_begin=self.begin, out_elem=fmt.ELEM_F32, **work)
        nv.merge_rows(self.out, tokens * k, self.position, tokens, k, d, self.y, elem=fmt.ELEM_F32, w=self.w, stream=stream)

    def check(self, x):
        """every stage against 64 bits on the stage's own input"""
        tokens, d, f, e, k = self.size
        position, source, begin = check_order(self.idx, e, self.position, self.source, self.begin)
        q, s = codes64(x)
        at = torch.from_numpy(source // k).cuda()
        assert torch.equal(self.rows.double(), q[at]) and torch.equal(self.scales.double(), s[at])
        want, off, _ = product64(self.rows, self.scales, self.gate_up, self.gate_up_scales, f, fmt.ACT_SILU, begin)
        assert ((self.acts.double() - want).abs() <= off + half_step(torch.float16, want) * 1.01).all()
        qa, sa = codes64(self.acts)
        want, off, _ = product64(qa, sa, self.down, self.down_scales, d, fmt.ACT_NONE, begin)
        assert ((self.out.double() - want).abs() <= off + half_step(torch.float32, want) * 1.01).all()
        terms = self.w.double()[:, :, None] * self.out.double()[torch.from_numpy(position).cuda()]
        assert ((self.y.double() - terms.sum(1)).abs() <= (k + 2) * U * terms.abs().sum(1) * 1.01).all()


def hidden(tokens, d, seed):
    return randn(seed, tokens, d).half()


@pytest.mark.parametrize("tokens,d,f,e", [(1, 256, 128, 32), (5, 320, 192, 40), (77, 256, 128, 32), (500, 512, 128, 24)])
def test_a_block_of_the_operators(tokens, d, f, e):
    block = Block(tokens, d, f, e, 8, 90 + tokens)
    x = hidden(tokens, d, 91)
    block.run(x)
    nv.int8_matmul_status()
    block.check(x)


def test_a_block_is_near_the_frameworks_own():
    """the same layer through layer_decode (its affine codes as they are): the distance is that of the 8-bit codes.  Each of
    the three quantisations (x, the activations, the weights' rows) moves a value by at most half a step of 1 / 127 of its row's
    largest; on random rows of this length that is about 1 % of a dot product's spread each, and 10 % bounds their sum"""
    tokens, d, f, e = 16, 512, 256, 16
    block = Block(tokens, d, f, e, 8, 95)
    x = hidden(tokens, d, 96)
    block.run(x)
    own = torch.empty_like(block.y)
    block.moe.layer_decode(0, x, tokens, h2_out=own)
    torch.cuda.synchronize()
    assert float((block.y - own).norm() / own.norm()) < 0.1


def test_a_captured_block_replays_on_new_rows_and_streams():
    """captured on a side stream, replayed on other inputs with the plain calls' bits, while a second block runs beside it"""
    tokens, d, f, e = 33, 256, 128, 16
    one, two = Block(tokens, d, f, e, 8, 97), Block(tokens, d, f, e, 8, 98)
    x = hidden(tokens, d, 99)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    one.run(x, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        one.run(x, stream=side)
    for seed in (100, 101, 102):
        new = hidden(tokens, d, seed)
        x.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(3):
                graph.replay()
        for _ in range(3):
            two.run(new, stream=other)
        torch.cuda.synchronize()
        one.check(new)
        two.check(new)


def test_a_wait_that_runs_out_is_reported_and_over():
    """one copy is left out: the call ends, the status says so once, the next call is right"""
    from nvmai_b200.moe import debug_set_wait_limit
    from nvmai_b200.row_ops import debug_drop_int8_copy
    rows, k, n = 300, 640, 130
    nv.int8_matmul_status()
    debug_set_wait_limit(2_000_000)
    try:
        for activation in (fmt.ACT_NONE, fmt.ACT_SILU):
            debug_drop_int8_copy()
            assert code_of(lambda: check_product(rows, k, n, activation)) == _lib.ETIMEOUT
            check_product(rows, k, n, activation)
    finally:
        debug_set_wait_limit(0)


def test_status_refuses_a_capture():
    stream = torch.cuda.Stream()
    x, q, s = torch.zeros(1, 64, device="cuda"), torch.zeros(64, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        nv.quantize_rows(x, 1, 64, q, s, elem=fmt.ELEM_F32, stream=stream)
        assert code_of(lambda: nv.int8_matmul_status(stream)) == _lib.EINVAL
    graph.replay()
    torch.cuda.synchronize()


FIRST_CALLS = """
import torch, nvmai_b200 as nv
from nvmai_b200 import format as fmt
t, k, e, d, n = 300, 4, 8, 128, 64
dev = dict(device="cuda")
g = torch.Generator(**dev).manual_seed(1)
idx = torch.randint(0, e, (t, k), generator=g, **dev).to(torch.int32)
x = torch.randn((t, d), generator=g, **dev)
b = torch.randint(-127, 128, (e * n, d), generator=g, dtype=torch.int8, **dev)
bs = torch.rand(e * n, generator=g, **dev)
i32 = lambda *s: torch.empty(s, dtype=torch.int32, **dev)
position, source, begin = i32(t, k), i32(t * k), i32(e + 1)
rows, out, y, dw = torch.zeros(t * k, d, **dev), torch.empty(t * k, n, **dev), torch.empty(t, n, **dev), torch.empty(t, k, **dev)
drows = torch.empty(t * k, n, **dev)
work = torch.empty(nv.int8_matmul_workspace(t * k, d, fmt.ELEM_F32), dtype=torch.uint8, **dev)
stream = torch.cuda.Stream()
def run():
    nv.sort_rows(idx, t, k, e, position, source, begin, x=x, d=d, elem=fmt.ELEM_F32, rows=rows, stream=stream)
    nv.int8_matmul(rows, b, bs, out, t * k, d, n, a_elem=fmt.ELEM_F32, num_experts=e, expert_begin=begin, out_elem=fmt.ELEM_F32,
                   workspace=work, workspace_bytes=work.numel(), stream=stream)
    nv.merge_rows(out, t * k, position, t, k, n, y, elem=fmt.ELEM_F32, stream=stream)
    nv.merge_rows_grad(y, out, t * k, position, None, t, k, n, drows, dw, elem=fmt.ELEM_F32, stream=stream)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream):
    run()
graph.replay()
torch.cuda.synchronize()
first = [v.clone() for v in (position, out, y, drows, dw)]
for v in (out, y, drows, dw):
    v.zero_()
torch.cuda.synchronize()
run()
nv.int8_matmul_status(stream)
assert all(torch.equal(a, b) for a, b in zip(first, (position, out, y, drows, dw)))
print("the same")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("pinned", [False, True])
def test_buffers_of_the_host_are_refused(pinned):
    host, dev = torch.zeros(64, dtype=torch.float32, pin_memory=pinned), torch.zeros(64, device="cuda")
    q = torch.zeros(64, dtype=torch.int8, device="cuda")
    for call in (lambda: nv.quantize_rows(host, 1, 64, q, dev, elem=fmt.ELEM_F32),
                 lambda: nv.merge_rows(dev, 1, host, 1, 1, 64, dev, elem=fmt.ELEM_F32),
                 lambda: nv.merge_rows_grad(host, dev, 1, dev, None, 1, 1, 64, dev, dev, elem=fmt.ELEM_F32),
                 lambda: nv.sort_rows(host, 1, 1, 4, q, dev, dev),
                 lambda: nv.int8_matmul(q, q, host, dev, 1, 64, 1, a_scales=dev, out_elem=fmt.ELEM_F32)):
        assert code_of(call) == _lib.EINVAL
    torch.cuda.synchronize()

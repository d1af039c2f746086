"""Arguments that the row operators refuse, before they touch a device (no GPU needed)."""
import pytest

from nvmai_b200 import _lib, build
from nvmai_b200 import format as fmt

A = 0x10000          # an address that a refused call never uses


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


SORT = dict(idx=A, tokens=4, top_k=2, num_experts=8, position=A, source=A, expert_begin=A, x=A, x_elem=fmt.ELEM_F16,
            x_stride=64, d=64, rows=A, rows_elem=fmt.ELEM_F16, rows_stride=64, row_scales=None, workspace=None,
            workspace_bytes=0, stream=None)
MERGE = dict(rows=A, elem=fmt.ELEM_F16, rows_stride=64, n_rows=8, position=A, w=A, w_elem=fmt.ELEM_F16, tokens=4, top_k=2,
             d=64, base=A, base_stride=64, y=A, y_stride=64, stream=None)
GRAD = dict(dy=A, elem=fmt.ELEM_F16, dy_stride=64, rows=A, rows_stride=64, n_rows=8, position=A, w=A, w_elem=fmt.ELEM_F16,
            tokens=4, top_k=2, d=64, drows=A, drows_stride=64, dw=A, stream=None)
QUANT = dict(x=A, elem=fmt.ELEM_F16, x_stride=64, rows=4, n=64, q=A, q_stride=64, scales=A, stream=None)
MATMUL = dict(a=A, a_elem=fmt.ELEM_I8, a_stride=64, a_scales=A, rows=4, k=64, b=A, b_stride=64, b_scales=A, n=8,
              num_experts=2, expert_begin=A, activation=fmt.ACT_NONE, out=A, out_elem=fmt.ELEM_F16, out_stride=8,
              workspace=None, workspace_bytes=0, stream=None)
E, R = _lib.EINVAL, _lib.ERANGE


@pytest.mark.parametrize("name,good,change,code", [
    ("sort_rows", SORT, dict(idx=None), E),
    ("sort_rows", SORT, dict(position=None), E),
    ("sort_rows", SORT, dict(source=None), E),
    ("sort_rows", SORT, dict(expert_begin=None), E),
    ("sort_rows", SORT, dict(top_k=0), R),
    ("sort_rows", SORT, dict(top_k=65), R),
    ("sort_rows", SORT, dict(num_experts=0), R),
    ("sort_rows", SORT, dict(num_experts=1025), R),
    ("sort_rows", SORT, dict(tokens=1 << 30), R),
    ("sort_rows", SORT, dict(tokens=1 << 25), R),
    ("sort_rows", SORT, dict(tokens=1 << 24), R),                             # without its workspace
    ("sort_rows", SORT, dict(tokens=1 << 24, workspace_bytes=1 << 40), E),
    ("sort_rows", SORT, dict(tokens=1 << 24, workspace=A + 8, workspace_bytes=1 << 40), E),
    ("sort_rows", SORT, dict(x=None), E),
    ("sort_rows", SORT, dict(rows=None), E),
    ("sort_rows", SORT, dict(d=0), E),
    ("sort_rows", SORT, dict(x_stride=63), E),
    ("sort_rows", SORT, dict(rows_stride=63), E),
    ("sort_rows", SORT, dict(x=A + 1), E),
    ("sort_rows", SORT, dict(rows=A + 1), E),
    ("sort_rows", SORT, dict(idx=A + 2), E),
    ("sort_rows", SORT, dict(x_elem=fmt.ELEM_I8), E),
    ("sort_rows", SORT, dict(rows_elem=fmt.ELEM_F32), E),
    ("sort_rows", SORT, dict(rows_elem=fmt.ELEM_I8), E),                      # codes without their scales
    ("sort_rows", SORT, dict(row_scales=A), E),                               # scales without codes
    ("sort_rows", SORT, dict(d=(1 << 30) + 8, x_stride=1 << 31, rows_stride=1 << 31), R),
    ("merge_rows", MERGE, dict(d=(1 << 30) + 8, rows_stride=1 << 31, base_stride=1 << 31, y_stride=1 << 31), R),
    ("merge_rows_grad", GRAD, dict(d=(1 << 30) + 8, dy_stride=1 << 31, rows_stride=1 << 31, drows_stride=1 << 31), R),
    ("quantize_rows", QUANT, dict(n=(1 << 30) + 8, x_stride=1 << 31, q_stride=1 << 31), R),
    ("merge_rows", MERGE, dict(rows=None), E),
    ("merge_rows", MERGE, dict(position=None), E),
    ("merge_rows", MERGE, dict(y=None), E),
    ("merge_rows", MERGE, dict(elem=fmt.ELEM_I8), E),
    ("merge_rows", MERGE, dict(w_elem=fmt.ELEM_I8), E),
    ("merge_rows", MERGE, dict(top_k=0), R),
    ("merge_rows", MERGE, dict(top_k=65), R),
    ("merge_rows", MERGE, dict(d=0), E),
    ("merge_rows", MERGE, dict(rows_stride=63), E),
    ("merge_rows", MERGE, dict(base_stride=63), E),
    ("merge_rows", MERGE, dict(y_stride=63), E),
    ("merge_rows", MERGE, dict(y=A + 1), E),
    ("merge_rows", MERGE, dict(w=A + 1), E),
    ("merge_rows", MERGE, dict(position=A + 2), E),
    ("merge_rows_grad", GRAD, dict(dy=None), E),
    ("merge_rows_grad", GRAD, dict(drows=None, dw=None), E),
    ("merge_rows_grad", GRAD, dict(rows=None), E),
    ("merge_rows_grad", GRAD, dict(position=None), E),
    ("merge_rows_grad", GRAD, dict(elem=fmt.ELEM_I8), E),
    ("merge_rows_grad", GRAD, dict(top_k=65), R),
    ("merge_rows_grad", GRAD, dict(d=0), E),
    ("merge_rows_grad", GRAD, dict(dy_stride=63), E),
    ("merge_rows_grad", GRAD, dict(drows_stride=63), E),
    ("merge_rows_grad", GRAD, dict(dw=A + 2), E),
    ("quantize_rows", QUANT, dict(x=None), E),
    ("quantize_rows", QUANT, dict(q=None), E),
    ("quantize_rows", QUANT, dict(scales=None), E),
    ("quantize_rows", QUANT, dict(elem=fmt.ELEM_I8), E),
    ("quantize_rows", QUANT, dict(n=0), E),
    ("quantize_rows", QUANT, dict(x_stride=63), E),
    ("quantize_rows", QUANT, dict(q_stride=63), E),
    ("quantize_rows", QUANT, dict(x=A + 1), E),
    ("int8_matmul", MATMUL, dict(a=None), E),
    ("int8_matmul", MATMUL, dict(b=None), E),
    ("int8_matmul", MATMUL, dict(b_scales=None), E),
    ("int8_matmul", MATMUL, dict(out=None), E),
    ("int8_matmul", MATMUL, dict(a_scales=None), E),                          # codes without their scales
    ("int8_matmul", MATMUL, dict(a_elem=fmt.ELEM_F16), E),                    # elements with scales
    ("int8_matmul", MATMUL, dict(a_elem=4), E),
    ("int8_matmul", MATMUL, dict(out_elem=fmt.ELEM_I8), E),
    ("int8_matmul", MATMUL, dict(activation=3), E),
    ("int8_matmul", MATMUL, dict(k=0), E),
    ("int8_matmul", MATMUL, dict(n=0), E),
    ("int8_matmul", MATMUL, dict(a_stride=48), E),
    ("int8_matmul", MATMUL, dict(b_stride=48), E),
    ("int8_matmul", MATMUL, dict(out_stride=7), E),
    ("int8_matmul", MATMUL, dict(a=A + 8), E),
    ("int8_matmul", MATMUL, dict(b=A + 8), E),
    ("int8_matmul", MATMUL, dict(a_stride=72), E),
    ("int8_matmul", MATMUL, dict(b_stride=72), E),
    ("int8_matmul", MATMUL, dict(num_experts=0), E),
    ("int8_matmul", MATMUL, dict(expert_begin=None), E),                      # several matrices, rows of nobody
    ("int8_matmul", MATMUL, dict(num_experts=1025), R),
    ("int8_matmul", MATMUL, dict(k=131072, a_stride=131072, b_stride=131072), R),
    ("int8_matmul", MATMUL, dict(n=1 << 30, out_stride=1 << 30), R),
    ("int8_matmul", MATMUL, dict(a_elem=fmt.ELEM_F16, a_scales=None), R),     # no workspace
    ("int8_matmul", MATMUL, dict(a_elem=fmt.ELEM_F16, a_scales=None, workspace_bytes=1 << 20), E),
    ("int8_matmul", MATMUL, dict(a_elem=fmt.ELEM_F16, a_scales=None, workspace=A + 8, workspace_bytes=1 << 20), E),
])
def test_refused_before_the_device_is_touched(lib, name, good, change, code):
    args = {**good, **change}
    assert getattr(lib, "nvmai_cuda_moe_" + name)(*args.values()) == code


@pytest.mark.parametrize("name,good,change", [
    ("merge_rows", MERGE, dict(tokens=0)),
    ("merge_rows_grad", GRAD, dict(tokens=0)),
    ("quantize_rows", QUANT, dict(rows=0)),
    ("int8_matmul", MATMUL, dict(rows=0)),
    ("int8_matmul", MATMUL, dict(rows=0, a=None, a_scales=None, out=None)),
])
def test_nothing_to_do_is_no_error(lib, name, good, change):
    assert getattr(lib, "nvmai_cuda_moe_" + name)(*{**good, **change}.values()) == _lib.OK


def test_workspaces_hold_counts_codes_and_scales():
    from nvmai_b200 import int8_matmul_workspace, sort_rows_workspace
    assert sort_rows_workspace(4096, 8, 256) == 0
    assert sort_rows_workspace(16384, 8, 256) == 148 * 256 * 4
    assert sort_rows_workspace(1 << 20, 8, 1024) == 2048 * 1024 * 4          # a block's pairs stay 4096
    assert int8_matmul_workspace(77, 100, fmt.ELEM_I8) == 0
    for elem in (fmt.ELEM_F16, fmt.ELEM_F32, fmt.ELEM_BF16):
        assert int8_matmul_workspace(77, 100, elem) >= 77 * 112 + 77 * 4
    assert int8_matmul_workspace(1 << 20, 1 << 16, fmt.ELEM_F16) > 1 << 36          # past 32 bits

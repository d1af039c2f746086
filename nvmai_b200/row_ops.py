"""Row operators: token rows sorted by expert and back, with gradients, and products in 8-bit integers.

Thin ctypes wrappers over the handle-free entry points of `include/nvmai_cuda_moe.h` (sort_rows .. int8_matmul),
which have no counterpart in the reference.  Buffers are as in `moe.py`; element types are `format.ELEM_*`, strides count
elements and default to dense rows.  The calls enqueue on `stream` and return; errors surface as `NvmaiError`.
"""
from __future__ import annotations

from . import _lib
from . import format as fmt
from ._lib import check
from .moe import _ptr, _stream


def sort_rows_workspace(tokens: int, top_k: int, num_experts: int) -> int:
    """Bytes of workspace that `sort_rows` needs."""
    return int(_lib.lib().nvmai_cuda_moe_sort_rows_workspace(tokens, top_k, num_experts))


def sort_rows(idx, tokens: int, top_k: int, num_experts: int, position, source, expert_begin, *, x=None, d: int = 0,
              elem: int = fmt.ELEM_F16, rows=None, rows_elem: int | None = None, row_scales=None, x_stride: int | None = None,
              rows_stride: int | None = None, workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """Pairs (token, slot) sorted by expert, and with `x` the token rows in that order (rows_elem ELEM_I8: as codes
    with `row_scales`).  The gradient of x is `merge_rows` of the rows' gradient without weights."""
    check(_lib.lib().nvmai_cuda_moe_sort_rows(_ptr(idx), tokens, top_k, num_experts, _ptr(position), _ptr(source),
                                              _ptr(expert_begin), _ptr(x), elem, d if x_stride is None else x_stride, d,
                                              _ptr(rows), elem if rows_elem is None else rows_elem,
                                              d if rows_stride is None else rows_stride, _ptr(row_scales),
                                              _ptr(workspace), workspace_bytes, _stream(stream)), "sort_rows")


def merge_rows(rows, n_rows: int, position, tokens: int, top_k: int, d: int, y, *, elem: int = fmt.ELEM_F16, w=None,
               w_elem: int = fmt.ELEM_F16, base=None, rows_stride: int | None = None, base_stride: int | None = None,
               y_stride: int | None = None, stream=None) -> None:
    """y[t] = base[t] + sum_k w[t][k] * rows[position[t][k]]; without `w` the gradient of `sort_rows`."""
    check(_lib.lib().nvmai_cuda_moe_merge_rows(_ptr(rows), elem, d if rows_stride is None else rows_stride, n_rows,
                                               _ptr(position), _ptr(w), w_elem, tokens, top_k, d, _ptr(base),
                                               d if base_stride is None else base_stride, _ptr(y),
                                               d if y_stride is None else y_stride, _stream(stream)), "merge_rows")


def merge_rows_grad(dy, rows, n_rows: int, position, w, tokens: int, top_k: int, d: int, drows, dw, *,
                    elem: int = fmt.ELEM_F16, w_elem: int = fmt.ELEM_F16, dy_stride: int | None = None,
                    rows_stride: int | None = None, drows_stride: int | None = None, stream=None) -> None:
    """Gradients of `merge_rows`: drows (type `elem`) and dw (fp32 [tokens][top_k]); either may be None."""
    check(_lib.lib().nvmai_cuda_moe_merge_rows_grad(_ptr(dy), elem, d if dy_stride is None else dy_stride, _ptr(rows),
                                                    d if rows_stride is None else rows_stride, n_rows, _ptr(position),
                                                    _ptr(w), w_elem, tokens, top_k, d, _ptr(drows),
                                                    d if drows_stride is None else drows_stride, _ptr(dw),
                                                    _stream(stream)), "merge_rows_grad")


def quantize_rows(x, rows: int, n: int, q, scales, *, elem: int = fmt.ELEM_F16, x_stride: int | None = None,
                  q_stride: int | None = None, stream=None) -> None:
    """8-bit codes and fp32 scales of rows: m = max |x|, scale m / 127, code rint(x * (127 / m))."""
    check(_lib.lib().nvmai_cuda_moe_quantize_rows(_ptr(x), elem, n if x_stride is None else x_stride, rows, n, _ptr(q),
                                                  n if q_stride is None else q_stride, _ptr(scales), _stream(stream)),
          "quantize_rows")


def int8_matmul_workspace(rows: int, k: int, a_elem: int) -> int:
    """Bytes of workspace that `int8_matmul` needs (0 for codes)."""
    return int(_lib.lib().nvmai_cuda_moe_int8_matmul_workspace(rows, k, a_elem))


def int8_matmul(a, b, b_scales, out, rows: int, k: int, n: int, *, a_elem: int = fmt.ELEM_I8, a_scales=None,
                num_experts: int = 1, expert_begin=None, activation: int = fmt.ACT_NONE, out_elem: int = fmt.ELEM_F16,
                a_stride: int | None = None, b_stride: int | None = None, out_stride: int | None = None, workspace=None,
                workspace_bytes: int = 0, stream=None) -> None:
    """Rows times 8-bit matrices [num_experts][n, or 2n with an activation][k] with a scale per channel; each row takes
    the matrix of its expert (`expert_begin` as `sort_rows` writes it).  a_elem other than ELEM_I8: the call quantises."""
    check(_lib.lib().nvmai_cuda_moe_int8_matmul(_ptr(a), a_elem, k if a_stride is None else a_stride, _ptr(a_scales), rows,
                                                k, _ptr(b), k if b_stride is None else b_stride, _ptr(b_scales), n,
                                                num_experts, _ptr(expert_begin), activation, _ptr(out), out_elem,
                                                n if out_stride is None else out_stride, _ptr(workspace),
                                                workspace_bytes, _stream(stream)), "int8_matmul")


def int8_matmul_status(stream=None) -> None:
    """Waits for `stream`; raises NvmaiError(ETIMEOUT) if an `int8_matmul` call on the device, on this stream or another, gave up
    a device-side wait that this stream has not been told of."""
    check(_lib.lib().nvmai_cuda_moe_int8_matmul_status(_stream(stream)), "int8_matmul_status")


def debug_drop_int8_copy() -> None:
    """Test hook: the next large `int8_matmul` leaves out one copy, so that its bounded waits run out."""
    check(_lib.lib().nvmai_cuda_moe_debug_drop_int8_copy(), "debug_drop_int8_copy")

"""Calls of the row operators with nothing to write are no error: buffers of no rows have no address (no GPU needed)."""
import pytest

from nvmai_b200 import _lib, build
from test_row_ops import GRAD


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("change", [
    dict(tokens=0, dy=None, position=None, drows=None, dw=None),             # dw of no tokens, drows not asked for
    dict(tokens=0, dy=None, position=None, dw=None),                         # drows of other tokens' rows, dw of none
    dict(n_rows=0, rows=None, drows=None, dw=None),                          # a rank that holds none of the experts: drows of no rows
    dict(n_rows=0, dw=None),
])
def test_gradients_of_nothing(lib, change):
    assert lib.nvmai_cuda_moe_merge_rows_grad(*{**GRAD, **change}.values()) == _lib.OK


@pytest.mark.parametrize("change", [dict(drows=None, dw=None), dict(n_rows=0, drows=None, dw=None, dy=None), dict(tokens=0, drows=None, dw=None, d=0)])
def test_what_is_wrong_stays_refused(lib, change):
    assert lib.nvmai_cuda_moe_merge_rows_grad(*{**GRAD, **change}.values()) == _lib.EINVAL

"""Results that lie over a layer's operand, without a GPU: refused before any
device work."""
import ctypes as C

import pytest


def _layer(**more):
    from proxima_amd import _capi
    plain = dict(type=2, out_type=2, bias_type=0, activation=-1, rows=4, k=8, groups=1, n=8, x=1 << 20, x_stride=8, w=4096,
                 w_stride=8, w_group_stride=64, y=1 << 21, y_stride=8)
    lib = _capi.lib
    return lib.pxg_grouped_linear_device(C.byref(_capi.LinearC(**{**plain, **more})), None), lib.pxg_last_error_parameter()


X = 1 << 20


@pytest.mark.parametrize("more", [
    dict(y=X), dict(y=X, residual=X, residual_stride=8), dict(y=X + 62), dict(y=X - 62),      # rows of 16 bytes, 64 in all
    dict(rows=1, y=X, x_stride=0, y_stride=0), dict(rows=1, y=X + 14), dict(rows=1, y=X - 14),
    dict(x_stride=24, y_stride=24, y=X + 14), dict(x_stride=24, y_stride=24, y=X + 48 * 2 + 34),  # into the next row
    dict(x_stride=24, y_stride=20, y=X + 16), dict(out_type=0, y=X - 124), dict(out_type=0, y=X + 60),
    dict(x_stride=24, y_stride=12, out_type=0, y=X + 20),
])
def test_a_result_over_x_is_refused(more):
    assert _layer(**more) == (7, b"y")


@pytest.mark.parametrize("more", [dict(h=X, h_stride=8), dict(h=X + 62, h_stride=8)])
def test_kept_rows_over_x_are_refused(more):
    assert _layer(**more) == (7, b"h")

"""Expert layers and packed rows without a GPU: what is refused before any
device work, and the sizes that the C ABI tells a caller."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from proxima_amd import _capi
    return _capi.lib


def _refused(lib, status, parameter):
    assert status == 7
    assert lib.pxg_last_error_parameter() == parameter


def test_packed_sizes(lib):
    for cols, wide, few in ((1, 128, 4), (128, 128, 4), (129, 256, 4), (512, 512, 4), (513, 640, 8), (4096, 4096, 32)):
        assert lib.pxg_block8_code_stride(cols) == wide
        assert lib.pxg_block8_scale_stride(cols) == few


def test_packing_refuses(lib):
    p = C.c_void_p(4096)
    _refused(lib, lib.pxg_block8_pack_device(3, p, 4, 8, 8, p, p, None), b"type")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 4, 0, 8, p, p, None), b"cols")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 4, 8, 7, p, p, None), b"stride")
    _refused(lib, lib.pxg_block8_pack_device(0, None, 4, 8, 8, p, p, None), b"x")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 4, 8, 8, None, p, None), b"codes")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 4, 8, 8, C.c_void_p(4104), p, None), b"codes")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 4, 8, 8, p, C.c_void_p(4098), None), b"scales")
    _refused(lib, lib.pxg_block8_pack_device(0, C.c_void_p(4097), 4, 8, 8, p, p, None), b"x")
    _refused(lib, lib.pxg_block8_pack_device(0, p, 1 << 31, 8, 8, p, p, None), b"rows")
    _refused(lib, lib.pxg_activation_pack_device(2, 0, p, 4, 8, 8, p, 8, p, p, None), b"activation")
    _refused(lib, lib.pxg_activation_grad_device(0, 0, p, 4, 8, 8, p, p, None, 8, None), b"out")
    # no rows: nothing is looked at and nothing is launched
    assert lib.pxg_block8_pack_device(0, None, 0, 8, 8, None, None, None) == 0
    assert lib.pxg_last_error_parameter() == b""


def test_products_refuse(lib):
    p = C.c_void_p(4096)
    f = lib.pxg_grouped_matmul_device
    _refused(lib, f(0, p, 4, 8, 8, p, 1, 8, 8, 64, None, 0, p, 8, None), b"type")
    _refused(lib, f(2, p, 4, 8, 8, p, 1, 8, 8, 64, None, 1, p, 8, None), b"out_type")
    _refused(lib, f(2, p, 4, 0, 8, p, 1, 8, 8, 64, None, 2, p, 8, None), b"k")
    _refused(lib, f(2, p, 4, 8, 8, p, 1, 0, 8, 64, None, 2, p, 8, None), b"n")
    _refused(lib, f(2, p, 4, 8, 8, p, 0, 8, 8, 64, None, 2, p, 8, None), b"groups")
    _refused(lib, f(2, p, 4, 8, 8, p, 2, 8, 8, 64, None, 2, p, 8, None), b"groups")  # without offsets
    _refused(lib, f(2, p, 4, 8, 8, p, 1, 8, 8, 64, C.c_void_p(4100), 2, p, 8, None), b"offsets")
    _refused(lib, f(2, p, 4, 8, 4, p, 1, 8, 8, 64, None, 2, p, 8, None), b"stride")
    _refused(lib, f(2, p, 4, 8, 1 << 23, p, 1, 8, 8, 64, None, 2, p, 8, None), b"stride")
    _refused(lib, f(2, p, 4, 8, 8, None, 1, 8, 8, 64, None, 2, p, 8, None), b"w")
    _refused(lib, f(2, p, 4, 8, 8, p, 1, 8, 8, 64, None, 2, None, 8, None), b"y")
    w = lib.pxg_grouped_matmul_grad_weight_device
    _refused(lib, w(2, p, 4, 8, 8, p, 8, 8, None, 1, 2, p, 8, 64, None, 0, None), b"offsets")
    _refused(lib, w(2, p, 4, 8, 8, p, 8, 8, p, 1, 2, p, 8, 64, C.c_void_p(4104), 0, None), b"workspace")
    b = lib.pxg_block8_matmul_device
    _refused(lib, b(p, p, 4, 8, p, p, 1, 8, None, 5, p, 8, None), b"type")
    _refused(lib, b(p, None, 4, 8, p, p, 1, 8, None, 2, p, 8, None), b"scales")
    _refused(lib, b(p, p, 4, 8, C.c_void_p(4100), p, 1, 8, None, 2, p, 8, None), b"w_codes")
    assert f(2, None, 0, 8, 8, p, 1, 8, 8, 64, None, 2, None, 8, None) == 0


def test_workspace_is_for_long_sums_into_small_matrices(lib):
    size = lib.pxg_grouped_matmul_grad_weight_workspace
    assert size(100_000, 128, 128, 1) > 0
    assert size(100_000, 128, 128, 1) % (4 * 128 * 128) == 0
    assert size(64, 128, 128, 1) == 0          # a short sum
    assert size(16_384, 2048, 2048, 64) == 0   # enough tiles as they are
    assert size(0, 128, 128, 1) == 0
    assert size(100, 0, 128, 1) == 0


def test_python_side_refuses_host_tensors():
    import torch

    import proxima_amd as px
    x, w = torch.zeros(4, 8), torch.zeros(1, 8, 8)
    offsets = torch.tensor([0, 4])
    for call in (lambda: px.block8_pack(x), lambda: px.grouped_matmul(x, w, offsets),
                 lambda: px.grouped_matmul_grad_input(x, w, offsets),
                 lambda: px.grouped_matmul_grad_weight(x, x, offsets), lambda: px.activation_pack(x, "gelu"),
                 lambda: px.block8_matmul(x, x), lambda: px.block8_unpack(x),
                 lambda: px.Block8(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 8),
                 lambda: px.activation_pack(x, "tanh")):
        with pytest.raises(ValueError):
            call()


def test_matrices_of_a_result_may_not_overlap(lib):
    p = C.c_void_p(4096)

    def plain(groups, n, k, stride, group_stride):
        return lib.pxg_grouped_matmul_grad_weight_device(2, p, 4, n, n, p, k, k, p, groups, 2, p, stride, group_stride,
                                                         None, 0, None)

    def packed(groups, n, k, stride, group_stride):
        return lib.pxg_grouped_matmul_grad_weight_block8_device(p, 4, n, n, p, p, k, p, groups, 2, p, stride,
                                                                group_stride, None, 0, None)

    for call in (plain, packed):
        # one matrix for all groups; a row, an element too near; rows of one group among another's; past 64 bits
        for groups, n, k, stride, apart in ((2, 8, 8, 8, 0), (2, 8, 8, 8, 56), (3, 8, 8, 8, 63), (3, 8, 8, 23, 8),
                                            (2, 8, 8, 16, 4), (2, 1, 8, 8, 7), (2, 8, 8, (1 << 63) + 8, 7)):
            _refused(lib, call(groups, n, k, stride, apart), b"dw_group_stride")


def test_kernels_that_are_not_there_are_refused(lib):
    for rows in (-1, 1, 32, 512):
        _refused(lib, lib.pxg_grouped_matmul_set_kernel(rows), b"rows")
    for rows in (16, 64, 128, 256, 0):
        assert lib.pxg_grouped_matmul_set_kernel(rows) == 0

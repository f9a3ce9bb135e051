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


def test_layers_refuse(lib):
    p, odd = C.c_void_p(4096), C.c_void_p(4097)

    def f(kind=2, x=p, rows=4, k=8, xs=8, w=p, groups=1, n=8, ws=8, offsets=None, bias_type=0, bias=p, bs=8, act=1,
          out=2, r=p, rs=8, h=p, hs=8, y=p, ys=8):
        return lib.pxg_grouped_linear_device(kind, x, rows, k, xs, w, groups, n, ws, 64, offsets, bias_type, bias, bs, act,
                                             out, r, rs, h, hs, y, ys, None)

    for more, parameter in (
            (dict(kind=0), b"type"), (dict(out=1), b"out_type"), (dict(k=0), b"k"), (dict(n=0), b"n"),
            (dict(groups=0), b"groups"), (dict(groups=2), b"groups"), (dict(xs=7), b"stride"),
            (dict(xs=1 << 23), b"stride"), (dict(w=None), b"w"), (dict(y=None), b"y"), (dict(x=odd), b"x"),
            (dict(bias_type=1), b"bias_type"), (dict(bias=C.c_void_p(4098)), b"bias"),
            (dict(groups=2, offsets=p, bs=7), b"stride"), (dict(act=2), b"activation"), (dict(act=-2), b"activation"),
            (dict(rs=7), b"stride"), (dict(r=odd), b"residual"), (dict(hs=7), b"stride"), (dict(h=odd), b"h"),
            (dict(ys=7), b"stride"), (dict(rows=1 << 31), b"rows")):
        _refused(lib, f(**more), parameter)
    assert f(rows=0, x=None, y=None, r=None, h=None) == 0

    def b(codes=p, scales=p, rows=4, k=8, wc=p, ws=p, groups=1, n=8, offsets=None, bias_type=0, bias=p, bs=8, act=1,
          out=2, r=p, rs=8, y=p, ys=8):
        return lib.pxg_block8_linear_device(codes, scales, rows, k, wc, ws, groups, n, offsets, bias_type, bias, bs, act,
                                            out, r, rs, y, ys, None)

    for more, parameter in (
            (dict(out=3), b"type"), (dict(scales=None), b"scales"), (dict(wc=C.c_void_p(4104)), b"w_codes"),
            (dict(bias_type=1), b"bias_type"), (dict(act=5), b"activation"), (dict(rs=4), b"stride"),
            (dict(groups=3), b"groups"), (dict(y=odd), b"y"), (dict(k=0), b"k")):
        _refused(lib, b(**more), parameter)
    assert b(rows=0, codes=None, scales=None, y=None, r=None) == 0


def test_layers_backward_pass_refuses(lib):
    p, odd = C.c_void_p(4096), C.c_void_p(4097)

    def f(act=1, kind=2, grad=p, rows=4, n=8, gs=8, h=p, hs=8, offsets=None, groups=1, dh=p, ds=8, bias_type=0, db=p,
          dbs=8, space=None, size=0):
        return lib.pxg_grouped_linear_grad_device(act, kind, grad, rows, n, gs, h, hs, offsets, groups, dh, ds, bias_type,
                                                  db, dbs, space, size, None)

    for more, parameter in (
            (dict(kind=3), b"type"), (dict(act=2), b"activation"), (dict(n=0), b"n"), (dict(groups=4), b"groups"),
            (dict(offsets=C.c_void_p(4100)), b"offsets"), (dict(grad=None), b"grad"), (dict(gs=7), b"stride"),
            (dict(h=None), b"h"), (dict(hs=7), b"stride"), (dict(dh=None), b"dh"), (dict(dh=odd), b"dh"),
            (dict(bias_type=1), b"bias_type"), (dict(db=C.c_void_p(4098)), b"dbias"),
            (dict(offsets=p, groups=2, dbs=7), b"stride"), (dict(space=C.c_void_p(4104)), b"workspace"),
            (dict(rows=1 << 31), b"rows")):
        _refused(lib, f(**more), parameter)
    assert f(act=-1, h=None, dh=None, db=None) == 0  # nothing to do
    size = lib.pxg_grouped_linear_grad_workspace
    assert size(100_000, 1024, 8) > 0 and size(100_000, 1024, 8) % (4 * 1024) == 0
    assert size(8, 1024, 8) == 0 and size(0, 8, 1) == 0 and size(8, 0, 1) == 0 and size(8, 8, 0) == 0


def test_whole_layers_refuse(lib):
    from proxima_amd._capi import ExpertMatrixC
    p, odd = C.c_void_p(4096), C.c_void_p(4097)
    m = ExpertMatrixC(4096, 8, 64, 4096)

    def f(kind=2, x=p, rows=4, k=8, xs=8, ids=p, picks=2, is_=2, gates=p, gs=2, experts=3, hidden=8, n=8, w1=m, up=None,
          w2=m, packed=0, act=1, bias_type=0, b1=p, b1s=8, b2=p, b2s=8, out=2, r=p, rs=8, y=p, ys=8, space=p,
          size=1 << 30):
        return lib.pxg_expert_layer_device(kind, x, rows, k, xs, ids, picks, is_, gates, gs, experts, hidden, n, w1, up, w2,
                                           packed, act, bias_type, b1, b1s, b2, b2s, out, r, rs, y, ys, space, size, None)

    for more, parameter in (
            (dict(kind=0), b"type"), (dict(kind=1, packed=1, out=1), b"type"), (dict(out=1), b"out_type"),
            (dict(rows=65537), b"rows"), (dict(picks=0), b"picks"), (dict(picks=17, is_=17, gs=17), b"picks"),
            (dict(experts=0), b"experts"), (dict(experts=65537), b"experts"), (dict(k=0), b"k"),
            (dict(k=(1 << 22) + 1), b"k"), (dict(hidden=0), b"hidden"), (dict(n=0), b"n"), (dict(act=2), b"activation"),
            (dict(x=None), b"x"), (dict(xs=7), b"stride"), (dict(gates=None), b"gates"), (dict(gs=1), b"stride"),
            (dict(ids=None), b"experts"), (dict(ids=C.c_void_p(4100)), b"experts"), (dict(w1=None), b"w1"),
            (dict(w1=ExpertMatrixC(None, 8, 64, None)), b"w1"), (dict(w2=ExpertMatrixC(4097, 8, 64, None)), b"w2"),
            (dict(up=ExpertMatrixC(4096, 7, 64, None)), b"stride"),
            (dict(w2=ExpertMatrixC(4096, 8, 64, None), packed=1), b"w2"),
            (dict(w1=ExpertMatrixC(4104, 8, 64, 4096), packed=1), b"w1"), (dict(bias_type=1), b"bias_type"),
            (dict(b1=C.c_void_p(4098)), b"bias1"), (dict(b2s=7), b"stride"), (dict(r=odd), b"residual"),
            (dict(rs=7), b"stride"), (dict(y=None), b"y"), (dict(space=None), b"workspace_bytes"),
            (dict(size=64), b"workspace_bytes"), (dict(space=C.c_void_p(4104)), b"workspace")):
        _refused(lib, f(**more), parameter)
    assert f(rows=0, x=None, ids=None, gates=None, r=None, y=None, space=None, size=0) == 0
    size = lib.pxg_expert_layer_workspace
    assert size(8, 2, 16, 512, 512, 0) > size(8, 2, 16, 512, 512, 2) > 8 * 2 * 512 * 2 * 2
    assert size(0, 2, 16, 512, 512, 0) == 0 and size(8, 17, 16, 512, 512, 0) == 0 and size(8, 2, 0, 512, 512, 0) == 0


def test_distillation_refuses(lib):
    p, odd = C.c_void_p(4096), C.c_void_p(4097)

    def f(kind=0, weight=p, x=p, rows=4, cols=8, xs=8, ids=p, is_=2, scores=p, ss=2, counts=p, top=2, t=1.0, loss=p, dx=p,
          ds=8, space=None, size=0):
        return lib.pxg_distill_loss_grad_device(kind, weight, x, rows, cols, xs, ids, is_, scores, ss, counts, top, t, loss,
                                                dx, ds, space, size, None)

    for more, parameter in (
            (dict(kind=3), b"type"), (dict(cols=0), b"cols"), (dict(top=0), b"top"), (dict(top=4097), b"top"),
            (dict(t=0.0), b"temperature"), (dict(t=float("nan")), b"temperature"), (dict(t=1e7), b"temperature"),
            (dict(x=None), b"logits"), (dict(xs=7), b"stride"), (dict(x=odd), b"logits"), (dict(ids=None), b"ids"),
            (dict(ids=C.c_void_p(4100)), b"ids"), (dict(is_=1), b"stride"), (dict(scores=None), b"scores"),
            (dict(counts=None), b"counts"), (dict(loss=None), b"loss"), (dict(weight=None), b"weight"),
            (dict(dx=None), b"dx"), (dict(ds=7), b"stride"), (dict(rows=1 << 31), b"rows"),
            (dict(cols=1 << 20, xs=1 << 20, ds=1 << 20), b"workspace_bytes"),
            (dict(space=C.c_void_p(4104)), b"workspace")):
        _refused(lib, f(**more), parameter)
    assert f(rows=0, weight=None, x=None, ids=None, scores=None, counts=None, loss=None, dx=None) == 0
    assert lib.pxg_distill_loss_device(0, None, 0, 8, 8, None, 2, None, 2, None, 2, 1.0, None, None, 0, None) == 0
    _refused(lib, lib.pxg_distill_loss_device(0, None, 4, 8, 8, p, 2, p, 2, p, 2, 1.0, p, None, 0, None), b"logits")
    size = lib.pxg_distill_workspace
    assert size(0, 4, 1 << 20, 2) > 0 and size(0, 4, 8, 2) == 0 and size(0, 0, 8, 2) == 0 and size(0, 4, 8, 0) == 0


def test_python_side_of_layers_and_losses_refuses_host_tensors():
    import torch

    import proxima_amd as px
    x, w = torch.zeros(4, 8), torch.zeros(2, 8, 8)
    ids, scores, counts = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: px.grouped_linear(x, w), lambda: px.block8_linear(x, x), lambda: px.grouped_linear_grad(x),
                 lambda: px.expert_layer(x, ids, w, w, scores), lambda: px.distill_loss(x, ids, scores, counts),
                 lambda: px.distill_loss_grad(counts, x, ids, scores, counts)):
        with pytest.raises(ValueError):
            call()

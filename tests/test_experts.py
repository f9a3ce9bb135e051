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


def _with(kind, defaults, more):
    """A C struct of these fields; pointers are numbers."""
    s = kind(**{**defaults, **more})
    return C.byref(s)


def test_layers_refuse(lib):
    from proxima_amd._capi import LinearC
    plain = dict(type=2, out_type=2, bias_type=0, activation=1, rows=4, k=8, groups=1, n=8, x=4096, x_stride=8, w=4096,
                 w_stride=8, w_group_stride=64, bias=4096, bias_stride=8, residual=4096, residual_stride=8, h=4096,
                 h_stride=8, y=4096, y_stride=8, x_scales=4096, w_scales=4096)
    for more, parameter in (
            (dict(type=0), b"type"), (dict(type=(1 << 32) + 2), b"type"), (dict(out_type=1), b"out_type"),
            (dict(k=0), b"k"), (dict(n=0), b"n"), (dict(groups=0), b"groups"), (dict(groups=2), b"groups"),
            (dict(x_stride=7), b"stride"), (dict(x_stride=1 << 23), b"stride"), (dict(w=None), b"w"),
            (dict(y=None), b"y"), (dict(x=4097), b"x"), (dict(bias_type=1), b"bias_type"),
            (dict(bias_type=1 << 32), b"bias_type"), (dict(bias=4098), b"bias"),
            (dict(groups=2, offsets=4096, bias_stride=7), b"stride"), (dict(activation=2), b"activation"),
            (dict(activation=-2), b"activation"), (dict(activation=1 << 32), b"activation"),
            (dict(residual_stride=7), b"stride"), (dict(residual=4097), b"residual"), (dict(h_stride=7), b"stride"),
            (dict(h=4097), b"h"), (dict(y_stride=7), b"stride"), (dict(rows=1 << 31), b"rows")):
        _refused(lib, lib.pxg_grouped_linear_device(_with(LinearC, plain, more), None), parameter)
    none = dict(rows=0, x=None, y=None, residual=None, h=None)
    assert lib.pxg_grouped_linear_device(_with(LinearC, plain, none), None) == 0
    for more, parameter in (
            (dict(out_type=3), b"type"), (dict(x_scales=None), b"x_scales"), (dict(w=4104), b"w"),
            (dict(w_scales=4098), b"w_scales"), (dict(bias_type=1), b"bias_type"), (dict(activation=5), b"activation"),
            (dict(residual_stride=4), b"stride"), (dict(groups=3), b"groups"), (dict(y=4097), b"y"), (dict(k=0), b"k")):
        _refused(lib, lib.pxg_block8_linear_device(_with(LinearC, plain, more), None), parameter)
    assert lib.pxg_block8_linear_device(_with(LinearC, plain, {**none, "x_scales": None}), None) == 0


def test_layers_backward_pass_refuses(lib):
    from proxima_amd._capi import LinearGradC
    plain = dict(type=2, bias_type=0, activation=1, rows=4, n=8, groups=1, grad=4096, grad_stride=8, h=4096, h_stride=8,
                 dh=4096, dh_stride=8, dbias=4096, dbias_stride=8)
    f = lib.pxg_grouped_linear_grad_device
    for more, parameter in (
            (dict(type=3), b"type"), (dict(activation=2), b"activation"), (dict(n=0), b"n"), (dict(groups=4), b"groups"),
            (dict(offsets=4100), b"offsets"), (dict(grad=None), b"grad"), (dict(grad_stride=7), b"stride"),
            (dict(h=None), b"h"), (dict(h_stride=7), b"stride"), (dict(dh=None), b"dh"), (dict(dh=4097), b"dh"),
            (dict(bias_type=1), b"bias_type"), (dict(dbias=4098), b"dbias"),
            (dict(offsets=4096, groups=2, dbias_stride=7), b"stride"), (dict(workspace=4104), b"workspace"),
            (dict(rows=1 << 31), b"rows")):
        _refused(lib, f(_with(LinearGradC, plain, more), None), parameter)
    assert f(_with(LinearGradC, plain, dict(activation=-1, h=None, dh=None, dbias=None)), None) == 0  # nothing to do
    size = lib.pxg_grouped_linear_grad_workspace
    assert size(100_000, 1024, 8) > 0 and size(100_000, 1024, 8) % 4 == 0
    assert size(8, 1024, 8) == 0 and size(0, 8, 1) == 0 and size(8, 0, 1) == 0 and size(8, 8, 0) == 0


def test_whole_layers_refuse(lib):
    from proxima_amd._capi import ExpertLayerC, ExpertMatrixC

    def m(data=4096, stride=8, scales=4096):
        return ExpertMatrixC(data, stride, 64, scales)

    plain = dict(type=2, out_type=2, bias_type=0, activation=1, packed=0, rows=4, k=8, picks=2, experts=3, hidden=8, n=8,
                 x=4096, x_stride=8, ids=4096, ids_stride=2, gates=4096, gates_stride=2, w1=m(), w2=m(), bias1=4096,
                 bias1_stride=8, bias2=4096, bias2_stride=8, residual=4096, residual_stride=8, y=4096, y_stride=8,
                 workspace=4096, workspace_bytes=1 << 30)
    f = lib.pxg_expert_layer_device
    for more, parameter in (
            (dict(type=0), b"type"), (dict(type=1, packed=1, out_type=1), b"type"), (dict(out_type=1), b"out_type"),
            (dict(rows=65537), b"rows"), (dict(picks=0), b"picks"), (dict(picks=17, ids_stride=17, gates_stride=17), b"picks"),
            (dict(experts=0), b"experts"), (dict(experts=65537), b"experts"), (dict(k=0), b"k"),
            (dict(k=(1 << 22) + 1), b"k"), (dict(hidden=0), b"hidden"), (dict(n=0), b"n"),
            (dict(activation=2), b"activation"), (dict(x=None), b"x"), (dict(x_stride=7), b"stride"),
            (dict(gates=None), b"gates"), (dict(gates_stride=1), b"stride"), (dict(ids=None), b"ids"),
            (dict(ids=4100), b"ids"), (dict(w1=m(None)), b"w1"), (dict(w2=m(4097)), b"w2"),
            (dict(up=m(4096, 7)), b"stride"), (dict(w2=m(scales=None), packed=1), b"w2"),
            (dict(w1=m(4104), packed=1), b"w1"), (dict(bias_type=1), b"bias_type"), (dict(bias1=4098), b"bias1"),
            (dict(bias2_stride=7), b"stride"), (dict(residual=4097), b"residual"), (dict(residual_stride=7), b"stride"),
            (dict(y=None), b"y"), (dict(workspace=None), b"workspace_bytes"),
            (dict(workspace_bytes=64), b"workspace_bytes"), (dict(workspace=4104), b"workspace")):
        _refused(lib, f(_with(ExpertLayerC, plain, more), None), parameter)
    none = dict(rows=0, x=None, ids=None, gates=None, residual=None, y=None, workspace=None, workspace_bytes=0)
    assert f(_with(ExpertLayerC, plain, none), None) == 0
    size = lib.pxg_expert_layer_workspace
    assert size(8, 2, 16, 512, 512, 0) > size(8, 2, 16, 512, 512, 2) > 8 * 2 * 512 * 2 * 2
    assert size(0, 2, 16, 512, 512, 0) == 0 and size(8, 17, 16, 512, 512, 0) == 0 and size(8, 2, 0, 512, 512, 0) == 0


def test_distillation_refuses(lib):
    from proxima_amd._capi import DistillC
    plain = dict(type=0, rows=4, cols=8, top=2, logits=4096, logits_stride=8, ids=4096, ids_stride=2, scores=4096,
                 scores_stride=2, counts=4096, temperature=1.0, loss=4096, weight=4096, dx=4096, dx_stride=8)
    f = lib.pxg_distill_loss_grad_device
    for more, parameter in (
            (dict(type=3), b"type"), (dict(cols=0), b"cols"), (dict(top=0), b"top"), (dict(top=4097), b"top"),
            (dict(temperature=0.0), b"temperature"), (dict(temperature=float("nan")), b"temperature"),
            (dict(temperature=1e7), b"temperature"), (dict(logits=None), b"logits"), (dict(logits_stride=7), b"stride"),
            (dict(logits=4097), b"logits"), (dict(ids=None), b"ids"), (dict(ids=4100), b"ids"),
            (dict(ids_stride=1), b"stride"), (dict(scores=None), b"scores"), (dict(counts=None), b"counts"),
            (dict(loss=None), b"loss"), (dict(weight=None), b"weight"), (dict(dx=None), b"dx"),
            (dict(dx_stride=7), b"stride"), (dict(rows=1 << 31), b"rows"),
            (dict(cols=1 << 20, logits_stride=1 << 20, dx_stride=1 << 20), b"workspace_bytes"),
            (dict(workspace=4104), b"workspace")):
        _refused(lib, f(_with(DistillC, plain, more), None), parameter)
    none = dict(rows=0, logits=None, ids=None, scores=None, counts=None, loss=None, weight=None, dx=None)
    for call in (f, lib.pxg_distill_loss_device):
        assert call(_with(DistillC, plain, none), None) == 0
    _refused(lib, lib.pxg_distill_loss_device(_with(DistillC, plain, dict(logits=None, weight=None, dx=None)), None),
             b"logits")
    size = lib.pxg_distill_workspace
    assert size(0, 4, 1 << 20, 2) > 0 and size(0, 4, 8, 2) == 0 and size(0, 0, 8, 2) == 0 and size(0, 4, 8, 0) == 0


def test_no_struct_is_refused(lib):
    for f in (lib.pxg_grouped_linear_device, lib.pxg_block8_linear_device, lib.pxg_grouped_linear_grad_device,
              lib.pxg_expert_layer_device, lib.pxg_distill_loss_device, lib.pxg_distill_loss_grad_device):
        _refused(lib, f(None, None), b"arguments")


def test_arguments_are_packed_as_the_structs_lie():
    from proxima_amd import _capi, experts
    for packer, kind in ((experts._LINEAR, _capi.LinearC), (experts._LINEAR_GRAD, _capi.LinearGradC),
                         (experts._EXPERT_LAYER, _capi.ExpertLayerC), (experts._DISTILL, _capi.DistillC)):
        assert packer.size == C.sizeof(kind)
        count = packer.size // 8
        s = kind.from_buffer_copy(packer.pack(*range(1, count + 1)))

        def values(t):
            for name, of in t._fields_:
                v = getattr(t, name)
                yield from values(v) if isinstance(v, C.Structure) else (v,)

        assert list(values(s)) == list(range(1, count + 1))


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

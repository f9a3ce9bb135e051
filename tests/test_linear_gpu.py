"""Layers with their epilogue (grouped_linear, block8_linear and their backward
pass) against plain 64-bit implementations.

Tolerances. h is a product and a bias: products' tolerance of
test_experts_gpu.py with one term more. An activation's slope is at most 1.13,
so h's error grows by that at most. Into f32 the activation is evaluated to
2^-20 of |h|; into 16 bits, with the hardware's exponential, to 2^-16 of its
value and 2^-22 of |h| (the kernel's own figures: 7.4e-6 of the tail, and a
difference from one). Adding the residual is one rounding more, and the result
is rounded once: y from h before h is rounded. Packed rows into 16 bits may be
multiplied on the 8-bit cores: their cut is test_expert_kernels_gpu.py's.

A gradient's slope is off by 2^-18 (f32) or 2^-16 (16 bits) at most, terms'
magnitudes being at most 2; dh is rounded once, and a bias' gradient is a sum of
terms before that rounding, in f32: no partial sum passes the sum of the terms'
magnitudes, and no term takes part in more additions than there are rows.
"""
import ctypes as C

import pytest

import test_expert_kernels_gpu as kernels
import test_experts_gpu as base

pytestmark = pytest.mark.gpu
take = kernels.take

ACTS = [None, "silu", "gelu"]


def _act64(torch, h, act):
    if act == "silu":
        return h * torch.sigmoid(h)
    return h * torch.special.ndtr(h) if act == "gelu" else h


def _slope64(torch, h, act):
    if act == "silu":
        return torch.sigmoid(h) * (1.0 + h * torch.sigmoid(-h))
    if act == "gelu":
        return torch.special.ndtr(h) + h * torch.exp(-h * h / 2.0) * 0.3989422804014327
    return torch.ones_like(h)


def _half(dtype):
    return 2.0 ** -25 if str(dtype).endswith("float16") and not str(dtype).endswith("bfloat16") else 0.0


def _check_layer(torch, got, kept, h, size, terms, bias, ends, act, residual, cut=0.0):
    """h, size: the product and its terms' magnitudes in 64 bits, zeros in rows of no group."""
    h, size = h.clone(), size.clone()
    if bias is not None:
        for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
            h[lo:hi] += bias[g].double()
            size[lo:hi] += bias[g].double().abs()
    err = 1.25 * (terms + 1) * 2.0 ** -24 * size + cut
    if kept is not None:
        unit = base._unit(kept.dtype)
        bound = err + unit * (h.abs() + err) + _half(kept.dtype)
        assert bool(((kept.double() - h).abs() <= bound).all())
    y = _act64(torch, h, act)
    if act is not None:
        fine = got.dtype is torch.float32
        err = 1.13 * err + (2.0 ** -20 * h.abs() if fine else 2.0 ** -16 * y.abs() + 2.0 ** -22 * h.abs())
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0 ** -24 * (y.abs() + err)
    unit = base._unit(got.dtype)
    bound = err + unit * (y.abs() + err) + _half(got.dtype)
    bad = (got.double() - y).abs() > bound
    assert not bool(bad.any()), float(((got.double() - y).abs() / bound.clamp(min=1e-300)).max())


def _extras(torch, x, w, seed, dtype, out, mode):
    """(bias, residual) by mode: 0 neither, 1 a bias in f32, 2 in the operands' type and a residual, 3 a residual."""
    g = base._dev(torch, 1000 + seed)
    bias = residual = None
    if mode in (1, 2):
        bias = torch.randn(w.shape[0], w.shape[1], generator=g, device="cuda").to(torch.float32 if mode == 1 else dtype)
    if mode in (2, 3):
        residual = torch.randn(x.shape[0], w.shape[1], generator=g, device="cuda").to(out)
    return bias, residual


@pytest.mark.parametrize("kernel", [0, 16, 64, 128, 256])
@pytest.mark.parametrize("n,k", [(1, 1), (64, 64), (301, 203), (136, 520), (520, 1096), (770, 257)])
@pytest.mark.parametrize("case", range(len(kernels.RAGGED)))
def test_layers_of_ragged_groups(gpu, take, kernel, n, k, case):
    import torch
    sizes = kernels.RAGGED[case]
    dtype = torch.bfloat16 if (case + k) % 2 else torch.float16
    out = torch.float32 if (case + n) % 3 == 0 else dtype
    x, w, _, offsets = base._make(torch, sizes, n, k, dtype, 70 + case, case % 3 * 2, case % 2 * 5)
    ends = offsets.tolist()
    act, mode, keep = ACTS[(case + kernel // 16) % 3], (case + n) % 4, case % 2 == 0
    bias, residual = _extras(torch, x, w, case, dtype, out, mode)
    h, size = base._per_row(torch, x, w, ends, True)
    take(kernel)
    got = gpu.grouped_linear(x, w, offsets, bias=bias, activation=act, residual=residual, out_dtype=out, keep=keep)
    kept = None
    if keep:
        got, kept = got
    _check_layer(torch, got, kept, h, size, k, bias, ends, act, residual)
    again = gpu.grouped_linear(x, w, offsets, bias=bias, activation=act, residual=residual, out_dtype=out)
    assert torch.equal(got, again)
    if x.shape[0] and kernel:
        last = kernels._last(gpu)
        assert last == kernel if k % 8 == 0 else last == (kernel if kernel == 16 else min(kernel, 128)) | kernels.UNALIGNED


@pytest.mark.parametrize("kernel", [0, 16, 64, 128, 256])
@pytest.mark.parametrize("n,k", [(1, 1), (301, 203), (136, 520), (520, 1096)])
@pytest.mark.parametrize("case", range(len(kernels.RAGGED)))
def test_packed_layers_of_ragged_groups(gpu, take, kernel, n, k, case):
    import torch
    sizes = kernels.RAGGED[case]
    x, w, _, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 90 + case, case % 3 * 2, case % 2 * 5)
    ends = offsets.tolist()
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv, wv = gpu.block8_unpack(p, torch.float32), gpu.block8_unpack(q, torch.float32).view(w.shape)
    h, size = base._per_row(torch, xv, wv, ends, True)
    cut = torch.zeros_like(h)
    for b in range(0, k, 128):
        top, _ = base._per_row(torch, xv[:, b:b + 128].abs().amax(1, keepdim=True),
                               wv[:, :, b:b + 128].abs().amax(2, keepdim=True), ends, True)
        cut += 128 * 2.0 ** -13 * top
    take(kernel)
    for i, out in enumerate((torch.bfloat16, torch.float16, torch.float32)):
        act, mode = ACTS[(case + i) % 3], (case + n + i) % 4
        bias, residual = _extras(torch, x, w, case, torch.bfloat16, out, mode)
        got = gpu.block8_linear(p, q, offsets, bias=bias, activation=act, residual=residual, out_dtype=out)
        _check_layer(torch, got, None, h, size, k, bias, ends, act, residual,
                     0.0 if out is torch.float32 or kernel not in (0, 256) else cut)


def test_a_layer_without_anything_is_the_product(gpu):
    import torch
    for sizes, n, k in (([5, 0, 70], 64, 136), ([700, 900], 512, 384), ([31], 77, 48)):
        x, w, _, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 3, 1, 2)
        for out in (torch.bfloat16, torch.float32):
            assert torch.equal(gpu.grouped_linear(x, w, offsets, out_dtype=out),
                               gpu.grouped_matmul(x, w, offsets, out_dtype=out))
        p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
        assert torch.equal(gpu.block8_linear(p, q, offsets), gpu.block8_matmul(p, q, offsets))


@pytest.mark.parametrize("n,k", [(72, 80), (129, 77), (256, 1024)])
def test_strided_layers_and_a_residual_in_place(gpu, n, k):
    import torch
    sizes = [60, 0, 300]
    x, w, _, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 6, 3, 9)
    ends = offsets.tolist()
    rows = x.shape[0]
    h, size = base._per_row(torch, x, w, ends, True)
    for pad in (1, 8, 40):
        def wide(t, fill=float("nan")):
            b = torch.full((*t.shape[:-1], t.shape[-1] + pad), fill, dtype=t.dtype, device="cuda")
            b[..., :t.shape[-1]] = t
            return b[..., :t.shape[-1]]

        for out in (torch.bfloat16, torch.float32):
            bias, residual = _extras(torch, x, w, pad, torch.bfloat16, out, 2)
            held = wide(residual, 3.0)
            got = gpu.grouped_linear(wide(x), wide(w), offsets, bias=wide(bias), activation="gelu", residual=held,
                                     out=held)
            assert got.data_ptr() == held.data_ptr()
            _check_layer(torch, got, None, h, size, k, bias, ends, "gelu", residual)
            full = held.as_strided((rows, n + pad), (n + pad, 1))
            assert bool((full[:, n:] == 3.0).all())
    one = gpu.grouped_linear(x[:1], w[0], bias=w[0, :, 0].contiguous(), activation="silu")
    assert torch.equal(one, gpu.grouped_linear(x[:1], w[0], bias=w[:1, :, 0].contiguous(), activation="silu"))
    assert gpu.grouped_linear(x[:0], w[0]).shape == (0, n)


def test_layers_keep_other_groups_out(gpu, take):
    import torch
    sizes = [140, 330, 0, 550]
    for kernel in (16, 64, 128, 256):
        take(kernel)
        x, w, residual, offsets = base._make(torch, sizes, 88, 72, torch.bfloat16, 9, 10, 20)
        ends = offsets.tolist()
        bias = torch.randn(4, 88, device="cuda")

        def every():
            y, h = gpu.grouped_linear(x, w, offsets, bias=bias, activation="gelu", residual=residual, keep=True)
            p = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, 72))
            return [y, h, gpu.block8_linear(*p, offsets, bias=bias, activation="silu", residual=residual)]

        clean = every()
        x[:ends[0]], x[ends[-1]:], x[ends[1]:ends[2]] = float("nan"), float("inf"), float("nan")
        w[1], w[2], bias[1], bias[2] = float("inf"), float("nan"), float("nan"), float("inf")
        dirty = every()
        none = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
        none[ends[0]:ends[-1]] = False
        for a, b in zip(clean, dirty):
            for lo, hi in ((0, ends[1]), (ends[2], x.shape[0])):
                assert torch.equal(a[lo:hi], b[lo:hi])
            assert bool(torch.isnan(b[ends[1]:ends[2]]).all())
        for y in (dirty[0], dirty[2]):
            assert torch.equal(y[none], residual[none])
        assert not bool(dirty[1][none].any())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_an_activation_s_far_values(gpu, act, dtype):
    # h of every magnitude, both signs, infinities and NaN, through a bias; the products are zero
    import torch
    dtype = getattr(torch, dtype)
    v = torch.tensor([0.0, 1e-30, 1e-6, 0.1, 1.0, 3.0, 8.0, 13.0, 30.0, 100.0, 300.0, 3e4], device="cuda")
    v = torch.cat([v, -v, torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda")])
    n = v.numel()
    operands = torch.bfloat16 if dtype is torch.float32 else dtype
    x, w = torch.zeros(3, 8, dtype=operands, device="cuda"), torch.zeros(n, 8, dtype=operands, device="cuda")
    y = gpu.grouped_linear(x, w, bias=v, activation=act, out_dtype=dtype)
    h = v.double()
    want = _act64(torch, h, act)
    bound = 2.0 ** -20 * h.abs() if dtype is torch.float32 else 2.0 ** -16 * want.abs() + 2.0 ** -22 * h.abs()
    bound = bound + base._unit(dtype) * (want.abs() + bound) + _half(dtype)
    for row in y.double():
        assert bool(((row - want).abs()[:n - 3] <= bound[:n - 3]).all())
        assert float(row[n - 3]) == float("inf") and bool(torch.isnan(row[n - 1]))
        assert bool(torch.isnan(row[n - 2])) or float(row[n - 2]) == 0.0  # -inf times zero, or its limit


# --- the backward pass ------------------------------------------------------------------
def _check_grad(torch, dh, dbias, grad, h, act, ends, none_dh=True):
    slope = _slope64(torch, h.double(), act) if act else torch.ones_like(grad, dtype=torch.float64)
    want = grad.double() * slope
    inside = torch.zeros(grad.shape[0], dtype=torch.bool, device="cuda")
    inside[ends[0]:ends[-1]] = True
    fast = grad.dtype is not torch.float32
    off = 0.0 if act is None else (2.0 ** -16 if fast else 2.0 ** -18) * grad.double().abs()
    if act is not None:
        bound = off + base._unit(grad.dtype) * (want.abs() + off) + _half(grad.dtype)
        bad = ((dh.double() - want).abs() > bound) & inside[:, None]
        assert not bool(bad.any())
        assert not bool(dh[~inside].any())
    for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        s = want[lo:hi].sum(0)
        size = want[lo:hi].abs().sum(0) + (off[lo:hi].sum(0) if act else 0.0)
        bound = (off[lo:hi].sum(0) if act else 0.0) + (hi - lo + 1) * 2.0 ** -24 * size
        bound = bound + base._unit(dbias.dtype) * (s.abs() + bound) + _half(dbias.dtype)
        assert bool(((dbias[g].double() - s).abs() <= bound).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("n", [1, 7, 64, 301, 520, 4096])
@pytest.mark.parametrize("case", range(len(kernels.RAGGED)))
def test_backward_pass_of_ragged_groups(gpu, dtype, n, case):
    import torch
    sizes, dtype = kernels.RAGGED[case], getattr(torch, dtype)
    g = base._dev(torch, case * 10 + n)
    before, after = case % 3, case % 2 * 4
    rows = sum(sizes) + before + after
    grad = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    h = (2.0 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    offsets = base._offsets(torch, sizes, before)
    ends = offsets.tolist()
    for act in ACTS:
        bias_dtype = dtype if case % 2 else torch.float32
        dh, dbias = gpu.grouped_linear_grad(grad, h if act else None, act, offsets, bias_dtype=bias_dtype)
        if act is None:
            assert dh is grad
        _check_grad(torch, dh, dbias, grad, h, act, ends)
        assert dbias.dtype is bias_dtype and dbias.shape == (len(sizes), n)


@pytest.mark.parametrize("sizes,n", [([20_000], 33), ([9000, 0, 12, 7001], 136), ([40_000, 3], 1000), ([300] * 90, 264)])
def test_backward_pass_of_long_groups(gpu, sizes, n):
    # sums in parts, and the same without a workspace
    import torch

    from proxima_amd._capi import LinearGradC
    g = base._dev(torch, n)
    rows = sum(sizes) + 11
    grad = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    h = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    offsets = base._offsets(torch, sizes, 4)
    ends = offsets.tolist()
    lib = gpu._lib
    need = lib.pxg_grouped_linear_grad_workspace(rows, n, len(sizes))
    assert need > 0
    dh, dbias = gpu.grouped_linear_grad(grad, h, "gelu", offsets)
    _check_grad(torch, dh, dbias, grad, h, "gelu", ends)
    again = gpu.grouped_linear_grad(grad, h, "gelu", offsets)
    assert torch.equal(dh, again[0]) and torch.equal(dbias, again[1])
    space = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")
    def call(out, other, given):
        a = LinearGradC(type=2, bias_type=0, activation=1, rows=rows, n=n, groups=len(sizes), grad=grad.data_ptr(),
                        grad_stride=n, h=h.data_ptr(), h_stride=n, offsets=offsets.data_ptr(), dh=out.data_ptr(),
                        dh_stride=n, dbias=other.data_ptr() if other is not None else None, dbias_stride=n,
                        workspace=space.data_ptr() if given else None, workspace_bytes=given)
        assert lib.pxg_grouped_linear_grad_device(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0

    for given in (0, need - 4, need):
        space.fill_(255)
        out, other = torch.empty_like(dh), torch.empty_like(dbias)
        call(out, other, given)
        assert torch.equal(out, dh)
        _check_grad(torch, out, other, grad, h, "gelu", ends)
        assert bool((space[given:] == 255).all())
    # without a bias
    out = torch.empty_like(dh)
    call(out, None, 0)
    assert torch.equal(out, dh)


def test_backward_pass_in_place_strided_and_of_offsets_of_any_value(gpu):
    import torch
    g = base._dev(torch, 5)
    for n in (264, 77):
        grad = torch.randn(200, n, generator=g, device="cuda").half()
        h = torch.randn(200, n, generator=g, device="cuda").half()
        for raw in ([0, 90, 40, 120, 200], [-5, 10, 10, 150, 1 << 40], [30, 20, 10, 5, 0], [500, 600, 700, 800, 900]):
            ends, top = [], 0
            for v in raw:
                top = max(top, min(max(v, 0), 200))
                ends.append(top)
            offsets = torch.tensor(raw, device="cuda")
            dh, dbias = gpu.grouped_linear_grad(grad, h, "silu", offsets)
            _check_grad(torch, dh, dbias, grad, h, "silu", ends)
            for which in range(2):
                hold = torch.full((2, 200, n + 9), 3.0, dtype=torch.float16, device="cuda")
                a, b = hold[0, :, :n], hold[1, :, :n]
                a.copy_(grad), b.copy_(h)
                got = gpu.grouped_linear_grad(a, b, "silu", offsets, out=(a, b)[which])
                assert torch.equal(got[0], dh) and torch.equal(got[1], dbias)
                assert bool((hold[..., n:] == 3.0).all())
                assert torch.equal((b, a)[which], (h, grad)[which])
        dh, dbias = gpu.grouped_linear_grad(grad, h, "gelu")
        assert dbias.shape == (n,)
        _check_grad(torch, dh, dbias[None], grad, h, "gelu", [0, 200])
    none = gpu.grouped_linear_grad(grad[:0], h[:0], "gelu", torch.tensor([0, 3, 9], device="cuda"))
    assert none[0].shape == (0, 77) and not bool(none[1].any())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_backward_pass_against_differences(gpu, act):
    # of the layer itself, by its bias: (f(h + d) - f(h - d)) / 2 d is off from f'(h) by d^2 max |f'''| / 6 (0.8 at
    # most for both) and by the two values' errors over 2 d
    import torch
    sizes, n, k, d = [70, 0, 130], 96, 64, 2.0 ** -6
    x, w, grad, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 2)
    bias = torch.randn(3, n, device="cuda")
    _, h = gpu.grouped_linear(x, w, offsets, bias=bias, activation=act, out_dtype=torch.float32, keep=True)
    dh, dbias = gpu.grouped_linear_grad(grad.float(), h, act, offsets)
    up = gpu.grouped_linear(x, w, offsets, bias=bias + d, activation=act, out_dtype=torch.float32).double()
    down = gpu.grouped_linear(x, w, offsets, bias=bias - d, activation=act, out_dtype=torch.float32).double()
    want = (up - down) / (2.0 * d)
    _, size = base._per_row(torch, x, w, offsets.tolist(), True)
    size += bias.abs().max() + d
    off = d * d * 0.8 / 6.0 + (1.13 * 1.25 * (k + 1) * 2.0 ** -24 * size + 2.0 ** -20 * size + 2.0 ** -23 * size) / d
    off += 2.0 ** -17  # the slope's own, and its rounding
    assert bool(((dh.double() - grad.double() * want).abs() <= grad.double().abs() * off).all())
    for g, (lo, hi) in enumerate(zip(offsets.tolist()[:-1], offsets.tolist()[1:])):
        s, bound = (grad.double() * want)[lo:hi].sum(0), (grad.double().abs() * (off + 130 * 2.0 ** -23))[lo:hi].sum(0)
        assert bool(((dbias[g].double() - s).abs() <= bound).all())


def test_a_network_of_them_is_differentiated(gpu):
    """Two layers with a residual as a torch.autograd.Function, against autograd in 64 bits on the same weights."""
    import torch

    class Network(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w1, b1, w2, offsets):
            a, h = gpu.grouped_linear(x, w1, offsets, bias=b1, activation="gelu", keep=True)
            ctx.save_for_backward(x, w1, w2, h, a, offsets)
            return gpu.grouped_linear(a, w2, offsets, residual=x)

        @staticmethod
        def backward(ctx, dy):
            x, w1, w2, h, a, offsets = ctx.saved_tensors
            dw2 = gpu.grouped_matmul_grad_weight(dy, a, offsets)
            dh, db1 = gpu.grouped_linear_grad(gpu.grouped_matmul_grad_input(dy, w2, offsets), h, "gelu", offsets)
            dw1 = gpu.grouped_matmul_grad_weight(dh, x, offsets)
            return dy + gpu.grouped_matmul_grad_input(dh, w1, offsets), dw1, db1, dw2, None

    sizes, dim, hidden = [70, 0, 33, 129], 64, 96
    x, w1, _, offsets = base._make(torch, sizes, hidden, dim, torch.float16, 2)
    _, w2, dy, _ = base._make(torch, sizes, dim, hidden, torch.float16, 3)
    b1 = torch.randn(len(sizes), hidden, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w1, b1, w2)]
    Network.apply(*leaves, offsets).backward(dy)
    x64, w164, b164, w264 = [t.detach().double().cpu().requires_grad_() for t in leaves]
    y, ends = [], offsets.tolist()
    for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        h = x64[lo:hi] @ w164[g].t() + b164[g]
        y.append(h * torch.special.ndtr(h) @ w264[g].t() + x64[lo:hi])
    torch.cat(y).backward(dy.double().cpu())
    # a, h, dh, da and the results are rounded to f16: five roundings of 2^-11 on any path, of sums whose terms'
    # magnitudes are at most sqrt(terms) of the result's own for these normal values
    for got, want in zip(leaves, (x64, w164, b164, w264)):
        want = want.grad.cuda()
        assert float((got.grad.double() - want).norm() / want.norm()) < 5 * 2.0 ** -11


def test_layers_in_a_graph_and_on_another_stream(gpu):
    import torch
    x, w, grad, offsets = base._make(torch, [100, 0, 60], 256, 128, torch.bfloat16, 11)
    bias = torch.randn(3, 256, device="cuda")

    def step():
        y, h = gpu.grouped_linear(x, w, offsets, bias=bias, activation="gelu", keep=True)
        dh, dbias = gpu.grouped_linear_grad(grad, h, "gelu", offsets)
        p = gpu.block8_pack(x)
        z = gpu.block8_linear(p, gpu.block8_pack(w.reshape(-1, 128)), offsets, bias=bias, residual=y)
        return [y, h, dh, dbias, z]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        fx, _, fg, fo = base._make(torch, [[100, 0, 60], [1, 150, 9], [0, 0, 160], [53, 53, 54]][seed], 256, 128,
                                   torch.bfloat16, 20 + seed)
        x.copy_(fx), grad.copy_(fg), offsets.copy_(fo)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_rows_millions_of_elements_apart_and_many(gpu):
    import torch
    sizes, n, k, far = [300, 0, 260], 264, 136, 1 << 22
    x, w, grad, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 23)

    def apart(t):
        hold = torch.empty(t.shape[0] * far, dtype=t.dtype, device="cuda").view(t.shape[0], far)[:, :t.shape[1]]
        return hold.copy_(t)

    residual = grad.clone()
    want, h = gpu.grouped_linear(x, w, offsets, activation="gelu", residual=residual, keep=True)
    assert torch.equal(gpu.grouped_linear(apart(x), w, offsets, activation="gelu", residual=apart(residual),
                                          out=apart(torch.zeros_like(grad))), want)
    plain = gpu.grouped_linear_grad(grad, h, "gelu", offsets)
    got = gpu.grouped_linear_grad(apart(grad), apart(h), "gelu", offsets, out=apart(torch.zeros_like(grad)))
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    torch.cuda.empty_cache()
    # rows past 2^32 bytes: what is not zero lies at the very end
    rows, n, tail = 1_060_000, 4096, 50
    grad = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    grad[-tail:] = torch.randn(tail, n, generator=base._dev(torch, 25), device="cuda").bfloat16()
    offsets = torch.tensor([0, rows - tail, rows], device="cuda")
    dh, dbias = gpu.grouped_linear_grad(grad, grad, "silu", offsets)
    small = gpu.grouped_linear_grad(grad[-tail:].clone(), grad[-tail:].clone(), "silu")
    assert torch.equal(dh[-tail:], small[0])
    assert not bool(dh[:rows - tail].any()) and not bool(dbias[0].any())
    want = small[0].double().sum(0)
    size = small[0].double().abs().sum(0)
    assert bool(((dbias[1].double() - want).abs() <= (2.0 ** -8 + tail * 2.0 ** -24) * size).all())


def test_layers_refuse(gpu):
    import torch
    x, w, grad, offsets = base._make(torch, [4, 5], 16, 24, torch.bfloat16, 1)
    bias, h = torch.zeros(2, 16, device="cuda"), grad.clone()
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, 24))
    f, b, r = gpu.grouped_linear, gpu.block8_linear, gpu.grouped_linear_grad
    mismatch = gpu.DimensionMismatch
    for call, error in [
        (lambda: f(x, w, offsets, bias=bias[:1]), mismatch),
        (lambda: f(x, w, offsets, bias=bias[0]), ValueError),
        (lambda: f(x, w, offsets, bias=bias.half()), ValueError),
        (lambda: f(x, w, offsets, bias=bias.cpu()), ValueError),
        (lambda: f(x, w, offsets, bias=bias[:1].expand(2, 16)), gpu.ProximaError),
        (lambda: f(x, w, offsets, activation="tanh"), ValueError),
        (lambda: f(x, w, offsets, residual=grad[:3]), mismatch),
        (lambda: f(x, w, offsets, residual=grad.float()), ValueError),
        (lambda: f(x, w, offsets, residual=grad, out_dtype=torch.float32), ValueError),
        (lambda: f(x, w, offsets, out=torch.zeros(9, 17, device="cuda")), mismatch),
        (lambda: f(x.float(), w, offsets), ValueError),
        (lambda: f(x, w, offsets, out_dtype=torch.float16), gpu.ProximaError),
        (lambda: b(p, q, offsets, bias=bias.half()), ValueError),
        (lambda: b(p, q, offsets, residual=grad.half()), ValueError),
        (lambda: b(x, q, offsets), ValueError),
        (lambda: r(grad, None, "gelu", offsets), ValueError),
        (lambda: r(grad, h, None, offsets), ValueError),
        (lambda: r(grad, h.float(), "gelu", offsets), ValueError),
        (lambda: r(grad, h[:3], "gelu", offsets), mismatch),
        (lambda: r(grad, h, "gelu", offsets, bias_dtype=torch.float16), ValueError),
        (lambda: f(x.clone().requires_grad_(), w, offsets), ValueError),
        (lambda: f(x, w, offsets, bias=bias.clone().requires_grad_()), ValueError),
        (lambda: f(x, w, offsets, residual=grad.clone().requires_grad_()), ValueError),
        (lambda: r(grad, h.clone().requires_grad_(), "gelu", offsets), ValueError),
    ]:
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("dtype,n,k", [("bfloat16", 2048, 192), ("float16", 2056, 200), ("bfloat16", 2049, 128)])
def test_large_results_are_written_past_the_caches(gpu, dtype, n, k):
    # y and h of 16 MB and more, of whole and of odd rows, which the next calls read
    import torch
    dtype = getattr(torch, dtype)
    sizes = [2600, 90, 0, 1900, 128]
    x, w, _, offsets = base._make(torch, sizes, n, k, dtype, 33, 4, 3)
    ends = offsets.tolist()
    bias, residual = _extras(torch, x, w, 5, dtype, dtype, 2)
    h, size = base._per_row(torch, x, w, ends, True)
    y, kept = gpu.grouped_linear(x, w, offsets, bias=bias, activation="gelu", residual=residual, keep=True)
    _check_layer(torch, y, kept, h, size, k, bias, ends, "gelu", residual)
    dh, dbias = gpu.grouped_linear_grad(y, kept, "silu", offsets)
    _check_grad(torch, dh, dbias, y, kept, "silu", ends)
    held = residual.clone()
    gpu.grouped_linear(x, w, offsets, bias=bias, activation="gelu", residual=held, out=held)
    assert torch.equal(held, y)

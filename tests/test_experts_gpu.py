"""Expert layers and packed rows (proxima_amd/experts.py) against plain 64-bit
implementations: the packed format value by value, the products of ragged
groups and their gradients at sizes where tiles, blocks and groups end badly,
and the activations with their packed input.

Tolerances. A product is summed in f32 on the matrix cores: each instruction
adds at most 32 (16-bit operands) or 128 (packed) products onto the
accumulator, with no more than one unit of 2^-24 of the largest partial sum
for each term and one for the accumulator; partial sums are at most S, the sum
of the terms' magnitudes, so the error is below 1.25 K 2^-24 S for K terms.
Then one rounding to the output's type: 2^-24, 2^-11 (f16; 2^-25 for its
subnormals) or 2^-8 (bf16) of the value. Activations are evaluated in f32 from
exact inputs: 2^-20 of the terms' magnitudes covers a dozen roundings and the
functions' own few ulp, then the same rounding.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _dev(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _unit(dtype):
    return UNIT[str(dtype).split(".")[1]]


def _offsets(torch, sizes, before=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]) + before, dtype=torch.int64, device="cuda")


def _close(got, want, magnitude, terms):
    """Products' tolerance (see above); `magnitude` is the sum of the terms' magnitudes."""
    got = got.double()
    bound = 1.25 * terms * 2.0 ** -24 * magnitude
    bound = bound + _unit_of(got, want, bound)
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), float(((got - want).abs() / bound.clamp(min=1e-300)).max())


def _unit_of(got, want, bound):
    return _unit_of.unit * (want.abs() + bound) + (2.0 ** -25 if _unit_of.unit == 2.0 ** -11 else 0.0)


def _check(got, want, magnitude, terms):
    _unit_of.unit = _unit(got.dtype)
    _close(got, want, magnitude, terms)


# --- the packed format --------------------------------------------------------------
def _values(bits):
    """The 256 e4m3 values, by the format's definition."""
    out = np.zeros(256)
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        v = m / 8.0 * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
        out[c] = np.nan if (c & 127) == 127 else (-v if s else v)
    return out[bits]


def _pack64(x):
    """(values, scale bytes) of packed rows, in 64 bits; x finite or not."""
    rows, cols = x.shape
    blocks = -(-cols // 128)
    out, scales = np.zeros((rows, cols)), np.full((rows, -(-blocks // 4) * 4), 127, np.uint8)
    for b in range(blocks):
        v = x[:, 128 * b:128 * b + 128].astype(np.float64)
        fine = np.isfinite(v)
        m = np.where(fine, np.abs(v), 0.0).max(1)
        e = np.full(rows, -126)
        for i, t in enumerate(m):
            while t > 448.0 * 2.0 ** float(e[i]):
                e[i] += 1
        scales[:, b] = e + 127
        u = np.where(fine, v, 0.0) / np.exp2(e.astype(float))[:, None]
        step = np.exp2(np.floor(np.log2(np.maximum(np.abs(u), 2.0 ** -6)))) / 8.0
        q = np.round(u / step) * step * np.exp2(e.astype(float))[:, None]  # np.round: ties to even
        out[:, 128 * b:128 * b + 128] = np.where(fine, q, np.nan)
    return out, scales


def _decoded(p):
    codes, scales = p.codes.cpu().numpy(), p.scales.cpu().numpy().astype(float)
    wide = np.repeat(np.exp2(scales - 127.0), 128, 1)[:, :codes.shape[1]]
    return _values(codes) * wide


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (2, 128), (5, 129), (4, 512), (7, 641), (130, 300)])
def test_pack_is_the_definition(gpu, dtype, rows, cols):
    import torch
    g = _dev(torch, rows * 1000 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(
        3.0 * torch.randn(rows, cols, generator=g, device="cuda"))
    x = x.to(getattr(torch, dtype))
    x[0, 0] = 0.0
    p = gpu.block8_pack(x)
    want, scales = _pack64(x.double().cpu().numpy())
    got = _decoded(p)
    assert np.array_equal(p.scales.cpu().numpy(), scales)
    # some f16 inputs are infinite, and packed as NaN
    assert np.array_equal(got[:, :cols], want, equal_nan=True)
    assert not got[:, cols:].any()
    back = gpu.block8_unpack(p, torch.float32).cpu().numpy()
    assert np.array_equal(back.astype(float), want, equal_nan=True)
    assert np.array_equal(gpu.block8_unpack(p).float().cpu().numpy(), back, equal_nan=True)  # exact in bf16


def test_pack_at_the_format_s_edges(gpu):
    import torch
    inf, nan = float("inf"), float("nan")
    rows = []
    for top in (0.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), 2.0 ** -140, 3.4e38, 2.0 ** -118, 1e-38,
                449.0, 896.0, 897.0):
        r = np.zeros(128, np.float32)
        r[5], r[6], r[7], r[77] = top, -top / 3, top / 448 * 2.0 ** -9, top / 448 * 2.0 ** -10
        rows.append(r)
    # every midpoint between neighbouring values, and one f32 step either side
    v = _values(np.arange(0, 127))
    mid = ((v[1:] + v[:-1]) / 2).astype(np.float32)
    for m in (mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(1e9))):
        rows.append(np.concatenate([m[:120], -m[119:125], [448.0, 0.0]]).astype(np.float32))
        rows.append(np.concatenate([m[6:], [448.0] * 8]).astype(np.float32))
    rows.append(np.array([nan, inf, -inf, 1.0] + [0.0] * 124, np.float32))
    rows.append(np.full(128, nan, np.float32))
    x = np.stack(rows)
    p = gpu.block8_pack(torch.from_numpy(x).cuda())
    want, scales = _pack64(x.astype(np.float64))
    assert np.array_equal(p.scales.cpu().numpy(), scales)
    assert np.array_equal(_decoded(p), want, equal_nan=True)


def test_pack_of_strided_rows_and_no_rows(gpu):
    import torch
    g = _dev(torch, 3)
    big = torch.randn(40, 515, generator=g, device="cuda").bfloat16()
    for x in (big[:, 3:260], big[::3, 1:130], big[5:6, 2:300]):
        a, b = gpu.block8_pack(x), gpu.block8_pack(x.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        out = torch.full((40, 515), 7.0, device="cuda")
        gpu.block8_unpack(a, out=out[:x.shape[0], 3:3 + x.shape[1]])
        assert torch.equal(out[:x.shape[0], 3:3 + x.shape[1]], gpu.block8_unpack(b, torch.float32))
        assert bool((out[:, :3] == 7.0).all()) and bool((out[:, 3 + x.shape[1]:] == 7.0).all())
    none = gpu.block8_pack(big[:0])
    assert none.rows == 0 and gpu.block8_unpack(none).shape == (0, 515)


# --- products -----------------------------------------------------------------------
SIZES = [
    [1], [5], [0, 3, 0], [64, 1, 63], [100, 0, 0, 29, 200], [0, 0], [17, 16, 15, 1, 1, 300], [257, 0, 255],
    [3] * 70, [0] * 65 + [9] + [0] * 5,
]
SHAPES = [(1, 1), (8, 8), (64, 64), (31, 65), (128, 200), (301, 203), (136, 520), (512, 256)]


def _make(torch, sizes, n, k, dtype, seed, before=0, after=0):
    g = _dev(torch, seed)
    rows = int(sum(sizes)) + before + after
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(len(sizes), n, k, generator=g, device="cuda") / k ** 0.5).to(dtype)
    grad = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    return x, w, grad, _offsets(torch, sizes, before)


def _per_row(torch, a, w, ends, transposed):
    """(result, magnitude) in 64 bits: each group's rows times its matrix (or that transposed), zeros elsewhere."""
    cols = w.shape[1] if transposed else w.shape[2]
    out = torch.zeros(a.shape[0], cols, dtype=torch.float64, device="cuda")
    size = out.clone()
    for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        if hi > lo:
            m = (w[g].double().t() if transposed else w[g].double()).contiguous()
            out[lo:hi] = a[lo:hi].double() @ m
            size[lo:hi] = a[lo:hi].double().abs() @ m.abs()
    return out, size


def _per_group(torch, grad, x, ends):
    out = torch.zeros(len(ends) - 1, grad.shape[1], x.shape[1], dtype=torch.float64, device="cuda")
    size = out.clone()
    for g, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        if hi > lo:
            m = grad[lo:hi].double().t().contiguous()
            out[g] = m @ x[lo:hi].double()
            size[g] = m.abs() @ x[lo:hi].double().abs()
    return out, size


def _check_products(torch, px, x, w, grad, offsets, ends, out_dtype):
    n, k = w.shape[1:]
    longest = max([b - a for a, b in zip(ends[:-1], ends[1:])] + [1])
    want, size = _per_row(torch, x, w, ends, True)
    _check(px.grouped_matmul(x, w, offsets, out_dtype=out_dtype), want, size, k)
    want, size = _per_row(torch, grad, w, ends, False)
    _check(px.grouped_matmul_grad_input(grad, w, offsets, out_dtype=out_dtype), want, size, n)
    want, size = _per_group(torch, grad, x, ends)
    _check(px.grouped_matmul_grad_weight(grad, x, offsets, out_dtype=out_dtype), want, size, longest)


@pytest.mark.parametrize("case", range(len(SIZES)))
@pytest.mark.parametrize("n,k", SHAPES)
def test_products_of_ragged_groups(gpu, case, n, k):
    import torch
    dtype = torch.bfloat16 if (case + n) % 2 else torch.float16
    out = torch.float32 if (case + k) % 3 == 0 else None
    x, w, grad, offsets = _make(torch, SIZES[case], n, k, dtype, case, before=case % 2 * 3, after=case % 3)
    _check_products(torch, gpu, x, w, grad, offsets, offsets.tolist(), out)


@pytest.mark.parametrize("case", range(len(SIZES)))
@pytest.mark.parametrize("n,k", SHAPES)
def test_packed_products_of_ragged_groups(gpu, case, n, k):
    import torch
    x, w, grad, offsets = _make(torch, SIZES[case], n, k, torch.bfloat16, 100 + case, case % 3, case % 2)
    ends = offsets.tolist()
    px, pw = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv = torch.from_numpy(_decoded(px)[:, :k].copy()).cuda()
    wv = torch.from_numpy(_decoded(pw)[:, :k].copy()).cuda().view(w.shape)
    want, size = _per_row(torch, xv, wv, ends, True)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _check(gpu.block8_matmul(px, pw, offsets, out_dtype=dtype), want, size, k)
    longest = max([b - a for a, b in zip(ends[:-1], ends[1:])] + [1])
    want, size = _per_group(torch, grad, xv, ends)
    for dtype in (torch.bfloat16, torch.float32):
        _check(gpu.grouped_matmul_grad_weight(grad, px, offsets, out_dtype=dtype), want, size, longest)


@pytest.mark.parametrize("sizes,n,k", [([700, 0, 900, 448], 768, 512), ([2048], 256, 1024), ([1, 2, 3, 4, 2500], 520, 264),
                                       ([300] * 9, 384, 128), ([5000, 100], 128, 128), ([1531], 1000, 333)])
def test_larger_products(gpu, sizes, n, k):
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        x, w, grad, offsets = _make(torch, sizes, n, k, dtype, 7, 5, 300)
        ends = offsets.tolist()
        _check_products(torch, gpu, x, w, grad, offsets, ends, None)
        _check_products(torch, gpu, x, w, grad, offsets, ends, torch.float32)
    x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 8, 300, 5)
    ends = offsets.tolist()
    px, pw = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv, wv = gpu.block8_unpack(px, torch.float32), gpu.block8_unpack(pw, torch.float32).view(w.shape)
    want, size = _per_row(torch, xv, wv, ends, True)
    _check(gpu.block8_matmul(px, pw, offsets, out_dtype=torch.float32), want, size, k)
    want, size = _per_group(torch, grad, xv, ends)
    _check(gpu.grouped_matmul_grad_weight(grad, px, offsets, out_dtype=torch.float32), want, size, max(sizes))


@pytest.mark.parametrize("sizes,n,k", [([9000], 128, 72), ([5000, 0, 130, 4000], 64, 200), ([20000], 33, 17),
                                       ([3, 8000], 256, 256)])
def test_weight_gradients_of_long_groups(gpu, sizes, n, k):
    # long sums into small matrices: parts of a group's rows, joined
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        x, w, grad, offsets = _make(torch, sizes, n, k, dtype, 14, 2, 9)
        assert gpu._lib.pxg_grouped_matmul_grad_weight_workspace(x.shape[0], n, k, len(sizes)) > 0
        ends = offsets.tolist()
        want, size = _per_group(torch, grad, x, ends)
        for out_dtype in (dtype, torch.float32):
            hold = torch.full((len(sizes), n, k + 5), 3.0, dtype=out_dtype, device="cuda")
            got = gpu.grouped_matmul_grad_weight(grad, x, offsets, out=hold[..., :k])
            _check(got, want, size, max(sizes))
            assert bool((hold[..., k:] == 3.0).all())
            assert torch.equal(got, gpu.grouped_matmul_grad_weight(grad, x, offsets, out_dtype=out_dtype))
    packed = gpu.block8_pack(x)
    grad = grad.bfloat16()
    want, size = _per_group(torch, grad, gpu.block8_unpack(packed, torch.float32), ends)
    _check(gpu.grouped_matmul_grad_weight(grad, packed, offsets, out_dtype=torch.float32), want, size, max(sizes))


def test_weight_gradients_with_less_workspace(gpu):
    import torch
    lib = gpu._lib
    sizes, n, k = [6000, 0, 2500, 64], 96, 136
    x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 31)
    want, size = _per_group(torch, grad, x, offsets.tolist())
    rows = x.shape[0]
    need = lib.pxg_grouped_matmul_grad_weight_workspace(rows, n, k, len(sizes))
    slot = 4 * n * k
    assert need > slot
    space = torch.full((need + slot,), 255, dtype=torch.uint8, device="cuda")  # NaN in f32
    for given in (0, slot - 4, slot, need - 4, need, need + slot):
        out = torch.empty(len(sizes), n, k, dtype=torch.float32, device="cuda")
        status = lib.pxg_grouped_matmul_grad_weight_device(
            2, grad.data_ptr(), rows, n, n, x.data_ptr(), k, k, offsets.data_ptr(), len(sizes), 0, out.data_ptr(), k,
            n * k, space.data_ptr() if given else None, given, torch.cuda.current_stream().cuda_stream)
        assert status == 0
        _check(out, want, size, max(sizes))
        assert bool((space[given:] == 255).all())


@pytest.mark.parametrize("sizes,n,k", [([24], 520, 2048), ([33], 2048, 1000), ([100], 256, 4096), ([20, 0, 45, 7], 1024, 1032),
                                       ([1] * 16, 2048, 1024), ([100] * 70, 264, 200), ([1] * 62 + [129], 136, 72),
                                       ([16] * 8, 1024, 2048)])
def test_few_rows_and_many_groups(gpu, sizes, n, k):
    # on either side of the products' choice for few rows, and of 62 groups
    import torch
    for dtype in (torch.bfloat16, torch.float16):
        x, w, grad, offsets = _make(torch, sizes, n, k, dtype, 21, 1, 2)
        _check_products(torch, gpu, x, w, grad, offsets, offsets.tolist(), torch.float32)
        _check_products(torch, gpu, x, w, grad, offsets, offsets.tolist(), None)
    x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 22, 2, 1)
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv, wv = gpu.block8_unpack(p, torch.float32), gpu.block8_unpack(q, torch.float32).view(w.shape)
    want, size = _per_row(torch, xv, wv, offsets.tolist(), True)
    _check(gpu.block8_matmul(p, q, offsets, out_dtype=torch.float32), want, size, k)


def test_rows_millions_of_elements_apart(gpu):
    # operands and results whose bytes pass 2^32 and whose tiles pass 2^31
    import torch
    sizes, n, k, far = [300, 0, 260], 264, 136, 1 << 22
    x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 23)
    ends = offsets.tolist()

    def apart(t):
        hold = torch.empty(t.shape[0] * far, dtype=t.dtype, device="cuda").view(t.shape[0], far)[:, :t.shape[1]]
        return hold.copy_(t)

    ws = apart(w.reshape(-1, k)).as_strided((3, n, k), (n * far, far, 1))
    xs, gs = apart(x), apart(grad)
    want, size = _per_row(torch, x, w, ends, True)
    _check(gpu.grouped_matmul(xs, ws, offsets, out=apart(torch.zeros_like(grad))), want, size, k)
    want, size = _per_row(torch, grad, w, ends, False)
    _check(gpu.grouped_matmul_grad_input(gs, ws, offsets, out=apart(torch.zeros_like(x))), want, size, n)
    want, size = _per_group(torch, grad, x, ends)
    out = apart(torch.zeros_like(w.reshape(-1, k))).as_strided((3, n, k), (n * far, far, 1))
    _check(gpu.grouped_matmul_grad_weight(gs, xs, offsets, out=out), want, size, max(sizes))
    p = gpu.block8_pack(xs)
    assert torch.equal(p.codes, gpu.block8_pack(x).codes)
    assert torch.equal(gpu.block8_unpack(p, out=apart(torch.zeros_like(x))), gpu.block8_unpack(p, torch.bfloat16))
    for act in ("silu", "gelu"):
        a, h8 = gpu.activation_pack(gs, act)
        b, g8 = gpu.activation_pack(grad, act)
        assert torch.equal(a, b) and torch.equal(h8.codes, g8.codes)
        assert torch.equal(gpu.activation_grad(gs, h8, act), gpu.activation_grad(grad, g8, act))


def test_a_million_rows(gpu):
    # rows, codes and gradients past 2^32 bytes; what is not zero lies at the very end
    import torch
    rows, n, k, tail = 1_060_000, 64, 4096, 50
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    _, w, grad, _ = _make(torch, [1, 1], n, k, torch.bfloat16, 24)
    x[-tail:] = torch.randn(tail, k, generator=_dev(torch, 25), device="cuda").bfloat16()
    offsets = torch.tensor([0, rows - tail, rows], device="cuda")
    last = [0, tail]
    want, size = _per_row(torch, x[-tail:], w[1:], last, True)
    y = gpu.grouped_matmul(x, w, offsets)
    _check(y[-tail:], want, size, k)
    assert not bool(y[:-tail].any())
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv, wv = gpu.block8_unpack(p, torch.float32)[-tail:].clone(), gpu.block8_unpack(q, torch.float32).view(w.shape)
    assert torch.equal(p.codes[-tail:], gpu.block8_pack(x[-tail:]).codes)
    want, size = _per_row(torch, xv, wv[1:], last, True)
    _check(gpu.block8_matmul(p, q, offsets, out_dtype=torch.float32)[-tail:], want, size, k)
    grad = torch.randn(rows, n, generator=_dev(torch, 26), device="cuda").bfloat16()
    for rhs, plain in ((x, x[-tail:].float()), (p, xv)):
        want, size = _per_group(torch, grad[-tail:], plain, last)
        got = gpu.grouped_matmul_grad_weight(grad, rhs, offsets, out_dtype=torch.float32)
        _check(got[1:], want, size, tail)
        assert not bool(got[0].any())
    dx = gpu.grouped_matmul_grad_input(grad, w, offsets)
    want, size = _per_row(torch, grad[-tail:], w[1:], last, False)
    _check(dx[-tail:], want, size, n)
    a, h8 = gpu.activation_pack(x, "gelu")
    assert torch.equal(h8.codes, p.codes)
    assert torch.equal(a[-tail:], gpu.activation_pack(x[-tail:], "gelu")[0])


def test_one_group_without_offsets(gpu):
    import torch
    x, w, grad, offsets = _make(torch, [190], 96, 160, torch.float16, 4)
    assert torch.equal(gpu.grouped_matmul(x, w[0]), gpu.grouped_matmul(x, w, offsets))
    assert torch.equal(gpu.grouped_matmul_grad_input(grad, w[0]), gpu.grouped_matmul_grad_input(grad, w, offsets))
    px, pw = gpu.block8_pack(x), gpu.block8_pack(w[0])
    assert torch.equal(gpu.block8_matmul(px, pw), gpu.block8_matmul(px, pw, offsets))
    assert gpu.grouped_matmul(x[:0], w[0]).shape == (0, 96)
    assert not bool(gpu.grouped_matmul_grad_weight(grad[:0], x[:0], offsets).any())


def test_offsets_of_any_value_are_clamped(gpu):
    import torch
    x, w, grad, _ = _make(torch, [50, 50, 50, 50], 72, 80, torch.bfloat16, 5)
    for raw in ([0, 90, 40, 120, 200], [-5, 10, 10, 150, 1 << 40], [30, 20, 10, 5, 0], [500, 600, 700, 800, 900],
                [-9, -8, -7, -6, -5]):
        ends, top = [], 0
        for v in raw:
            top = max(top, min(max(v, 0), 200))
            ends.append(top)
        _check_products(torch, gpu, x, w, grad, torch.tensor(raw, device="cuda"), ends, torch.float32)
        px, pw = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, 80))
        xv, wv = gpu.block8_unpack(px, torch.float32), gpu.block8_unpack(pw, torch.float32).view(w.shape)
        want, size = _per_row(torch, xv, wv, ends, True)
        _check(gpu.block8_matmul(px, pw, torch.tensor(raw, device="cuda"), out_dtype=torch.float32), want, size, 80)


@pytest.mark.parametrize("n,k", [(72, 80), (129, 77), (256, 256)])
def test_strided_operands_and_outputs(gpu, n, k):
    import torch
    sizes = [60, 0, 130]
    x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 6)
    for pad in (1, 8, 40):
        def wide(t):
            b = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device="cuda")
            b[..., :t.shape[-1]] = t
            return b[..., :t.shape[-1]]

        xs, ws, gs = wide(x), wide(w), wide(grad)
        for fn, args, plain in ((gpu.grouped_matmul, (xs, ws), (x, w)),
                                (gpu.grouped_matmul_grad_input, (gs, ws), (grad, w)),
                                (gpu.grouped_matmul_grad_weight, (gs, xs), (grad, x))):
            want = fn(*plain, offsets)
            hold = torch.full((*want.shape[:-1], want.shape[-1] + pad), 3.0, dtype=want.dtype, device="cuda")
            got = fn(*args, offsets, out=hold[..., :want.shape[-1]])
            tol = 2.0 ** -8 * want.float().abs() + 1e-3  # another path may sum in another order
            assert bool(((got.float() - want.float()).abs() <= tol).all())
            assert bool((hold[..., want.shape[-1]:] == 3.0).all())
    every = gpu.grouped_matmul(x, w, offsets)
    some = torch.zeros(2 * x.shape[0], k, dtype=x.dtype, device="cuda")
    some[::2] = x
    assert torch.equal(gpu.grouped_matmul(some[::2], w, offsets), every)


def test_products_keep_other_groups_out(gpu):
    # NaN and infinities in one group's rows and matrix, in rows of no group and past the columns reach nothing else
    import torch
    sizes = [40, 30, 0, 50]
    for n, k in ((88, 72), (130, 250)):
        x, w, grad, offsets = _make(torch, sizes, n, k, torch.bfloat16, 9, 10, 20)
        ends = offsets.tolist()
        clean = [gpu.grouped_matmul(x, w, offsets), gpu.grouped_matmul_grad_input(grad, w, offsets),
                 gpu.grouped_matmul_grad_weight(grad, x, offsets),
                 gpu.grouped_matmul_grad_weight(grad, gpu.block8_pack(x), offsets)]
        packed = gpu.block8_matmul(gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k)), offsets)
        for t in (x, grad):
            t[:ends[0]] = float("nan")
            t[ends[-1]:] = float("inf")
            t[ends[1]:ends[2]] = float("nan")
        w[1] = float("inf")
        w[2] = float("nan")
        dirty = [gpu.grouped_matmul(x, w, offsets), gpu.grouped_matmul_grad_input(grad, w, offsets),
                 gpu.grouped_matmul_grad_weight(grad, x, offsets),
                 gpu.grouped_matmul_grad_weight(grad, gpu.block8_pack(x), offsets)]
        packed2 = gpu.block8_matmul(gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k)), offsets)
        for a, b in zip(clean[:2] + [packed], dirty[:2] + [packed2]):
            for lo, hi in ((0, ends[1]), (ends[2], x.shape[0])):
                assert torch.equal(a[lo:hi], b[lo:hi])
            assert bool(torch.isnan(b[ends[1]:ends[2]]).all())
        for a, b in zip(clean[2:], dirty[2:]):
            for e in (0, 2, 3):
                assert torch.equal(a[e], b[e])
            assert bool(torch.isnan(b[1]).all())


def test_results_repeat_and_follow_the_stream(gpu):
    import torch
    x, w, grad, offsets = _make(torch, [700, 30, 0, 900], 512, 384, torch.bfloat16, 10)

    def every():
        p = gpu.block8_pack(x)
        return [gpu.grouped_matmul(x, w, offsets), gpu.grouped_matmul_grad_input(grad, w, offsets),
                gpu.grouped_matmul_grad_weight(grad, x, offsets), gpu.grouped_matmul_grad_weight(grad, p, offsets),
                gpu.block8_matmul(p, gpu.block8_pack(w.reshape(-1, 384)), offsets)]

    first = every()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = every()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_products_in_a_graph(gpu):
    import torch
    x, w, grad, offsets = _make(torch, [100, 0, 60], 256, 128, torch.bfloat16, 11)

    def step():
        y = gpu.grouped_matmul(x, w, offsets)
        a, kept = gpu.activation_pack(y, "gelu")
        dy = gpu.activation_grad(grad, kept, "gelu")
        p = gpu.block8_pack(x)
        return [y, a, gpu.grouped_matmul_grad_input(dy, w, offsets), gpu.grouped_matmul_grad_weight(dy, p, offsets),
                gpu.block8_matmul(p, gpu.block8_pack(w.reshape(-1, 128)), offsets)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        fx, _, fg, fo = _make(torch, [[100, 0, 60], [1, 150, 9], [0, 0, 160], [53, 53, 54]][seed], 256, 128,
                              torch.bfloat16, 20 + seed)
        x.copy_(fx), grad.copy_(fg), offsets.copy_(fo)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# --- the 8-bit matrix cores ------------------------------------------------------------
# Products into 16 bits of many rows a group are multiplied in 8 bits. The cores
# align the products that they sum together to the largest of them and cut each
# below 2^-11 of it (two products of the type's extremes are off by 2^-10.9 of
# the larger, never more in 10^5 trials), so products whose magnitudes are
# within 2^5 of each other are summed exactly, and others within
# 2^-11 of their block's largest product each.
LARGE = [([600], 256, 512), ([300, 700], 512, 1024), ([0, 900, 40], 264, 384), ([2500, 3, 1200, 900], 1024, 640),
         ([4096], 2048, 2048)]


def _runs_in_8_bits(px, torch, sizes, n, k):
    """Whether the result differs from the exactly summed one on values that the cores cut."""
    x, w, _, offsets = _make(torch, sizes, n, k, torch.bfloat16, 15)
    p, q = px.block8_pack(x), px.block8_pack(w.reshape(-1, k))
    return not torch.equal(px.block8_matmul(p, q, offsets),
                           px.block8_matmul(p, q, offsets, out_dtype=torch.float32).bfloat16())


@pytest.mark.parametrize("sizes,n,k", LARGE)
def test_products_in_8_bits_of_exact_sums(gpu, sizes, n, k):
    # values of +-1, +-1.5, +-2 and +-4 with a power of two for every block: sums are exact, to the last bit
    import torch
    if sizes == [4096]:
        assert _runs_in_8_bits(gpu, torch, sizes, n, k)
    g = _dev(torch, n + k)
    rows = sum(sizes) + 7
    values = torch.tensor([1.0, 1.5, 2.0, 4.0, -1.0, -1.5, -2.0, -4.0], device="cuda")

    def draw(r):
        v = values[torch.randint(0, 8, (r, k), generator=g, device="cuda")]
        scale = torch.exp2(torch.randint(-2, 3, (r, (k + 127) // 128), generator=g, device="cuda").float())
        return v * scale.repeat_interleave(128, 1)[:, :k]

    x, w = draw(rows), draw(len(sizes) * n)
    offsets = _offsets(torch, sizes, 3)
    ends = offsets.tolist()
    p, q = gpu.block8_pack(x), gpu.block8_pack(w)
    assert torch.equal(gpu.block8_unpack(p, torch.float32), x)
    want, _ = _per_row(torch, x, w.view(len(sizes), n, k), ends, True)
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(gpu.block8_matmul(p, q, offsets, out_dtype=dtype), want.float().to(dtype))


@pytest.mark.parametrize("sizes,n,k", LARGE)
def test_products_in_8_bits(gpu, sizes, n, k):
    import torch
    x, w, _, offsets = _make(torch, sizes, n, k, torch.bfloat16, 16, 5, 11)
    ends = offsets.tolist()
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    xv, wv = gpu.block8_unpack(p, torch.float32), gpu.block8_unpack(q, torch.float32).view(w.shape)
    want, size = _per_row(torch, xv, wv, ends, True)
    cut = torch.zeros_like(want)  # 128 products of a block, each within 2^-11 of the largest of them at most
    for b in range(0, k, 128):
        top, _ = _per_row(torch, xv[:, b:b + 128].abs().amax(1, keepdim=True),
                          wv[:, :, b:b + 128].abs().amax(2, keepdim=True), ends, True)
        cut += 128 * 2.0 ** -11 * top
    for dtype in (torch.bfloat16, torch.float16):
        got = gpu.block8_matmul(p, q, offsets, out_dtype=dtype).double()
        bound = cut + 1.25 * k * 2.0 ** -24 * size
        assert bool(((got - want).abs() <= bound + _unit(dtype) * (want.abs() + bound)).all())
        # and as a whole: the cuts are of either sign, so far below the sum of their bounds
        assert float((got - want).norm() / want.norm()) < 2 * _unit(dtype)


def test_products_in_8_bits_of_short_groups(gpu):
    # many matrices with 40 rows each: the 8-bit cores also there
    import torch
    sizes, n, k = [40, 0, 61, 33] * 8, 2048, 1024
    assert _runs_in_8_bits(gpu, torch, sizes, n, k)
    test_products_in_8_bits(gpu, sizes, n, k)
    test_products_in_8_bits_of_exact_sums(gpu, sizes, n, k)


# --- activations --------------------------------------------------------------------
def _act64(torch, h, act):
    """(f, f', the magnitudes of their terms) in 64 bits."""
    if act == "silu":
        s = torch.sigmoid(h)
        return h * s, s + h * s * (1 - s), (h * s).abs(), s + (h * s * (1 - s)).abs()
    p = 0.5 * torch.erfc(-h / 2.0 ** 0.5)
    d = h * torch.exp(-h * h / 2) / (2 * torch.pi) ** 0.5
    return h * p, p + d, h.abs(), 1.0 + d.abs()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 200), (64, 1000), (129, 1024), (2, 4099)])
def test_activation_and_its_packed_backward(gpu, act, dtype, rows, cols):
    import torch
    dt = getattr(torch, dtype)
    g = _dev(torch, rows + cols)
    h = (4.0 * torch.randn(rows, cols, generator=g, device="cuda")).to(dt)
    grad = torch.randn(rows, cols, generator=g, device="cuda").to(dt)
    a, p = gpu.activation_pack(h, act)
    q = gpu.block8_pack(h)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    f, _, size, _ = _act64(torch, h.double(), act)
    bound = 2.0 ** -20 * size + 2.0 ** -60
    assert bool(((a.double() - f).abs() <= bound + _rounding(a, f, bound)).all())
    kept = torch.from_numpy(_decoded(p)[:, :cols].copy()).cuda()
    _, slope, _, size = _act64(torch, kept, act)
    got = gpu.activation_grad(grad, p, act)
    want = grad.double() * slope
    bound = 2.0 ** -20 * grad.double().abs() * size + 2.0 ** -60
    assert bool(((got.double() - want).abs() <= bound + _rounding(got, want, bound)).all())
    # against differences of the forward pass, at the kept values
    step = 2.0 ** -12
    hi, _, _, _ = _act64(torch, kept + step, act)
    lo, _, _, _ = _act64(torch, kept - step, act)
    near = grad.double() * (hi - lo) / (2 * step)
    bound = bound + grad.double().abs() * step ** 2  # a third derivative below 6
    assert bool(((got.double() - near).abs() <= bound + _rounding(got, near, bound)).all())


def _rounding(got, want, bound):
    u = _unit(got.dtype)
    return u * (want.abs() + bound) + (2.0 ** -25 if u == 2.0 ** -11 else 0.0)


def test_activation_extremes(gpu):
    import torch
    h = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 90.0, -90.0, 1e4, -1e4, 3e38, -3e38, float("inf"),
                       float("nan")]], device="cuda")
    for act in ("silu", "gelu"):
        a, p = gpu.activation_pack(h, act)
        assert not bool(torch.isnan(a[0, :13]).any()) and bool(torch.isnan(a[0, 13]))
        assert torch.equal(a[0, 8:13:2], h[0, 8:13:2]) and not bool((a[0, 9:12:2] != 0).any())
        one = torch.ones_like(h)
        for i in range(12):  # each alone in its block, so that it is kept as itself
            x = h[:, i:i + 1].contiguous()
            d = gpu.activation_grad(one[:, :1].contiguous(), gpu.activation_pack(x, act)[1], act)
            want = 0.5 if abs(float(x)) < 1 else float(x > 0)
            assert abs(float(d) - want) < 1e-6, (act, float(x), float(d))


def test_strided_activation(gpu):
    import torch
    g = _dev(torch, 12)
    big = torch.randn(50, 700, generator=g, device="cuda").half()
    h, grad = big[::2, 5:405], big[1::2, 3:403]
    a, p = gpu.activation_pack(h, "silu")
    b, q = gpu.activation_pack(h.contiguous(), "silu")
    assert torch.equal(a, b) and torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    assert torch.equal(gpu.activation_grad(grad, p, "silu"), gpu.activation_grad(grad.contiguous(), q, "silu"))


# --- gradients against differences ----------------------------------------------------
def test_layer_gradients_against_differences(gpu):
    # L = sum(grad * y): exactly linear in x and in w, so differences of the forward pass in f32 outputs are exact up
    # to its own tolerance; one element of each group is moved
    import torch
    x, w, grad, offsets = _make(torch, [40, 0, 33, 60], 48, 64, torch.float16, 13)
    ends = offsets.tolist()
    dx = gpu.grouped_matmul_grad_input(grad, w, offsets, out_dtype=torch.float32)
    dw = gpu.grouped_matmul_grad_weight(grad, x, offsets, out_dtype=torch.float32)

    def loss(x, w):
        return float((grad.double() * gpu.grouped_matmul(x, w, offsets, out_dtype=torch.float32).double()).sum())

    base = float((grad.double().abs() * gpu.grouped_matmul(x.abs(), w.abs(), offsets,
                                                           out_dtype=torch.float32).double()).sum())
    tol = 4 * 1.25 * 64 * 2.0 ** -24 * base
    for e, t in ((0, 3), (2, 41), (3, 100)):
        assert ends[e] <= t < ends[e + 1]
        hi, lo = x.clone(), x.clone()
        hi[t, 5], lo[t, 5] = 16.0, -16.0
        assert abs((loss(hi, w) - loss(lo, w)) / 32.0 - float(dx[t, 5])) <= tol
        hi, lo = w.clone(), w.clone()
        hi[e, 7, 9], lo[e, 7, 9] = 16.0, -16.0
        assert abs((loss(x, hi) - loss(x, lo)) / 32.0 - float(dw[e, 7, 9])) <= tol


# --- all of them together ---------------------------------------------------------------
def test_the_adapter_example_learns(gpu, capsys):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_adapters.py")
    spec = importlib.util.spec_from_file_location("expert_adapters", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    before, after = module.main(docs=20_000, train=16_384, steps=150)
    with capsys.disabled():
        print(f"recall {before:.3f} -> {after:.3f} ", end="")
    assert after > before + 0.3


# --- refusals ------------------------------------------------------------------------
def test_refusals(gpu):
    import torch
    px = gpu
    x, w, grad, offsets = _make(torch, [4, 5], 16, 24, torch.bfloat16, 1)
    p, pw = px.block8_pack(x), px.block8_pack(w.reshape(-1, 24))
    bad = [
        lambda: px.grouped_matmul(x.float(), w.float(), offsets),
        lambda: px.grouped_matmul(x, w.half(), offsets),
        lambda: px.grouped_matmul(x, w[:1], offsets),
        lambda: px.grouped_matmul(x[:, :20], w, offsets),
        lambda: px.grouped_matmul(x.t(), w, offsets),
        lambda: px.grouped_matmul(x.cpu(), w, offsets),
        lambda: px.grouped_matmul(x, w, offsets.int()),
        lambda: px.grouped_matmul(x, w, offsets.cpu()),
        lambda: px.grouped_matmul(x, w, offsets[:1]),
        lambda: px.grouped_matmul(x, w),
        lambda: px.grouped_matmul(x, w, offsets, out_dtype=torch.float16),
        lambda: px.grouped_matmul(x, w, offsets, out=torch.empty(9, 17, device="cuda", dtype=x.dtype)),
        lambda: px.grouped_matmul_grad_input(grad[:, 1:], w, offsets),
        lambda: px.grouped_matmul_grad_weight(grad[1:], x, offsets),
        lambda: px.grouped_matmul_grad_weight(grad, x.half(), offsets),
        lambda: px.grouped_matmul_grad_weight(grad.half(), p, offsets),
        lambda: px.grouped_matmul_grad_weight(grad, x, None),
        lambda: px.block8_matmul(p, px.block8_pack(w.reshape(-1, 48)), offsets),
        lambda: px.block8_matmul(p, px.Block8(pw.codes[:31], pw.scales[:31], 24), offsets),
        lambda: px.block8_matmul(x, pw, offsets),
        lambda: px.block8_pack(x.long()),
        lambda: px.block8_pack(x[0]),
        lambda: px.block8_pack(x[:, :0]),
        lambda: px.block8_unpack(px.Block8(p.codes, p.scales, 200)),
        lambda: px.activation_pack(x, "relu"),
        lambda: px.activation_grad(grad, p, "gelu"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, px.ProximaError)):
            call()
            print("not refused:", i)
    assert px.grouped_matmul(x, w, offsets).shape == (9, 16)  # still serves

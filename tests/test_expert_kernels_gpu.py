"""Every kernel of the products at every kind of case, and the cases for which
each is chosen: the entry points take the kernel that is estimated fastest, so
that small cases alone would leave the large tiles' loops untried. Tolerances
are those of test_experts_gpu.py. Packed rows into 16 bits may run on the 8-bit
cores, which cut every product toward zero by less than 2^(E - 13), E the sum of
two codes' exponents at most: 2^E is no more than the product of the largest
magnitudes of the two blocks, so a block's 128 products are off by 128 2^-13 of
that at most.
"""
import pytest

import test_experts_gpu as base

pytestmark = pytest.mark.gpu

EIGHT_BIT, UNALIGNED, PARTS = 1 << 16, 1 << 17, 1 << 18
KERNELS = [16, 64, 128, 256]


@pytest.fixture
def take(gpu):
    """take(rows): the kernel of the products from here on."""
    def ask(rows):
        assert gpu._lib.pxg_grouped_matmul_set_kernel(rows) == 0
    yield ask
    ask(0)


def _last(px):
    return px._lib.pxg_grouped_matmul_last_kernel()


def _check_16_bits(torch, px, p, q, w_shape, offsets, dtype):
    k = p.cols
    ends = offsets.tolist()
    xv, wv = px.block8_unpack(p, torch.float32), px.block8_unpack(q, torch.float32).view(w_shape)
    want, size = base._per_row(torch, xv, wv, ends, True)
    cut = torch.zeros_like(want)
    for b in range(0, k, 128):
        top, _ = base._per_row(torch, xv[:, b:b + 128].abs().amax(1, keepdim=True),
                               wv[:, :, b:b + 128].abs().amax(2, keepdim=True), ends, True)
        cut += 128 * 2.0 ** -13 * top
    got = px.block8_matmul(p, q, offsets, out_dtype=dtype).double()
    bound = cut + 1.25 * k * 2.0 ** -24 * size
    unit = base._unit(dtype)
    bound = bound + unit * (want.abs() + bound) + (2.0 ** -25 if dtype is torch.float16 else 0.0)
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound.clamp(min=1e-300)).max())


RAGGED = base.SIZES + [[600, 0, 130, 257, 1], [1024], [128, 512, 5, 300, 0, 256]]
WIDTHS = [(1, 1), (64, 64), (301, 203), (136, 520), (512, 768), (520, 1096), (770, 257)]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("n,k", WIDTHS)
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_every_kernel_takes_every_case(gpu, take, kernel, n, k, case):
    import torch
    sizes = RAGGED[case]
    dtype = torch.bfloat16 if (case + k) % 2 else torch.float16
    out = torch.float32 if (case + n) % 3 == 0 else None
    x, w, grad, offsets = base._make(torch, sizes, n, k, dtype, 70 + case, case % 3 * 2, case % 2 * 5)
    take(kernel)
    base._check_products(torch, gpu, x, w, grad, offsets, offsets.tolist(), out)
    aligned = n % 8 == 0 and k % 8 == 0
    if x.shape[0]:
        gpu.grouped_matmul(x, w, offsets)
        if k % 8 == 0:
            assert _last(gpu) == kernel
        else:  # rows that are not whole 16-byte pieces: 64 and 128 only
            assert _last(gpu) & UNALIGNED and (kernel == 16 or _last(gpu) & 0xFFFF == min(kernel, 128))
        if aligned:
            gpu.grouped_matmul_grad_input(grad, w, offsets)
            assert _last(gpu) == kernel
            gpu.grouped_matmul_grad_weight(grad, x, offsets)
            assert kernel == 16 or _last(gpu) & 0xFFFF == kernel


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("n,k", WIDTHS)
@pytest.mark.parametrize("case", range(0, len(RAGGED), 2))
def test_every_kernel_takes_every_packed_case(gpu, take, kernel, n, k, case):
    import torch
    sizes = RAGGED[case]
    x, w, grad, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 90 + case, case % 3 * 2, case % 2 * 5)
    ends = offsets.tolist()
    p, q = gpu.block8_pack(x), gpu.block8_pack(w.reshape(-1, k))
    take(kernel)
    xv, wv = gpu.block8_unpack(p, torch.float32), gpu.block8_unpack(q, torch.float32).view(w.shape)
    want, size = base._per_row(torch, xv, wv, ends, True)
    base._check(gpu.block8_matmul(p, q, offsets, out_dtype=torch.float32), want, size, k)
    assert not x.shape[0] or kernel == 256 or _last(gpu) == kernel
    assert not _last(gpu) & EIGHT_BIT or not x.shape[0]
    for dtype in (torch.bfloat16, torch.float16):
        _check_16_bits(torch, gpu, p, q, w.shape, offsets, dtype)
        assert not x.shape[0] or _last(gpu) == (256 | EIGHT_BIT if kernel == 256 else kernel)
    want, size = base._per_group(torch, grad, xv, ends)
    longest = max(sizes + [1])
    for dtype in (torch.bfloat16, torch.float32):
        base._check(gpu.grouped_matmul_grad_weight(grad, p, offsets, out_dtype=dtype), want, size, longest)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("n,k", [(88, 72), (520, 1096), (130, 250)])
def test_every_kernel_keeps_other_groups_out(gpu, take, kernel, n, k):
    # NaN and infinities in one group's rows and matrix and in rows of no group
    import torch
    sizes = [140, 330, 0, 550]
    x, w, grad, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 9, 10, 20)
    ends = offsets.tolist()
    take(kernel)

    def every():
        p = gpu.block8_pack(x)
        return ([gpu.grouped_matmul(x, w, offsets), gpu.grouped_matmul_grad_input(grad, w, offsets),
                 gpu.block8_matmul(p, gpu.block8_pack(w.reshape(-1, k)), offsets)],
                [gpu.grouped_matmul_grad_weight(grad, x, offsets), gpu.grouped_matmul_grad_weight(grad, p, offsets)])

    clean = every()
    for a, b in zip(sum(clean, []), sum(every(), [])):
        assert torch.equal(a, b)
    for t in (x, grad):
        t[:ends[0]], t[ends[-1]:], t[ends[1]:ends[2]] = float("nan"), float("inf"), float("nan")
    w[1], w[2] = float("inf"), float("nan")
    dirty = every()
    for a, b in zip(clean[0], dirty[0]):
        for lo, hi in ((0, ends[1]), (ends[2], x.shape[0])):
            assert torch.equal(a[lo:hi], b[lo:hi])
        assert bool(torch.isnan(b[ends[1]:ends[2]]).all())
    for a, b in zip(clean[1], dirty[1]):
        for e in (0, 2, 3):
            assert torch.equal(a[e], b[e])
        assert bool(torch.isnan(b[1]).all())


@pytest.mark.parametrize("kernel", [64, 128, 256])
@pytest.mark.parametrize("sizes,n,k", [([9000], 128, 72), ([5000, 0, 130, 4000], 64, 200), ([20_000], 33, 17),
                                       ([16_000], 1100, 264), ([3, 8000], 264, 1024), ([12_000, 40, 30], 700, 99)])
def test_long_groups_in_parts_of_every_tile(gpu, take, kernel, sizes, n, k):
    # parts' sums in their slots and joined, also past 512 rows of a matrix; with less workspace than asked for
    import torch
    x, w, grad, offsets = base._make(torch, sizes, n, k, torch.bfloat16, 14, 2, 9)
    take(kernel)
    packed = gpu.block8_pack(x)
    plain = gpu.block8_unpack(packed, torch.float32)
    for rhs, values in ((x, x), (packed, plain)):
        want, size = base._per_group(torch, grad, values, offsets.tolist())
        for dtype in (torch.bfloat16, torch.float32):
            hold = torch.full((len(sizes), n, k + 5), 3.0, dtype=dtype, device="cuda")
            got = gpu.grouped_matmul_grad_weight(grad, rhs, offsets, out=hold[..., :k])
            assert _last(gpu) & PARTS and _last(gpu) & 0xFFFF in (kernel, 128)
            base._check(got, want, size, max(sizes))
            assert bool((hold[..., k:] == 3.0).all())
            assert torch.equal(got, gpu.grouped_matmul_grad_weight(grad, rhs, offsets, out_dtype=dtype))
    want, size = base._per_group(torch, grad, x, offsets.tolist())
    rows = x.shape[0]
    need, slot = gpu._lib.pxg_grouped_matmul_grad_weight_workspace(rows, n, k, len(sizes)), 4 * n * k
    space = torch.full((need + 64,), 255, dtype=torch.uint8, device="cuda")  # NaN in f32
    for given in (0, 2 * slot, need - 4, need):
        out = torch.empty(len(sizes), n, k, dtype=torch.float32, device="cuda")
        assert gpu._lib.pxg_grouped_matmul_grad_weight_device(
            2, grad.data_ptr(), rows, n, n, x.data_ptr(), k, k, offsets.data_ptr(), len(sizes), 0, out.data_ptr(), k,
            n * k, space.data_ptr() if given else None, given, torch.cuda.current_stream().cuda_stream) == 0
        base._check(out, want, size, max(sizes))
        assert bool((space[given:] == 255).all())


# --- what the estimates choose -------------------------------------------------------------
UNEVEN = [2600, 90, 0, 1900, 128, 1400, 1274, 800]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("sizes,n,k,kernels", [
    (UNEVEN, 4096, 1024, (256, 256, 256)),
    (UNEVEN, 1024, 4096, (256, 256, 256)),
    ([512] * 8, 1024, 1024, (128, 128, None)),
    ([3000], 1500, 1500, (128 | UNALIGNED, 128 | UNALIGNED, None)),
    ([7800, 500, 0, 900, 40, 1200] + [594] * 9 + [598], 2048, 2048, (256, 256, 256 | PARTS)),
])
def test_large_products_take_large_tiles(gpu, dtype, sizes, n, k, kernels):
    import torch
    dtype = getattr(torch, dtype)
    x, w, grad, offsets = base._make(torch, sizes, n, k, dtype, 33, 4, 3)
    ends = offsets.tolist()
    forward, back, weight = kernels
    for out in (None, torch.float32):
        want, size = base._per_row(torch, x, w, ends, True)
        base._check(gpu.grouped_matmul(x, w, offsets, out_dtype=out), want, size, k)
        assert forward is None or _last(gpu) == forward
        want, size = base._per_row(torch, grad, w, ends, False)
        base._check(gpu.grouped_matmul_grad_input(grad, w, offsets, out_dtype=out), want, size, n)
        assert back is None or _last(gpu) == back
        want, size = base._per_group(torch, grad, x, ends)
        base._check(gpu.grouped_matmul_grad_weight(grad, x, offsets, out_dtype=out), want, size, max(sizes))
        assert weight is None or _last(gpu) & weight == weight
    if dtype is torch.bfloat16:
        p = gpu.block8_pack(x)
        want, size = base._per_group(torch, grad, gpu.block8_unpack(p, torch.float32), ends)
        for out in (None, torch.float32):
            base._check(gpu.grouped_matmul_grad_weight(grad, p, offsets, out_dtype=out), want, size, max(sizes))
            assert weight is None or _last(gpu) & weight == weight


def test_small_and_large_products_choose(gpu):
    import torch
    seen = set()
    for rows, n, k in ((1, 4096, 4096), (200, 512, 512), (4096, 1024, 1024), (8192, 4096, 4096)):
        x, w, grad, offsets = base._make(torch, [rows], n, k, torch.bfloat16, 5)
        p, q = gpu.block8_pack(x), gpu.block8_pack(w[0])
        for call in (lambda: gpu.grouped_matmul(x, w, offsets), lambda: gpu.grouped_matmul_grad_input(grad, w, offsets),
                     lambda: gpu.grouped_matmul_grad_weight(grad, x, offsets), lambda: gpu.block8_matmul(p, q),
                     lambda: gpu.block8_matmul(p, q, out_dtype=torch.float32)):
            call()
            seen.add(_last(gpu))
    assert {16, 64, 128, 256, 256 | EIGHT_BIT} <= {s & ~PARTS for s in seen}

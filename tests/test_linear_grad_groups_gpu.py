"""The layers' backward pass where one of many groups, or the rows behind the
last of them, hold most rows, against the formula in 64 bits with the tolerances
of test_linear_gpu.py."""
import pytest

import test_experts_gpu as base
import test_linear_gpu as linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,act", [("bfloat16", "gelu"), ("float16", "silu"), ("float32", "gelu"), ("bfloat16", None)])
@pytest.mark.parametrize("n", [264, 301])
@pytest.mark.parametrize("groups,longest,behind", [(128, 5000, 0), (256, 5000, 77), (130, 0, 5000), (70, 2000, 3000)])
def test_most_rows_in_one_place(gpu, groups, longest, behind, n, dtype, act):
    import torch
    dtype = getattr(torch, dtype)
    g = base._dev(torch, groups + n)
    sizes = [i % 5 for i in range(groups)]
    sizes[groups // 3] += longest
    rows = sum(sizes) + behind
    grad = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    h = (2.0 * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)
    if behind:
        grad[-behind:] = float("nan")  # padding is not looked at
    offsets = base._offsets(torch, sizes, 0)
    ends = offsets.tolist()
    dh, dbias = gpu.grouped_linear_grad(grad, h if act else None, act, offsets)
    if behind and act:
        assert not bool(dh[-behind:].any())
    clean = grad.clone()
    clean[rows - behind:] = 0.0
    linear._check_grad(torch, dh if act else clean, dbias, clean, h, act, ends)
    again = gpu.grouped_linear_grad(grad, h if act else None, act, offsets)
    assert torch.equal(again[1], dbias)

"""Expert layers in a training program: no gradient is lost unseen under
autograd, a torch.autograd.Function made of them is differentiated by their
gradients, and gradients may be written among others."""
import pytest

import test_experts_gpu as base

pytestmark = pytest.mark.gpu


def test_operands_that_require_grad_are_refused(gpu):
    import torch
    x, w, grad, offsets = base._make(torch, [4, 5], 16, 24, torch.bfloat16, 1)
    p = gpu.block8_pack(x)
    tracked = [t.clone().requires_grad_() for t in (x, w, grad)]
    tx, tw, tg = tracked
    calls = [
        lambda: gpu.grouped_matmul(tx, w, offsets),
        lambda: gpu.grouped_matmul(x, tw, offsets),
        lambda: gpu.grouped_matmul(x, tw * 2, offsets),  # not a leaf
        lambda: gpu.grouped_matmul_grad_input(tg, w, offsets),
        lambda: gpu.grouped_matmul_grad_input(grad, tw, offsets),
        lambda: gpu.grouped_matmul_grad_weight(tg, x, offsets),
        lambda: gpu.grouped_matmul_grad_weight(grad, tx, offsets),
        lambda: gpu.grouped_matmul_grad_weight(tg, p, offsets),
        lambda: gpu.grouped_matmul(x, w, offsets, out=tg),
        lambda: gpu.block8_pack(tx),
        lambda: gpu.block8_unpack(p, out=tx),
        lambda: gpu.activation_pack(tx, "gelu"),
        lambda: gpu.activation_grad(tx, p, "gelu"),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="requires grad"):
            call()
        with torch.no_grad():
            call()
    assert all(t.grad is None for t in tracked)


def test_a_function_of_them_is_differentiated(gpu):
    import torch

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, offsets):
            ctx.save_for_backward(x, w, offsets)
            return gpu.grouped_matmul(x, w, offsets)

        @staticmethod
        def backward(ctx, grad):
            x, w, offsets = ctx.saved_tensors
            return (gpu.grouped_matmul_grad_input(grad, w, offsets),
                    gpu.grouped_matmul_grad_weight(grad, x, offsets), None)

    x, w, grad, offsets = base._make(torch, [70, 0, 33], 48, 64, torch.float16, 2)
    x.requires_grad_(), w.requires_grad_()
    Product.apply(x, w, offsets).backward(grad)
    with torch.no_grad():
        assert torch.equal(x.grad, gpu.grouped_matmul_grad_input(grad, w, offsets))
        assert torch.equal(w.grad, gpu.grouped_matmul_grad_weight(grad, x, offsets))


def test_gradients_into_matrices_that_lie_between_one_another(gpu):
    import torch
    x, w, grad, offsets = base._make(torch, [70, 0, 33], 48, 64, torch.bfloat16, 3)
    want = gpu.grouped_matmul_grad_weight(grad, x, offsets)
    between = torch.zeros(48, 3, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    apart = torch.zeros(3, 50, 72, dtype=torch.bfloat16, device="cuda")[:, :48, :64]
    for out in (between, apart):
        gpu.grouped_matmul_grad_weight(grad, x, offsets, out=out)
        assert torch.equal(out, want)
    one = torch.zeros(1, 48, 64, dtype=torch.bfloat16, device="cuda").expand(3, 48, 64)
    with pytest.raises(gpu.ProximaError, match="dw_group_stride"):
        gpu.grouped_matmul_grad_weight(grad, x, offsets, out=one)

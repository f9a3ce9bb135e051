"""Layers whose result is their residual, lies between their operand's rows, or
would lie over the operand."""
import pytest

import test_experts_gpu as base
import test_tokens_gpu as tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(1, 64), (3, 72), (500, 264), (3000, 1024)])
def test_a_layer_s_result_beside_its_operand(gpu, rows, n):
    import torch
    g = base._dev(torch, rows)
    k = n
    hold = torch.zeros(rows, k + n + 8, dtype=torch.bfloat16, device="cuda")
    x, y = hold[:, :k], hold[:, k:k + n]
    x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
    w = (torch.randn(n, k, generator=g, device="cuda") / k ** 0.5).bfloat16()
    want = gpu.grouped_linear(x.clone(), w, activation="silu", residual=x.clone())
    assert torch.equal(gpu.grouped_linear(x, w, activation="silu", residual=x, out=y), want) and torch.equal(y, want)
    # over it: as the residual, one column or one row on
    for out in (x, hold[:, 1:n + 1]) + ((hold.view(-1)[8:8 + n][None],) if rows == 1 else ()):
        before = hold.clone()
        with pytest.raises(gpu.ProximaError):
            gpu.grouped_linear(x, w, activation="silu", residual=x, out=out)
        assert torch.equal(hold, before)
    # the residual itself, which is a copy of x
    r = x.clone()
    assert gpu.grouped_linear(x, w, activation="silu", residual=r, out=r) is r and torch.equal(r, want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,picks,experts,n,hidden", [(1, 1, 4, 64, 72), (8, 2, 3, 2048, 96), (40, 3, 5, 203, 520), (150, 2, 6, 136, 64)])
def test_an_expert_layer_s_result_is_its_input(gpu, rows, picks, experts, n, hidden, dtype):
    import torch
    dtype = getattr(torch, dtype)
    x, ids, gates, w1, up, w2, b1, b2, r = tokens._make(torch, rows, picks, experts, n, hidden, n, dtype, rows)
    want = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", up=up, bias1=b1, bias2=b2, residual=x)
    assert gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", up=up, bias1=b1, bias2=b2, residual=x, out=x) is x
    assert torch.equal(x, want)

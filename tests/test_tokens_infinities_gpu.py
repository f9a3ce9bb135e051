"""expert_layer with infinities that belong to a token, against the formula in 64
bits. (Those of other tokens and experts: test_tokens_gpu.py.)"""
import pytest

import test_experts_gpu as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "packed"])
@pytest.mark.parametrize("rows", [1, 9, 40])
def test_infinities_of_a_token_s_own_experts(gpu, rows, dtype):
    """An infinity in W2, or between the products, makes the sums that it is in infinite, or not a number where the
    formula says so; values that 8 bits hold exactly, whose further planes are empty, are no exception."""
    import torch
    packed, dtype = dtype == "packed", torch.bfloat16 if dtype == "packed" else getattr(torch, dtype)
    k, hidden, n = 8, 24, 40
    g = base._dev(torch, rows)
    x = torch.randint(1, 9, (rows, k), generator=g, device="cuda").to(dtype)
    w1 = torch.zeros(4, hidden, k, device="cuda", dtype=dtype)
    w1[:, torch.arange(hidden), torch.arange(hidden) % k] = 1.0  # a is x, of 4 bits
    w1[:, 5, 5] = 1.0 + 2.0 ** -7                                # and of more, once
    w2 = (0.5 * torch.randint(1, 7, (4, n, hidden), generator=g, device="cuda")).to(dtype)
    huge = torch.finfo(torch.bfloat16).max if packed else float("inf")  # packed, that is 2^128
    w2[0, 3, 2], w2[0, 17, 5], w2[1, 30, 7], w2[1, 31, 6] = huge, -huge, -huge, huge
    w2[2, 20, 1], w2[2, 20, 2] = huge, -huge
    b1 = torch.zeros(4, hidden, device="cuda")
    b1[3, 4], b1[3, 11] = float("inf"), -3.0
    w2[3, 9, 4], w2[3, 10, 4], w2[3, 11, 4], w2[3, 12, 4], w2[3, 13, 4] = 0.0, -1.0, 2.5, huge, -huge
    ids = (3 - torch.arange(rows, device="cuda")[:, None]) % 4
    gates = torch.ones(rows, 1, device="cuda")
    gates[1::4] = -0.5
    m1, m2 = w1, w2
    if packed:
        m1, m2 = (gpu.block8_pack(w.reshape(-1, w.shape[2])) for w in (w1, w2))
        w1, w2 = (gpu.block8_unpack(p, torch.float32).view(w.shape) for p, w in ((m1, w1), (m2, w2)))
        assert bool(torch.isinf(w2).any())
    e = ids[:, 0]
    a = gates.double() * ((w1[e].double() * x[:, None].double()).sum(2) + b1[e].double())
    want = (a[:, None] * w2[e].double()).sum(2)
    inf, nan = torch.isinf(want), torch.isnan(want)
    assert bool(inf.any()) and bool(nan.any())
    # 24 terms of at most 8.1 x 3 (packed, what stands in a block beside 2^128 is less), summed in f32
    bound = 1.25 * 24 * 2.0 ** -24 * 24 * 25
    for out in (dtype, torch.float32):
        got = gpu.expert_layer(x, ids, m1, m2, gates, bias1=b1, out_dtype=out).double()
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[inf], want[inf])
        rest = ~inf & ~nan
        assert bool(((got - want)[rest].abs() <= bound + base._unit(out) * (want[rest].abs() + bound)).all())

"""The 16-bit activations at every finite value of their type, tails included,
relative to the value itself.

Tolerance: the exponentials' arguments reach 90 (SiLU) and 169 / 2 (GELU at 13),
and half a unit of f32 in them is 90 2^-24 = 5.4e-6 of the result; a dozen
roundings and the functions' own ulp are 2^-20 = 9.5e-7 more: 1e-5. Then one
rounding to the type. Results so small that f32's smallest normal number enters
into them (exp or its reciprocal below 2^-126, times |h| below 2^7) may be zero:
2^-119.
"""
import pytest

import test_experts_gpu as base

pytestmark = pytest.mark.gpu


def _all_values(torch, dtype):
    h = torch.arange(-32768, 32768, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    return h[torch.isfinite(h)]


def _tails(torch, h, act):
    """(f, f', the larger of the slope's terms) in 64 bits, without cancellation in the tails."""
    if act == "silu":
        s, c = torch.sigmoid(h), torch.sigmoid(-h)
        return h * s, s * (1 + h * c), s * torch.maximum(torch.ones_like(h), (h * c).abs())
    p = 0.5 * torch.special.erfc(-h / 2.0 ** 0.5)
    d = h * torch.exp(-h * h / 2) / (2 * torch.pi) ** 0.5
    return h * p, p + d, torch.maximum(p, d.abs())


def _within(torch, got, want, terms):
    allowed = 1e-5 * terms + 2.0 ** -119
    unit = base._unit(got.dtype)
    allowed = allowed + unit * (want.abs() + allowed) + (2.0 ** -25 if got.dtype is torch.float16 else 2.0 ** -134)
    off = (got.double() - want).abs()
    return bool((off <= allowed).all()), float((off / allowed).max())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_activations_of_every_value(gpu, act, dtype):
    import torch
    h = _all_values(torch, getattr(torch, dtype))
    h = h.reshape(-1, 1).contiguous()
    a, _ = gpu.activation_pack(h, act)
    f, _, _ = _tails(torch, h.double(), act)
    limit = torch.finfo(a.dtype).max
    fits = f.abs() <= limit
    ok, worst = _within(torch, a[fits], f[fits], f[fits].abs())
    assert ok, worst


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_slopes_of_every_kept_value(gpu, act, dtype):
    # one column: each value alone in its block, kept with four bits
    import torch
    dt = getattr(torch, dtype)
    h = _all_values(torch, dt).reshape(-1, 1).contiguous()
    p = gpu.block8_pack(h)
    kept = gpu.block8_unpack(p, torch.float32).double()
    # magnitudes that round to 2^128 are infinity when unpacked, and nothing else is
    over = torch.isinf(kept)
    assert torch.equal(over, h.double().abs() >= 1.9375 * 2.0 ** 127)
    assert torch.equal(torch.sign(kept[over]), torch.sign(h[over].double()))
    _, slope, terms = _tails(torch, kept, act)
    got = gpu.activation_grad(torch.ones_like(h), p, act)
    ok, worst = _within(torch, got[~over], slope[~over], terms[~over])
    assert ok, worst

"""expert_layer at sizes whose kernels have 2^32 work-items and more, against the
formula in 64 bits with the tolerances of test_tokens_gpu.py."""
import pytest

import test_experts_gpu as base
import test_tokens_gpu as tokens

pytestmark = pytest.mark.gpu


def test_as_many_workgroups_as_the_sizes_allow(gpu):
    # 1024 experts in use of 8192 tiles of W1 each, 512 threads a workgroup
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = tokens._make(torch, 64, 16, 1024, 8, 16, 8, torch.bfloat16, 1)
    hidden = 131072
    g = base._dev(torch, 2)
    ids = torch.randperm(1024, generator=g, device="cuda").view(64, 16)
    w1 = torch.randn(1024, hidden, 8, generator=g, device="cuda", dtype=torch.bfloat16) / 8 ** 0.5
    w2 = torch.randn(1024, 8, hidden, generator=g, device="cuda", dtype=torch.bfloat16) / hidden ** 0.5
    r = r.bfloat16()
    got = gpu.expert_layer(x, ids, w1, w2, gates, activation="silu", bias2=b2, residual=r)
    # the tokens of the first experts, of the middle and of the last
    some = torch.cat([torch.nonzero((ids == e).any(1))[0] for e in (0, 1, 511, 512, 1022, 1023)])
    tokens._check(torch, got[some], tokens._layer64(torch, x[some], ids[some], w1, w2, gates[some], "silu", None, None, b2,
                                                    r[some], torch.bfloat16))


@pytest.mark.parametrize("rows,out", [(3, "bfloat16"), (20, "float32")])
def test_results_as_wide_as_two_launches(gpu, rows, out):
    # 2^22 tiles of 16 columns and some, 1024 threads a workgroup
    import torch
    n, out = (1 << 26) + 41, getattr(torch, out)
    x, ids, gates, w1, up, w2, b1, b2, r = tokens._make(torch, rows, 2, 2, 8, 8, 16, torch.bfloat16, rows)
    w2 = torch.randn(2, n, 8, generator=base._dev(torch, 3), device="cuda", dtype=torch.bfloat16)
    got = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", bias1=b1, out_dtype=out)
    for a in range(0, n, 1 << 24):
        part = slice(a, min(a + (1 << 24), n))
        tokens._check(torch, got[:, part], tokens._layer64(torch, x, ids, w1, w2[:, part], gates, "gelu", None, b1, None,
                                                           None, out))


@pytest.mark.parametrize("packed", [False, True])
def test_as_many_tokens_as_there_may_be(gpu, packed):
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = tokens._make(torch, 65536, 16, 40, 24, 40, 16, torch.bfloat16, 4)
    m1, m2, m3 = w1, w2, up
    if packed:
        m1, m2, m3 = (gpu.block8_pack(w.reshape(-1, w.shape[2])) for w in (w1, w2, up))
        w1, w2, up = (gpu.block8_unpack(p, torch.float32).view(w.shape) for p, w in ((m1, w1), (m2, w2), (m3, up)))
    got = gpu.expert_layer(x, ids, m1, m2, gates, activation="gelu", up=m3, bias1=b1, bias2=b2)
    tokens._check(torch, got, tokens._layer64(torch, x, ids, w1, w2, gates, "gelu", up, b1, b2, None, torch.bfloat16))

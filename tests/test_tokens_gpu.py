"""expert_layer against the formula in 64 bits.

Tolerances. A first product of k terms, with its bias, is off by e1 = 1.25 (k + 1)
2^-24 S1, S1 the sum of its terms' magnitudes (test_experts_gpu.py). The
activation's slope is at most 1.13, its evaluation off by 2^-20 of |h| (f32
results) or 2^-16 of f(h) and 2^-22 of |h| (16 bits). a = g f(h) up takes that
times |g up| and f's magnitude times |g| up's error, three roundings of 2^-24, and
what its planes lose: 2^-17 for 16-bit results, nothing for f32. The second product
adds up all experts' and hidden columns' terms, at most `used` hidden of them, each
off by a's error times |w2|, and 1.25 terms 2^-24 of the terms' magnitudes; biases,
gates and the residual are a few terms more. Then one rounding to the result's type.
"""
import pytest

import test_experts_gpu as base
from test_linear_gpu import _act64, _half

pytestmark = pytest.mark.gpu


def _layer64(torch, x, ids, w1, w2, gates, act, up, b1, b2, residual, out_dtype):
    """(y, how far off it may be) in 64 bits; an id outside the experts is none."""
    rows, picks = ids.shape
    experts, hidden, k = w1.shape
    n = w2.shape[1]
    y = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
    off, size, terms = y.clone(), y.clone(), torch.zeros(rows, 1, dtype=torch.float64, device="cuda")
    fine = out_dtype is torch.float32
    gates = gates.double()
    for e in range(experts):
        hit = ids == e
        token = torch.nonzero(hit.any(1))[:, 0]
        if token.numel() == 0:
            continue
        g = (torch.where(hit, gates, 0.0).sum(1))[token][:, None]
        gs = (torch.where(hit, gates.abs(), 0.0).sum(1))[token][:, None]
        xe = x[token].double()
        m = w1[e].double().t().contiguous()
        h, hs = xe @ m, xe.abs() @ m.abs()
        if b1 is not None:
            h, hs = h + b1[e].double(), hs + b1[e].double().abs()
        e1 = 1.25 * (k + 1) * 2.0 ** -24 * hs
        a = _act64(torch, h, act)
        ea = e1 if act is None else 1.13 * e1 + (2.0 ** -20 * h.abs() if fine else 2.0 ** -16 * a.abs() + 2.0 ** -22 * h.abs())
        if up is not None:
            m = up[e].double().t().contiguous()
            u, eu = xe @ m, 1.25 * k * 2.0 ** -24 * (xe.abs() @ m.abs())
            a, ea = a * u, ea * (u.abs() + eu) + a.abs() * eu
        ea = gs * ea + (gs + picks * gs) * 2.0 ** -23 * a.abs()
        a = g * a
        ea = ea + (0.0 if fine else 2.0 ** -17) * (a.abs() + ea)
        m = w2[e].double().t().contiguous()
        y[token] += a @ m
        off[token] += ea @ m.abs()
        size[token] += (a.abs() + ea) @ m.abs()
        terms[token] += hidden
        if b2 is not None:
            y[token] += g * b2[e].double()
            size[token] += gs * b2[e].double().abs()
            terms[token] += 2 * picks
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    off = off + 1.25 * (terms + 2) * 2.0 ** -24 * size
    return y, off


def _check(torch, got, want):
    y, off = want
    bound = off + base._unit(got.dtype) * (y.abs() + off) + _half(got.dtype)
    bad = (got.double() - y).abs() > bound
    assert not bool(bad.any()), float(((got.double() - y).abs() / bound.clamp(min=1e-300)).max())


def _make(torch, rows, picks, experts, k, hidden, n, dtype, seed, spread=True):
    g = base._dev(torch, seed)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    w1 = (torch.randn(experts, hidden, k, generator=g, device="cuda") / k ** 0.5).to(dtype)
    up = (torch.randn(experts, hidden, k, generator=g, device="cuda") / k ** 0.5).to(dtype)
    w2 = (torch.randn(experts, n, hidden, generator=g, device="cuda") / hidden ** 0.5).to(dtype)
    ids = torch.rand(rows, experts, generator=g, device="cuda").topk(min(picks, experts), 1)[1]
    if picks > experts:
        ids = torch.randint(0, experts, (rows, picks), generator=g, device="cuda")
    gates = torch.rand(rows, picks, generator=g, device="cuda")
    b1 = torch.randn(experts, hidden, generator=g, device="cuda")
    b2 = torch.randn(experts, n, generator=g, device="cuda")
    return x, ids.contiguous(), gates, w1, up, w2, b1, b2, torch.randn(rows, n, generator=g, device="cuda")


SIZES = [  # rows, picks, experts, k, hidden, n
    (1, 1, 1, 1, 1, 1), (1, 1, 8, 128, 256, 128), (1, 8, 64, 64, 64, 64), (2, 3, 5, 72, 130, 40), (16, 2, 4, 200, 96, 301),
    (17, 1, 1, 203, 77, 33), (31, 4, 40, 1000, 520, 260), (33, 2, 3, 520, 1100, 17), (64, 8, 8, 65, 63, 129),
    (64, 1, 2, 256, 136, 264), (65, 2, 6, 136, 264, 72), (150, 5, 70, 99, 101, 103), (5, 16, 300, 64, 80, 96),
    (8, 2, 16, 2048, 512, 256), (3, 4, 2, 40, 48, 56), (130, 16, 9, 48, 64, 40),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_layers_of_few_tokens(gpu, case, gated, dtype):
    import torch
    dtype = getattr(torch, dtype)
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, *SIZES[case], dtype, case)
    up = up if gated else None
    for i, out in enumerate((dtype, torch.float32)):
        act = [None, "silu", "gelu"][(case + i) % 3]
        b1_, b2_ = [(None, None), (b1, b2), (b1.to(dtype), None), (None, b2.to(dtype))][(case + 2 * i + gated) % 4]
        r_ = r.to(out) if (case + i) % 2 else None
        got = gpu.expert_layer(x, ids, w1, w2, gates, activation=act, up=up, bias1=b1_, bias2=b2_, residual=r_, out_dtype=out)
        assert got.dtype is out
        _check(torch, got, _layer64(torch, x, ids, w1, w2, gates, act, up, b1_, b2_, r_, out))
        assert torch.equal(got, gpu.expert_layer(x, ids, w1, w2, gates, activation=act, up=up, bias1=b1_, bias2=b2_,
                                                 residual=r_, out_dtype=out))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_packed_layers_of_few_tokens(gpu, case, gated):
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, *SIZES[case], torch.bfloat16, 50 + case)
    p1, p2, p3 = (gpu.block8_pack(w.reshape(-1, w.shape[2])) for w in (w1, w2, up))
    v1, v2, v3 = (gpu.block8_unpack(p, torch.float32).view(w.shape) for p, w in ((p1, w1), (p2, w2), (p3, up)))
    for i, out in enumerate((torch.bfloat16, torch.float32)):
        act = [None, "silu", "gelu"][(case + i) % 3]
        b1_, b2_ = [(None, None), (b1, b2)][(case + i) % 2]
        got = gpu.expert_layer(x, ids, p1, p2, gates, activation=act, up=p3 if gated else None, bias1=b1_, bias2=b2_,
                               residual=r.to(out), out_dtype=out)
        _check(torch, got, _layer64(torch, x, ids, v1, v2, gates, act, v3 if gated else None, b1_, b2_, r.to(out), out))


def test_ids_that_are_no_expert_s_and_ids_twice(gpu):
    import torch
    for seed, dtype in enumerate((torch.bfloat16, torch.float16)):
        x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 40, 4, 7, 136, 200, 72, dtype, 70 + seed)
        big = 1 << 40
        ids[0] = torch.tensor([-1, 7, big, -big], device="cuda")       # none
        ids[1] = torch.tensor([3, 3, 3, 3], device="cuda")             # one, four times
        ids[2] = torch.tensor([-1, 6, 6, 8], device="cuda")
        ids[3] = torch.tensor([(1 << 32) + 1, 0, -1, -1], device="cuda")
        r = r.to(dtype)
        got = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", up=up, bias1=b1, bias2=b2, residual=r)
        _check(torch, got, _layer64(torch, x, ids, w1, w2, gates, "gelu", up, b1, b2, r, dtype))
        assert torch.equal(got[0], r[0])
        none = gpu.expert_layer(x, torch.full_like(ids, -1), w1, w2, gates, bias1=b1, bias2=b2)
        assert not bool(none.any())


def test_far_values_between_the_products(gpu):
    # what is between the products passes f16's range both ways, the results do not
    import torch
    g = base._dev(torch, 5)
    for scale in (2.0 ** -20, 2.0 ** 18):
        x = torch.randn(6, 64, generator=g, device="cuda").half()
        w1 = torch.randn(3, 80, 64, generator=g, device="cuda").half()
        up = torch.randn(3, 80, 64, generator=g, device="cuda").half()
        w2 = (torch.randn(3, 40, 80, generator=g, device="cuda") * 2.0 ** -8).half()
        gates = torch.full((6, 2), scale, device="cuda")
        ids = torch.randint(0, 3, (6, 2), generator=g, device="cuda")
        for out in (torch.float16, torch.float32):
            got = gpu.expert_layer(x, ids, w1, w2, gates, activation="silu", up=up, out_dtype=out)
            want = _layer64(torch, x, ids, w1, w2, gates, "silu", up, None, None, None, out)
            if out is torch.float32 or scale < 1.0:
                _check(torch, got, want)
            else:
                over = want[0].abs() > 65520.0 + want[1]
                assert bool(torch.isinf(got[over]).all()) and bool(over.any())


@pytest.mark.parametrize("packed", [False, True])
def test_other_tokens_experts_keep_out(gpu, packed):
    # NaN and infinities in a token's row, its gates and its experts reach no token that has none of them
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 40, 2, 8, 128, 136, 80, torch.bfloat16, 6)
    ids = ids % 6
    ids[7], ids[20] = 6, 7
    ids[21] = torch.tensor([1, -1], device="cuda")

    def run():
        m = [gpu.block8_pack(w.reshape(-1, w.shape[2])) if packed else w for w in (w1, w2, up)]
        return gpu.expert_layer(x, ids, m[0], m[1], gates, activation="gelu", up=m[2], bias1=b1, bias2=b2,
                                residual=r, out_dtype=torch.float32)

    clean = run()
    w1[6], w2[6], up[6], b1[6], b2[6] = float("inf"), float("nan"), float("-inf"), float("nan"), float("inf")
    w2[7] = float("inf")
    x[33], gates[34] = float("nan"), float("inf")
    gates[21, 1] = float("nan")  # of no expert
    dirty = run()
    hurt = torch.zeros(40, dtype=torch.bool, device="cuda")
    hurt[[7, 20, 33, 34]] = True
    assert torch.equal(clean[~hurt], dirty[~hurt])
    assert not bool(torch.isfinite(dirty[hurt]).any())


def test_strided_operands_and_a_residual_in_place(gpu):
    import torch
    for seed, (k, hidden, n) in enumerate(((128, 136, 80), (129, 77, 45))):
        x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 20, 3, 6, k, hidden, n, torch.bfloat16, 80 + seed)
        for pad in (1, 3, 8):
            def wide(t):
                fill = 0 if t.dtype is torch.int64 else float("nan")
                b = torch.full((*t.shape[:-1], t.shape[-1] + pad), fill, dtype=t.dtype, device="cuda")
                b[..., :t.shape[-1]] = t
                return b[..., :t.shape[-1]]

            held = torch.full((20, n + pad), 3.0, dtype=torch.bfloat16, device="cuda")
            held[:, :n] = r.bfloat16()
            got = gpu.expert_layer(wide(x), wide(ids), wide(w1), wide(w2), wide(gates), activation="gelu", up=wide(up),
                                   bias1=wide(b1), bias2=wide(b2), residual=held[:, :n], out=held[:, :n])
            _check(torch, got, _layer64(torch, x, ids, w1, w2, gates, "gelu", up, b1, b2, r.bfloat16(), torch.bfloat16))
            assert got.data_ptr() == held.data_ptr() and bool((held[:, n:] == 3.0).all())
        # every other row; experts that lie between one another
        some = torch.zeros(40, k, dtype=x.dtype, device="cuda")
        some[::2] = x
        between = w1.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(gpu.expert_layer(some[::2], ids, between, w2, gates), gpu.expert_layer(x, ids, w1, w2, gates))


def test_the_layer_is_what_the_grouped_layers_make(gpu):
    # routing, both products, gates and the sum over picks by the batch's operators
    import torch
    x, ids, gates, w1, _, w2, b1, b2, r = _make(torch, 48, 2, 10, 256, 320, 192, torch.bfloat16, 7)
    order = torch.sort(ids.reshape(-1), stable=True)[1]
    offsets = torch.searchsorted(ids.reshape(-1)[order], torch.arange(11, device="cuda"))
    a = gpu.grouped_linear(x[order // 2], w1, offsets, bias=b1, activation="gelu")
    z = gpu.grouped_linear(a, w2, offsets, bias=b2, out_dtype=torch.float32)
    want = r.clone().index_add_(0, order // 2, z * gates.reshape(-1)[order][:, None])
    got = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", bias1=b1, bias2=b2, residual=r,
                           out_dtype=torch.float32)
    # the grouped layers round a to bf16: half a step of 2^-8 of each of 2 x 320 terms
    _, off = _layer64(torch, x, ids, w1, w2, gates, "gelu", None, b1, b2, r, torch.float32)
    terms = torch.zeros_like(got, dtype=torch.float64)
    for g, (lo, hi) in enumerate(zip(offsets.tolist()[:-1], offsets.tolist()[1:])):
        m = w2[g].double().abs().t().contiguous()
        terms.index_add_(0, (order // 2)[lo:hi], (a[lo:hi].double().abs() @ m) * gates.reshape(-1)[order][lo:hi, None])
    assert bool(((got.double() - want.double()).abs() <= 3 * off + 2.0 ** -8 * 1.01 * terms + 2.0 ** -20).all())


def test_tokens_in_a_graph_and_on_another_stream(gpu):
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 24, 2, 12, 256, 512, 128, torch.bfloat16, 8)

    def step():
        y = gpu.expert_layer(x, ids, w1, w2, gates, activation="silu", up=up, bias2=b2, residual=x[:, :128].contiguous())
        return [y, gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", bias1=b1, out_dtype=torch.float32)]

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
        fx, fi, fg, *_ = _make(torch, 24, 2, 12, 256, 512, 128, torch.bfloat16, 20 + seed)
        x.copy_(fx), ids.copy_(fi if seed else torch.full_like(fi, -1)), gates.copy_(fg)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_matrices_and_rows_past_4_gb(gpu):
    # experts 6 GB apart, rows millions of elements apart; many experts, of which the last are in use
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 5, 2, 3, 64, 128, 48, torch.bfloat16, 9)
    want = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", residual=r.bfloat16())

    def apart(t, far):
        m = t.reshape(-1, t.shape[-1])
        hold = torch.zeros(m.shape[0] * far, dtype=t.dtype, device="cuda").view(m.shape[0], far)[:, :m.shape[1]]
        hold.copy_(m)
        return hold if t.dim() == 2 else hold.as_strided(t.shape, (t.shape[1] * far, far, 1))

    far = 1 << 22
    got = gpu.expert_layer(apart(x, far), apart(ids, 99), apart(w1, far), apart(w2, far), apart(gates, 77),
                           activation="gelu", residual=apart(r.bfloat16(), far), out=apart(torch.zeros_like(r).bfloat16(), far))
    assert torch.equal(got, want)
    del got
    torch.cuda.empty_cache()
    many = 65536
    big1 = torch.zeros(many, 128, 64, dtype=torch.bfloat16, device="cuda")
    big2 = torch.zeros(many, 48, 128, dtype=torch.bfloat16, device="cuda")
    big1[-3:], big2[-3:] = w1, w2
    assert torch.equal(gpu.expert_layer(x, ids + many - 3, big1, big2, gates, activation="gelu", residual=r.bfloat16()), want)


def test_rows_past_a_block_of_tokens(gpu):
    # each block of 64 tokens for itself: the same rows give the same results wherever they are
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 64, 2, 6, 72, 88, 40, torch.bfloat16, 10)
    one = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", bias1=b1, bias2=b2, out_dtype=torch.float32)
    many = gpu.expert_layer(x.repeat(40, 1), ids.repeat(40, 1), w1, w2, gates.repeat(40, 1), activation="gelu", bias1=b1,
                            bias2=b2, out_dtype=torch.float32)
    want = _layer64(torch, x, ids, w1, w2, gates, "gelu", None, b1, b2, None, torch.float32)
    _check(torch, one, want)
    for i in range(40):
        _check(torch, many[64 * i:64 * i + 64], want)
    assert gpu.expert_layer(x[:0], ids[:0], w1, w2, gates[:0]).shape == (0, 40)


def test_tokens_refuse(gpu):
    import torch
    x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, 4, 2, 3, 16, 24, 8, torch.bfloat16, 11)
    p1, p2 = gpu.block8_pack(w1.reshape(-1, 16)), gpu.block8_pack(w2.reshape(-1, 24))
    f, mismatch = gpu.expert_layer, gpu.DimensionMismatch
    for call, error in [
        (lambda: f(x.float(), ids, w1, w2, gates), ValueError),
        (lambda: f(x.half(), ids, w1, w2, gates), ValueError),
        (lambda: f(x, ids.int(), w1, w2, gates), ValueError),
        (lambda: f(x, ids[:3], w1, w2, gates), mismatch),
        (lambda: f(x, ids, w1, w2, gates[:, :1]), mismatch),
        (lambda: f(x, ids, w1, w2, gates.double()), ValueError),
        (lambda: f(x, ids.repeat(1, 9), w1, w2, gates.repeat(1, 9)), gpu.ProximaError),
        (lambda: f(x, ids, w1[:2], w2, gates), mismatch),
        (lambda: f(x, ids, w1, w2[:, :, :9], gates), mismatch),
        (lambda: f(x[:, :9], ids, w1, w2, gates), mismatch),
        (lambda: f(x, ids, w1, w2, gates, up=up[:, :9]), mismatch),
        (lambda: f(x, ids, w1, w2, gates, up=p1), ValueError),
        (lambda: f(x, ids, p1, w2, gates), ValueError),
        (lambda: f(x, ids, p1, p2, gates, up=up), ValueError),
        (lambda: f(x.half(), ids, p1, p2, gates), ValueError),
        (lambda: f(x, ids, gpu.block8_pack(w1.reshape(-1, 16)[:70]), p2, gates), mismatch),
        (lambda: f(x, ids, p1, gpu.block8_pack(w2.reshape(-1, 24)[:23]), gates), mismatch),
        (lambda: f(x, ids, w1, w2, gates, activation="relu"), ValueError),
        (lambda: f(x, ids, w1, w2, gates, bias1=b1[:, :9]), mismatch),
        (lambda: f(x, ids, w1, w2, gates, bias1=b1, bias2=b2.bfloat16()), ValueError),
        (lambda: f(x, ids, w1, w2, gates, bias2=b2.half()), ValueError),
        (lambda: f(x, ids, w1, w2, gates, residual=r), ValueError),
        (lambda: f(x, ids, w1, w2, gates, residual=r[:3], out_dtype=torch.float32), mismatch),
        (lambda: f(x, ids, w1, w2, gates, out_dtype=torch.float16), gpu.ProximaError),
        (lambda: f(x, ids, w1, w2, gates, out=torch.zeros(4, 9, device="cuda")), mismatch),
        (lambda: f(x, ids, w1, w2, gates.clone().requires_grad_()), ValueError),
        (lambda: f(x, ids, w1.clone().requires_grad_(), w2, gates), ValueError),
        (lambda: f(x, ids, w1, w2, gates, bias1=b1.clone().requires_grad_()), ValueError),
        (lambda: f(x, ids.cpu(), w1, w2, gates), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_two_streams_at_once_and_a_residual_in_place_of_a_sliced_sum(gpu):
    import torch
    a, b = (_make(torch, rows, 2, 16, 256, 2048, 256, torch.bfloat16, 40 + rows) for rows in (9, 40))
    runs = []
    for x, ids, gates, w1, up, w2, b1, b2, r in (a, b):
        def run(out, x=x, ids=ids, gates=gates, w1=w1, up=up, w2=w2, b1=b1, b2=b2, r=r):
            out.copy_(r)
            return gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", up=up, bias1=b1, bias2=b2, residual=out, out=out)
        want = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", up=up, bias1=b1, bias2=b2,
                                residual=r.bfloat16())
        _check(torch, want, _layer64(torch, x, ids, w1, w2, gates, "gelu", up, b1, b2, r.bfloat16(), torch.bfloat16))
        runs.append((run, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        held = []
        for _ in range(6):
            for run, want, stream in runs:
                with torch.cuda.stream(stream):
                    held.append((run(torch.empty_like(want)), want))
        torch.cuda.synchronize()
        for got, want in held:
            assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 16, 21, 32, 33, 70])
@pytest.mark.parametrize("n", [2040, 2048, 2500, 4096, 4101])
def test_every_shape_of_the_second_product(gpu, rows, n):
    # 8 or 16 rows of a matrix to a workgroup, 8 or 16 wavefronts, with slices or not
    import torch
    for i, dtype in enumerate((torch.bfloat16, torch.float16)):
        hidden = (200, 331)[(rows + i) % 2]
        x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, rows, 3, 7, 72, hidden, n, dtype, rows + n)
        w2[6] = float("inf")  # another token's
        ids[ids == 6] = -1
        ids[-1] = 6
        out = (dtype, torch.float32)[(rows + n + i) % 2]
        got = gpu.expert_layer(x, ids, w1, w2, gates, activation="gelu", bias2=b2, residual=r.to(out), out_dtype=out)
        fine = w2.clone()
        fine[6] = 0.0
        y, off = _layer64(torch, x, ids, w1, fine, gates, "gelu", None, None, b2, r.to(out), out)
        _check(torch, got[:-1], (y[:-1], off[:-1]))
        assert not bool(torch.isfinite(got[-1]).any())
        if i == 0:
            p1, p2 = gpu.block8_pack(w1.reshape(-1, 72)), gpu.block8_pack(fine.reshape(-1, hidden))
            v1 = gpu.block8_unpack(p1, torch.float32).view(w1.shape)
            v2 = gpu.block8_unpack(p2, torch.float32).view(w2.shape)
            got = gpu.expert_layer(x, ids, p1, p2, gates, activation="silu", out_dtype=out)
            _check(torch, got, _layer64(torch, x, ids, v1, v2, gates, "silu", None, None, None, None, out))


def test_the_example_serves_a_few_queries_as_a_batch(gpu):
    import importlib.util
    import os

    import torch
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_adapters.py")
    spec = importlib.util.spec_from_file_location("expert_adapters", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    g = base._dev(torch, 3)
    x = torch.randn(300, 128, generator=g, device="cuda")
    router = example.Router(x, 8, 2)
    w1 = torch.randn(8, 256, 128, generator=g, device="cuda") / 128 ** 0.5
    w2 = torch.randn(8, 128, 256, generator=g, device="cuda") / 256 ** 0.5
    packed = tuple(gpu.block8_pack(w.reshape(-1, w.shape[2])) for w in (w1, w2))
    few = torch.cat([example.serve_few(router, packed, x[i:i + 7].contiguous()) for i in range(0, 300, 7)])
    v1, v2 = (gpu.block8_unpack(p, torch.float32).view(w.shape) for p, w in zip(packed, (w1, w2)))
    ids, ones = router.cells(x), torch.ones(300, 1, device="cuda")
    _check(torch, few, _layer64(torch, x.bfloat16(), ids, v1, v2, ones, "gelu", None, None, None, x, torch.float32))
    # the batch packs its rows in 8 bits twice: half a step of 2^-3 each
    batch = example.serve(router, packed, x)
    assert float((few - batch).norm() / (batch - x).norm()) < 2 * 2.0 ** -4


def test_rows_that_begin_between_words(gpu):
    # every operand at an odd element of its storage, by itself and together; what lies around them is not a number
    import torch

    def shifted(t, by):
        hold = torch.full((t.numel() + 2 * by + 8,), 0 if t.dtype is torch.int64 else float("nan"), dtype=t.dtype, device="cuda")
        v = hold[by:by + t.numel()].view(t.shape)
        return v.copy_(t)

    for rows, k, hidden, n in ((5, 64, 72, 40), (20, 65, 33, 2049), (3, 1001, 130, 7), (40, 128, 127, 4096)):
        x, ids, gates, w1, up, w2, b1, b2, r = _make(torch, rows, 2, 4, k, hidden, n, torch.float16, rows)
        for which in range(5):
            on = [shifted(t, 1) if which in (i, 4) else t for i, t in enumerate((x, w1, w2, up))]
            rr = shifted(r.half(), 3)
            got = gpu.expert_layer(on[0], ids, on[1], on[2], gates, activation="gelu", up=on[3], bias1=shifted(b1, 1),
                                   bias2=shifted(b2, 1), residual=rr, out=shifted(torch.zeros_like(rr), 1))
            _check(torch, got, _layer64(torch, x, ids, w1, w2, gates, "gelu", up, b1, b2, rr, torch.float16))
            h = gpu.grouped_linear(on[0], on[1][1], bias=shifted(b1[1].contiguous(), 1), activation="silu")
            want = x.double() @ w1[1].double().t().contiguous() + b1[1].double()
            size = x.double().abs() @ w1[1].double().abs().t().contiguous() + b1[1].double().abs()
            want, err = _act64(torch, want, "silu"), 1.13 * 1.25 * (k + 1) * 2.0 ** -24 * size + 2.0 ** -16 * size
            bound = err + 2.0 ** -11 * (want.abs() + err) + 2.0 ** -25
            assert bool(((h.double() - want).abs() <= bound).all())

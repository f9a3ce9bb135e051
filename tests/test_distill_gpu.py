"""distill_loss and its gradient against the formula in 64 bits.

Tolerances. Logits are exact inputs; d = x - max is rounded once (2^-24 of |d|).
exp(d / T) is off by 2^-22 of itself and, of the exponent's rounding, by 2^-23
|d| / T (1 + log2 e): its scaled form is corrected in f32; for 16-bit logits the
product's own rounding, 2^-24 log2 e |d| / T, stays. A row's sum adds at most
ceil(cols / 64) + 40 such terms in a chain, each addition off by 2^-24 of it. Hence
q is off by r_q = 2^-21 + 2^-22 (|d| / T + 1) * 2 + (cols / 64 + 40) 2^-24 of itself
for the largest |d| that counts, and log q by that; p alike with `top` terms. dx is
k (q - p), one rounding of each, and to its type.
"""
import math

import pytest

import test_experts_gpu as base

pytestmark = pytest.mark.gpu

INF = float("inf")


def _exact(torch, x, ids, scores, counts, t, weight=None):
    """(loss, its bound, dx, its bound) in 64 bits."""
    rows, cols = x.shape
    x32 = x.dtype is torch.float32
    top = ids.shape[1]
    x, s = x.double() / t, scores.double() / t
    at = torch.arange(top, device="cuda")
    valid = (at < counts[:, None].clamp(0, top)) & (ids >= 0) & (ids < cols)
    s = torch.where(valid, s, -INF)
    best = s.amax(1, keepdim=True)
    some = best > -INF
    ds = torch.where(s == -INF, 0.0, s - torch.where(some, best, 0.0))
    p = torch.where(s == -INF, 0.0, torch.exp(ds))
    mass = torch.where(some, p.sum(1, keepdim=True), 1.0)
    p, logp = p / mass, ds - torch.log(mass)
    m = x.amax(1, keepdim=True)
    m0 = torch.where(m == -INF, 0.0, m)
    e = torch.exp(x - m0)
    total = e.sum(1, keepdim=True)
    q = torch.where(total > 0, e / torch.where(total > 0, total, 1.0), 0.0)
    here = torch.where(valid, ids, 0)
    dx_here = torch.gather(x, 1, here) - m0
    logq = dx_here - torch.log(torch.where(total == 0, 1.0, total))
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)

    def relative(d, terms):  # |d| / T
        return 2.0 ** -21 + 2.0 ** -21 * (d.abs() + 1.0) + (terms / 64 + 40) * 2.0 ** -24

    finite = torch.where(torch.isfinite(x), x, m0)
    rq = relative(finite - m0, cols) + (0.0 if x32 else 2.0 ** -17)
    # the sum's own relative error: that of its terms, weighted
    rsum = torch.where(total > 0, (q * rq).sum(1, keepdim=True), 0.0)
    rp = relative(ds, top * 64)
    rmass = (p * rp).sum(1, keepdim=True)
    off_p = p * (rp + rmass)
    lq = torch.where(p > 0, logq.clamp(-1e30, 1e30), 0.0)
    off_loss = (off_p * (logp.abs() + lq.abs()) +
                p * (rp + rmass + relative(torch.where(p > 0, dx_here.clamp(-1e30, 1e30), 0.0), cols) + rsum +
                     2.0 ** -22 * (logp.abs() + lq.abs()))).sum(1) + (top + 8) * 2.0 ** -24 * (p * (logp.abs() + lq.abs())).sum(1)
    if weight is None:
        return loss, off_loss, None, None
    ps = torch.zeros_like(x).scatter_add_(1, here, torch.where(valid, p, 0.0))
    offs = torch.zeros_like(x).scatter_add_(1, here, torch.where(valid, off_p + top * 2.0 ** -24 * p, 0.0))
    k = weight.double()[:, None] / t
    alive = some.double()
    dx = k * (q - ps) * alive
    # exponentials below f32's normal range, 2^-126, are zeros: of a sum of at least 1, q is off by that
    off = k.abs() * (q * (rq + rsum) + offs + 2.0 ** -22 * (q + ps) + 2.0 ** -126) * alive
    return loss, off_loss, dx, off


def _check(torch, got, want, off):
    unit = base._unit(got.dtype)
    tiny = {2.0 ** -11: 2.0 ** -25, 2.0 ** -8: 2.0 ** -133, 2.0 ** -24: 2.0 ** -126}[unit]
    same = got.double() == want  # infinities
    bound = off + unit * (want.abs() + off) + tiny
    bad = ((got.double() - want).abs() > bound) & ~same
    assert not bool(bad.any()) and not bool(torch.isnan(got).any()), float(
        ((got.double() - want).abs() / bound)[~same].max())


def _make(torch, rows, cols, top, dtype, t, seed, masked=0.05):
    g = base._dev(torch, seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * 2.0 * t
    x[torch.rand(rows, cols, generator=g, device="cuda") < masked] = -INF
    scores = torch.randn(rows, top, generator=g, device="cuda") * 2.0 * t
    ids = torch.stack([torch.randperm(cols, generator=g, device="cuda")[:top] if top <= cols else
                       torch.randint(0, cols, (top,), generator=g, device="cuda") for _ in range(rows)])
    counts = torch.randint(-1, top + 3, (rows,), generator=g, device="cuda").int()
    weight = torch.randn(rows, generator=g, device="cuda")
    return x.to(dtype), ids, scores, counts, weight


def _both(torch, px, x, ids, scores, counts, weight, t):
    loss, off, dx, off_dx = _exact(torch, x, ids, scores, counts, t, weight)
    one = px.distill_loss(x, ids, scores, counts, temperature=t)
    _check(torch, one, loss, off)
    got, grad = px.distill_loss_grad(weight, x, ids, scores, counts, temperature=t)
    assert grad.dtype is x.dtype
    _check(torch, got, loss, off)
    _check(torch, grad, dx, off_dx)
    return got, grad


SIZES = [  # rows, cols, top
    (1, 1, 1), (3, 2, 5), (5, 7, 3), (9, 63, 10), (4, 255, 64), (70, 1000, 10), (5, 1024, 65), (2, 2050, 200), (6, 4093, 1),
    (140, 5000, 33), (130, 8190, 7), (3, 9000, 100), (129, 16390, 12), (5, 33000, 40), (2, 70001, 300), (130, 32760, 9),
    (128, 50000, 20), (1, 1_000_003, 17), (133, 66000, 4), (2, 300, 4096),
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_distillation(gpu, case, dtype):
    import torch
    t = [1.0, 0.05, 2.0][case % 3]
    _both(torch, gpu, *_make(torch, *SIZES[case], getattr(torch, dtype), t, case), t)


@pytest.mark.parametrize("cols", [40, 3000, 9001])
def test_rows_that_have_little(gpu, cols):
    # no entries; scores of -inf; logits of -inf, everywhere or at the entries; ids that are no column's or come twice
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        x, ids, scores, counts, weight = _make(torch, 12, cols, 8, dtype, 1.0, cols, 0.0)
        counts[:] = 8
        counts[0], counts[1], counts[2], counts[3] = 0, -7, 100, 1
        scores[4] = -INF
        scores[5, ::2] = -INF
        x[6] = -INF
        x[7] = -INF
        counts[7] = 0
        x[8, ids[8, 3]] = -INF
        ids[9] = ids[9, 0]
        ids[10] = torch.tensor([-1, cols, 1 << 40, -(1 << 40), (1 << 32) + 1, 3, 3, 5], device="cuda")
        ids[11] = -1
        loss, grad = _both(torch, gpu, x, ids, scores, counts, weight, 1.0)
        for row in (0, 1, 4, 7, 11):
            assert float(loss[row]) == 0.0 and not bool(grad[row].any())
        assert float(loss[6]) == INF and float(loss[8]) == INF
        # an entry of p = 0 at a logit of -inf adds nothing
        scores[8, 3] = -INF
        _both(torch, gpu, x, ids, scores, counts, weight, 1.0)
        assert bool(torch.isfinite(gpu.distill_loss(x, ids, scores, counts)[8]))


def test_only_a_row_s_own_not_a_numbers(gpu):
    import torch
    for rows, cols in ((6, 300), (140, 12000), (3, 40000)):
        x, ids, scores, counts, weight = _make(torch, rows, cols, 5, torch.bfloat16, 1.0, cols)
        counts[:] = 5
        clean = gpu.distill_loss_grad(weight, x, ids, scores, counts)
        x[1, 17], scores[2, 4] = float("nan"), float("nan")
        dirty = gpu.distill_loss_grad(weight, x, ids, scores, counts)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[1:3] = False
        for a, b in zip(clean, dirty):
            assert torch.equal(a[keep], b[keep])
        assert bool(torch.isnan(dirty[0][1:3]).all()) and bool(torch.isnan(dirty[1][1]).all())
        # unused entries are not looked at
        counts[:] = 3
        few = gpu.distill_loss_grad(weight, x, ids, scores, counts)
        assert bool(torch.isfinite(few[0][2])) and bool(torch.isfinite(few[1][2].float()).all())


@pytest.mark.parametrize("rows,cols", [(5, 300), (130, 9000), (3, 20011)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_far_logits_and_temperatures(gpu, rows, cols, dtype):
    import torch
    dtype = getattr(torch, dtype)
    for scale, t in ((1000.0, 1.0), (1e-3, 1e-4), (30000.0, 1e3), (1.0, 1e6), (3.0, 0.01)):
        x, ids, scores, counts, weight = _make(torch, rows, cols, 6, torch.float32, 1.0, int(t * 100) + cols, 0.01)
        x = (x.clamp(-2, 2) / 2.0 * scale).to(dtype)
        _both(torch, gpu, x, ids, scores * scale / 8.0, counts, weight, t)


def test_gradient_against_differences(gpu):
    # of the loss in f32: (l(x + d) - l(x - d)) / 2 d is off by d^2 / 6 times the third derivative in one logit, at
    # most 1 / 4 T^3, and by the losses' own bounds over d
    import torch
    rows, cols, top, t, d = 4, 90, 6, 1.5, 2.0 ** -5
    x, ids, scores, counts, weight = _make(torch, rows, cols, top, torch.float32, t, 3, 0.0)
    counts[:] = torch.tensor([6, 3, 0, 1], device="cuda")
    _, dx = gpu.distill_loss_grad(weight, x, ids, scores, counts, temperature=t)
    _, off, _, _ = _exact(torch, x, ids, scores, counts, t)
    for c in list(range(0, cols, 7)) + ids[0].tolist():
        up, down = x.clone(), x.clone()
        up[:, c] += d
        down[:, c] -= d
        width = up[:, c].double() - down[:, c].double()
        slope = (gpu.distill_loss(up, ids, scores, counts, temperature=t).double() -
                 gpu.distill_loss(down, ids, scores, counts, temperature=t).double()) / width
        bound = d * d / 6.0 / 4.0 / t ** 3 + 2.5 * off / d + 2.0 ** -20
        assert bool(((dx[:, c].double() - weight.double() * slope).abs() <= weight.double().abs() * bound + 2.0 ** -20).all())


def test_strided_in_place_and_not_aligned(gpu):
    import torch
    for rows, cols in ((6, 301), (130, 5003), (129, 40001), (4, 40003)):
        for dtype in (torch.float32, torch.bfloat16):
            x, ids, scores, counts, weight = _make(torch, rows, cols, 5, dtype, 1.0, cols)
            want = gpu.distill_loss_grad(weight, x, ids, scores, counts)
            loss, off, dx, off_dx = _exact(torch, x, ids, scores, counts, 1.0, weight)
            for shift in (1, 3, 8):
                hold = torch.full((rows, cols + 13), 7.0, dtype=dtype, device="cuda")
                into = torch.full((rows, cols + 9), 7.0, dtype=dtype, device="cuda")
                mine = hold[:, shift:shift + cols]
                mine.copy_(x)
                wide_ids = torch.zeros(rows, 9, dtype=torch.int64, device="cuda")
                wide_ids[:, :5] = ids
                wide_scores = torch.full((rows, 7), float("nan"), device="cuda")
                wide_scores[:, :5] = scores
                args = (wide_ids[:, :5], wide_scores[:, :5], counts)
                for out in (into[:, 2:2 + cols], mine):
                    got = gpu.distill_loss_grad(weight, mine, *args, out=out)
                    assert got[1].data_ptr() == out.data_ptr()
                    _check(torch, got[0], loss, off)
                    _check(torch, got[1], dx, off_dx)
                assert bool((hold[:, :shift] == 7.0).all()) and bool((hold[:, shift + cols:] == 7.0).all())
                assert bool((into[:, :2] == 7.0).all()) and bool((into[:, 2 + cols:] == 7.0).all())
            x2 = x.clone()
            got = gpu.distill_loss_grad(weight, x2, ids, scores, counts, out=x2)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_what_an_index_returns_is_the_teacher(gpu):
    import torch
    g = base._dev(torch, 1)
    docs = torch.nn.functional.normalize(torch.randn(3000, 64, generator=g, device="cuda"), dim=1)
    queries = torch.nn.functional.normalize(torch.randn(50, 64, generator=g, device="cuda"), dim=1)
    index = gpu.FlatIndex(gpu.VectorSpace(64, gpu.Metric.COSINE), 3000)
    index.insert_device(range(3000), docs)
    ids = torch.zeros(50, 20, dtype=torch.int64, device="cuda")
    dist = torch.zeros(50, 20, device="cuda")
    count = torch.zeros(50, dtype=torch.int32, device="cuda")
    index.search_device(queries, 20, ids, dist, count)
    student = torch.nn.functional.normalize(queries + 0.1 * torch.randn(50, 64, generator=g, device="cuda"), dim=1)
    logits = (student @ docs.t()).contiguous()
    weight = torch.full((50,), 1.0 / 50, device="cuda")
    _both(torch, gpu, logits, ids, -dist, count, weight, 0.05)
    # the teacher's own logits over its results only: nothing to learn
    masked = torch.full((50, 3000), -INF, device="cuda").scatter_(1, ids, -dist)
    loss, grad = gpu.distill_loss_grad(weight, masked, ids, -dist, count, temperature=0.05)
    assert float(loss.abs().max()) < 20 * 2.0 ** -19 and float(grad.abs().max()) < 2.0 ** -18 / 50 / 0.05


def test_distillation_in_a_graph_on_a_stream_and_again(gpu):
    import torch
    for rows, cols in ((32, 2000), (6, 60000)):
        x, ids, scores, counts, weight = _make(torch, rows, cols, 9, torch.bfloat16, 1.0, 4)

        def step():
            return [gpu.distill_loss(x, ids, scores, counts), *gpu.distill_loss_grad(weight, x, ids, scores, counts)]

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
            for a, b in zip((x, ids, scores, counts, weight), _make(torch, rows, cols, 9, torch.bfloat16, 1.0, 30 + seed)):
                a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_rows_past_4_gb(gpu):
    import torch
    rows, cols, tail = 70_000, 40_000, 3
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    small, ids, scores, counts, weight = _make(torch, tail, cols, 5, torch.bfloat16, 1.0, 5)
    x[-tail:] = small
    more = [torch.zeros(rows, *t.shape[1:], dtype=t.dtype, device="cuda") for t in (ids, scores, counts, weight)]
    for a, b in zip(more, (ids, scores, counts, weight)):
        a[-tail:] = b
    loss, dx = gpu.distill_loss_grad(more[3], x, *more[:3], out=x)
    want = _exact(torch, small, ids, scores, counts, 1.0, weight)
    _check(torch, loss[-tail:], *want[:2])
    _check(torch, dx[-tail:], *want[2:])
    assert not bool(loss[:-tail].any()) and not bool(dx[:1000].any())
    del dx
    # logits millions of columns apart
    far = 1 << 30
    hold = torch.zeros(far + cols, dtype=torch.float32, device="cuda").as_strided((2, cols), (far, 1))
    hold.copy_(small[:2])
    got = gpu.distill_loss_grad(weight[:2], hold, ids[:2], scores[:2], counts[:2], out=hold)
    want = _exact(torch, small[:2].float(), ids[:2], scores[:2], counts[:2], 1.0, weight[:2])
    _check(torch, got[0], *want[:2])
    _check(torch, got[1], *want[2:])


def test_many_short_rows(gpu):
    import torch
    x, ids, scores, counts, weight = _make(torch, 200, 6, 2, torch.float32, 1.0, 8)
    n = 2_200_000 // 200
    args = [t.repeat(n, *[1] * (t.dim() - 1)) for t in (weight, x, ids, scores, counts)]
    loss, dx = gpu.distill_loss_grad(*args)
    one = gpu.distill_loss_grad(weight, x, ids, scores, counts)
    assert bool((loss.view(n, 200) == one[0]).all()) and bool((dx.view(n, 200, 6) == one[1]).all())
    none = gpu.distill_loss_grad(weight[:0], x[:0], ids[:0], scores[:0], counts[:0])
    assert none[0].shape == (0,) and none[1].shape == (0, 6)


def test_distillation_refuses(gpu):
    import torch
    x, ids, scores, counts, weight = _make(torch, 4, 20, 3, torch.float32, 1.0, 9)
    f, b, mismatch = gpu.distill_loss, gpu.distill_loss_grad, gpu.DimensionMismatch
    for call, error in [
        (lambda: f(x.double(), ids, scores, counts), ValueError),
        (lambda: f(x.t(), ids, scores, counts), ValueError),
        (lambda: f(x, ids.int(), scores, counts), ValueError),
        (lambda: f(x, ids[:3], scores, counts), mismatch),
        (lambda: f(x, ids, scores[:, :2], counts), mismatch),
        (lambda: f(x, ids, scores.half(), counts), ValueError),
        (lambda: f(x, ids, scores, counts.long()), ValueError),
        (lambda: f(x, ids, scores, counts[:3]), mismatch),
        (lambda: f(x, ids, scores, counts.cpu()), ValueError),
        (lambda: f(x, ids, scores, counts, temperature=0.0), gpu.ProximaError),
        (lambda: f(x, ids, scores, counts, temperature=-1.0), gpu.ProximaError),
        (lambda: f(x, ids, scores, counts, temperature=math.nan), gpu.ProximaError),
        (lambda: f(x, ids, scores, counts, temperature=math.inf), gpu.ProximaError),
        (lambda: f(x, ids[:, :0], scores[:, :0], counts), gpu.ProximaError),
        (lambda: f(x, ids.repeat(1, 1400), scores.repeat(1, 1400), counts), gpu.ProximaError),
        (lambda: b(weight[:3], x, ids, scores, counts), mismatch),
        (lambda: b(weight.double(), x, ids, scores, counts), ValueError),
        (lambda: b(weight, x, ids, scores, counts, out=x.half()), ValueError),
        (lambda: b(weight, x, ids, scores, counts, out=x[:, :19]), mismatch),
        (lambda: f(x.clone().requires_grad_(), ids, scores, counts), ValueError),
        (lambda: b(weight, x.clone().requires_grad_(), ids, scores, counts), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_an_encoder_is_trained_by_an_index_and_served_token_by_token(gpu):
    """The operators as they are used together: a layer of experts with a residual makes embeddings, an index' answers
    are the target, the loss' gradient goes back through both products, and the trained matrices serve single tokens.
    All gradients against autograd in 64 bits."""
    import torch
    g = base._dev(torch, 11)
    dim, hidden, experts, docs, sizes, t = 64, 128, 4, 500, [40, 0, 21, 67], 0.5
    rows = sum(sizes)
    corpus = torch.nn.functional.normalize(torch.randn(docs, dim, generator=g, device="cuda"), dim=1)
    index = gpu.FlatIndex(gpu.VectorSpace(dim, gpu.Metric.INNER_PRODUCT), docs)
    index.insert_device(range(docs), corpus)
    x = torch.randn(rows, dim, generator=g, device="cuda").half()
    w1 = (torch.randn(experts, hidden, dim, generator=g, device="cuda") / dim ** 0.5).half()
    w2 = (torch.randn(experts, dim, hidden, generator=g, device="cuda") / hidden ** 0.5).half()
    b1, b2 = (torch.randn(experts, n, generator=g, device="cuda") * 0.1 for n in (hidden, dim))
    offsets = base._offsets(torch, sizes)
    teacher = torch.nn.functional.normalize(x.float() + torch.randn(rows, dim, generator=g, device="cuda"), dim=1)
    ids = torch.zeros(rows, 10, dtype=torch.int64, device="cuda")
    dist = torch.zeros(rows, 10, device="cuda")
    count = torch.zeros(rows, dtype=torch.int32, device="cuda")
    index.search_device(teacher.contiguous(), 10, ids, dist, count)
    keys = corpus.half()

    a, h = gpu.grouped_linear(x, w1, offsets, bias=b1, activation="gelu", keep=True)
    y = gpu.grouped_linear(a, w2, offsets, bias=b2, residual=x)
    logits = gpu.grouped_linear(y, keys, out_dtype=torch.float32)
    weight = torch.full((rows,), 1.0 / rows, device="cuda")
    loss, dlogits = gpu.distill_loss_grad(weight, logits, ids, -dist, count, temperature=t)
    scale = 1024.0  # f16 gradients of a mean
    dy = gpu.grouped_matmul_grad_input((dlogits * scale).half(), keys)
    dw2 = gpu.grouped_matmul_grad_weight(dy, a, offsets, out_dtype=torch.float32) / scale
    _, db2 = gpu.grouped_linear_grad(dy, offsets=offsets)
    dh, db1 = gpu.grouped_linear_grad(gpu.grouped_matmul_grad_input(dy, w2, offsets), h, "gelu", offsets)
    dw1 = gpu.grouped_matmul_grad_weight(dh, x, offsets, out_dtype=torch.float32) / scale
    db1, db2 = db1 / scale, db2 / scale

    leaves = [v.double().cpu().requires_grad_() for v in (w1, b1, w2, b2)]
    v1, c1, v2, c2 = leaves
    out, ends = [], offsets.tolist()
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        z = x[lo:hi].double().cpu()
        k = z @ v1[e].t() + c1[e]
        out.append(k * torch.special.ndtr(k) @ v2[e].t() + c2[e] + z)
    logq = torch.log_softmax(torch.cat(out) @ keys.double().cpu().t() / t, 1)
    logp = torch.log_softmax(-dist.double().cpu() / t, 1)
    want = (logp.exp() * (logp - logq.gather(1, ids.cpu()))).sum(1)
    want.mean().backward()
    # a, h, y, the logits' gradient, dy, da, dh: seven roundings of 2^-11 of normal values on any path
    assert float((loss.double().cpu() - want.detach()).norm() / want.detach().norm()) < 7 * 2.0 ** -11
    for got, leaf in zip((dw1, db1, dw2, db2), leaves):
        assert float((got.double().cpu() - leaf.grad).norm() / leaf.grad.norm()) < 7 * 2.0 ** -11

    # a few of the rows, each with its expert, as single tokens
    expert = torch.repeat_interleave(torch.arange(experts, device="cuda"), torch.tensor(sizes, device="cuda"))
    some = torch.randperm(rows, generator=g, device="cuda")[:9]
    ones = torch.ones(9, 1, device="cuda")
    served = gpu.expert_layer(x[some], expert[some, None], w1, w2, ones, activation="gelu", bias1=b1, bias2=b2,
                              residual=x[some])
    # the batch rounds a to f16 between the products (2^-11), and both their results
    assert float((served.double() - y[some].double()).norm() / y[some].double().norm()) < 3 * 2.0 ** -11


def test_two_streams_and_two_graphs_at_once(gpu):
    import torch
    cases = [_make(torch, rows, cols, 8, torch.bfloat16, 1.0, cols) for rows, cols in ((70, 3000), (5, 90000))]
    wants = [gpu.distill_loss_grad(w, x, i, s, c) for x, i, s, c, w in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    graphs, held = [], []
    torch.cuda.synchronize()
    for (x, i, s, c, w), stream in zip(cases, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held.append(gpu.distill_loss_grad(w, x, i, s, c))
        graphs.append(graph)
    for _ in range(6):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [gpu.distill_loss_grad(w, x, i, s, c) for x, i, s, c, w in cases]
        torch.cuda.synchronize()
        for got in (held, eager):
            for a, b in zip(got, wants):
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])

"""distill_loss and its gradient with every number of threads to a row and of
16-byte vectors to a thread, against the formula in 64 bits with the tolerances
of test_distill_gpu.py. Which row takes which: 64 threads up to 256 vectors of
more than 1024 rows, 256 up to 1024 vectors and, of more than 512 rows, up to
2048, 1024 threads up to 8192; a row of `cols` counts (cols + 2 e - 2) // e
vectors of e elements, as many as it can touch at any alignment."""
import pytest

import test_distill_gpu as base

pytestmark = pytest.mark.gpu

VARIANTS = [(64, 1), (64, 2), (64, 3), (64, 4)] + [(256, n) for n in range(1, 9)] + [(1024, n) for n in range(2, 9)]


def _rows(threads, each):
    return 1100 if threads == 64 else 600 if (threads, each) > (256, 4) and threads == 256 else 3


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("threads,each", VARIANTS)
def test_every_number_of_vectors(gpu, threads, each, dtype):
    import torch
    dtype = getattr(torch, dtype)
    e = 4 if dtype is torch.float32 else 8
    rows = _rows(threads, each)
    # the longest row of the variant, and one whose last vectors are few threads'
    for i, vectors in enumerate((threads * each, threads * (each - 1) + threads // 3)):
        cols = vectors * e - 2 * e + 2 + (e - 1) * i
        assert (cols + 2 * e - 2) // e == vectors
        t = (1.0, 0.05)[i]
        x, ids, scores, counts, weight = base._make(torch, rows, cols, 7, dtype, t, 100 * each + i)
        base._both(torch, gpu, x, ids, scores, counts, weight, t)
        # rows that begin at any element, in place and apart
        hold = torch.full((rows, cols + 5), 7.0, dtype=dtype, device="cuda")
        mine = hold[:, 3:3 + cols]
        mine.copy_(x)
        loss, off, dx, off_dx = base._exact(torch, x, ids, scores, counts, t, weight)
        for out in (torch.empty(rows, cols + 2, dtype=dtype, device="cuda")[:, 1:1 + cols], mine):
            got = gpu.distill_loss_grad(weight, mine, ids, scores, counts, temperature=t, out=out)
            base._check(torch, got[0], loss, off)
            base._check(torch, got[1], dx, off_dx)
        assert bool((hold[:, :3] == 7.0).all()) and bool((hold[:, 3 + cols:] == 7.0).all())


@pytest.mark.parametrize("rows,cols,top", [(2000, 700, 200), (1100, 250, 4096), (5, 9000, 4096), (3, 70_000, 4096)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_entries(gpu, rows, cols, top, dtype):
    # most of them, or all, with ids that come several times where there are more entries than columns
    import torch
    x, ids, scores, counts, weight = base._make(torch, rows, cols, top, getattr(torch, dtype), 1.0, top + cols)
    counts[::3] = top
    if top <= cols:
        ids[1, : top // 2] = ids[1, 0]
    base._both(torch, gpu, x, ids, scores, counts, weight, 1.0)

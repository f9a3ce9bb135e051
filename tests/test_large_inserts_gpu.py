"""Inserts of more rows than one launch may give a workgroup of 256 threads each
(2^24): every row is stored and found; and calls that no launch holds."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROWS, DIM = 2 ** 24 + 100, 4


@pytest.mark.parametrize("kind", ["flat", "ivfpq"])
def test_more_rows_than_a_launch(gpu, kind):
    import torch
    px = gpu
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(ROWS, DIM, generator=g, device="cuda")
    space = px.VectorSpace(DIM, px.Metric.EUCLIDEAN)
    if kind == "flat":
        index = px.FlatIndex(space, ROWS)
    else:  # untrained: its search scans every row
        index = px.IvfPqIndex(space, px.IvfPqConfig(4, 2).with_train_threshold(1 << 62))
    ids = np.arange(5, ROWS + 5, dtype=np.uint64)
    index.insert_device(ids, x)
    assert len(index) == ROWS
    at = np.array([0, 1, 99, 100, 2 ** 22 - 1, 2 ** 22, 2 ** 23 + 7, 2 ** 24 - 1, 2 ** 24, ROWS - 1])
    got, dist, count = index.search_batch(x[torch.from_numpy(at).cuda()].cpu().numpy(), 2)
    assert (count == 2).all()
    assert np.array_equal(got[:, 0], ids[at]) and not dist[:, 0].any()
    bad = x[:20].clone()
    bad[13, 2] = float("nan")
    with pytest.raises(px.NonFinite):
        index.insert_device(np.arange(20, dtype=np.uint64) + 2 * ROWS, bad)


def test_calls_that_a_launch_cannot_hold_are_refused(gpu):
    # one workgroup of 64 threads for each vector: 2^26 vectors are 2^32 work-items, which would wrap around
    px = gpu
    q = px.ScalarQuantizer.train(px.VectorSpace(1, px.Metric.EUCLIDEAN), np.array([-1.0, 1.0], np.float32))
    x = np.linspace(-1, 1, 2 ** 26 + 3, dtype=np.float32)
    codes = np.full(x.size, 77, np.uint8)

    def encode(n):
        return px._lib.pxg_sq_encode(px._ptr(x), n, 1, 1, 0, px._ptr(q.min), px._ptr(q.inverse_scale), px._ptr(codes))

    with pytest.raises(px.Capacity, match="fewer rows or queries"):
        px._check(encode(x.size))
    assert (codes == 77).all()
    assert encode(2 ** 26 - 1) == 0
    assert codes[0] == 0 and codes[2 ** 26 - 2] == 255 and (np.diff(codes[:2 ** 26 - 1].astype(int)) >= 0).all()

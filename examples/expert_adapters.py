"""Adapters in front of an index: one small network per cell of a k-means
router, trained with 8-bit activation checkpoints and served in 8 bits.

Documents are embeddings in a FlatIndex. Queries come from another encoder,
which here distorts them differently in every region, so that plain search
finds little. k-means over the queries makes the cells; a query's cell is its
nearest centroid (another FlatIndex); the cell's adapter, y = x + W2 gelu(W1 x),
maps the query to where the documents are:

- training sorts a batch by cell and runs the cells' ragged groups in one
  product each way; what the backward pass needs of the layers' inputs is kept
  in 8 bits (activation_pack, block8_pack);
- serving packs the trained matrices once: batches are multiplied in 8 bits, a
  few queries at a time take the layer whole (expert_layer).

    python examples/expert_adapters.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import proxima_amd as px  # noqa: E402


def corpus(docs, queries, dim, regions, seed):
    """Unit documents around `regions` centres, and each region's queries through its own distortion."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    centres = normal(regions, dim)
    region = torch.randint(0, regions, (docs,), generator=g, device="cuda")
    d = torch.nn.functional.normalize(centres[region] + normal(docs, dim), dim=1)
    target = torch.randint(0, docs, (queries,), generator=g, device="cuda")
    mix = 0.2 * torch.eye(dim, device="cuda") + normal(regions, dim, dim) / dim ** 0.5
    q = torch.empty(queries, dim, device="cuda")
    for r in range(regions):
        rows = region[target] == r
        q[rows] = d[target[rows]] @ mix[r]
    return d, q + 0.01 * normal(queries, dim), target


class Router:
    """Cells of a k-means clustering; a row's cell is its nearest centroid."""

    def __init__(self, points, cells, seed):
        self.centroids = torch.zeros(cells, points.shape[1], device="cuda")
        assign = torch.zeros(points.shape[0], dtype=torch.int32, device="cuda")
        px.kmeans_device(points, cells, 10, seed, self.centroids, assign, None)
        self.index = px.FlatIndex(px.VectorSpace(points.shape[1], px.Metric.EUCLIDEAN), cells)
        self.index.insert_device(range(cells), self.centroids)

    def cells(self, x):
        """The cell of each row of x, [rows, 1]."""
        n = x.shape[0]
        ids = torch.zeros(n, 1, dtype=torch.int64, device="cuda")
        dist = torch.zeros(n, 1, device="cuda")
        count = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.index.search_device(x, 1, ids, dist, count)
        return ids

    def __call__(self, x):
        """(order, offsets): the rows of x sorted by cell, and where each cell's begin."""
        cell, order = torch.sort(self.cells(x)[:, 0], stable=True)
        return order, torch.searchsorted(cell, torch.arange(self.centroids.shape[0] + 1, device="cuda"))


class Adapters:
    """y = x + W2 gelu(W1 x), a pair of matrices per cell; master weights in f32."""

    def __init__(self, cells, dim, hidden, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.w1 = torch.randn(cells, hidden, dim, generator=g, device="cuda") / dim ** 0.5
        self.w2 = torch.zeros(cells, dim, hidden, device="cuda")
        self.moments = [(torch.zeros_like(w), torch.zeros_like(w)) for w in (self.w1, self.w2)]
        self.steps = 0

    def train_step(self, x, target, offsets, rate):
        """One step towards `target`, rows sorted by cell; the mean squared error before it."""
        xb = x.bfloat16()
        w1, w2 = self.w1.bfloat16(), self.w2.bfloat16()
        # forward; the inputs of both layers are kept in 8 bits
        h = px.grouped_matmul(xb, w1, offsets)
        a, kept_h = px.activation_pack(h, "gelu")
        y = x + px.grouped_matmul(a, w2, offsets, out_dtype=torch.float32)
        kept_x, kept_a = px.block8_pack(xb), px.block8_pack(a)
        # backward
        diff = y - target
        dy = (diff * (2.0 / x.shape[0])).bfloat16()
        dw2 = px.grouped_matmul_grad_weight(dy, kept_a, offsets, out_dtype=torch.float32)
        dh = px.activation_grad(px.grouped_matmul_grad_input(dy, w2, offsets), kept_h, "gelu")
        dw1 = px.grouped_matmul_grad_weight(dh, kept_x, offsets, out_dtype=torch.float32)
        # Adam on the master weights
        self.steps += 1
        for w, dw, (m, v) in zip((self.w1, self.w2), (dw1, dw2), self.moments):
            m.lerp_(dw, 0.1)
            v.lerp_(dw * dw, 0.01)
            scale = rate * (1 - 0.99 ** self.steps) ** 0.5 / (1 - 0.9 ** self.steps)
            w.addcdiv_(m, v.sqrt().add_(1e-8), value=-scale)
        return float(diff.square().sum(1).mean())

    def packed(self):
        """The matrices in 8 bits, for serving."""
        return tuple(px.block8_pack(w.reshape(-1, w.shape[2])) for w in (self.w1, self.w2))


def serve(router, matrices, x):
    """Adapted queries, in the order they came, all products in 8 bits."""
    w1, w2 = matrices
    order, offsets = router(x)
    sorted_x = x[order]
    h = px.block8_matmul(px.block8_pack(sorted_x), w1, offsets)
    a, _ = px.activation_pack(h, "gelu")
    y = sorted_x + px.block8_matmul(px.block8_pack(a), w2, offsets, out_dtype=torch.float32)
    out = torch.empty_like(x)
    out[order] = y
    return out


def serve_few(router, matrices, x):
    """The same for a few queries: the layer whole, from their cells, without sorting or packing them."""
    w1, w2 = matrices
    gates = torch.ones(x.shape[0], 1, device="cuda")
    return px.expert_layer(x.bfloat16(), router.cells(x), w1, w2, gates, activation="gelu", residual=x,
                           out_dtype=torch.float32)


def recall(index, queries, target, k=10):
    """The share of queries whose document is among the k nearest."""
    n = queries.shape[0]
    ids = torch.zeros(n, k, dtype=torch.int64, device="cuda")
    dist = torch.zeros(n, k, device="cuda")
    count = torch.zeros(n, dtype=torch.int32, device="cuda")
    index.search_device(queries.contiguous(), k, ids, dist, count)
    return float((ids == target[:, None]).any(1).float().mean())


def main(docs=50_000, train=32_768, test=1000, dim=128, hidden=256, cells=8, steps=300, batch=4096):
    d, q, target = corpus(docs, train + test, dim, cells, 1)
    index = px.FlatIndex(px.VectorSpace(dim, px.Metric.COSINE), docs)
    index.insert_device(range(docs), d)
    router = Router(q[:train].contiguous(), cells, 2)
    adapters = Adapters(cells, dim, hidden, 3)
    before = recall(index, q[train:], target[train:])
    for step in range(steps):
        rows = torch.randint(0, train, (batch,), device="cuda")
        x = q[rows]
        order, offsets = router(x)
        loss = adapters.train_step(x[order], d[target[rows[order]]], offsets, 3e-3 * (1 - step / steps))
        if step % 50 == 0:
            print(f"step {step}: mean squared error {loss:.4f}", flush=True)
    matrices = adapters.packed()
    after = recall(index, serve(router, matrices, q[train:].contiguous()), target[train:])
    few = torch.cat([serve_few(router, matrices, q[i:i + 4].contiguous()) for i in range(train, train + 64, 4)])
    print(f"recall@10 without adapters {before:.3f}, with adapters served in 8 bits {after:.3f}, "
          f"of 64 queries served by fours {recall(index, few, target[train:train + 64]):.3f}")
    return before, after


if __name__ == "__main__":
    main()

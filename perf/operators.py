"""The operators of expert layers over packed 8-bit rows, as cases that can be timed and compared.

Three families, each called as a program that trains or serves the layers in front of an index would:

- `block8`: rows of activations are packed (e4m3 codes, one power-of-two scale for each block of 128 columns) and
  multiplied with weights packed beforehand, for one matrix or for one per group of rows;
- `forward`, `backward`: products in 16 bits grouped by expert, the groups ragged and some empty, and both gradients;
- `checkpoint`, `layer`: an activation whose input is kept in 8 bits for its backward pass, and an expert layer whose
  weight gradient is taken from its packed input.

Where `own` is false, the same is computed in elementary torch operations in 32 bits and rounded once at the end.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 128


def listed():
    return [
        # one row answered at once: the weights are read, nothing else counts
        {"name": "block8_one_row", "kind": "block8", "rows": 1, "k": 4096, "n": 4096, "groups": 1, "type": "bf16"},
        # a small batch, nothing a multiple of a tile or of a block
        {"name": "block8_odd", "kind": "block8", "rows": 333, "k": 1000, "n": 1500, "groups": 1, "type": "f16"},
        # a large batch of rows through one matrix
        {"name": "block8_large", "kind": "block8", "rows": 8192, "k": 4096, "n": 4096, "groups": 1, "type": "bf16"},
        # a few rows spread over many experts
        {"name": "block8_few_rows", "kind": "block8", "rows": 16, "k": 2048, "n": 1024, "groups": 32, "type": "bf16"},
        # a batch routed to experts, unevenly
        {"name": "block8_experts", "kind": "block8", "rows": 4096, "k": 2048, "n": 2048, "groups": 16,
         "type": "bf16"},
        # a few rows through experts kept in 16 bits
        {"name": "forward_few_rows", "kind": "forward", "rows": 8, "k": 2048, "n": 2048, "groups": 16,
         "type": "bf16"},
        # a training batch's forward pass
        {"name": "forward_large", "kind": "forward", "rows": 16384, "k": 2048, "n": 2048, "groups": 32,
         "type": "bf16"},
        # both gradients of a training batch
        {"name": "backward_large", "kind": "backward", "rows": 16384, "k": 2048, "n": 2048, "groups": 16,
         "type": "bf16", "wtype": "bf16"},
        # both gradients at odd sizes: rows of 602 and 406 bytes
        {"name": "backward_odd", "kind": "backward", "rows": 1511, "k": 301, "n": 203, "groups": 7, "type": "f16",
         "wtype": "f32"},
        # an activation between two small layers
        {"name": "checkpoint_small", "kind": "checkpoint", "rows": 64, "k": 1000, "act": "silu", "type": "f32"},
        # the activation of a training batch
        {"name": "checkpoint_large", "kind": "checkpoint", "rows": 16384, "k": 4096, "act": "gelu", "type": "bf16"},
        # a training step of an expert layer that keeps its input in 8 bits
        {"name": "layer_step", "kind": "layer", "rows": 8192, "k": 1024, "n": 4096, "groups": 8, "type": "bf16",
         "wtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["block8", "block8", "forward", "backward", "checkpoint", "layer"])
    if kind == "checkpoint":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "k": _log(rng, 100, 4096),
                "act": rng.choice(["silu", "gelu"]), "type": rng.choice(sorted(DTYPES))}

    def width():
        w = _log(rng, 100, 4096)
        return w if rng.random() < 0.4 else max(128, w // 64 * 64)

    k, n = width(), width()
    groups = rng.choice([1, _log(rng, 2, 64)]) if kind == "block8" else _log(rng, 1, 64)
    groups = max(1, min(groups, (1 << 27) // (n * k)))
    cost = {"block8": 2, "forward": 2, "backward": 4, "layer": 6}[kind]
    rows = _log(rng, 1, max(1, min(16384, 200_000_000_000 // (cost * n * k))))
    c = {"kind": kind, "rows": rows, "k": k, "n": n, "groups": groups,
         "type": "bf16" if kind == "layer" else rng.choice(["bf16", "bf16", "f16"])}
    if kind in ("backward", "layer"):
        c["wtype"] = rng.choice(["f32", c["type"]])
    return c


# --- inputs ---------------------------------------------------------------------------
def _rows(g, rows, cols, dtype):
    """Activations: a few columns are much larger than the others, as a layer's outputs have them."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.exp(torch.randn(cols, generator=g, device=DEV) * 0.7)
    return x.to(dtype)


def _sizes(g, rows, groups):
    """Rows of each group: a router's uneven shares, the rarest experts empty."""
    share = torch.softmax(torch.randn(groups, generator=g, device=DEV) * 1.2, 0)
    if groups >= 4:
        share[share < 0.15 / groups] = 0.0
    pick = torch.multinomial(share, rows, replacement=True, generator=g)
    return torch.bincount(pick, minlength=groups)


def _weights(g, groups, n, k, dtype):
    w = torch.empty(groups, n, k, dtype=dtype, device=DEV)
    for e in range(groups):
        w[e] = torch.randn(n, k, generator=g, device=DEV) / math.sqrt(k)
    return w


def _inputs(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["type"]]
    s = {"x": _rows(g, c["rows"], c["k"], dt)}
    if c["kind"] == "checkpoint":
        s["grad"] = _rows(g, c["rows"], c["k"], dt)
        return s
    sizes = _sizes(g, c["rows"], c["groups"])
    s["sizes"] = sizes.tolist()
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), sizes.cumsum(0)])
    s["w"] = _weights(g, c["groups"], c["n"], c["k"], dt)
    if c["kind"] in ("backward", "layer"):
        s["grad"] = _rows(g, c["rows"], c["n"], dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "block8":  # the weights are packed once, when a model is loaded
        w = s.pop("w")
        s["w_codes"], s["w_scales"] = _pack(w.reshape(-1, case["k"]))
    return s


# --- plain forms ----------------------------------------------------------------------
def _pack(x):
    """Codes [rows, cols rounded up to 128] and scale bytes [rows, blocks rounded up to 4] of x's rows."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    m, ex = torch.frexp(v.abs().amax(2))  # m in [0.5, 1); 448 is 0.875 * 2^9
    e = torch.where(m <= 0.875, ex - 9, ex - 8).clamp(-126, 127)
    e = torch.where(m == 0.0, torch.full_like(e, -126), e)
    inverse = ((127 - e) << 23).to(torch.int32).view(torch.float32)  # 2^-e
    codes = (v * inverse[:, :, None]).to(torch.float8_e4m3fn).view(rows, -1).view(torch.uint8)
    scales = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return codes, scales


def _unpack(codes, scales, cols):
    rows, wide = codes.shape
    blocks = wide // BLOCK
    scale = (scales[:, :blocks].to(torch.int32) << 23).view(torch.float32)
    v = codes.view(torch.float8_e4m3fn).float().view(rows, blocks, BLOCK) * scale[:, :, None]
    return v.view(rows, wide)[:, :cols]


def _forward(x, w, sizes, out_type):
    """Each group's rows times the transpose of its matrix [n, k]."""
    y = torch.empty(x.shape[0], w.shape[1], dtype=out_type, device=x.device)
    a = 0
    for e, size in enumerate(sizes):
        if size:
            y[a:a + size] = x[a:a + size].float() @ w[e].float().T
            a += size
    return y


def _grad_input(grad, w, sizes):
    dx = torch.empty(grad.shape[0], w.shape[2], dtype=grad.dtype, device=grad.device)
    a = 0
    for e, size in enumerate(sizes):
        if size:
            dx[a:a + size] = grad[a:a + size].float() @ w[e].float()
            a += size
    return dx


def _grad_weight(grad, x, sizes, out_type):
    dw = torch.zeros(len(sizes), grad.shape[1], x.shape[1], dtype=out_type, device=grad.device)
    a = 0
    for e, size in enumerate(sizes):
        if size:
            dw[e] = grad[a:a + size].float().T @ x[a:a + size].float()
            a += size
    return dw


def _act(h, act):
    if act == "silu":
        return h / (1.0 + torch.exp(-h))
    return 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))


def _act_slope(h, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-h))
        return s * (1.0 + h * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain(s, c):
    x = s["x"]
    if c["kind"] == "block8":
        xv = _unpack(*_pack(x), c["k"])
        w = _unpack(s["w_codes"], s["w_scales"], c["k"]).view(c["groups"], c["n"], c["k"])
        return {"y": _forward(xv, w, s["sizes"], x.dtype)}
    if c["kind"] == "forward":
        return {"y": _forward(x, s["w"], s["sizes"], x.dtype)}
    if c["kind"] == "backward":
        return {"dx": _grad_input(s["grad"], s["w"], s["sizes"]),
                "dw": _grad_weight(s["grad"], x, s["sizes"], DTYPES[c["wtype"]])}
    if c["kind"] == "checkpoint":
        a = _act(x.float(), c["act"]).to(x.dtype)
        kept = _pack(x)
        slope = _act_slope(_unpack(*kept, c["k"]), c["act"])
        return {"a": a, "dx": (s["grad"].float() * slope).to(x.dtype)}
    y = _forward(x, s["w"], s["sizes"], x.dtype)
    kept = _pack(x)
    return {"y": y, "dx": _grad_input(s["grad"], s["w"], s["sizes"]),
            "dw": _grad_weight(s["grad"], _unpack(*kept, c["k"]), s["sizes"], DTYPES[c["wtype"]])}


# --- the framework's kernels ----------------------------------------------------------
def _own(s, c):
    import proxima_amd as px

    x = s["x"]
    if c["kind"] == "block8":
        w = px.Block8(s["w_codes"], s["w_scales"], c["k"])
        return {"y": px.block8_matmul(px.block8_pack(x), w, s["offsets"], out_dtype=x.dtype)}
    if c["kind"] == "forward":
        return {"y": px.grouped_matmul(x, s["w"], s["offsets"])}
    if c["kind"] == "backward":
        return {"dx": px.grouped_matmul_grad_input(s["grad"], s["w"], s["offsets"]),
                "dw": px.grouped_matmul_grad_weight(s["grad"], x, s["offsets"], out_dtype=DTYPES[c["wtype"]])}
    if c["kind"] == "checkpoint":
        a, kept = px.activation_pack(x, c["act"])
        return {"a": a, "dx": px.activation_grad(s["grad"], kept, c["act"])}
    y = px.grouped_matmul(x, s["w"], s["offsets"])
    kept = px.block8_pack(x)
    return {"y": y, "dx": px.grouped_matmul_grad_input(s["grad"], s["w"], s["offsets"]),
            "dw": px.grouped_matmul_grad_weight(s["grad"], kept, s["offsets"], out_dtype=DTYPES[c["wtype"]])}


def run(state):
    return (_own if own else _plain)(state, state["case"])


def work(case):
    c = case
    size = 4 if c["type"] == "f32" else 2
    rows, k = c["rows"], c["k"]
    if c["kind"] == "checkpoint":  # x, the gradient, a and dx; the slope and the activation
        return {"bytes": 4 * rows * k * size, "flops": 30.0 * rows * k}
    n, groups = c["n"], c["groups"]
    used = min(groups, rows)
    product = 2.0 * rows * n * k
    if c["kind"] == "block8":
        return {"bytes": rows * (k + n) * size + used * n * k * (1 + 1 / BLOCK), "flops": product}
    if c["kind"] == "forward":
        return {"bytes": rows * (k + n) * size + used * n * k * size, "flops": product}
    wsize = 4 if c["wtype"] == "f32" else 2
    both = rows * (2 * k + n) * size + used * n * k * size + groups * n * k * wsize
    if c["kind"] == "backward":
        return {"bytes": both, "flops": 2 * product}
    return {"bytes": both + rows * n * size, "flops": 3 * product}


# --- the same in 64 bits --------------------------------------------------------------
def _rounded64(x):
    """x's values after packing: each to the nearest multiple (ties to even) of its binade's step at 3 fraction bits,
    the steps no finer than 2^-9 of the block's scale, the scale the least power of two that brings the block
    within 448."""
    rows, cols = x.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    for a in range(0, cols, BLOCK):
        v = x[:, a:a + BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        scale = torch.full_like(top, 2.0 ** -126)
        some = top > 0
        guess = torch.exp2(torch.floor(torch.log2(torch.where(some, top, torch.ones_like(top)) / 448.0)) - 1.0)
        for _ in range(3):
            guess = torch.where(top > 448.0 * guess, guess * 2.0, guess)
        scale = torch.where(some, torch.maximum(guess, scale), scale)
        u = v / scale
        binade = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))))
        step = binade / 8.0
        out[:, a:a + BLOCK] = torch.round(u / step) * step * scale
    return out


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    x = s["x"]
    if c["kind"] == "checkpoint":
        h, kept, grad = x.double(), _rounded64(x), s["grad"].double()
        if c["act"] == "silu":
            a, p = h * torch.sigmoid(h), torch.sigmoid(kept)
            return {"a": a, "dx": grad * (p + kept * p * (1.0 - p))}
        normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device=DEV), 1.0)
        density = torch.exp(-kept.square() / 2.0) / math.sqrt(2.0 * math.pi)
        return {"a": h * normal.cdf(h), "dx": grad * (normal.cdf(kept) + kept * density)}
    out = {}
    n, k = c["n"], c["k"]
    if c["kind"] == "block8":
        x64 = _rounded64(x)
    else:
        x64 = x.double()
    if c["kind"] != "backward":
        out["y"] = torch.zeros(c["rows"], n, dtype=torch.float64, device=DEV)
    if c["kind"] in ("backward", "layer"):
        kept = _rounded64(x) if c["kind"] == "layer" else x64
        out["dx"] = torch.zeros(c["rows"], k, dtype=torch.float64, device=DEV)
        out["dw"] = torch.zeros(c["groups"], n, k, dtype=torch.float64, device=DEV)
    ends = s["offsets"].tolist()
    for e in range(c["groups"]):
        r = slice(ends[e], ends[e + 1])
        if ends[e] == ends[e + 1]:
            continue
        w = _rounded64(s["w"][e]) if c["kind"] == "block8" else s["w"][e].double()
        if "y" in out:
            out["y"][r] = torch.mm(x64[r], w.t().contiguous())
        if "dx" in out:
            grad = s["grad"][r].double()
            out["dx"][r] = torch.mm(grad, w)
            out["dw"][e] = torch.mm(grad.t().contiguous(), kept[r])
    return out

"""Layers with their epilogue, whole expert layers for a few tokens and distillation, as cases that can be timed and
compared.

Four kinds, each called as a program that trains or serves the layers in front of an index would:

- `linear`: a layer of ragged groups of rows, y = f(x w_g^T + b_g) + r, in 16 bits (a training pass also keeps
  h = x w_g^T + b_g) or over packed 8-bit rows;
- `linear_grad`: its backward pass up to the products, dh = dy f'(h) and the bias' gradient;
- `tokens`: a whole expert layer for a few tokens, each with a few experts and their gates, the matrices in 16 or 8 bits;
- `distill`: the loss of an encoder that is trained to rank as a teacher does, whose best results (ids, scores and how
  many, as a search returns them) are the target, alone or with its gradient.

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
        # one query through a dense layer: the matrix is read, nothing else counts
        {"name": "linear_one_row", "kind": "linear", "rows": 1, "pad": 0, "k": 4096, "n": 4096, "groups": 1,
         "type": "bf16", "out": "bf16", "bias": "bf16", "act": "gelu", "residual": False, "keep": False,
         "packed": False},
        # a small batch, nothing a multiple of a tile; the layer's input passes by it
        {"name": "linear_odd", "kind": "linear", "rows": 333, "pad": 0, "k": 1000, "n": 1500, "groups": 1,
         "type": "f16", "out": "f16", "bias": "f32", "act": "silu", "residual": True, "keep": False, "packed": False},
        # a training batch's forward pass through experts, what the backward pass needs kept
        {"name": "linear_train", "kind": "linear", "rows": 8192, "pad": 0, "k": 1024, "n": 4096, "groups": 8,
         "type": "bf16", "out": "bf16", "bias": "f32", "act": "gelu", "residual": False, "keep": True,
         "packed": False},
        # a batch served in 8 bits through a layer's second matrices, added to its input
        {"name": "linear_packed", "kind": "linear", "rows": 4096, "pad": 96, "k": 2048, "n": 2048, "groups": 16,
         "type": "bf16", "out": "bf16", "bias": "bf16", "act": "none", "residual": True, "keep": False,
         "packed": True},
        # the backward pass of a training batch
        {"name": "linear_grad_large", "kind": "linear_grad", "rows": 16384, "pad": 0, "n": 4096, "groups": 8,
         "type": "bf16", "act": "gelu"},
        # the same at odd sizes: rows of 602 bytes
        {"name": "linear_grad_odd", "kind": "linear_grad", "rows": 1511, "pad": 37, "n": 301, "groups": 7,
         "type": "f16", "act": "silu"},
        # one query through its cell's adapter, as small as these layers get: latency
        {"name": "tokens_one", "kind": "tokens", "rows": 1, "picks": 1, "experts": 8, "k": 128, "hidden": 256,
         "n": 128, "type": "bf16", "out": "f32", "act": "gelu", "gated": False, "bias": "none", "residual": True,
         "packed": False},
        # a few tokens through gated experts in 16 bits
        {"name": "tokens_few", "kind": "tokens", "rows": 8, "picks": 2, "experts": 16, "k": 2048, "hidden": 4096,
         "n": 2048, "type": "bf16", "out": "bf16", "act": "silu", "gated": True, "bias": "none", "residual": True,
         "packed": False},
        # a serving batch through many experts in 8 bits
        {"name": "tokens_packed", "kind": "tokens", "rows": 32, "picks": 4, "experts": 64, "k": 2048, "hidden": 1024,
         "n": 2048, "type": "bf16", "out": "bf16", "act": "gelu", "gated": False, "bias": "f32", "residual": False,
         "packed": True},
        # a small batch against the other documents of a batch
        {"name": "distill_small", "kind": "distill", "rows": 64, "cols": 1000, "top": 10, "type": "f32",
         "grad": True, "temperature": 0.05},
        # a training batch against a whole corpus
        {"name": "distill_large", "kind": "distill", "rows": 4096, "cols": 50000, "top": 100, "type": "bf16",
         "grad": True, "temperature": 1.0},
        # a few validation queries against a large corpus
        {"name": "distill_long", "kind": "distill", "rows": 16, "cols": 1000000, "top": 10, "type": "bf16",
         "grad": False, "temperature": 0.05},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.4 else max(64, w // 64 * 64)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear_grad", "tokens", "tokens", "distill", "distill"])
    if kind == "distill":
        cols, kind_of = _log(rng, 100, 1000000), rng.choice(sorted(DTYPES))
        most = (100_000_000 if kind_of == "f32" else 200_000_000) // cols
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(8192, most))), "cols": cols,
                "top": _log(rng, 1, min(200, cols // 2)), "type": kind_of,
                "grad": rng.random() < 0.7, "temperature": rng.choice([0.05, 1.0, 2.0])}
    if kind == "tokens":
        experts = _log(rng, 1, 64)
        c = {"kind": kind, "rows": _log(rng, 1, 64), "picks": rng.randint(1, min(8, experts)), "experts": experts,
             "k": _width(rng, 100, 4096), "hidden": _width(rng, 100, 4096), "n": _width(rng, 100, 4096),
             "type": rng.choice(["bf16", "bf16", "f16"]), "act": rng.choice(["silu", "gelu"]),
             "gated": rng.random() < 0.4, "bias": rng.choice(["none", "f32"]), "residual": rng.random() < 0.5,
             "packed": rng.random() < 0.4}
        while c["experts"] * c["hidden"] * (2 * c["k"] + c["n"]) > 1 << 28:
            c["hidden"] //= 2
        if c["packed"]:
            c["type"] = "bf16"
        c["out"] = rng.choice([c["type"], "f32"])
        return c
    n, groups = _width(rng, 100, 4096), _log(rng, 1, 64)
    pad = rng.choice([0, rng.randint(1, 100)])
    if kind == "linear_grad":
        return {"kind": kind, "rows": _log(rng, 1, 16384), "pad": pad, "n": n, "groups": groups,
                "type": rng.choice(sorted(DTYPES)), "act": rng.choice(["none", "silu", "gelu"])}
    k = _width(rng, 100, 4096)
    groups = max(1, min(groups, (1 << 27) // (n * k)))
    packed = rng.random() < 0.3
    c = {"kind": kind, "rows": _log(rng, 1, max(1, min(16384, 68_000_000_000 // (2 * n * k)))),
         "pad": pad if groups > 1 else 0, "k": k, "n": n, "groups": groups,
         "type": "bf16" if packed else rng.choice(["bf16", "bf16", "f16"]),
         "act": rng.choice(["none", "silu", "gelu"]), "residual": rng.random() < 0.5,
         "keep": not packed and rng.random() < 0.4, "packed": packed}
    c["out"] = rng.choice([c["type"], c["type"], "f32"])
    c["bias"] = rng.choice(["none", "f32", c["type"]])
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


def _groups(s, g, c):
    """The batch's groups; the rows behind the last are padding."""
    sizes = _sizes(g, c["rows"], c["groups"])
    s["sizes"] = sizes.tolist()
    s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), sizes.cumsum(0)])


def _linear_inputs(s, g, c):
    dt = DTYPES[c["type"]]
    rows = c["rows"] + c["pad"]
    s["x"] = _rows(g, rows, c["k"], dt)
    _groups(s, g, c)
    s["w"] = _weights(g, c["groups"], c["n"], c["k"], dt)
    s["bias"] = s["residual"] = None
    if c["bias"] != "none":
        s["bias"] = (0.5 * torch.randn(c["groups"], c["n"], generator=g, device=DEV)).to(DTYPES[c["bias"]])
    if c["residual"]:
        s["residual"] = _rows(g, rows, c["n"], DTYPES[c["out"]])


def _grad_inputs(s, g, c):
    dt = DTYPES[c["type"]]
    rows = c["rows"] + c["pad"]
    _groups(s, g, c)
    s["grad"] = _rows(g, rows, c["n"], dt)
    s["h"] = _rows(g, rows, c["n"], dt) if c["act"] != "none" else None


def _token_inputs(s, g, c):
    dt = DTYPES[c["type"]]
    rows, experts, picks = c["rows"], c["experts"], c["picks"]
    s["x"] = _rows(g, rows, c["k"], dt)
    s["w1"] = _weights(g, experts, c["hidden"], c["k"], dt)
    s["up"] = _weights(g, experts, c["hidden"], c["k"], dt) if c["gated"] else None
    s["w2"] = _weights(g, experts, c["n"], c["hidden"], dt)
    s["bias1"] = s["bias2"] = s["residual"] = None
    if c["bias"] != "none":
        s["bias1"] = (0.5 * torch.randn(experts, c["hidden"], generator=g, device=DEV)).to(DTYPES[c["bias"]])
        s["bias2"] = (0.5 * torch.randn(experts, c["n"], generator=g, device=DEV)).to(DTYPES[c["bias"]])
    if c["residual"]:
        s["residual"] = _rows(g, rows, c["n"], DTYPES[c["out"]])
    # a router's choice: some experts are liked by all tokens
    like = torch.randn(rows, experts, generator=g, device=DEV) + torch.randn(experts, generator=g, device=DEV)
    top, s["experts"] = torch.topk(like, picks, dim=1)
    s["gates"] = torch.softmax(top, 1)


def _distill_inputs(s, g, c):
    rows, cols, top = c["rows"], c["cols"], c["top"]
    t = c["temperature"]
    dt = DTYPES[c["type"]]
    # similarities that a softmax at this temperature tells apart; a few documents are masked
    x = torch.randn(rows, cols, generator=g, device=DEV) * (2.0 * t)
    x[torch.rand(rows, cols, generator=g, device=DEV) < 0.01] = -math.inf
    s["logits"] = x.to(dt)
    # the teacher sees what the student sees, and more
    x += torch.randn(rows, cols, generator=g, device=DEV) * t
    s["scores"], s["ids"] = torch.topk(x, top, dim=1)
    # some searches found less, a few nothing
    count = torch.randint(-top // 8, 3 * top + 1, (rows,), generator=g, device=DEV).clamp(0, top)
    masked = (s["scores"] == -math.inf).int().argmax(1)
    s["counts"] = torch.where(s["scores"][:, -1] == -math.inf, torch.minimum(count, masked), count).to(torch.int32)
    unused = torch.arange(top, device=DEV) >= s["counts"][:, None]
    s["ids"][unused] = 0
    s["scores"][unused] = 0.0
    if c["grad"]:  # the mean's weights, scaled as mixed-precision training scales them
        s["weight"] = torch.rand(rows, generator=g, device=DEV) * 64.0 + 64.0


_INPUTS = {"linear": _linear_inputs, "linear_grad": _grad_inputs, "tokens": _token_inputs, "distill": _distill_inputs}


def _inputs(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {}
    _INPUTS[c["kind"]](s, g, c)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case.get("packed"):  # the weights are packed once, when a model is loaded; rows are packed by the layer before
        for name in ("x", "w") if case["kind"] == "linear" else ("w1", "up", "w2"):
            if s[name] is not None:
                s[name] = _pack(s[name].reshape(-1, s[name].shape[-1]))
    if case["kind"] == "tokens":  # the plain form's plan: the tokens of each expert in use, and which pick it is
        s["plan"] = []
        for e in torch.unique(s["experts"]).tolist():
            s["plan"].append((e, *torch.nonzero(s["experts"] == e, as_tuple=True)))
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


def _unpack(packed, cols):
    codes, scales = packed
    rows, wide = codes.shape
    blocks = wide // BLOCK
    scale = (scales[:, :blocks].to(torch.int32) << 23).view(torch.float32)
    v = codes.view(torch.float8_e4m3fn).float().view(rows, blocks, BLOCK) * scale[:, :, None]
    return v.view(rows, wide)[:, :cols]


def _act(h, act):
    if act == "silu":
        return h / (1.0 + torch.exp(-h))
    if act == "gelu":
        return 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))
    return h


def _act_slope(h, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-h))
        return s * (1.0 + h * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_linear(s, c):
    x = _unpack(s["x"], c["k"]) if c["packed"] else s["x"]
    w = _unpack(s["w"], c["k"]).view(c["groups"], c["n"], c["k"]) if c["packed"] else s["w"]
    rows = c["rows"] + c["pad"]
    h = torch.zeros(rows, c["n"], device=DEV)
    a = 0
    for e, size in enumerate(s["sizes"]):
        if size:
            h[a:a + size] = x[a:a + size].float() @ w[e].float().T
            if s["bias"] is not None:
                h[a:a + size] += s["bias"][e].float()
            a += size
    y = _act(h, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(DTYPES[c["out"]])}
    if c["keep"]:
        out["h"] = h.to(DTYPES[c["out"]])
    return out


def _plain_grad(s, c):
    dh = s["grad"].float()
    if c["act"] != "none":
        dh = dh * _act_slope(s["h"].float(), c["act"])
    dbias = torch.zeros(c["groups"], c["n"], device=DEV)
    a = 0
    for e, size in enumerate(s["sizes"]):
        if size:
            dbias[e] = dh[a:a + size].sum(0)
            a += size
    dh = dh.to(s["grad"].dtype)
    if c["act"] != "none" and c["pad"]:
        dh[a:] = 0.0
    return {"dh": dh, "dbias": dbias}


def _plain_tokens(s, c):
    k, hidden, n = c["k"], c["hidden"], c["n"]

    def matrix(name, e, rows, cols):
        if not c["packed"]:
            return s[name][e].float()
        codes, scales = s[name]
        return _unpack((codes[e * rows:(e + 1) * rows], scales[e * rows:(e + 1) * rows]), cols)

    y = s["residual"].float().clone() if s["residual"] is not None else torch.zeros(c["rows"], n, device=DEV)
    for e, token, pick in s["plan"]:
        x = s["x"][token].float()
        h = x @ matrix("w1", e, hidden, k).T
        if s["bias1"] is not None:
            h = h + s["bias1"][e].float()
        a = _act(h, c["act"])
        if c["gated"]:
            a = a * (x @ matrix("up", e, hidden, k).T)
        z = a @ matrix("w2", e, n, hidden).T
        if s["bias2"] is not None:
            z = z + s["bias2"][e].float()
        y[token] += s["gates"][token, pick][:, None] * z
    return {"y": y.to(DTYPES[c["out"]])}


def _plain_distill(s, c):
    x = s["logits"].float() / c["temperature"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    valid = torch.arange(c["top"], device=DEV) < s["counts"][:, None]
    t = torch.where(valid, s["scores"] / c["temperature"], -math.inf)
    best = t.amax(1, keepdim=True)
    t = torch.where(valid, t - torch.where(best == -math.inf, 0.0, best), -math.inf)
    p = torch.exp(t)
    mass = p.sum(1, keepdim=True)
    some = mass > 0.0
    mass = torch.where(some, mass, 1.0)
    p = p / mass
    logq = torch.gather(x, 1, s["ids"]) - top - torch.log(total)
    terms = p * (t - torch.log(mass) - logq)
    out = {"loss": torch.where(p > 0.0, terms, 0.0).sum(1)}
    if c["grad"]:
        dx = torch.where(some, e / total, 0.0).scatter_add_(1, s["ids"], -p)
        out["dx"] = (dx * (s["weight"] / c["temperature"])[:, None]).to(s["logits"].dtype)
    return out


_PLAIN = {"linear": _plain_linear, "linear_grad": _plain_grad, "tokens": _plain_tokens, "distill": _plain_distill}


# --- the framework's kernels ----------------------------------------------------------
def _own(s, c):
    import proxima_amd as px

    if c["kind"] == "linear":
        act, out = None if c["act"] == "none" else c["act"], DTYPES[c["out"]]
        if c["packed"]:
            x, w = px.Block8(*s["x"], c["k"]), px.Block8(*s["w"], c["k"])
            return {"y": px.block8_linear(x, w, s["offsets"], bias=s["bias"], activation=act, residual=s["residual"],
                                          out_dtype=out)}
        got = px.grouped_linear(s["x"], s["w"], s["offsets"], bias=s["bias"], activation=act, residual=s["residual"],
                                out_dtype=out, keep=c["keep"])
        return {"y": got[0], "h": got[1]} if c["keep"] else {"y": got}
    if c["kind"] == "linear_grad":
        dh, dbias = px.grouped_linear_grad(s["grad"], s["h"], None if c["act"] == "none" else c["act"], s["offsets"])
        return {"dh": dh, "dbias": dbias}
    if c["kind"] == "tokens":
        if c["packed"]:
            w1, w2 = px.Block8(*s["w1"], c["k"]), px.Block8(*s["w2"], c["hidden"])
            up = px.Block8(*s["up"], c["k"]) if c["gated"] else None
        else:
            w1, w2, up = s["w1"], s["w2"], s["up"]
        return {"y": px.expert_layer(s["x"], s["experts"], w1, w2, s["gates"], activation=c["act"], up=up,
                                     bias1=s["bias1"], bias2=s["bias2"], residual=s["residual"],
                                     out_dtype=DTYPES[c["out"]])}
    if c["grad"]:
        loss, dx = px.distill_loss_grad(s["weight"], s["logits"], s["ids"], s["scores"], s["counts"],
                                        temperature=c["temperature"])
        return {"loss": loss, "dx": dx}
    return {"loss": px.distill_loss(s["logits"], s["ids"], s["scores"], s["counts"], temperature=c["temperature"])}


def run(state):
    c = state["case"]
    return _own(state, c) if own else _PLAIN[c["kind"]](state, c)


_SIZES = {"bf16": 2, "f16": 2, "f32": 4, "none": 0}


def work(case):
    c = case
    size = _SIZES[c["type"]]
    if c["kind"] == "distill":  # the logits, their gradient and the entries; a difference, an exponential, sums
        elements = c["rows"] * c["cols"]
        return {"bytes": elements * size * (2 if c["grad"] else 1) + c["rows"] * c["top"] * 12,
                "flops": elements * (10.0 if c["grad"] else 5.0)}
    if c["kind"] == "linear_grad":
        rows = c["rows"] + c["pad"]
        if c["act"] == "none":
            return {"bytes": rows * c["n"] * size + c["groups"] * c["n"] * 4, "flops": 1.0 * rows * c["n"]}
        return {"bytes": 3 * rows * c["n"] * size + c["groups"] * c["n"] * 4, "flops": 30.0 * rows * c["n"]}
    element = 1 + 1 / BLOCK if c["packed"] else size
    if c["kind"] == "tokens":
        pairs = c["rows"] * c["picks"]
        matrices = c["hidden"] * (c["k"] * (2 if c["gated"] else 1) + c["n"])
        # experts that some token chose, were all liked alike
        used = c["experts"] * (1.0 - (1.0 - c["picks"] / c["experts"]) ** c["rows"])
        return {"bytes": used * matrices * element + c["rows"] * (c["k"] * size + c["n"] * _SIZES[c["out"]]),
                "flops": 2.0 * pairs * matrices}
    rows, n, k, out = c["rows"] + c["pad"], c["n"], c["k"], _SIZES[c["out"]]
    used = min(c["groups"], c["rows"])
    return {"bytes": c["rows"] * k * element + used * n * (k * element + _SIZES[c["bias"]])
            + rows * n * out * (1 + c["residual"] + c["keep"]), "flops": 2.0 * c["rows"] * n * k}


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


def _normal(h):
    return torch.special.ndtr(h)


def _act64(h, act):
    return h * torch.sigmoid(h) if act == "silu" else h * _normal(h) if act == "gelu" else h


def exact(case, seed):
    c = case
    s = _inputs(c, seed)
    if c["kind"] == "distill":
        return _exact_distill(s, c)
    if c["kind"] == "tokens":
        return _exact_tokens(s, c)
    ends = s["offsets"].tolist()
    rows = c["rows"] + c["pad"]
    if c["kind"] == "linear_grad":
        dh, h = s["grad"].double(), s["h"]
        if c["act"] == "silu":
            h = h.double()
            dh = dh * torch.sigmoid(h) * (1.0 + h * torch.sigmoid(-h))
        elif c["act"] == "gelu":
            h = h.double()
            dh = dh * (_normal(h) + h * torch.exp(-h.square() / 2.0) / math.sqrt(2.0 * math.pi))
        dbias = torch.stack([dh[a:b].sum(0) for a, b in zip(ends, ends[1:])])
        if c["act"] != "none":
            dh[ends[-1]:] = 0.0
        return {"dh": dh, "dbias": dbias}
    h = torch.zeros(rows, c["n"], dtype=torch.float64, device=DEV)
    x = _rounded64(s["x"]) if c["packed"] else s["x"].double()
    for e in range(c["groups"]):
        r = slice(ends[e], ends[e + 1])
        if ends[e] == ends[e + 1]:
            continue
        w = _rounded64(s["w"][e]) if c["packed"] else s["w"][e].double()
        h[r] = torch.mm(x[r], w.t().contiguous())
        if s["bias"] is not None:
            h[r] += s["bias"][e].double()
    y = _act64(h, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return {"y": y, "h": h} if c["keep"] else {"y": y}


def _exact_tokens(s, c):
    picked = s["experts"].tolist()
    gates = s["gates"].double()
    y = torch.zeros(c["rows"], c["n"], dtype=torch.float64, device=DEV)
    for e in sorted({e for row in picked for e in row}):
        token = [t for t, row in enumerate(picked) if e in row]
        gate = torch.stack([gates[t, picked[t].index(e)] for t in token])
        w1, w2 = s["w1"][e], s["w2"][e]
        w1, w2 = (_rounded64(w1), _rounded64(w2)) if c["packed"] else (w1.double(), w2.double())
        x = s["x"][token].double()
        h = torch.mm(x, w1.t().contiguous())
        if s["bias1"] is not None:
            h = h + s["bias1"][e].double()
        a = _act64(h, c["act"])
        if c["gated"]:
            up = _rounded64(s["up"][e]) if c["packed"] else s["up"][e].double()
            a = a * torch.mm(x, up.t().contiguous())
        z = torch.mm(a, w2.t().contiguous())
        if s["bias2"] is not None:
            z = z + s["bias2"][e].double()
        y[token] += gate[:, None] * z
    return {"y": y + s["residual"].double() if s["residual"] is not None else y}


def _exact_distill(s, c):
    rows, cols = s["logits"].shape
    loss = torch.zeros(rows, dtype=torch.float64, device=DEV)
    dx = torch.zeros(rows, cols, dtype=torch.float64, device=DEV) if c["grad"] else None
    counts = s["counts"].tolist()
    some = max(1, 50_000_000 // cols)
    for a in range(0, rows, some):
        r = slice(a, min(rows, a + some))
        logq = torch.log_softmax(s["logits"][r].double() / c["temperature"], 1)
        p = torch.zeros(logq.shape[0], c["top"], dtype=torch.float64, device=DEV)
        logp = torch.zeros_like(p)
        for i, n in enumerate(counts[r]):
            if n:
                logp[i, :n] = torch.log_softmax(s["scores"][a + i, :n].double() / c["temperature"], 0)
                p[i, :n] = torch.exp(logp[i, :n])
        loss[r] = torch.where(p > 0.0, p * (logp - logq.gather(1, s["ids"][r])), 0.0).sum(1)
        if c["grad"]:
            d = torch.exp(logq)
            d[s["counts"][r] == 0] = 0.0
            d.scatter_add_(1, s["ids"][r], -p)
            dx[r] = d * (s["weight"][r].double() / c["temperature"])[:, None]
    return {"loss": loss, "dx": dx} if c["grad"] else {"loss": loss}

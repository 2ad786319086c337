"""What the transformer-layer operators of ``muspace_b200.ops`` are measured on.

Around every deformable attention of an encoder or decoder layer stand the same
few operators: projections and feed-forward products with a bias, an activation
and a residual (``linear_act``), the normalisation of what comes out
(``layer_norm``), and, in training, activations kept in 8 bits for the backward
pass (``checkpoint="int8"``, ``checkpoint_pack`` / ``checkpoint_unpack``).

``run`` computes a case in its plain form (``own`` false: elementary torch
operations in 32 bits, rounded once at the end) or by the framework's calls
(``own`` true). ``exact`` gives the same outputs in 64 bits.

Definitions:

* linear: ``y = act(x W^T + b) + r``; act is the identity, relu, gelu (by erf) or silu.
* layer norm: ``y = (x - mean) / sqrt(var + eps) * w + b`` over the last dim.
* 8-bit checkpoint of x: blocks of 32 along the last dim (the last one may be
  short); a block is held as integers ``q = rint(x / 2^e)`` (ties to even), e
  the smallest integer >= -126 with ``max|x| <= 127 * 2^e`` (-126 for a block
  of zeros). With ``checkpoint="int8"`` the forward result is that of x, and
  the gradients are those at the input that the checkpoint holds.

Training cases use smooth activations: at the kink of relu, a pre-activation
that rounds to the other side changes a gradient by a whole term in any
implementation. Relu is measured forward.
"""

import math

import torch

own = False

EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # one decoder query through an attention-sized projection: the smallest call, all latency
        linear("linear-1-token", 1, 256, 512, "bf16", "relu"),
        # one token through a wide layer with its residual: a 32 MB weight read once
        linear("linear-1-token-wide", 1, 4096, 4096, "bf16", "silu", residual=True),
        # training BEVFormer's feed-forward: 200 x 200 BEV queries, 256 -> 512
        linear("linear-bev-ffn-train", 40000, 256, 512, "bf16", "gelu", train=True),
        # value projection of 6 camera images' feature maps (6 x 30825 pixels), 256 -> 256
        linear("linear-value-proj", 184950, 256, 256, "bf16", "none"),
        # training a wide layer: where the matrix units are the bound
        linear("linear-wide-train", 8192, 4096, 8192, "bf16", "gelu", residual=True, train=True),
        # training Deformable-DETR's feed-forward in float32: 22223 queries, 256 -> 1024
        linear("linear-detr-ffn-train-f32", 22223, 256, 1024, "f32", "silu", train=True),
        # the norm of one token
        norm("norm-1-token", 1, 4096, "bf16"),
        # training the norm after BEVFormer's attention: short rows
        norm("norm-bev-train", 40000, 256, "bf16", train=True),
        # training the norm of a wide layer: long rows
        norm("norm-wide-train", 8192, 8192, "bf16", train=True),
        # the feed-forward of linear-bev-ffn-train with its input kept in 8 bits
        linear("checkpoint-bev-ffn-train", 40000, 256, 512, "bf16", "gelu", train=True, checkpoint=True),
        # odd sizes in float32, input kept in 8 bits
        linear("checkpoint-odd-train-f32", 2221, 771, 517, "f32", "silu", residual=True, train=True, checkpoint=True),
        # Deformable-DETR's norm (2 images) with its input kept in 8 bits
        norm("checkpoint-norm-train-f32", 44446, 256, "f32", train=True, checkpoint=True),
    ]


def linear(name, rows, k, n, dtype, act, residual=False, train=False, checkpoint=False):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act,
            "residual": residual, "train": train, "checkpoint": checkpoint}


def norm(name, rows, k, dtype, train=False, checkpoint=False):
    return {"name": name, "op": "norm", "rows": rows, "k": k, "dtype": dtype, "train": train,
            "checkpoint": checkpoint}


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "pack"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    train = rng.random() < 0.6
    checkpoint = train and rng.random() < 0.4
    if op == "linear":
        rows, k, n = spread(1, 184950), spread(24, 4096), spread(24, 8192)
        while rows * k * n > 8192 * 4096 * (4096 if dtype == "bf16" else 1024):
            rows = max(1, rows // 3)
        if rng.random() < 0.6:  # most layers have widths of whole vectors
            k, n = max(32, k // 32 * 32), max(32, n // 32 * 32)
        act = rng.choice(["none", "gelu", "silu"] if train else ["none", "relu", "gelu", "silu"])
        case = linear("", rows, k, n, dtype, act, rng.random() < 0.5, train, checkpoint)
    elif op == "norm":
        k = spread(24, 8192)
        rows = spread(1, min(184950, 8192 * 8192 // k // (1 if dtype == "bf16" else 2)))
        if rng.random() < 0.6:
            k = max(32, k // 32 * 32)
        case = norm("", rows, k, dtype, train, checkpoint)
    else:
        k = spread(24, 8192)
        case = {"op": "pack", "rows": spread(1, min(184950, 8192 * 4096 // k)), "k": k, "dtype": dtype}
    case.pop("name", None)
    return case


def _dtype(case):
    return {"bf16": torch.bfloat16, "f32": torch.float32}[case["dtype"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, k = _dtype(case), case["rows"], case["k"]
    train = case.get("train", False)

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(mean)

    x = normal(rows, k)
    if case["op"] != "linear":
        # a residual stream: rows of different scale, an offset, a few strong channels
        x *= torch.exp(normal(rows, 1, scale=0.5))
        x += 0.2
        x[:, :: max(1, k // 4)] *= 6.0
    state = {"case": case, "x": x.to(dtype)}
    if case["op"] == "linear":
        n = case["n"]
        state["w"] = normal(n, k, scale=k ** -0.5).to(dtype)
        state["b"] = normal(n, scale=0.1).to(dtype)
        state["r"] = normal(rows, n).to(dtype) if case["residual"] else None
        out = n
    elif case["op"] == "norm":
        state["w"] = normal(k, scale=0.2, mean=1.0).to(dtype)
        state["b"] = normal(k, scale=0.1).to(dtype)
        out = k
    if train:
        state["g"] = normal(rows, out).to(dtype)
        for name in ("x", "w", "b", "r"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's calls ----------------------------------------------------------


def _run_own(state):
    from muspace_b200.ops import checkpoint_pack, checkpoint_unpack, layer_norm, linear_act

    case, x = state["case"], state["x"]
    if case["op"] == "pack":
        return {"x": checkpoint_unpack(checkpoint_pack(x))}
    keep = "int8" if case["checkpoint"] else None
    if case["op"] == "linear":
        y = linear_act(x, state["w"], state["b"], state["r"], activation=case["act"], checkpoint=keep)
    else:
        y = layer_norm(x, state["w"], state["b"], eps=EPS, checkpoint=keep)
    if not case["train"]:
        return {"y": y}
    names = [m for m in ("x", "w", "b", "r") if state.get(m) is not None]
    grads = torch.autograd.grad(y, [state[m] for m in names], state["g"])
    return {"y": y, **{"d" + m: g for m, g in zip(names, grads)}}


# ---- the plain form ------------------------------------------------------------------


def _plain_act(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * torch.sigmoid(z) if name == "silu" else z


def _plain_slope(name, z):
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def _plain_kept(x):
    """What an 8-bit checkpoint of x (float32) holds."""
    rows, k = x.shape
    pad = -k % BLOCK
    blocks = torch.nn.functional.pad(x, (0, pad)).reshape(rows, -1, BLOCK)
    m, p = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 127 / 128, p - 7, p - 6).clamp(min=-126)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    q = torch.round(torch.ldexp(blocks, -e))
    return torch.ldexp(q, e).reshape(rows, -1)[:, :k]


def _run_plain(state):
    case, dtype = state["case"], state["x"].dtype
    with torch.no_grad():
        x = state["x"].float()
        if case["op"] == "pack":
            return {"x": _plain_kept(x).to(dtype)}
        outs = (_plain_linear if case["op"] == "linear" else _plain_norm)(case, state, x)
        return {m: v.to(dtype) for m, v in outs.items()}


def _plain_linear(case, state, x):
    w, b, r = state["w"].float(), state["b"].float(), state["r"]
    z = x @ w.t() + b
    y = _plain_act(case["act"], z)
    if r is not None:
        y = y + r.float()
    if not case["train"]:
        return {"y": y}
    if case["checkpoint"]:
        x = _plain_kept(x)
        z = x @ w.t() + b
    g = state["g"].float()
    dz = g if case["act"] == "none" else g * _plain_slope(case["act"], z)
    outs = {"y": y, "dx": dz @ w, "dw": dz.t() @ x, "db": dz.sum(0)}
    return outs if r is None else {**outs, "dr": g}


def _plain_norm(case, state, x):
    w, b = state["w"].float(), state["b"].float()

    def normalised(x):
        c = x - x.mean(-1, keepdim=True)
        scale = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
        return c * scale, scale

    h, scale = normalised(x)
    y = h * w + b
    if not case["train"]:
        return {"y": y}
    if case["checkpoint"]:
        h, scale = normalised(_plain_kept(x))
    g = state["g"].float()
    gw = g * w
    dx = scale * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx, "dw": (g * h).sum(0), "db": g.sum(0)}


# ---- 64 bits ---------------------------------------------------------------------------


def _held(x):
    """The 8-bit checkpoint by its definition, block by block of columns."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        top = part.abs().max(dim=1, keepdim=True).values
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 127))
        e = torch.where(top > 127 * torch.exp2(e), e + 1, e)  # the logarithm may be an ulp off
        e = torch.where(top <= 127 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        out[:, at:at + BLOCK] = torch.round(part / torch.exp2(e)) * torch.exp2(e)
    return out


def exact(case, seed):
    import torch.nn.functional as F

    state = {m: v.detach().double() if isinstance(v, torch.Tensor) else v for m, v in prepare(case, seed).items()}
    x = state["x"]
    if case["op"] == "pack":
        return {"x": _held(x)}
    acts = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}

    def forward(x, w, b):
        if case["op"] == "linear":
            return acts[case["act"]](F.linear(x, w, b))
        return F.layer_norm(x, (case["k"],), w, b, EPS)

    with torch.no_grad():
        y = forward(x, state["w"], state["b"])
        if state.get("r") is not None:
            y = y + state["r"]
    if not case["train"]:
        return {"y": y}
    leaves = [(_held(x) if case["checkpoint"] else x).requires_grad_(True),
              state["w"].requires_grad_(True), state["b"].requires_grad_(True)]
    dx, dw, db = torch.autograd.grad(forward(*leaves), leaves, state["g"])
    outs = {"y": y, "dx": dx, "dw": dw, "db": db}
    return outs if state.get("r") is None else {**outs, "dr": state["g"]}


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    rows, k = case["rows"], case["k"]
    if case["op"] == "pack":  # x in, codes and exponents out and in again, x out
        return {"bytes": 2 * rows * k * e + 2 * rows * (k + -(-k // BLOCK)), "flops": 4 * rows * k}
    if case["op"] == "norm":
        if not case["train"]:
            return {"bytes": (2 * rows * k + 2 * k) * e, "flops": 8 * rows * k}
        # x, g, w, b in; y, dx, dw, db out
        return {"bytes": (4 * rows * k + 4 * k) * e, "flops": 20 * rows * k}
    n = case["n"]
    data = rows * k + n * k + n + rows * n + (rows * n if case["residual"] else 0)  # x, w, b, r in; y out
    flops = 2 * rows * k * n
    if case["train"]:
        data += rows * n + rows * k + n * k + n  # g in; dx, dw, db out
        data += rows * n if case["residual"] else 0
        flops *= 3
    return {"bytes": data * e, "flops": flops}

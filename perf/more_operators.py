"""What the operators between a layer's blocks are measured on: dropout, norms
with the residual they belong to, and the gated feed-forward product.

Between the attention and the feed-forward of an encoder or decoder layer, and
between one layer and the next, a block's output is dropped out, scaled by a
gate, added to the residual stream and normalised (``dropout``, ``add_norm``,
``norm_add``); a gated feed-forward multiplies two projections of the same rows
(``gated_linear``).

``run`` computes a case in its plain form (``own`` false: elementary torch
operations in 32 bits, rounded once at the end) or by the framework's calls
(``own`` true). ``exact`` gives the same outputs in 64 bits.

Definitions (rows are those of the last dimension, counted over all others):

* Random bits: Philox-4x32 with ten rounds (Salmon and others, 2011), key
  ``(seed mod 2^32, seed div 2^32)``, counter ``(column div 8, row, sequence mod
  2^32, sequence div 2^32)``. Its four words are the 16-bit numbers of eight
  neighbouring columns, the low half of the first word first. An element is kept
  where its number is at least ``t = round(65536 p)``.
* dropout: ``D(x) = x * 65536 / (65536 - t)`` where kept, else 0.
* norm: ``(x - mean) / sqrt(var + eps) * w + b`` ("layer"), or ``x /
  sqrt(mean(x^2) + eps) * w + b`` ("rms").
* add_norm: ``s = alpha * r + gate * D(h)``, ``y = norm(s)``; s is an output where asked for.
* norm_add: ``s = alpha * r + gate * D(norm(h))``.
* gated_linear: ``D(act(x Wg^T + bg) * (x Wu^T + bu))``; the weight is Wg above Wu,
  the bias bg before bu; act is gelu (by erf) or silu.
"""

import math

import numpy as np
import torch

own = False

EPS = 1e-5


def listed():
    return [
        # dropout of one decoder query's features: the smallest call, all latency
        drop("dropout-1-query", 1, 256, "bf16", 0.1),
        # training: dropout inside BEVFormer's feed-forward, 200 x 200 BEV queries, 512 wide
        drop("dropout-bev-ffn-train", 40000, 512, "bf16", 0.1, train=True),
        # one token of a wide layer: the sum stays the residual stream, its norm enters the next block
        norm("add-norm-1-token", "add_norm", 1, 4096, "bf16", "rms", out_sum=True),
        # training BEVFormer's post-norm: attention output onto the BEV queries, dropout, norm
        norm("add-norm-bev-train", "add_norm", 40000, 256, "bf16", "layer", p=0.1, train=True),
        # training a wide pre-norm layer: a gate per channel, the sum and its norm both go on
        norm("add-norm-wide-train", "add_norm", 8192, 8192, "bf16", "rms", gate="channel", out_sum=True, train=True),
        # odd sizes in float32, everything on
        norm("add-norm-odd-train-f32", "add_norm", 2221, 771, "f32", "layer", p=0.25, gate="channel", alpha=1.5,
             out_sum=True, train=True),
        # training: normed branch of 6 camera images' feature rows (6 x 30825 pixels), a gate per image, float16
        norm("norm-add-cameras-train-f16", "norm_add", 184950, 256, "f16", "layer", p=0.1, gate="image", images=6,
             train=True),
        # 900 decoder queries of a detection head
        norm("norm-add-900-queries", "norm_add", 900, 256, "f32", "layer", gate="channel"),
        # one token through a wide gated layer: a 64 MB weight read once
        gated("gated-1-token-wide", 1, 4096, 4096, "bf16", "silu"),
        # training a gated feed-forward on BEVFormer's queries, with dropout inside
        gated("gated-bev-ffn-train", 40000, 256, 512, "bf16", "gelu", p=0.1, train=True),
        # training a wide gated layer: where the matrix units are the bound
        gated("gated-wide-train", 8192, 4096, 4096, "bf16", "silu", train=True),
        # training a gated feed-forward on Deformable-DETR's 22223 queries in float32
        gated("gated-detr-ffn-train-f32", 22223, 256, 512, "f32", "silu", train=True),
    ]


def drop(name, rows, n, dtype, p, train=False):
    return {"name": name, "op": "dropout", "rows": rows, "n": n, "dtype": dtype, "p": p, "train": train}


def norm(name, op, rows, n, dtype, kind, p=0.0, gate="none", images=1, alpha=1.0, out_sum=False, train=False):
    return {"name": name, "op": op, "rows": rows, "n": n, "dtype": dtype, "kind": kind, "p": p, "gate": gate,
            "images": images, "alpha": alpha, "out_sum": out_sum, "train": train}


def gated(name, rows, k, n, dtype, act, p=0.0, train=False):
    return {"name": name, "op": "gated", "rows": rows, "k": k, "n": n, "dtype": dtype, "act": act, "p": p,
            "train": train}


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))

    op = rng.choice(["dropout", "add_norm", "add_norm", "norm_add", "gated", "gated"])
    train = rng.random() < 0.6
    p = rng.choice([0.0, 0.1, 0.1, 0.25, 0.5])
    if op == "gated":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        rows, k, n = spread(1, 184950), spread(24, 4096), spread(24, 4096)
        while rows * k * n > 8192 * 4096 * (4096 if dtype == "bf16" else 512):
            rows = max(1, rows // 3)
        if rng.random() < 0.6:  # most layers have widths of whole vectors
            k, n = max(32, k // 32 * 32), max(32, n // 32 * 32)
        case = gated("", rows, k, n, dtype, rng.choice(["gelu", "silu"]), p, train)
    else:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        n = spread(24, 8192)
        if rng.random() < 0.6:
            n = max(32, n // 32 * 32)
        rows = spread(1, min(184950, 8192 * 8192 // n // (2 if dtype == "f32" else 1)))
        if op == "dropout":
            case = drop("", rows, n, dtype, p or 0.1, train)
        else:
            gate, images = rng.choice(["none", "channel", "image", "full"]), 1
            if gate == "image":
                images = rng.choice([2, 3, 6])
                rows = max(1, rows // images) * images
            if gate == "full":
                rows = max(1, rows // 2)
            case = norm("", op, rows, n, dtype, rng.choice(["layer", "rms"]), p, gate, images,
                        rng.choice([1.0, 1.0, 1.5]), op == "add_norm" and rng.random() < 0.6, train)
    case.pop("name", None)
    return case


def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, n = _dtype(case), case["rows"], case["n"]
    train = case["train"]
    # a program counts its steps in the seed and its dropouts in the sequence
    state = {"case": case, "seed": 1234567890123 + 977 * seed, "sequence": 3 + seed % 5}

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(mean)

    if case["op"] == "dropout":
        state["x"] = normal(rows, n).to(dtype)
        names = ["x"]
    elif case["op"] == "gated":
        k = case["k"]
        state["x"] = normal(rows, k).to(dtype)
        state["w"] = normal(2 * n, k, scale=k ** -0.5).to(dtype)
        state["b"] = normal(2 * n, scale=0.1).to(dtype)
        names = ["x", "w", "b"]
    else:
        images = case["images"]
        shape = (images, rows // images, n) if images > 1 else (rows, n)
        # a residual stream: rows of different scale, an offset, a few strong channels
        r = normal(*shape)
        r *= torch.exp(normal(*shape[:-1], 1, scale=0.5))
        r += 0.2
        r[..., :: max(1, n // 4)] *= 6.0
        state["h"], state["r"] = normal(*shape).to(dtype), r.to(dtype)
        state["w"] = normal(n, scale=0.2, mean=1.0).to(dtype)
        state["b"] = normal(n, scale=0.1).to(dtype)
        names = ["h", "r", "w", "b"]
        if case["gate"] != "none":
            gate_shape = {"channel": (n,), "image": (images, 1, n), "full": shape}[case["gate"]]
            state["gate"] = normal(*gate_shape, scale=0.3, mean=0.7).to(dtype)
            names.append("gate")
    if train:
        out_shape = (*state["x"].shape[:-1], n) if "x" in state else shape
        state["g"] = normal(*out_shape).to(dtype)
        if case.get("out_sum"):
            state["gs"] = normal(*out_shape).to(dtype)
        for name in names:
            state[name].requires_grad_(True)
    state["names"] = names
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the framework's calls ----------------------------------------------------------


def _run_own(state):
    from muspace_b200.ops import add_norm, dropout, gated_linear, norm_add

    case = state["case"]
    if case["op"] == "dropout":
        y = dropout(state["x"], case["p"], seed=state["seed"], sequence=state["sequence"])
    elif case["op"] == "gated":
        y = gated_linear(state["x"], state["w"], state["b"], activation=case["act"], dropout=case["p"],
                         seed=state["seed"], sequence=state["sequence"])
    else:
        how = {"gate": state.get("gate"), "residual_scale": case["alpha"], "kind": case["kind"], "eps": EPS,
               "dropout": case["p"], "seed": state["seed"], "sequence": state["sequence"]}
        if case["op"] == "add_norm":
            y = add_norm(state["h"], state["r"], state["w"], state["b"], return_sum=case["out_sum"], **how)
        else:
            y = norm_add(state["h"], state["r"], state["w"], state["b"], **how)
    y, s = y if case.get("out_sum") else (y, None)
    outs = {"y": y} if s is None else {"y": y, "s": s}
    if not case["train"]:
        return outs
    leaves = [state[m] for m in state["names"]]
    grads = torch.autograd.grad([*outs.values()], leaves, [state["g"]] if s is None else [state["g"], state["gs"]])
    return {**outs, **{"d" + m: g for m, g in zip(state["names"], grads)}}


# ---- the plain form ------------------------------------------------------------------


def _plain_kept(rows, n, p, seed, sequence, device):
    """Which elements are kept, as a mask [rows, n], and what they are multiplied by."""
    t = round(65536 * p)
    low = 0xFFFFFFFF
    c0 = torch.arange(-(-n // 8), device=device)[None, :].expand(rows, -1)
    c1 = torch.arange(rows, device=device)[:, None].expand_as(c0)
    c2 = torch.full_like(c0, sequence & low)
    c3 = torch.full_like(c0, sequence >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):  # products of 32 bits wrap in int64, their bits are right
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    numbers = torch.stack([half for c in (c0, c1, c2, c3) for half in (c & 0xFFFF, c >> 16)], -1)
    return numbers.reshape(rows, -1)[:, :n] >= t, 65536 / (65536 - t)


def _plain_dropper(state, rows, n):
    """D of [rows, n], and of a gradient."""
    case = state["case"]
    if not case["p"]:
        return lambda v: v
    device = state[state["names"][0]].device
    kept, scale = _plain_kept(rows, n, case["p"], state["seed"], state["sequence"], device)
    return lambda v: torch.where(kept, v.reshape(rows, n) * scale, 0.0).reshape(v.shape)


def _plain_norm(kind, x):
    """The normalised rows, and their scale."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    scale = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * scale, scale


def _plain_norm_grad(kind, d, normed, scale):
    """The gradient of a norm's input, of that at its normalised rows."""
    along = normed * (d * normed).mean(-1, keepdim=True)
    return scale * (d - along - (d.mean(-1, keepdim=True) if kind == "layer" else 0))


def _plain_act(name, z):
    """Value and slope."""
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def _sum_to(v, shape):
    """The sums of v over what is broadcast from `shape`."""
    over = [i for i in range(v.dim()) if i - v.dim() + len(shape) < 0 or shape[i - v.dim() + len(shape)] != v.shape[i]]
    return (v.sum(over, keepdim=True) if over else v).reshape(shape)


def _run_plain(state):
    case = state["case"]
    with torch.no_grad():
        outs = {"dropout": _plain_dropout, "gated": _plain_gated}.get(case["op"], _plain_residual)(case, state)
        return {m: v.to(_dtype(case)) for m, v in outs.items()}


def _plain_dropout(case, state):
    dropped = _plain_dropper(state, case["rows"], case["n"])
    outs = {"y": dropped(state["x"].float())}
    if case["train"]:
        outs["dx"] = dropped(state["g"].float())
    return outs


def _plain_residual(case, state):
    h, r, w, b = (state[m].float() for m in ("h", "r", "w", "b"))
    gate = state["gate"].float() if "gate" in state else None
    alpha, kind, n = case["alpha"], case["kind"], case["n"]
    dropped = _plain_dropper(state, case["rows"], n)
    gated_by = (lambda v: v) if gate is None else (lambda v: v * gate)
    if case["op"] == "add_norm":
        branch = dropped(h)
        s = alpha * r + gated_by(branch)
        normed, scale = _plain_norm(kind, s)
        outs = {"y": normed * w + b}
        if case["out_sum"]:
            outs["s"] = s
        if not case["train"]:
            return outs
        g = state["g"].float()
        ds = _plain_norm_grad(kind, g * w, normed, scale)
        if case["out_sum"]:
            ds = ds + state["gs"].float()
        outs.update(dh=dropped(gated_by(ds)), dr=alpha * ds, dw=_sum_to(g * normed, w.shape), db=_sum_to(g, b.shape))
    else:
        normed, scale = _plain_norm(kind, h)
        branch = dropped(normed * w + b)
        outs = {"y": alpha * r + gated_by(branch)}
        if not case["train"]:
            return outs
        ds = state["g"].float()
        d = dropped(gated_by(ds))
        outs.update(dh=_plain_norm_grad(kind, d * w, normed, scale), dr=alpha * ds, dw=_sum_to(d * normed, w.shape),
                    db=_sum_to(d, b.shape))
    if gate is not None:
        outs["dgate"] = _sum_to(ds * branch, gate.shape)
    return outs


def _plain_gated(case, state):
    x, w, b = (state[m].float() for m in ("x", "w", "b"))
    n = case["n"]
    z = x @ w.t() + b
    y, slope = _plain_act(case["act"], z[:, :n])
    dropped = _plain_dropper(state, case["rows"], n)
    outs = {"y": dropped(y * z[:, n:])}
    if case["train"]:
        g = dropped(state["g"].float())
        dz = torch.cat([g * z[:, n:] * slope, g * y], 1)
        outs.update(dx=dz @ w, dw=dz.t() @ x, db=dz.sum(0))
    return outs


# ---- 64 bits ---------------------------------------------------------------------------


def _factors(rows, n, p, seed, sequence, device):
    """0 or the scale for each element: the generator by its definition, in numpy."""
    threshold = round(65536 * p)
    word = np.uint64(0xFFFFFFFF)
    groups = (n + 7) // 8
    at = np.arange(rows * groups, dtype=np.uint64)
    x = [at % np.uint64(groups), at // np.uint64(groups), np.full_like(at, sequence % 2 ** 32),
         np.full_like(at, sequence // 2 ** 32)]
    key = [seed % 2 ** 32, seed // 2 ** 32]
    for _ in range(10):
        one, two = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(two >> np.uint64(32)) ^ x[1] ^ np.uint64(key[0]), two & word,
             (one >> np.uint64(32)) ^ x[3] ^ np.uint64(key[1]), one & word]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    numbers = np.stack(x, 1).astype("<u4").view("<u2").reshape(rows, groups * 8)[:, :n]
    kept = torch.from_numpy(np.ascontiguousarray(numbers >= threshold)).to(device)
    return kept.double() * (65536 / (65536 - threshold))


def exact(case, seed):
    import torch.nn.functional as F

    state = prepare(case, seed)
    shape = (*state["x" if "x" in state else "h"].shape[:-1], case["n"])
    factors = 1.0
    if case["p"]:
        factors = _factors(case["rows"], case["n"], case["p"], state["seed"], state["sequence"], "cuda").reshape(shape)
    names = state["names"]
    leaves = {m: state[m].detach().double().requires_grad_(case["train"]) for m in names}

    def normed(x):
        w, b = leaves["w"], leaves["b"]
        if case["kind"] == "layer":
            return F.layer_norm(x, (case["n"],), w, b, EPS)
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w + b

    if case["op"] == "dropout":
        outs = {"y": leaves["x"] * factors}
    elif case["op"] == "gated":
        gate, up = F.linear(leaves["x"], leaves["w"], leaves["b"]).chunk(2, -1)
        outs = {"y": getattr(F, case["act"])(gate) * up * factors}
    else:
        gate = leaves.get("gate", 1.0)
        if case["op"] == "add_norm":
            s = case["alpha"] * leaves["r"] + gate * (leaves["h"] * factors)
            outs = {"y": normed(s), "s": s} if case["out_sum"] else {"y": normed(s)}
        else:
            outs = {"y": case["alpha"] * leaves["r"] + gate * (normed(leaves["h"]) * factors)}
    if not case["train"]:
        return outs
    seeds = [state["g"].double()] + ([state["gs"].double()] if "s" in outs else [])
    grads = torch.autograd.grad([*outs.values()], [leaves[m] for m in names], seeds)
    return {**{m: v.detach() for m, v in outs.items()}, **{"d" + m: g for m, g in zip(names, grads)}}


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    rows, n = case["rows"], case["n"]
    if case["op"] == "dropout":  # x in, y out; g in, dx out
        return {"bytes": (4 if case["train"] else 2) * rows * n * e, "flops": (4 if case["train"] else 2) * rows * n}
    if case["op"] == "gated":
        k = case["k"]
        data, flops = rows * k + 2 * n * k + 2 * n + rows * n, 4 * rows * k * n  # x, w, b in; y out
        if case["train"]:  # g in; dx, dw, db out
            data, flops = data + rows * n + rows * k + 2 * n * k + 2 * n, 3 * flops
        return {"bytes": data * e, "flops": flops}
    gate = {"none": 0, "channel": n, "image": case["images"] * n, "full": rows * n}[case["gate"]]
    out = 2 if case["out_sum"] else 1
    data, flops = (2 + out) * rows * n + 2 * n + gate, 12 * rows * n  # h, r, w, b, gate in; y, s out
    if case["train"]:  # g, gs in; dh, dr, dw, db, dgate out
        data, flops = data + (out + 2) * rows * n + 2 * n + gate, 32 * rows * n
    return {"bytes": data * e, "flops": flops}

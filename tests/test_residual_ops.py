"""dropout, add_norm and norm_add against plain 64-bit formulas.

Masks are compared exactly with the generator written in numpy. Tolerances, per
element, from the arithmetic: an output is rounded once to its type; before that it
carries errors of float32 arithmetic, taken as 2^-20 of the sum of the magnitudes of
its terms (as in test_layer_ops, from which `near` comes). A sum s is off by 2^-20
of |alpha r| + |gate D(h)| =: size at most, its mean by the row's largest such
error, and rstd, relatively, by rstd times it; so a normalised value k is off by
2^-20 rstd (size + max size) (1 + |k|). The gradients of add_norm are those at s as it
is stored, in its type.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from muspace_b200 import clear_dispatch_report, get_last_dispatch_report
from muspace_b200.ops import add_norm, dropout, gated_linear, layer_norm, norm_add
from muspace_b200.runtime import native
import test_layer_ops
from test_layer_ops import BF16, F16, F32, SUM

DTYPES = [BF16, F16, F32]
IDS = ["bf16", "f16", "f32"]
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
# half of float16's smallest step: numbers below 2^-14 are that far apart, however small; the other types' is below 2^-130
LEAST = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}


def near(got, expected, terms, dtype):
    test_layer_ops.near(got, expected, terms + LEAST[dtype] / SUM, dtype)


# ---- 64-bit formulas ------------------------------------------------------------------


def philox(counter, key):
    """Ten rounds of Philox-4x32 on arrays of uint64 that hold 32 bits."""
    x, k, word = list(counter), list(key), np.uint64(0xFFFFFFFF)
    for _ in range(10):
        one, two = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(two >> np.uint64(32)) ^ x[1] ^ np.uint64(k[0]), two & word,
             (one >> np.uint64(32)) ^ x[3] ^ np.uint64(k[1]), one & word]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return x


def factors(rows, n, p, seed, sequence, first_row=0):
    """0 or the scale for each element [rows, n], rows counted from `first_row`."""
    threshold, groups = round(65536 * p), -(-n // 8)
    at = np.arange(rows * groups, dtype=np.uint64)
    x = philox([at % np.uint64(groups), at // np.uint64(groups) + np.uint64(first_row),
                np.full_like(at, sequence % 2 ** 32), np.full_like(at, sequence // 2 ** 32)],
               [seed % 2 ** 32, seed // 2 ** 32])
    numbers = np.stack([half for w in x for half in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1)
    kept = torch.from_numpy(numbers.reshape(rows, groups * 8)[:, :n] >= threshold)
    return kept.double() * (65536 / max(65536 - threshold, 1))


def test_generator_known_answers():
    """The published vectors of Philox-4x32-10."""
    zero = [np.zeros(1, np.uint64)] * 4
    assert [int(w[0]) for w in philox(zero, [0, 0])] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = [np.full(1, 0xFFFFFFFF, np.uint64)] * 4
    assert [int(w[0]) for w in philox(ones, [0xFFFFFFFF] * 2)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def normed64(kind, x, eps=1e-5):
    c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    return c * rstd, rstd


def norm_grad64(kind, d, k, rstd):
    """The gradient of a norm's input from d, that of its normalised rows, and the size of its terms."""
    m1 = d.mean(-1, keepdim=True) if kind == "layer" else 0
    m2 = (d * k).mean(-1, keepdim=True)
    size = rstd * (d.abs() + d.abs().mean(-1, keepdim=True) + k.abs() * (d * k).abs().mean(-1, keepdim=True))
    return rstd * (d - m1 - k * m2), size, m2


def summed(v, shape):
    v = v.reshape(*([1] * (len(shape) - v.dim())), *v.shape)
    over = [i for i in range(v.dim()) if i < v.dim() - len(shape) or shape[i - v.dim() + len(shape)] != v.shape[i]]
    return (v.sum(over, keepdim=True) if over else v).reshape(shape)


def inputs(shape, dtype, device, gate=None, seed=0, param=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    n, param = shape[-1], param or dtype
    out = {"h": r(*shape), "r": r(*shape) * torch.exp(0.5 * r(*shape[:-1], 1)) + 0.2, "w": 1 + 0.2 * r(n), "b": 0.1 * r(n),
           "gy": r(*shape), "gs": r(*shape)}
    if gate is not None:
        out["gate"] = 0.7 + 0.3 * r(*gate)
    return {m: t.to(param if m in ("w", "b", "gate") else dtype).to(device) for m, t in out.items()}


SEED, SEQUENCE = 2 ** 45 + 12345, 2 ** 33 + 7


def check(op, data, kind="layer", p=0.25, alpha=1.5, want_sum=True, use=("y", "s"), need="hrwbG", seed=SEED, eps=1e-5):
    """Forward and backward of one call against the formulas; returns outputs and gradients."""
    h, dtype = data["h"], data["h"].dtype
    shape, n = h.shape, h.shape[-1]
    rows = h.numel() // max(n, 1)
    names = {"h": "h", "r": "r", "w": "w", "b": "b", "G": "gate"}
    names = {c: m for c, m in names.items() if data.get(m) is not None}
    t = {m: data[m].detach().requires_grad_(c in need) for c, m in names.items()}
    how = dict(gate=t.get("gate"), residual_scale=alpha, kind=kind, dropout=p, seed=seed, sequence=SEQUENCE, eps=eps)
    if op == "add_norm":
        got = add_norm(t["h"], t["r"], t.get("w"), t.get("b"), return_sum=want_sum, **how)
        got = dict(zip("ys", got)) if want_sum else {"y": got}
    else:
        got = {"s": norm_add(t["h"], t["r"], t.get("w"), t.get("b"), **how)}
    x = {m: v.detach().double() for m, v in t.items()}
    f = factors(rows, n, p, int(seed), SEQUENCE).to(h.device).reshape(shape) if p else torch.ones(shape, device=h.device).double()
    w, b, gate = x.get("w", torch.ones(n, device=h.device).double()), x.get("b", torch.zeros(n, device=h.device).double()), x.get("gate", torch.ones((), device=h.device).double())
    r = x["r"].expand(shape)
    used = {m: data["g" + m].double() for m in use if m in got}
    if op == "add_norm":
        branch = x["h"] * f
        s = alpha * r + gate * branch
        size = (alpha * r).abs() + (gate * branch).abs()
        k, rstd = normed64(kind, s, eps)
        top = size.amax(-1, keepdim=True) if n else size
        off = rstd * (size + top) * (1 + k.abs())  # of k, over 2^-20
        near(got["y"].detach(), k * w + b, off * w.abs() + (k * w).abs() + b.abs(), dtype)
        if want_sum:
            near(got["s"].detach(), s, size, dtype)
        with torch.no_grad():  # the sum as it is stored
            s = (got["s"] if want_sum else add_norm(t["h"], t["r"], return_sum=True, **how)[1]).double()
        size = s.abs()
        k, rstd = normed64(kind, s, eps)
        top = size.amax(-1, keepdim=True) if n else size
        off = SUM * rstd * (size + top) * (1 + k.abs())
        ds, loose = torch.zeros_like(s), torch.zeros_like(s)
        expected, terms = {}, {}
        if "y" in used:
            g = used["y"]
            ds, ds_size, m2 = norm_grad64(kind, g * w, k, rstd)
            loose = rstd * (off * m2.abs() + k.abs() * ((g * w).abs() * off).mean(-1, keepdim=True))
            loose = loose + SUM * ds_size * (2 + rstd * top)
            expected["w"], terms["w"] = summed(g * k, (n,)), summed((g * k).abs() + g.abs() * off / SUM, (n,))
            expected["b"], terms["b"] = summed(g, (n,)), summed(g.abs(), (n,))
        if "s" in used:
            ds, loose = ds + used["s"], loose + SUM * used["s"].abs()
        loose = loose / SUM + ds.abs()
        # a broadcast residual: the rows' gradients are rounded before they are summed
        rounds = 1 + (x["r"].shape != shape) * HALF[dtype] / SUM
        expected.update(h=gate * f * ds, r=summed(alpha * ds, x["r"].shape))
        terms.update(h=(gate * f).abs() * loose, r=summed(abs(alpha) * loose * rounds, x["r"].shape))
        if "gate" in x:
            expected["G"], terms["G"] = summed(ds * branch, gate.shape), summed(loose * branch.abs(), gate.shape)
    else:
        k, rstd = normed64(kind, x["h"], eps)
        top = x["h"].abs().amax(-1, keepdim=True) if n else x["h"].abs()
        off = rstd * 2 * top * (1 + k.abs())
        normal = k * w + b
        branch = normal * f
        normal_size = (off * w.abs() + (k * w).abs() + b.abs()) * f
        s = alpha * r + gate * branch
        near(got["s"].detach(), s, (alpha * r).abs() + gate.abs() * normal_size, dtype)
        g = used["s"]
        d = gate * f * g
        dh, dh_size, m2 = norm_grad64(kind, d * w, k, rstd)
        loose = rstd * (off * m2.abs() + k.abs() * ((d * w).abs() * off).mean(-1, keepdim=True))
        expected = {"h": dh, "r": summed(alpha * g, x["r"].shape), "w": summed(d * k, (n,)), "b": summed(d, (n,))}
        rounds = 1 + (x["r"].shape != shape) * HALF[dtype] / SUM
        terms = {"h": loose + dh_size * (2 + rstd * top), "r": summed((alpha * g).abs() * rounds, x["r"].shape),
                 "w": summed((d * k).abs() + d.abs() * off, (n,)), "b": summed(d.abs(), (n,))}
        if "gate" in x:
            expected["G"], terms["G"] = summed(g * branch, gate.shape), summed(g.abs() * normal_size, gate.shape)
    leaves = {c: t[m] for c, m in names.items() if c in need and (c in expected)}
    grads = {}
    if used and leaves:
        grads = dict(zip(leaves, torch.autograd.grad([got[m] for m in used], [*leaves.values()],
                                                     [data["g" + m] for m in used])))
    for c, value in grads.items():
        near(value, expected[c], terms[c], leaves[c].dtype)
    return {m: v.detach() for m, v in got.items()}, grads


# ---- dropout ------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 256), (3, 7), (1, 4099), (129, 64), (1000, 257), (40, 1000), (3000, 512),
                                    (2, 2500007), (1, 2500008), (100000, 3)])
def test_dropout_is_the_generator(cuda_device, rows, n, dtype):
    gen = torch.Generator().manual_seed(n)
    x, g = (torch.randn(rows, n, generator=gen).to(dtype).to(cuda_device) for _ in range(2))
    for p, seed, sequence in ((0.1, SEED, SEQUENCE), (0.5, 0, 0), (0.97, 2 ** 63 - 1, 2 ** 63 - 1)):
        f = factors(rows, n, p, seed, sequence).to(cuda_device)
        leaf = x.clone().requires_grad_(True)
        y = dropout(leaf, p, seed=seed, sequence=sequence)
        (d,) = torch.autograd.grad(y, [leaf], g)
        for got, of in ((y.detach(), x), (d, g)):
            assert got.dtype == dtype and torch.equal(got == 0, (f == 0) | (of == 0))
            # one product with the scale rounded to float32, one rounding to the type
            assert bool(((got.double() - of.double() * f).abs() <= (of.double() * f).abs() * (HALF[dtype] + 2.0 ** -23)
                        + LEAST[dtype]).all())


@pytest.mark.gpu
def test_dropout_of_nothing_and_of_everything(cuda_device):
    x = torch.randn(70, 300, device=cuda_device, dtype=BF16)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    assert torch.equal(dropout(x, 0.0, seed=1).nan_to_num(7.0), x.nan_to_num(7.0))
    assert torch.equal(dropout(x, 2.0 ** -18, seed=1).nan_to_num(7.0), x.nan_to_num(7.0))  # to the nearest 2^-16
    leaf = x.clone().requires_grad_(True)
    y = dropout(leaf, 1.0, seed=1)
    assert not bool(y.any()) and not bool(torch.autograd.grad(y, [leaf], x)[0].any())
    bad = torch.full((50, 64), float("inf"), device=cuda_device)
    y = dropout(bad, 0.5, seed=3)
    f = factors(50, 64, 0.5, 3, 0).to(cuda_device)
    assert torch.equal(y == 0, f == 0) and torch.equal(y == math.inf, f > 0)
    assert torch.equal(dropout(bad * float("nan"), 0.5, seed=3).isnan(), f > 0)
    for shape in ((0, 8), (5, 0), (0, 0), (2, 0, 3)):
        leaf = torch.empty(shape, device=cuda_device, requires_grad=True)
        y = dropout(leaf, 0.3, seed=2)
        assert y.shape == shape and torch.autograd.grad(y, [leaf], torch.empty(shape, device=cuda_device))[0].shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_strides_and_shapes(cuda_device, dtype):
    wide = torch.randn(70, 301, device=cuda_device).to(dtype)
    for x in (wide[:, 5:105], wide[::2, :100], wide.T, wide[:1, :64].expand(35, 64), wide[:, 1:65], wide[0]):
        want = dropout(x.clone(memory_format=torch.contiguous_format), 0.3, seed=5)
        assert torch.equal(dropout(x, 0.3, seed=5), want)
    x = torch.randn(3, 4, 5, 40, device=cuda_device).to(dtype)
    y = dropout(x, 0.3, seed=5)
    assert torch.equal(y.view(60, 40), dropout(x.view(60, 40), 0.3, seed=5))
    assert torch.equal(dropout(x.permute(2, 0, 1, 3), 0.3, seed=5), dropout(x.permute(2, 0, 1, 3).contiguous(), 0.3, seed=5))
    leaf = x.clone().requires_grad_(True)
    dropout(leaf, 0.3, seed=5).sum().backward()  # an expanded gradient
    assert torch.equal(leaf.grad, dropout(torch.ones_like(x), 0.3, seed=5))


@pytest.mark.gpu
def test_dropout_rate_and_independence(cuda_device):
    """Counts within five standard deviations; sequences, seeds and rows differ."""
    rows, n = 4000, 1000
    x = torch.ones(rows, n, device=cuda_device)
    kept = [dropout(x, 0.1, seed=s, sequence=q) != 0 for s, q in ((1, 0), (1, 1), (2, 0))]
    t = round(65536 * 0.1) / 65536
    for k in kept:
        assert abs(float(k.double().mean()) - (1 - t)) <= 5 * math.sqrt(t * (1 - t) / (rows * n))
        columns = k.double().mean(0)
        assert float((columns - (1 - t)).abs().max()) <= 6 * math.sqrt(t * (1 - t) / rows)
    for a, b in ((0, 1), (0, 2), (1, 2)):
        both = float((kept[a] & kept[b]).double().mean())
        assert abs(both - (1 - t) ** 2) <= 5 * math.sqrt((1 - t) ** 2 * (1 - (1 - t) ** 2) / (rows * n))


@pytest.mark.gpu
def test_dropout_past_two_to_the_31_elements(cuda_device):
    rows, n = 263000, 8200  # 2.16e9 elements
    x = torch.randn(rows, n, device=cuda_device, dtype=BF16)
    y = dropout(x, 0.5, seed=11, sequence=4)
    f = factors(50, n, 0.5, 11, 4, first_row=rows - 50).to(cuda_device)
    last = x[-50:].double()
    assert torch.equal(y[-50:].double(), last * f)  # the scale is 2
    w = torch.randn(n, device=cuda_device, dtype=BF16)
    leaf = x.requires_grad_(True)
    out = norm_add(leaf, y, w, dropout=0.5, seed=11, sequence=4)
    k, rstd = normed64("layer", last)
    branch = k * w.double() * f
    terms = rstd * 2 * last.abs().amax(-1, keepdim=True) * (1 + k.abs()) * w.double().abs() * f + branch.abs()
    near(out[-50:].detach(), y[-50:].double() + branch, terms + y[-50:].double().abs(), BF16)
    del out
    (d,) = torch.autograd.grad(add_norm(leaf, y, w), [leaf], x.detach())
    # a layer norm's gradient sums to 0 over a row, but for its rounding
    assert bool(d[-50:].any(-1).all()) and bool((d[-50:].double().sum(-1).abs() <= 2.0 ** -8 * d[-50:].double().abs().sum(-1)).all())


@pytest.mark.gpu
def test_dropout_seed_on_the_device(cuda_device):
    x = torch.randn(100, 96, device=cuda_device, dtype=BF16)
    seed = torch.tensor(SEED, device=cuda_device)
    assert torch.equal(dropout(x, 0.4, seed=seed, sequence=3), dropout(x, 0.4, seed=SEED, sequence=3))
    assert torch.equal(dropout(x, 0.4, seed=seed.view(1), sequence=3), dropout(x, 0.4, seed=SEED, sequence=3))
    leaf = x.clone().requires_grad_(True)
    y = dropout(leaf, 0.4, seed=seed)
    (d,) = torch.autograd.grad(y, [leaf], x)
    assert torch.equal(d, dropout(x, 0.4, seed=SEED))
    y = dropout(leaf, 0.4, seed=seed)
    seed += 1  # a mask that can no longer be made again
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [leaf], x)


@pytest.mark.gpu
def test_captured_training_step_draws_anew(cuda_device):
    """A captured forward and backward with the seed on the device: each replay has the masks of its seed."""
    data = inputs((200, 96), F32, cuda_device, gate=(96,))
    seed = torch.zeros((), dtype=torch.int64, device=cuda_device)
    leaves = [data[m].requires_grad_(True) for m in ("h", "r", "w", "b", "gate")]

    def step(seed):
        h, r, w, b, gate = leaves
        y = norm_add(dropout(h, 0.2, seed=seed), r, w, b, gate=gate, dropout=0.3, seed=seed, sequence=1)
        y, s = add_norm(y, r, w, b, dropout=0.3, seed=seed, sequence=2, return_sum=True)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [data["gy"], data["gs"]])]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(seed)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(seed)
    for value in (5, 6):
        seed.fill_(value)
        graph.replay()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step(value)):
            assert torch.equal(a, b)


# ---- norms with their residual ---------------------------------------------------------------


SHAPES = [(1, 1), (1, 256), (5, 3), (17, 40), (900, 256), (129, 257), (300, 512), (77, 771), (40, 1024), (33, 1600),
          (20, 2056), (9, 4096), (400, 4000), (7, 5001), (12, 8192), (3, 8200), (4, 9001)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_norms_match_the_formulas(cuda_device, shape, op, kind, dtype):
    check(op, inputs(shape, dtype, cuda_device, gate=shape[-1:], seed=sum(shape)), kind)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("shape,gate", [((1300, 1032), None), ((2369, 2048), (2048,)), ((1250, 4096), (4096,)),
                                        ((1190, 8192), None), ((6, 400, 2000), (6, 1, 2000)), ((5, 301, 4104), (5, 301, 4104)),
                                        ((300, 5, 1040), (300, 1, 1040)), ((1185, 5000), (5000,))])
def test_many_long_rows(cuda_device, shape, gate, op, dtype):
    """Several rows to each block, and several blocks to a sample."""
    data = inputs(shape, dtype, cuda_device, gate=gate)
    check(op, data)
    check(op, data, kind="rms", p=0.0, alpha=1.0)
    if op == "add_norm":
        check(op, data, use=("y",), need="hrwb")
        check(op, data, use=("s",))
        check(op, data, use=("y",), need="wb")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("n", [64, 100, 513, 1024, 2500, 9000])
def test_gates(cuda_device, n, op, dtype):
    """Per channel, per sample, per row, one per element, one per row, and broadcast along the first dimension."""
    shape = (3, 11, n)
    for gate in ((n,), (1, n), (1, 1, n), (3, 1, n), (3, 11, n), (3, 11, 1), (3, 1, 1), (11, n), (1, 11, n), (1,), ()):
        check(op, inputs(shape, dtype, cuda_device, gate=gate, seed=n))
    check(op, inputs((2, 3, 5, n), dtype, cuda_device, gate=(2, 3, 1, n)))
    check(op, inputs((2, 3, 5, n), dtype, cuda_device, gate=(2, 1, 5, n)))
    check(op, inputs((9, 1, n), dtype, cuda_device, gate=(9, 1, n)))
    check(op, inputs((n,), dtype, cuda_device, gate=(n,)))


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("groups,per", [(700, 2), (40, 9), (3, 400), (2, 1500)])
def test_gates_of_many_samples(cuda_device, groups, per, op):
    check(op, inputs((groups, per, 72), F32, cuda_device, gate=(groups, 1, 72)))
    check(op, inputs((groups, per, 600), BF16, cuda_device, gate=(groups, 1, 600)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("n", [256, 90, 1500])
def test_without_this_or_that(cuda_device, n, op, dtype):
    """No weight, no bias, no gate, no dropout, no scale; float32 parameters beside narrow rows."""
    full = inputs((60, n), dtype, cuda_device, gate=(n,), seed=n)
    for leave in (("w",), ("b",), ("w", "b"), ("gate",), ("w", "b", "gate")):
        check(op, {m: v for m, v in full.items() if m not in leave})
    plain = {m: v for m, v in full.items() if m != "gate"}
    check(op, plain, p=0.0, alpha=1.0)
    check(op, plain, p=0.0, alpha=-0.5, kind="rms")
    check(op, plain, p=1.0, alpha=2.0)
    check(op, inputs((60, n), dtype, cuda_device, gate=(n,), param=F32))
    mixed = inputs((60, n), dtype, cuda_device, gate=(n,), param=F32)
    check(op, {**mixed, "gate": mixed["gate"].to(dtype)})
    check(op, {**full, "gate": full["gate"].float()})
    check(op, {**full, "gate": torch.randn(60, n, device=cuda_device)})


@pytest.mark.gpu
@pytest.mark.parametrize("op,gate", [("add_norm", (64,)), ("norm_add", (64,)), ("add_norm", None), ("norm_add", None)])
@pytest.mark.parametrize("need", ["h", "r", "w", "b", "hr", "wb", "hw", "hrw", "G", "rG", "wbG"])
def test_some_gradients(cuda_device, op, gate, need):
    if gate is None and need == "G":
        need = "hrwb"
    for p, alpha in ((0.25, 1.5), (0.0, 1.0)):
        check(op, inputs((50, 64), BF16, cuda_device, gate=gate), need=need, p=p, alpha=alpha)
        check(op, inputs((50, 64), F32, cuda_device, gate=gate), need=need, p=p, alpha=alpha, kind="rms")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [128, 1000, 9000])
def test_add_norm_when_one_output_is_used(cuda_device, n, dtype):
    data = inputs((30, n), dtype, cuda_device, gate=(n,))
    check("add_norm", data, use=("y",))
    check("add_norm", data, use=("s",))
    check("add_norm", data, want_sum=False)
    h, r, w = (data[m].clone().requires_grad_(True) for m in ("h", "r", "w"))
    _, s = add_norm(h, r, w, return_sum=True)
    assert torch.autograd.grad(s, [h, r, w], data["gs"], allow_unused=True)[2] is None  # the sum does not see the weight
    out = add_norm(h, r, w)
    out.backward(data["gy"])
    assert torch.equal(h.grad, r.grad)
    h.grad.zero_()  # gradients of leaves do not share memory
    assert bool(r.grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("shape", [(0, 8), (5, 0), (0, 0), (0, 3, 8), (3, 0, 8)])
def test_empty(cuda_device, op, shape):
    for gate in (None, shape[-1:], (*([1] * (len(shape) - 1)), shape[-1])):
        data = inputs(shape, F32, cuda_device, gate=gate)
        _, grads = check(op, data, p=0.2)
        for c, m in (("w", "w"), ("b", "b"), ("G", "gate")):
            if c in grads:
                assert grads[c].shape == data[m].shape and not bool(grads[c].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strides_offsets_and_broadcast_residuals(cuda_device, dtype):
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(cuda_device)  # noqa: E731
    for rows, n, layouts in ((35, 104, [lambda: rand(35, 300)[:, 5:109], lambda: rand(70, 120)[::2, :104],
                                        lambda: rand(104, 35).T, lambda: rand(1, 104).expand(35, 104),
                                        lambda: rand(35 * 104 + 1)[1:].view(35, 104)]),):
        for op in ("add_norm", "norm_add"):
            for i, layout in enumerate(layouts):
                data = inputs((rows, n), dtype, cuda_device, gate=(n,), seed=i)
                for m in ("h", "r", "gy", "gs"):
                    data[m] = layout()
                # the formulas' expanded tensors are leaves of their own
                data["h"], data["r"] = data["h"].detach(), data["r"].detach()
                check(op, data)
            data = inputs((5, 7, n), dtype, cuda_device, gate=(5, 1, n))
            data["r"] = rand(7, n)
            check(op, data)
            data["r"] = rand(n)
            check(op, data)
            data["gate"] = rand(5, 1, 2 * n)[..., ::2]
            data["w"] = rand(2 * n)[::2]
            check(op, data)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("n", [64, 67, 1600])
def test_not_finite_stays_in_its_row(cuda_device, op, n):
    data = inputs((40, n), F32, cuda_device, gate=(n,))
    run = lambda d: (add_norm if op == "add_norm" else norm_add)(  # noqa: E731
        d["h"], d["r"], d["w"], d["b"], gate=d["gate"], dropout=0.5, seed=SEED)
    clean = run(data)
    f = factors(40, n, 0.5, SEED, 0).to(cuda_device)
    bad = {**data, "h": data["h"].clone()}
    bad["h"][3, 5], bad["h"][4, 6] = float("nan"), float("inf")
    got = run(bad)
    rows = [i for i in range(40) if i not in (3, 4)]
    assert torch.equal(got[rows], clean[rows])
    if op == "add_norm":  # a dropped element does not reach the sum
        for row, col in ((3, 5), (4, 6)):
            assert bool(got[row].isnan().all()) == bool(f[row, col] > 0)
            if f[row, col] == 0:
                assert torch.equal(got[row], clean[row])
    else:
        assert torch.equal(got[3].isnan(), f[3] > 0)
    # a dropped infinity of the block's output reaches no gradient of the gate either
    leaf = data["gate"].clone().requires_grad_(True)
    fill = torch.where(f > 0, data["h"], torch.full_like(data["h"], float("inf")))
    if op == "add_norm":
        y = add_norm(fill, data["r"], data["w"], data["b"], gate=leaf, dropout=0.5, seed=SEED)
        assert bool(torch.autograd.grad(y, [leaf], data["gy"])[0].isfinite().all())


@pytest.mark.gpu
def test_large_offsets_keep_their_digits(cuda_device):
    """A mean of 1000 beside a spread of 1: two passes over the row, no cancellation."""
    data = inputs((100, 320), F32, cuda_device)
    data["r"] = data["r"] + 1000
    check("add_norm", data, alpha=1.0, p=0.0)
    data["h"] = data["h"] + 1000
    check("norm_add", data)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
def test_gradient_against_differences(cuda_device, op):
    """Central differences of the forward in float32 along random directions, step
    2^-6: its square times third derivatives of order ten is below 2^-8 of the size."""
    data = inputs((33, 64), F32, cuda_device, gate=(64,))
    names = ["h", "r", "w", "b", "gate"]

    def run(values):
        h, r, w, b, gate = values
        how = dict(gate=gate, residual_scale=1.5, dropout=0.25, seed=SEED)
        return add_norm(h, r, w, b, **how) if op == "add_norm" else norm_add(h, r, w, b, **how)

    leaves = [data[m].clone().requires_grad_(True) for m in names]
    grads = torch.autograd.grad(run(leaves), leaves, data["gy"])
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(cuda_device)
        step = 2.0 ** -6
        up, down = ([t.detach() + s * step * v if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1))
        loss = [float((run(a).double() * data["gy"].double()).sum()) for a in (up, down)]
        along = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double().square().sum() * v.double().square().sum()).sqrt())
        assert abs((loss[0] - loss[1]) / (2 * step) - along) <= 2.0 ** -8 * size


@pytest.mark.gpu
def test_one_mask_in_all_operators(cuda_device):
    """The same seed, sequence, rows and columns drop the same elements."""
    for n in (256, 77, 2000):
        h, zero = torch.randn(64, n, device=cuda_device), torch.zeros(64, n, device=cuda_device)
        kept = dropout(h, 0.3, seed=9, sequence=2)
        _, s = add_norm(h, zero, return_sum=True, dropout=0.3, seed=9, sequence=2)
        assert torch.equal(s, kept)
        assert torch.equal(norm_add(h, zero, dropout=0.3, seed=9, sequence=2) == 0, kept == 0)


@pytest.mark.gpu
def test_repeats_its_bits(cuda_device):
    for shape, gate in (((4000, 256), (256,)), ((6, 500, 256), (6, 1, 256)), ((300, 2048), (2048,)), ((20, 9000), (9000,))):
        for dtype in (BF16, F32):
            data = inputs(shape, dtype, cuda_device, gate=gate)
            for op in ("add_norm", "norm_add"):
                first, second = (check(op, data) for _ in range(2))
                for a, b in zip(first, second):
                    assert all(torch.equal(a[m], b[m]) for m in a)


@pytest.mark.gpu
def test_on_a_side_stream(cuda_device):
    data = inputs((700, 256), BF16, cuda_device, gate=(256,))

    def run():
        leaves = [data[m].detach().requires_grad_(True) for m in ("h", "r", "w", "b", "gate")]
        h, r, w, b, gate = leaves
        y = add_norm(dropout(h, 0.1, seed=3), r, w, b, gate=gate, dropout=0.1, seed=3, sequence=1)
        return [y.detach(), *torch.autograd.grad(y, leaves, data["gy"])]

    expected = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1000000)
        other = run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(other, expected))


@pytest.mark.gpu
def test_double_backward_and_tangents_are_refused(cuda_device):
    from torch.autograd import forward_ad

    x = torch.randn(4, 8, device=cuda_device, requires_grad=True)
    for call in (lambda t: dropout(t, 0.5, seed=1), lambda t: add_norm(t, x.detach()), lambda t: norm_add(t, x.detach())):
        (d,) = torch.autograd.grad(call(x).square().sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.sum().backward()
        with forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x.detach(), torch.ones_like(x)))


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_traces_record_the_calls(cuda_device):
    data = inputs((3, 20, 48), F32, cuda_device, gate=(3, 1, 48))
    w2, b2 = torch.randn(128, 48, device=cuda_device), torch.randn(128, device=cuda_device)

    def block(h, r, w, b, gate):
        y, s = add_norm(dropout(h, 0.2, seed=1), r, w, b, gate=gate, dropout=0.1, seed=2, return_sum=True)
        return gated_linear(norm_add(y, s, w, b, dropout=0.1, seed=3), w2, b2, dropout=0.1, seed=4)

    args = tuple(data[m] for m in ("h", "r", "w", "b", "gate"))
    traced = torch.jit.trace(block, args, check_trace=False)
    other = tuple(torch.randn_like(t) for t in args)
    assert torch.equal(traced(*other), block(*other))


# ---- refusals, on the CPU ---------------------------------------------------------------------


def test_dropout_refusals():
    x = torch.randn(4, 8)
    for error, args, how in (
            (TypeError, (1.0, 0.5), dict(seed=1)), (TypeError, (x.double(), 0.5), dict(seed=1)),
            (TypeError, (x, "0.5"), dict(seed=1)), (TypeError, (x, True), dict(seed=1)),
            (ValueError, (x, -0.1), dict(seed=1)), (ValueError, (x, 1.01), dict(seed=1)),
            (ValueError, (x, math.nan), dict(seed=1)), (ValueError, (x, 0.5), dict(seed=None)),
            (ValueError, (x, 0.0), dict(seed=None)),
            (TypeError, (x, 0.5), dict(seed=1.5)), (TypeError, (x, 0.5), dict(seed=True)),
            (ValueError, (x, 0.5), dict(seed=-1)), (ValueError, (x, 0.5), dict(seed=2 ** 63)),
            (TypeError, (x, 0.5), dict(seed=torch.tensor(1.0))), (ValueError, (x, 0.5), dict(seed=torch.tensor([1, 2]))),
            (TypeError, (x, 0.5), dict(seed=1, sequence=0.5)), (ValueError, (x, 0.5), dict(seed=1, sequence=-1)),
            (ValueError, (x[0, 0], 0.5), dict(seed=1)),
            (RuntimeError, (x, 0.5), dict(seed=1)), (RuntimeError, (x, 0.5), dict(seed=1, backend="cpu"))):
        with pytest.raises(error):
            dropout(*args, **how)


@pytest.mark.parametrize("op", [add_norm, norm_add])
def test_residual_norm_refusals(op):
    h, w = torch.randn(4, 8), torch.randn(8)
    bad = (
        (TypeError, (h, None), {}), (TypeError, (1, h), {}), (TypeError, (h, h.bfloat16()), {}),
        (TypeError, (h.long(), h.long()), {}), (TypeError, (h, h, w.bfloat16()), {}), (TypeError, (h, h, 1.0), {}),
        (TypeError, (h.bfloat16(), h.bfloat16(), w, w.bfloat16()), {}),
        (ValueError, (h, h, w[:4]), {}), (ValueError, (h, h, w, w[None]), {}), (ValueError, (h, h[:, :4]), {}),
        (ValueError, (h, h[None]), {}), (ValueError, (h[0, 0], h[0, 0]), {}),
        (ValueError, (h, h), dict(kind="batch")), (TypeError, (h, h), dict(gate=0.5)),
        (TypeError, (h, h), dict(gate=w.bfloat16())), (ValueError, (h, h), dict(gate=w[:4])),
        (ValueError, (h, h), dict(gate=torch.ones(2, 4, 8))), (ValueError, (h, h), dict(gate=torch.ones(1, 4, 8))),
        (ValueError, (h, h), dict(gate=torch.ones(1, 1, 8))), (ValueError, (h, h), dict(gate=torch.ones(3, 8))),
        (ValueError, (h, h), dict(dropout=0.1)), (ValueError, (h, h), dict(dropout=1.5, seed=1)),
        (TypeError, (h, h), dict(dropout=0.1, seed="x")),
        (RuntimeError, (h, h), {}), (RuntimeError, (h, h), dict(backend="reference")))
    for error, args, how in bad:
        with pytest.raises(error):
            op(*args, **how)
    clear_dispatch_report()
    with pytest.raises(RuntimeError, match="residual norm kernels need CUDA tensors"):
        op(h, h)
    assert get_last_dispatch_report().operator == op.__name__ and get_last_dispatch_report().selected_backend == "error"


@pytest.mark.gpu
def test_tensors_of_two_devices_are_refused(cuda_device):
    h = torch.randn(4, 8, device=cuda_device)
    for call in (lambda: dropout(h, 0.5, seed=torch.tensor(1)), lambda: add_norm(h, h.cpu()),
                 lambda: norm_add(h, h, gate=torch.ones(8)), lambda: add_norm(h, h, dropout=0.5, seed=torch.tensor(3))):
        with pytest.raises(RuntimeError, match="is on cpu"):
            call()


def test_c_entry_refusals():
    module = native.load_native_module()
    p = 4096  # aligned, never dereferenced

    def fails(name, message, **fields):
        args = native.ResidualNormArgs(**fields)
        entry = getattr(module.lib, name)
        import ctypes
        entry.restype, entry.argtypes = ctypes.c_int, [ctypes.POINTER(native.ResidualNormArgs), ctypes.c_void_p]
        assert entry(args, None) == 1 and message in module.last_error()

    for name in ("msda_add_norm_forward", "msda_norm_add_backward"):
        assert getattr(module.lib, name)(None, None) == 1 and "args is null" in module.last_error()
    good = dict(rows=4, cols=8, gate_groups=1, input=p, residual=p, output=p, sum=p)
    for name in ("msda_add_norm_forward", "msda_norm_add_forward"):
        fails(name, "dtype must be", **{**good, "dtype": 3})
        fails(name, "weight_dtype", **{**good, "dtype": 1, "weight_dtype": 2})
        fails(name, "kind must be", **{**good, "kind": 2})
        fails(name, "threshold must be", **{**good, "threshold": 65537})
        fails(name, "gate_groups must divide rows", **{**good, "gate": p, "gate_groups": 3})
        fails(name, "strides", **{**good, "residual_stride": -1})
        fails(name, "residual is null", **{**good, "residual": None})
    fails("msda_norm_add_forward", "sum is null", **{**good, "sum": None})
    fails("msda_add_norm_forward", "output is null", **{**good, "output": None})
    back = dict(rows=4, cols=8, gate_groups=1, input=p, sum=p, rstd=p, mean=p, grad_output=p, grad_sum=p, grad_input=p)
    fails("msda_add_norm_backward", "are null", **{**back, "grad_output": None, "grad_sum": None})
    fails("msda_add_norm_backward", "need grad_output", **{**back, "grad_output": None, "grad_weight": p})
    fails("msda_add_norm_backward", "mean is null", **{**back, "mean": None})
    fails("msda_norm_add_backward", "grad_sum is null", **{**back, "grad_sum": None})
    fails("msda_add_norm_backward", "workspace has 0 bytes", **{**back, "grad_weight": p})


# ---- rows that their storage type cannot hold ------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("n", [64, 100, 256, 520, 1500, 5001, 8192, 9000])
def test_add_norm_gradients_are_those_of_its_output(cuda_device, n, kind, dtype):
    """Of the norm alone, where the sum is not returned: rows whose offset is large beside their spread, and
    float16 rows whose sum is beyond 65504, have the derivative of what the forward computed.

    A row is kept for the backward pass as its sum or normalised, rounded to its type: the sum only where
    its mean is at most four times its spread. So a normalised value k is off by HALF (4 + |k|) at most,
    besides the float32 errors of the sum; call that e. Its mean and rstd follow: rstd is off by
    mean(|k| e) + mean(e^2), relatively, and k by e + mean(e) + |k| times that."""
    offsets = [0, 0, 0.5, -1, 3, -3, 5, 10, 100, -1000, 1000, 4096]
    data = inputs((len(offsets) + 2, n), dtype, cuda_device, gate=(n,), seed=n)
    for i, offset in enumerate(offsets):
        if offset:
            data["r"][i] = offset
    if dtype == F16:
        data["r"][-2:] = 60000
        data["h"][-2:] = 40000 + 2000 * data["h"][-2:]
    for p, gated in ((0.0, False), (0.25, True)):
        x = {m: v.double() for m, v in data.items()}
        f = factors(len(x["h"]), n, p, SEED, SEQUENCE).to(cuda_device) if p else torch.ones_like(x["h"])
        gate = x["gate"] if gated else torch.ones_like(x["gate"])
        s = x["r"] + gate * x["h"] * f
        size = x["r"].abs() + (gate * x["h"] * f).abs()
        k, rstd = normed64(kind, s)
        e = HALF[dtype] * (4 + k.abs()) + SUM * rstd * (size + size.amax(-1, keepdim=True)) * (1 + k.abs())
        rho = (k.abs() * e).mean(-1, keepdim=True) + e.square().mean(-1, keepdim=True)
        off = e + e.mean(-1, keepdim=True) + k.abs() * rho
        g = x["gy"]
        ds, ds_size, m2 = norm_grad64(kind, g * x["w"], k, rstd)
        loose = (rho + 2 * SUM) * ds_size + rstd * (off * m2.abs() + k.abs() * ((g * x["w"]).abs() * off).mean(-1, keepdim=True))
        branch = x["h"] * f
        expected = [gate * f * ds, ds, (g * k).sum(0), g.sum(0), (ds * branch).sum(0)]
        errors = [gate.abs() * f * loose, loose, (g.abs() * off).sum(0), 0 * g.sum(0), (loose * branch.abs()).sum(0)]
        terms = [(gate * f * ds).abs(), ds.abs(), (g * k).abs().sum(0), g.abs().sum(0), (ds * branch).abs().sum(0)]
        names = ["h", "r", "w", "b", "gate"][:4 + gated]
        leaves = [data[m].clone().requires_grad_(True) for m in names]
        y = add_norm(*leaves[:4], gate=leaves[4] if gated else None, kind=kind, dropout=p, seed=SEED, sequence=SEQUENCE)
        assert bool(y.isfinite().all())
        for i, got in enumerate(torch.autograd.grad(y, leaves, data["gy"])):
            near(got, expected[i], terms[i] + errors[i] / SUM, dtype)


@pytest.mark.gpu
def test_kept_rows_by_offset_repeat_and_stay_apart(cuda_device):
    """A row with a large offset changes nothing of the gradients of the rows beside it, and its own are those
    of the row without the offset, which the norm takes off."""
    for n in (64, 256, 1024, 9000):
        data = inputs((40, n), BF16, cuda_device)
        data["r"].zero_()
        plain = data["r"].clone()
        data["r"][7] = 2048
        run = lambda r: torch.autograd.grad(  # noqa: E731
            add_norm(h, r, data["w"], data["b"]), [h], data["gy"])[0]
        h = data["h"].requires_grad_(True)
        a, b = run(data["r"]), run(plain)
        rest = [i for i in range(40) if i != 7]
        assert torch.equal(a[rest], b[rest]) and torch.equal(a, run(data["r"]))
        # the float32 sum beside 2048 is off by 2^-13 in units of h, k by that and its rounding to bfloat16 (as b's h by its own)
        assert bool(((a[7] - b[7]).double().abs() <= 0.05 * b[7].double().abs() + 0.05 * float(b[7].double().square().mean().sqrt())).all())


def test_c_entry_refuses_keeping_what_is_no_forward_of_add_norm():
    module = native.load_native_module()
    p = 4096  # aligned, never dereferenced
    import ctypes
    for name, more in (("msda_norm_add_forward", {}), ("msda_add_norm_backward", dict(rstd=p, mean=p, grad_output=p, grad_input=p)),
                       ("msda_add_norm_forward", dict(sum=None, mean=p, rstd=p)), ("msda_add_norm_forward", dict(rstd=None))):
        args = native.ResidualNormArgs(**{**dict(rows=4, cols=8, gate_groups=1, input=p, residual=p, output=p, sum=p, kind=16), **more})
        entry = getattr(module.lib, name)
        entry.restype, entry.argtypes = ctypes.c_int, [ctypes.POINTER(native.ResidualNormArgs), ctypes.c_void_p]
        assert entry(args, None) == 1 and "MSDA_NORM_KEEP" in module.last_error()


@pytest.mark.parametrize("cols,rows,per_block", [(128, 2000, 16), (96, 2368, 16), (100, 2000, 8), (256, 2000, 8)])
def test_backward_units_are_whole_passes_of_a_block(cols, rows, per_block):
    """Two float32 rows of partial sums (weight and bias) to each block, and a block's rows are a multiple of those
    that it has under way: 16 where two rows of up to 128 columns share a warp."""
    import ctypes
    module = native.load_native_module()
    query = module.lib.msda_add_norm_backward_workspace
    query.restype, query.argtypes = ctypes.c_int, [ctypes.POINTER(native.ResidualNormArgs), ctypes.POINTER(ctypes.c_size_t)]
    size, p = ctypes.c_size_t(), 4096  # aligned, never dereferenced
    args = native.ResidualNormArgs(dtype=1, weight_dtype=1, gate_dtype=1, rows=rows, cols=cols, gate_groups=1, sum=p, rstd=p,
                                   mean=p, grad_output=p, grad_input=p, grad_weight=p, grad_bias=p)
    assert query(args, size) == 0
    blocks = size.value // (2 * cols * 4)
    assert size.value == blocks * 2 * cols * 4 and blocks == -(-rows // per_block)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(30, 64), (6, 5, 67), (3, 700), (2, 3, 9000)], ids=lambda s: "x".join(map(str, s)))
def test_a_gradient_that_comes_in_is_left_as_it_was(cuda_device, shape, dtype):
    """Slices and expanded gradients, which the residual's gradient is where the scale is 1: what lies beside and
    behind them stays."""
    n = shape[-1]
    data = inputs(shape, dtype, cuda_device, gate=(n,))
    guard = torch.randn(4, *shape[:-1], n + 5, device=cuda_device).to(dtype)
    slice_of, before = guard[2][..., 2:n + 2], guard.clone()
    single = torch.randn(100 * n, device=cuda_device).to(dtype)
    expanded, kept = single[50 * n:51 * n].expand(shape), single.clone()
    for op in (add_norm, norm_add):
        for need in ("hrwb", "rwb", "r", "hr"):
            for gated in (False, True):
                for grad in (slice_of, expanded):
                    names = [{"h": "h", "r": "r", "w": "w", "b": "b"}[c] for c in need] + ["gate"] * gated
                    leaves = {m: data[m].clone().requires_grad_(m in names) for m in ("h", "r", "w", "b", "gate")}
                    call = lambda: op(leaves["h"], leaves["r"], leaves["w"], leaves["b"],  # noqa: E731
                                      gate=leaves["gate"] if gated else None, dropout=0.1, seed=4)
                    got = torch.autograd.grad(call(), [leaves[m] for m in names], grad)
                    clean = torch.autograd.grad(call(), [leaves[m] for m in names], grad.clone(memory_format=torch.contiguous_format))
                    for a, b in zip(got, clean):  # one rounding each, of float32 sums in two orders
                        a, b = a.double(), b.double()
                        assert bool(((a - b).abs() <= 2 * HALF[dtype] * b.abs() + 2 * LEAST[dtype] + 2.0 ** -14 * b.abs().max()).all())
                    assert torch.equal(guard, before) and torch.equal(single, kept)
                    if op is norm_add:
                        assert torch.equal(got[names.index("r")], grad)
    # the whole way through autograd: a sum's gradient is one number, expanded
    for op in (add_norm, norm_add):
        leaves = [data[m].clone().requires_grad_(True) for m in ("h", "r", "w", "b")]
        op(*leaves).sum().backward()
        if op is norm_add:
            assert torch.equal(leaves[1].grad, torch.ones_like(leaves[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["add_norm", "norm_add"])
@pytest.mark.parametrize("shape", [(40, 1), (2, 6, 1), (1, 1), (1,), (0, 1)])
def test_single_columns_with_every_gate(cuda_device, op, shape):
    for gate in ((), (1,), (*([1] * len(shape)),), shape):
        data = inputs(shape, F32, cuda_device, gate=gate)
        _, grads = check(op, data)
        assert grads["G"].shape == gate

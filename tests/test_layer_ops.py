"""linear_act, layer_norm and 8-bit checkpoints against plain 64-bit formulas.

Tolerances, per element, from the arithmetic: an output is rounded once to its
type (half an ulp: up to 2^-8 of it for bfloat16, 2^-24 for float32, 2^-11 for
float16; twice that is allowed for the latter two), and before that carries the
error of float32 sums, taken as 2^-20 of the sum of the terms' magnitudes. In a
bfloat16 backward pass dz is rounded to bfloat16 before it is multiplied (2^-8 of
each term), with a slope rounded to float16 (2^-11).
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from muspace_b200 import clear_dispatch_report, get_last_dispatch_report
from muspace_b200.ops import Checkpoint8, checkpoint_pack, checkpoint_unpack, layer_norm, linear_act
from muspace_b200.runtime import native

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16
OUT = {BF16: 2.0 ** -8, F32: 2.0 ** -23, F16: 2.0 ** -10}
SUM = 2.0 ** -20


# ---- 64-bit formulas ------------------------------------------------------------------


def act64(name, z):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z / math.sqrt(2))
    return z * torch.sigmoid(z) if name == "silu" else z


def slope64(name, z):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def held64(x):
    """What a checkpoint of x holds, block by block: nothing above 63 * 2^122, the last code below float32's end."""
    out = x.double().clone()
    for at in range(0, x.shape[-1], 32):
        part = out[..., at:at + 32]
        top = part.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, -126)
        for shift in (128, 64, 32, 16, 8, 4, 2, 1):  # the largest e that is still too small, by bisection
            e = torch.where(top > 127 * torch.exp2(e + shift - 1), e + shift, e)
        out[..., at:at + 32] = torch.round(part / torch.exp2(e)) * torch.exp2(e)
    return out.clamp(-63 * 2.0 ** 122, 63 * 2.0 ** 122)


def norm64(x, w, b, eps):
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    return c * rstd * w + b, c * rstd, rstd


def near(got, expected, terms, dtype, extra=0.0):
    """|got - expected| within the type's rounding of it and the error of the sum whose terms' magnitudes add up to `terms`."""
    assert got.dtype == dtype and got.shape == expected.shape
    got = got.double()
    bound = OUT[dtype] * expected.abs() + (SUM + extra) * terms + 1e-37
    bad = (got - expected).abs() > bound
    assert not bool(bad.any()), (
        f"{int(bad.sum())} of {bad.numel()} outside; worst {float(((got - expected).abs() / bound).max()):.3g} of the bound")


# ---- linear -----------------------------------------------------------------------------


def linear_inputs(rows, k, n, dtype, device, seed=0, residual=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, w, b = r(rows, k), r(n, k) / math.sqrt(max(k, 1)), 0.3 * r(n)
    out = [t.to(dtype).to(device) for t in (x, w, b, r(rows, n), r(rows, n))]
    if not residual:
        out[3] = None
    return out


def check_linear(x, w, b, r, g, activation, checkpoint=None, need=(True, True, True)):
    """Forward and backward of one call against the formulas; returns the outputs."""
    dtype = x.dtype
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = linear_act(*leaves, activation=activation, checkpoint=checkpoint)
    named = [(m, t) for m, t in zip("xwbr", leaves) if t is not None]
    grads = dict(zip((m for m, _ in named), torch.autograd.grad(y, [t for _, t in named], g)))
    x6, w6, g6 = x.double(), w.double(), g.double()
    b6 = b.double() if b is not None else torch.zeros(w.size(0), dtype=torch.float64, device=x.device)
    z = x6 @ w6.T + b6
    size = x6.abs() @ w6.abs().T + b6.abs()
    expected = act64(activation, z) + (r.double() if r is not None else 0)
    near(y, expected, 2 * size + 1 + (r.double().abs() if r is not None else 0), dtype)
    if checkpoint:
        x6 = held64(x)
        z = x6 @ w6.T + b6
        size = x6.abs() @ w6.abs().T + b6.abs()
    dz = g6 * slope64(activation, z)
    # an error of z moves the slope by at most 1.2 of it; bfloat16: dz to 2^-8, the slope to 2^-11
    loose = dz.abs() * (0 if dtype == F32 else 2.0 ** -8) + g6.abs() * (2 * SUM * size + (0 if dtype == F32 else 2.0 ** -11))
    for name, value, error, terms in (
            ("x", dz @ w6, loose @ w6.abs(), dz.abs() @ w6.abs()),
            ("w", dz.T @ x6, loose.T @ x6.abs(), dz.abs().T @ x6.abs()),
            ("b", dz.sum(0), loose.sum(0), dz.abs().sum(0))):
        if name in grads:
            near(grads[name], value, terms + error / SUM, dtype)
    if r is not None:
        assert torch.equal(grads["r"], g)
    return y, grads


SHAPES = [(1, 1, 1), (1, 256, 512), (2, 4096, 300), (3, 7, 5), (17, 40, 33), (127, 64, 63), (128, 128, 128),
          (129, 65, 257), (300, 517, 259), (1000, 96, 40), (513, 1000, 8), (200, 256, 1024), (5000, 256, 136)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_matches_the_formulas(cuda_device, rows, k, n, dtype):
    args = linear_inputs(rows, k, n, dtype, cuda_device, seed=rows + k + n)
    check_linear(*args, "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("k", [72, 640])
def test_linear_activations_and_checkpoints(cuda_device, activation, checkpoint, k, dtype):
    check_linear(*linear_inputs(321, k, 200, dtype, cuda_device, seed=k), activation, checkpoint)
    check_linear(*linear_inputs(130, k + 3, 77, dtype, cuda_device, seed=k, residual=False), activation, checkpoint)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(2048, 1024, 1152), (2050, 2100, 1152), (1024, 2048, 2304)])
def test_linear_long_sums_of_whole_tiles(cuda_device, rows, k, n, dtype):
    """So many tiles that no sum is split, over k that is and is not a multiple of 1024."""
    check_linear(*linear_inputs(rows, k, n, dtype, cuda_device, seed=k), "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("rows,k,n", [(300, 72, 200), (130, 67, 77)])
def test_linear_backward_without_a_slope(cuda_device, rows, k, n, activation, dtype):
    """The C entry computes z again where it is given no slope: the gradients are the formulas' too."""
    x, w, b, _, g = linear_inputs(rows, k, n, dtype, cuda_device, seed=k)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    args = native.LinearArgs(0 if dtype == F32 else 1, {"relu": 1, "gelu": 2, "silu": 3}[activation], rows, k, n, k, k, 0,
                             0, n, x.data_ptr(), w.data_ptr(), b.data_ptr(), None, None, None, g.data_ptr(), None, None,
                             dx.data_ptr(), dw.data_ptr(), db.data_ptr())
    native.load_native_module().plain_call("msda_linear_act_backward")(x.device, args)
    x6, w6, g6 = x.double(), w.double(), g.double()
    z = x6 @ w6.T + b.double()
    size = x6.abs() @ w6.abs().T + b.double().abs()
    dz = g6 * slope64(activation, z)
    loose = dz.abs() * (0 if dtype == F32 else 2.0 ** -8) + g6.abs() * 2 * SUM * size
    if activation == "relu":  # where z is within its error of 0, the slope may be either
        loose = loose + g6.abs() * (z.abs() <= 2 * SUM * size)
    near(dx, dz @ w6, dz.abs() @ w6.abs() + loose @ w6.abs() / SUM, dtype)
    near(dw, dz.T @ x6, dz.abs().T @ x6.abs() + loose.T @ x6.abs() / SUM, dtype)
    near(db, dz.sum(0), dz.abs().sum(0) + loose.sum(0) / SUM, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation", [0, 1, 2, 3])
@pytest.mark.parametrize("rows,k,n", [(300, 72, 200), (300, 72, 77), (1, 72, 200)])
def test_linear_slope_of_the_c_entry(cuda_device, rows, k, n, activation, dtype):
    x, w, b, r, _ = linear_inputs(rows, k, n, dtype, cuda_device, seed=n)
    y = torch.empty_like(r)
    slope = torch.full((rows, n), float("nan"), device=cuda_device, dtype=F32 if dtype == F32 else F16)
    args = native.LinearArgs(0 if dtype == F32 else 1, activation, rows, k, n, k, k, n, n, 0, x.data_ptr(), w.data_ptr(),
                             b.data_ptr(), r.data_ptr(), y.data_ptr(), slope.data_ptr())
    native.load_native_module().plain_call("msda_linear_act_forward")(x.device, args)
    name = ["none", "relu", "gelu", "silu"][activation]
    z = x.double() @ w.double().T + b.double()
    size = x.double().abs() @ w.double().abs().T + b.double().abs()
    near(y, act64(name, z) + r.double(), 2 * size + 1 + r.double().abs(), dtype)
    expected = slope64(name, z) if activation else torch.ones_like(z)
    terms = 2 * size + 1
    if name == "relu":
        terms = terms + (z.abs() <= 2 * SUM * size) / SUM
    near(slope, expected, terms, slope.dtype, extra=0.0 if dtype == F32 else 2.0 ** -23)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("k", [64, 640])
def test_linear_relu(cuda_device, dtype, k):
    """Integers: every pre-activation is exact, so the kink falls the same way everywhere."""
    gen = torch.Generator().manual_seed(3)
    x, w, b, r, g = (torch.randint(-2, 3, s, generator=gen).to(dtype).to(cuda_device)
                     for s in ((150, k), (70, k), (70,), (150, 70), (150, 70)))
    check_linear(x, w, b, r, g, "relu")
    z = x.double() @ w.double().T
    y = linear_act(x, w, activation="relu")
    assert bool((z == 0).any()) and torch.equal(y.double(), z.clamp(min=0).to(dtype).double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(0, 8, 16), (5, 0, 16), (5, 8, 0), (0, 0, 0)])
def test_linear_empty(cuda_device, rows, k, n, dtype):
    x, w, b, r, g = linear_inputs(rows, k, n, dtype, cuda_device)
    y, grads = check_linear(x, w, b, r, g, "silu")
    assert y.shape == (rows, n) and grads["x"].shape == (rows, k) and grads["w"].shape == (n, k)
    if k == 0:
        near(y, act64("silu", b.double()) + r.double(), y.double().abs() + 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_linear_strides_offsets_and_leading_shapes(cuda_device, dtype):
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(cuda_device)  # noqa: E731
    wide = rand(70, 300)
    layouts = {
        "column slice": (wide[:, 5:105], rand(60, 100)),
        "every other row": (wide[::2, :100], rand(60, 100)),
        "transposed": (rand(100, 35).T, rand(100, 60).T),
        "broadcast rows": (rand(1, 100).expand(35, 100), rand(60, 100)),
        "weight rows off 16 bytes": (rand(35, 100), rand(61, 101)[1:, 1:]),
        "odd base": (rand(35 * 100 + 1)[1:].view(35, 100), rand(60, 100)),
    }
    for name, (x, w) in layouts.items():
        b, r, g = rand(w.size(0)), rand(x.size(0), w.size(0)), rand(w.size(0), x.size(0)).T
        check_linear(x, w, b, r, g, "gelu")
    x = rand(3, 4, 5, 100)
    w, b = rand(24, 100), rand(24)
    y = linear_act(x, w, b)
    assert y.shape == (3, 4, 5, 24)
    assert torch.equal(y.view(-1, 24), linear_act(x.reshape(-1, 100), w, b))
    assert torch.equal(linear_act(x[0, 0, 0], w, b), linear_act(x[0, 0, :1], w, b)[0])
    turned = x.permute(2, 0, 1, 3)
    assert torch.equal(linear_act(turned, w, b), linear_act(turned.contiguous(), w, b))


@pytest.mark.gpu
def test_linear_residual_broadcast_sums_its_gradient(cuda_device):
    x, w, b, _, g = linear_inputs(40, 32, 24, F32, cuda_device)
    row = torch.randn(24, device=cuda_device, requires_grad=True)
    y = linear_act(x, w, b, row, activation="silu")
    near(y, act64("silu", x.double() @ w.double().T + b.double()) + row.detach().double(),
         2 * (x.double().abs() @ w.double().abs().T) + 10, F32)
    (grad,) = torch.autograd.grad(y, [row], g)
    near(grad, g.double().sum(0), g.double().abs().sum(0), F32)


@pytest.mark.gpu
@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
@pytest.mark.parametrize("activation,checkpoint,k", [("none", None, 64), ("gelu", None, 64), ("gelu", None, 640),
                                                    ("silu", "int8", 64), ("none", "int8", 64)])
def test_linear_some_gradients(cuda_device, needs, activation, checkpoint, k):
    x, w, b, r, g = linear_inputs(100, k, 48, BF16, cuda_device)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    every = torch.autograd.grad(linear_act(*full, r, activation=activation, checkpoint=checkpoint), full, g)
    some = [t.clone().requires_grad_(q) for t, q in zip((x, w, b), needs)]
    y = linear_act(*some, r, activation=activation, checkpoint=checkpoint)
    got = torch.autograd.grad(y, [t for t in some if t.requires_grad], g)
    for a, e in zip(got, [e for e, q in zip(every, needs) if q]):
        assert torch.equal(a, e)


@pytest.mark.gpu
def test_linear_expanded_gradient(cuda_device):
    x, w, b, _, _ = linear_inputs(50, 40, 24, BF16, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    linear_act(*leaves).sum().backward()
    ones = torch.ones(50, 24, dtype=BF16, device=cuda_device)
    for t, e in zip(leaves, torch.autograd.grad(linear_act(*leaves), leaves, ones)):
        assert torch.equal(t.grad, e)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(150, 72, 200), (2, 72, 200), (40, 640, 96)])
def test_linear_infinities_and_nans_stay_in_their_rows(cuda_device, dtype, rows, k, n):
    x, w, b, r, g = linear_inputs(rows, k, n, dtype, cuda_device)
    clean = linear_act(x, w, b, r)
    bad = x.clone()
    bad[0, 3], bad[1, 5] = float("inf"), float("nan")
    y = linear_act(bad, w, b, r)
    assert torch.equal(y[0].double(), math.inf * w[:, 3].double().sign())
    assert bool(y[1].isnan().all()) and torch.equal(y[2:], clean[2:])
    wide = w.clone()
    wide[2, 1] = -float("inf")
    y = linear_act(x, wide, b, r)
    assert torch.equal(y[:, 2].double(), -math.inf * x[:, 1].double().sign())
    keep = [i for i in range(n) if i != 2]
    assert torch.equal(y[:, keep], clean[:, keep])
    # backward: an infinite gradient element reaches its row of dx, its row of dw, its db
    gi = g.clone()
    gi[0, 4] = float("inf")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear_act(*leaves, r), leaves, gi)
    assert torch.equal(dx[0].double(), math.inf * w[4].double().sign()) and bool(dx[1:].isfinite().all())
    assert torch.equal(dw[4].double(), math.inf * x[0].double().sign()) and float(db[4]) == math.inf
    others = [i for i in range(n) if i != 4]
    assert bool(dw[others].isfinite().all()) and bool(db[others].isfinite().all())


@pytest.mark.gpu
def test_linear_float32_range(cuda_device):
    """Float32's largest values are above bfloat16's; small ones keep their 24 bits."""
    for scale in (3.4e38, 1e30, 1e-25):
        x = torch.randn(64, 40, dtype=torch.float64).clamp(-1, 1) * scale
        x[0, 0] = scale
        w = torch.zeros(40, 40, dtype=torch.float64)
        w[torch.arange(40), torch.arange(40).flip(0)] = 0.5
        x, w = x.float().to(cuda_device), w.float().to(cuda_device)
        assert torch.allclose(linear_act(x, w).double(), x.double() @ w.double().T, rtol=2.0 ** -22, atol=0)


@pytest.mark.gpu
def test_linear_float16(cuda_device):
    x, w, b, r, g = linear_inputs(60, 40, 24, F16, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = linear_act(*leaves, activation="silu")
    z = x.detach().double() @ w.detach().double().T + b.detach().double()
    near(y.detach(), act64("silu", z) + r.detach().double(), z.abs() + 10, F16)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, g)
    assert {t.dtype for t in (dx, dw, db, dr)} == {F16}
    dz = g.double() * slope64("silu", z)
    near(dx, dz @ w.detach().double(), dz.abs() @ w.detach().double().abs(), F16)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_linear_gradient_against_differences(cuda_device, checkpoint):
    """Central differences of the forward in float32 along random directions. Inputs
    on a grid that an 8-bit checkpoint holds exactly, so it changes nothing; step
    2^-5: its square times the third derivative (of order one) is 2^-10 of the
    result's size, the forward's rounding over the step less."""
    gen = torch.Generator().manual_seed(9)
    rand = lambda *s: (torch.randint(-64, 65, s, generator=gen) / 64).to(cuda_device)  # noqa: E731
    x, w, b, r, g = rand(33, 64), rand(40, 64) / 8, rand(40), rand(33, 40), rand(33, 40)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear_act(*leaves, activation="gelu", checkpoint=checkpoint), leaves, g)
    for i in range(4):
        v = rand(*leaves[i].shape)
        step = 2.0 ** -5 / (8 if i < 2 else 1)
        up, down = ([t.detach() + s * step * v if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1))
        loss = [(linear_act(*a, activation="gelu").double() * g.double()).sum() for a in (up, down)]
        along = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double().square().sum() * v.double().square().sum()).sqrt())
        assert abs(float(loss[0] - loss[1]) / (2 * step) - along) <= 2.0 ** -9 * size


@pytest.mark.gpu
def test_linear_repeats_its_bits(cuda_device):
    for dtype in (BF16, F32):
        for rows, k, n in ((4000, 256, 512), (33, 2048, 96), (2, 4096, 256)):
            args = linear_inputs(rows, k, n, dtype, cuda_device)
            first, second = (check_linear(*args, "silu") for _ in range(2))
            assert torch.equal(first[0], second[0])
            assert all(torch.equal(first[1][m], second[1][m]) for m in first[1])


@pytest.mark.gpu
def test_layer_ops_on_a_side_stream_and_in_a_graph(cuda_device):
    x, w, b, r, g = linear_inputs(700, 256, 96, F32, cuda_device)
    scale, shift = torch.rand(96, device=cuda_device), torch.rand(96, device=cuda_device)

    def both():
        return layer_norm(linear_act(x, w, b, r, activation="gelu"), scale, shift)

    expected = both()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1000000)
        other = both()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, expected)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    x.mul_(2)
    graph.replay()
    assert torch.equal(captured, both()) and not torch.equal(captured, expected)


@pytest.mark.gpu
def test_layer_ops_past_two_to_the_31_elements(cuda_device):
    """Rows whose offsets need 64 bits equal the same rows of a small call, forward and backward."""
    rows, width = 263000, 8200  # 2.16e9 outputs
    x = torch.randn(rows, 32, device=cuda_device, dtype=BF16)
    w = torch.randn(width, 32, device=cuda_device, dtype=BF16) / 4
    y = linear_act(x, w, activation="gelu")
    tail = slice(rows - 300, rows)
    assert torch.equal(y[tail], linear_act(x[tail], w, activation="gelu"))
    scale = torch.rand(width, device=cuda_device, dtype=BF16)
    leaf = y.requires_grad_(True)
    n = layer_norm(leaf, scale)
    assert torch.equal(n[tail].detach(), layer_norm(leaf.detach()[tail], scale))
    (d,) = torch.autograd.grad(n, [leaf], y.detach())
    small = leaf.detach()[tail].clone().requires_grad_(True)
    assert torch.equal(d[tail], torch.autograd.grad(layer_norm(small, scale), [small], small.detach())[0])
    del n, d
    kept = checkpoint_pack(leaf)
    assert torch.equal(checkpoint_unpack(kept)[tail], checkpoint_unpack(checkpoint_pack(leaf.detach()[tail])))


# ---- layer norm ---------------------------------------------------------------------------


def norm_inputs(rows, n, dtype, device, seed=0, offset=0.2, wtype=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    x = r(rows, n) * torch.exp(0.5 * r(rows, 1)) + offset
    w, b, g = 1 + 0.2 * r(n), 0.1 * r(n), r(rows, n)
    wtype = wtype or dtype
    return x.to(dtype).to(device), w.to(wtype).to(device), b.to(wtype).to(device), g.to(dtype).to(device)


def check_norm(x, w, b, g, checkpoint=None, eps=1e-5):
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps, checkpoint=checkpoint)
    given = [t for t in leaves if t is not None]
    grads = list(torch.autograd.grad(y, given, g))
    n = x.size(-1)
    w6 = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    b6 = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    y6, h, rstd = norm64(x.double(), w6, b6, eps)
    # h carries the mean's error, which is of the size of the row's largest value
    spread = lambda x, h, rstd: h.abs() + x.double().abs().amax(-1, keepdim=True) * rstd + 1  # noqa: E731
    near(y, y6, spread(x, h, rstd) * w6.abs() + b6.abs(), x.dtype)
    if checkpoint:
        x = held64(x)
        _, h, rstd = norm64(x, w6, b6, eps)
    size = spread(x, h, rstd)
    g6 = g.double()
    gw = g6 * w6
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    terms = rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) + size * 3 * (gw * size).abs().mean(-1, keepdim=True))
    near(grads.pop(0), dx, terms, y.dtype)
    if w is not None:
        near(grads.pop(0), (g6 * h).sum(0), (g6.abs() * size).sum(0), w.dtype)
    if b is not None:
        near(grads.pop(0), g6.sum(0), g6.abs().sum(0), b.dtype)
    return y


WIDTHS = [1, 2, 8, 31, 32, 33, 256, 257, 264, 512, 513, 1000, 1024, 2048, 2056, 4096, 4099, 8192, 8200, 16385]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("n", WIDTHS)
def test_layer_norm_matches_the_formulas(cuda_device, n, checkpoint, dtype):
    rows = 700 if n <= 2048 else 160
    check_norm(*norm_inputs(rows, n, dtype, cuda_device, seed=n), checkpoint)
    check_norm(*norm_inputs(1, n, dtype, cuda_device, seed=n + 1), checkpoint)


@pytest.mark.gpu
def test_layer_norm_many_rows(cuda_device):
    check_norm(*norm_inputs(40001, 256, BF16, cuda_device))
    check_norm(*norm_inputs(30011, 96, F32, cuda_device), "int8")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [48, 50, 640, 5000])
def test_layer_norm_float32_weights_and_missing_ones(cuda_device, n):
    x, w, b, g = norm_inputs(65, n, BF16, cuda_device, wtype=F32)
    check_norm(x, w, b, g)
    check_norm(x, w, None, g)
    check_norm(x, None, b, g)
    check_norm(x, None, None, g)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [200, 3000, 20000])
def test_layer_norm_keeps_its_digits_beside_a_large_mean(cuda_device, n):
    x, w, b, g = norm_inputs(9, n, F32, cuda_device, offset=1000.0)
    check_norm(x, w, b, g)


@pytest.mark.gpu
def test_layer_norm_strides_and_shapes(cuda_device):
    x, w, b, g = norm_inputs(60, 400, BF16, cuda_device)
    for view in (x[:, 8:136], x[:, 3:131], x[::3, :128], x.T[:128].T, x[:1, :128].expand(60, 128)):
        check_norm(view, w[:128], b[5:133], g[:view.size(0), :128])
        check_norm(view, w[:128], b[5:133], g[:view.size(0), :128], "int8")
    y = layer_norm(x.view(3, 20, 400), w, b)
    assert torch.equal(y.view(60, 400), layer_norm(x, w, b))
    assert torch.equal(layer_norm(x[0], w, b), y[0, 0])
    leaf = x.clone().requires_grad_(True)
    layer_norm(leaf, w, b).sum().backward()
    (e,) = torch.autograd.grad(layer_norm(leaf, w, b), [leaf], torch.ones_like(x))
    assert torch.equal(leaf.grad, e)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [64, 700, 9000])
def test_layer_norm_constant_rows_and_what_is_not_finite(cuda_device, n):
    x, w, b, g = norm_inputs(12, n, F32, cuda_device)
    clean = layer_norm(x, w, b)
    x[3] = 2.5  # no variance: h = 0
    x[5, 7], x[6, 1] = float("nan"), float("inf")
    y = layer_norm(x, w, b)
    assert torch.equal(y[3], b)
    assert bool(y[5].isnan().all()) and bool(y[6].isnan().all())
    keep = [0, 1, 2, 4, 7, 8, 9, 10, 11]
    assert torch.equal(y[keep], clean[keep])
    leaf = x.clone().requires_grad_(True)
    for checkpoint in (None, "int8"):
        (dx,) = torch.autograd.grad(layer_norm(leaf, w, b, checkpoint=checkpoint), [leaf], g)
        assert bool(dx[5].isnan().all()) and bool(dx[6].isnan().all())
        assert bool(dx[[3] + keep].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(0, 16), (4, 0)])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_layer_norm_empty(cuda_device, rows, n, checkpoint):
    x, w, b, g = norm_inputs(rows, n, BF16, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, checkpoint=checkpoint)
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    assert y.shape == dx.shape == (rows, n) and not bool(dw.any()) and not bool(db.any())


@pytest.mark.gpu
@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True)])
def test_layer_norm_some_gradients(cuda_device, needs):
    for n in (64, 1000, 20000):
        x, w, b, g = norm_inputs(40, n, F32, cuda_device)
        full = [t.clone().requires_grad_(True) for t in (x, w, b)]
        every = torch.autograd.grad(layer_norm(*full), full, g)
        some = [t.clone().requires_grad_(q) for t, q in zip((x, w, b), needs)]
        (got,) = torch.autograd.grad(layer_norm(*some), [t for t in some if t.requires_grad], g)
        assert torch.equal(got, every[needs.index(True)])


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences(cuda_device):
    """As for the linear layer; the third derivative of a row of 48 values of order one is of order one."""
    gen = torch.Generator().manual_seed(9)
    rand = lambda *s: torch.randn(*s, generator=gen).to(cuda_device)  # noqa: E731
    x, w, b, g = rand(40, 48), rand(48), rand(48), rand(40, 48)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    step = 2.0 ** -7
    for i in range(3):
        v = rand(*leaves[i].shape)
        up, down = ([t.detach() + s * step * v if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1))
        loss = [(layer_norm(*a).double() * g.double()).sum() for a in (up, down)]
        along = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double().square().sum() * v.double().square().sum()).sqrt())
        assert abs(float(loss[0] - loss[1]) / (2 * step) - along) <= 2.0 ** -9 * size


@pytest.mark.gpu
def test_layer_norm_repeats_its_bits(cuda_device):
    for n in (256, 1000, 5000):
        x, w, b, g = norm_inputs(5000, n, BF16, cuda_device)
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        first, second = (torch.autograd.grad(layer_norm(*leaves), leaves, g) for _ in range(2))
        assert all(torch.equal(p, q) for p, q in zip(first, second))


# ---- 8-bit checkpoints ----------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32, F16], ids=["bf16", "f32", "f16"])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (7, 33), (2, 3, 100), (1000, 256), (257, 771), (40,)])
def test_checkpoint_holds_what_its_definition_says(cuda_device, shape, dtype):
    gen = torch.Generator().manual_seed(len(shape))
    x = torch.randn(*shape, generator=gen) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=gen))
    x = x.to(dtype).to(cuda_device)
    kept = checkpoint_pack(x)
    assert kept.codes.shape == x.shape and kept.codes.dtype == torch.int8
    assert kept.exponents.shape == (*shape[:-1], -(-shape[-1] // 32)) and kept.dtype == dtype
    expected = held64(x)
    assert torch.equal(checkpoint_unpack(kept, F32).double(), expected)
    assert torch.equal(checkpoint_unpack(kept).double(), expected.to(dtype).double())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [32, 35, 256])
def test_checkpoint_edges(cuda_device, n):
    """Zeros, powers of two, the borders 127 and its neighbour, ties, the ends of the range."""
    x = torch.zeros(12, n)
    x[1, 0], x[2, 0], x[3, 0] = 127.0, 127.0 + 2.0 ** -16, 128.0
    x[4, :5] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5])
    x[5, 0], x[6, 0], x[7, 0] = 3.4028234e38, 2.0 ** -149, 2.0 ** -126
    x[8, :2] = torch.tensor([1e-40, -1e-38])
    x[9, 0], x[10, 1] = -255.0, 2.0 ** 100
    x[11] = torch.linspace(-1, 1, n)
    x = x.to(cuda_device)
    kept = checkpoint_pack(x)
    assert torch.equal(checkpoint_unpack(kept).double(), held64(x))
    assert [int(v) for v in kept.exponents[:5, 0]] == [1, 127, 128, 128, 127]


@pytest.mark.gpu
def test_checkpoint_not_finite_and_strides(cuda_device):
    x = torch.randn(6, 96, device=cuda_device)
    clean = checkpoint_unpack(checkpoint_pack(x))
    bad = x.clone()
    bad[1, 40], bad[2, 0] = float("inf"), float("nan")
    got = checkpoint_unpack(checkpoint_pack(bad))
    assert bool(got[1, 32:64].isnan().all()) and bool(got[2, :32].isnan().all())
    got[1, 32:64], got[2, :32] = clean[1, 32:64], clean[2, :32]
    assert torch.equal(got, clean)
    for view in (x[:, 1:70], x.T, x[::2], x[:, :1].expand(6, 50), x.view(2, 3, 96).transpose(0, 1)):
        a, e = checkpoint_pack(view), checkpoint_pack(view.contiguous())
        assert torch.equal(a.codes, e.codes) and torch.equal(a.exponents, e.exponents)
    empty = checkpoint_unpack(checkpoint_pack(x[:0]))
    assert empty.shape == (0, 96)
    assert checkpoint_unpack(checkpoint_pack(x[:, :0])).shape == (6, 0)


@pytest.mark.gpu
def test_checkpoint_keeps_nothing_larger(cuda_device):
    """What a training step keeps between forward and backward: the input in 8.25 bits, nothing of the output's size."""
    x = torch.randn(4096, 512, device=cuda_device, dtype=BF16)
    w = torch.randn(1024, 512, device=cuda_device, dtype=BF16, requires_grad=True)
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
        linear_act(x, w, activation="gelu", checkpoint="int8")
        layer_norm(x.clone().requires_grad_(True), checkpoint="int8")
    held = [t for t in saved if t.data_ptr() != w.data_ptr()]
    assert sum(t.numel() * t.element_size() for t in held) == 2 * (4096 * 512 + 4096 * 16)


# ---- refusals (no GPU) ------------------------------------------------------------------------


def test_layer_ops_need_cuda_tensors_and_say_so():
    x, w = torch.zeros(2, 8), torch.zeros(3, 8)
    calls = {"linear_act": lambda **k: linear_act(x, w, **k), "layer_norm": lambda **k: layer_norm(x, **k),
             "checkpoint_pack": lambda **k: checkpoint_pack(x, **k),
             "checkpoint_unpack": lambda **k: checkpoint_unpack(
                 Checkpoint8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8), F32), **k)}
    for name, call in calls.items():
        clear_dispatch_report()
        with pytest.raises(RuntimeError, match="need CUDA tensors"):
            call()
        last = get_last_dispatch_report()
        assert last.operator == name and last.selected_backend == "error"
        with pytest.raises(RuntimeError, match="unknown backend"):
            call(backend="other")


def test_linear_refuses_bad_arguments():
    x, w, b = torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(3)
    with pytest.raises(TypeError, match="input must be a tensor"):
        linear_act([1.0], w)
    with pytest.raises(TypeError, match="float16, bfloat16 or float32"):
        linear_act(x.double(), w.double())
    with pytest.raises(TypeError, match="weight must have the dtype"):
        linear_act(x, w.bfloat16())
    with pytest.raises(TypeError, match="residual must have the dtype"):
        linear_act(x, w, b, torch.zeros(2, 3, dtype=BF16))
    with pytest.raises(ValueError, match="activation must be one of"):
        linear_act(x, w, activation="tanh")
    with pytest.raises(ValueError, match="checkpoint must be"):
        linear_act(x, w, checkpoint="fp8")
    with pytest.raises(ValueError, match="weight two"):
        linear_act(x, torch.zeros(8))
    with pytest.raises(ValueError, match="input has 8 features, weight takes 9"):
        linear_act(x, torch.zeros(3, 9))
    with pytest.raises(ValueError, match="bias must have shape"):
        linear_act(x, w, torch.zeros(4))
    with pytest.raises(ValueError, match="cannot be broadcast"):
        linear_act(x, w, b, torch.zeros(2, 4))


def test_layer_norm_refuses_bad_arguments():
    x = torch.zeros(2, 8)
    with pytest.raises(TypeError, match="float16, bfloat16 or float32"):
        layer_norm(x.double())
    with pytest.raises(TypeError, match="or float32"):
        layer_norm(x.bfloat16(), torch.zeros(8, dtype=F16))
    with pytest.raises(TypeError, match="one dtype"):
        layer_norm(x.bfloat16(), torch.zeros(8), torch.zeros(8, dtype=BF16))
    with pytest.raises(ValueError, match="weight must have shape"):
        layer_norm(x, torch.zeros(7))
    with pytest.raises(ValueError, match="at least one dimension"):
        layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="checkpoint must be"):
        layer_norm(x, checkpoint=8)


def test_checkpoint_refuses_bad_arguments():
    codes, exps = torch.zeros(2, 40, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8)
    with pytest.raises(TypeError, match="float16, bfloat16 or float32"):
        checkpoint_pack(torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="int8"):
        checkpoint_unpack(Checkpoint8(codes.float(), exps, F32))
    with pytest.raises(TypeError, match="dtype must be"):
        checkpoint_unpack(Checkpoint8(codes, exps, F32), torch.float64)
    with pytest.raises(ValueError, match="one byte for each block"):
        checkpoint_unpack(Checkpoint8(codes, exps[:, :1], F32))


def _refused(name, args, match):
    module = native.load_native_module()
    fn = getattr(module.lib, name)
    fn.restype = ctypes.c_int
    fn.argtypes = list(native._PLAIN_SIGNATURES[name]) + [ctypes.c_void_p]
    assert fn(*args, None) == 1
    assert match in module.last_error()


def test_plain_entries_refuse_before_any_launch():
    p = 4096  # never dereferenced: every call fails its checks
    good = dict(dtype=1, activation=2, rows=64, in_features=8, out_features=16, input_stride=8, weight_stride=8,
                output_stride=16, grad_output_stride=16, input=p, weight=p, output=p, grad_output=p)
    for change, match in ((dict(dtype=5), "dtype must be"), (dict(activation=9), "activation must be"),
                          (dict(rows=-1), "non-negative"), (dict(rows=2 ** 31), "rows exceeds"),
                          (dict(input_stride=-8), "strides"), (dict(weight=None), "weight is null"),
                          (dict(output=None), "output is null"), (dict(output_stride=8), "must not overlap"),
                          (dict(input_stride=9), "workspace has 0 bytes")):
        args = native.LinearArgs(**{**good, **change})
        _refused("msda_linear_act_forward", [ctypes.byref(args)], match)
    for change, match in ((dict(codes=p), "codes and exponents"), (dict(grad_output=None), "grad_output is null"),
                          (dict(input=None), "input is null"), (dict(grad_input=p), "workspace has 0 bytes"),
                          (dict(grad_input=p, workspace=p + 8, workspace_bytes=1 << 30), "256-byte aligned")):
        args = native.LinearArgs(**{**good, **change})
        _refused("msda_linear_act_backward", [ctypes.byref(args)], match)
    norm = dict(dtype=1, weight_dtype=0, rows=4, cols=8, input_stride=8, grad_output_stride=8, eps=1e-5, input=p,
                output=p, mean=p, rstd=p, grad_output=p)
    for change, match in ((dict(dtype=0, weight_dtype=1), "weight_dtype must be dtype or float32"),
                          (dict(cols=-2), "non-negative"), (dict(rstd=None), "mean and rstd"),
                          (dict(output=None), "output is null"), (dict(codes=p), "codes and exponents")):
        args = native.LayerNormArgs(**{**norm, **change})
        _refused("msda_layer_norm_forward", [ctypes.byref(args)], match)
    args = native.LayerNormArgs(**{**norm, "grad_weight": p})
    _refused("msda_layer_norm_backward", [ctypes.byref(args)], "workspace has 0 bytes")
    _refused("msda_checkpoint_pack", [3, p, 1, 1, 1, p, p], "dtype must be")
    _refused("msda_checkpoint_pack", [0, None, 1, 1, 1, p, p], "input is null")
    _refused("msda_checkpoint_unpack", [0, p, p, 1, 1, None], "output is null")


def test_plain_entries_accept_empty_problems():
    module = native.load_native_module()
    args = native.LinearArgs(dtype=0, rows=0, in_features=8, out_features=8)
    args.weight = 4096
    fn = module.lib.msda_linear_act_forward
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.POINTER(native.LinearArgs), ctypes.c_void_p]
    assert fn(ctypes.byref(args), None) == 0
    empty = native.LayerNormArgs(rows=0, cols=8)
    fn = module.lib.msda_layer_norm_forward
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.POINTER(native.LayerNormArgs), ctypes.c_void_p]
    assert fn(ctypes.byref(empty), None) == 0

"""gated_linear against plain 64-bit formulas.

Tolerances, per element, from the arithmetic, on top of one rounding of the result
(in `near`): a pre-activation is a float32 sum, off by 2^-20 of the sum of its terms'
magnitudes; an activation passes that on with a slope of at most 1.2, its slope with
one of at most 1. The bfloat16 kernels' activations are off by 2^-12 of their terms'
size besides. In training the factors are rounded (beside bfloat16 to float16 under an
exponent of eight, 2^-11), and dz to the rows' type (2^-8 in bfloat16), but for db.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from muspace_b200 import clear_dispatch_report, get_last_dispatch_report
from muspace_b200.ops import dropout, gated_linear, linear_act
from muspace_b200.runtime import native
from test_layer_ops import BF16, F16, F32, SUM, act64, near, slope64
from test_residual_ops import SEED, SEQUENCE, factors

STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}  # half a step of dz in storage
FACTOR = {BF16: 2.0 ** -11, F32: 2.0 ** -24}  # and of a factor
FAST = {BF16: 2.0 ** -12, F32: 0.0}  # of an activation


def inputs(rows, k, n, dtype, device, seed=0, bias=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    out = [t.to(dtype).to(device) for t in (r(rows, k), r(2 * n, k) / math.sqrt(max(k, 1)), 0.3 * r(2 * n), r(rows, n))]
    if not bias:
        out[2] = None
    return out


def check(x, w, b, g, activation="silu", p=0.0, need="xwb", seed=SEED):
    """Forward and backward of one call against the formulas; returns the outputs."""
    dtype, rows, n = x.dtype, x.size(0), w.size(0) // 2
    leaves = {m: t.detach().requires_grad_(m in need) for m, t in zip("xwb", (x, w, b)) if t is not None}
    y = gated_linear(leaves["x"], leaves["w"], leaves.get("b"), activation=activation, dropout=p, seed=seed,
                     sequence=SEQUENCE)
    x6, w6, g6 = x.double(), w.double(), g.double()
    b6 = b.double() if b is not None else torch.zeros(2 * n, dtype=torch.float64, device=x.device)
    f = factors(rows, n, p, int(seed), SEQUENCE).to(x.device) if p else torch.ones(rows, n, device=x.device).double()
    z, size = x6 @ w6.T + b6, x6.abs() @ w6.abs().T + b6.abs()
    zg, zu, size_g, size_u = z[:, :n], z[:, n:], size[:, :n], size[:, n:]
    act, slope = act64(activation, zg), slope64(activation, zg)
    fast = FAST[dtype] / SUM
    off_act, off_slope = 1.2 * size_g + fast * act.abs(), size_g + fast * 1.2
    expected = f * act * zu
    near(y.detach(), expected, f * (off_act * zu.abs() + act.abs() * size_u) + expected.abs(), dtype)
    wanted = [m for m in leaves if m in need]
    grads = dict(zip(wanted, torch.autograd.grad(y, [leaves[m] for m in wanted], g)))
    dz = torch.cat([g6 * f * slope * zu, g6 * f * act], 1)
    loose = SUM * torch.cat([g6.abs() * f * (off_slope * zu.abs() + slope.abs() * size_u), g6.abs() * f * off_act], 1)
    loose = loose + FACTOR[dtype] * dz.abs()
    rounded = loose + STEP[dtype] * dz.abs() * 1.01
    for name, value, error, terms in (("x", dz @ w6, rounded @ w6.abs(), dz.abs() @ w6.abs()),
                                      ("w", dz.T @ x6, rounded.T @ x6.abs(), dz.abs().T @ x6.abs()),
                                      ("b", dz.sum(0), loose.sum(0), dz.abs().sum(0))):
        if name in grads:
            near(grads[name], value, terms + error / SUM, dtype)
    return y.detach(), grads


SHAPES = [(1, 1, 1), (1, 256, 512), (1, 4096, 300), (2, 1000, 96), (3, 7, 5), (7, 512, 64), (17, 40, 33), (40, 640, 96),
          (127, 64, 63), (128, 128, 128), (129, 65, 257), (300, 517, 259), (600, 1024, 40), (513, 1000, 8),
          (200, 256, 512), (5000, 256, 136), (2048, 512, 576), (2050, 1100, 520), (700, 2048, 1152), (9000, 64, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_gated_matches_the_formulas(cuda_device, rows, k, n, p, dtype):
    check(*inputs(rows, k, n, dtype, cuda_device, seed=rows + k + n), "gelu" if p else "silu", p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("rows,k,n", [(1, 72, 200), (321, 72, 200), (321, 640, 200), (130, 67, 77), (4000, 128, 256)])
def test_gated_activations(cuda_device, rows, k, n, activation, dtype):
    check(*inputs(rows, k, n, dtype, cuda_device, seed=k), activation, 0.1)
    check(*inputs(rows, k, n, dtype, cuda_device, seed=k, bias=False), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 150, 3000])
def test_gated_relu(cuda_device, rows, dtype):
    """Integers: every pre-activation is exact, so the kink falls the same way everywhere."""
    gen = torch.Generator().manual_seed(3)
    x, w, b, g = (torch.randint(-2, 3, s, generator=gen).to(dtype).to(cuda_device)
                  for s in ((rows, 64), (144, 64), (144,), (rows, 72)))
    check(x, w, b, g, "relu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_gated_inference_and_training_agree(cuda_device, dtype):
    """The kernel without factors gives the bits of the one with them."""
    for rows, k, n in ((1, 256, 128), (5, 256, 128), (300, 256, 128), (4000, 256, 512), (4000, 200, 136), (90, 40, 33)):
        x, w, b, _ = inputs(rows, k, n, dtype, cuda_device)
        for activation in ("none", "relu", "gelu", "silu"):
            kept = gated_linear(x, w.clone().requires_grad_(True), b, activation=activation, dropout=0.2, seed=5)
            got = gated_linear(x, w, b, activation=activation, dropout=0.2, seed=5)
            if dtype == BF16 and rows <= 8:  # inference takes few rows in another order: two roundings of one sum
                assert torch.allclose(kept.double(), got.double(), rtol=2.0 ** -7, atol=2.0 ** -12)
            else:
                assert torch.equal(kept.detach(), got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(40, 64), (40, 67), (3000, 512), (3000, 520)])
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -12, 2.0 ** 20, 2.0 ** 60])
def test_gated_factors_of_any_size(cuda_device, rows, n, scale):
    """Bfloat16's factors are halves under an exponent: pre-activations far outside of
    float16's range lose no more than others, whatever their neighbours in other eights are."""
    x, w, b, g = inputs(rows, 64, n, BF16, cuda_device)
    w[n:] *= scale  # up, and with it the gate's gradient
    b[n:] *= scale
    w[n + 16:n + 24] /= scale
    b[n + 16:n + 24] /= scale
    check(x, w, b, g, "silu", 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(40, 72), (3000, 512)])
def test_gated_infinite_factors_leave_their_neighbours(cuda_device, rows, n):
    x, w, b, g = inputs(rows, 64, n, BF16, cuda_device)
    clean = [t.clone().requires_grad_(True) for t in (x, w, b)]
    expected = torch.autograd.grad(gated_linear(*clean), clean, g)
    bad = w.clone()
    bad[n + 3] = math.inf  # one column of up: its factor P is not finite
    leaves = [x.clone().requires_grad_(True), bad.requires_grad_(True), b.clone().requires_grad_(True)]
    dw, db = torch.autograd.grad(gated_linear(*leaves), leaves, g)[1:]
    keep = [i for i in range(2 * n) if i != 3]
    assert torch.equal(dw[keep], expected[1][keep]) and torch.equal(db[keep], expected[2][keep])
    assert not bool(dw[3].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 200), (6, 64, 77), (400, 64, 200), (400, 64, 77), (3000, 512, 640)])
def test_gated_drops_what_dropout_drops(cuda_device, rows, k, n, dtype):
    x, w, b, _ = inputs(rows, k, n, dtype, cuda_device)
    y = gated_linear(x, w, b, dropout=0.3, seed=torch.tensor(SEED, device=cuda_device), sequence=9)
    ones = dropout(torch.ones(rows, n, device=cuda_device), 0.3, seed=SEED, sequence=9)
    plain = gated_linear(x, w, b)
    assert torch.equal(y == 0, (ones == 0) | (plain == 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(0, 8, 16), (5, 0, 16), (300, 0, 16), (5, 8, 0), (0, 0, 0)])
def test_gated_empty(cuda_device, rows, k, n, dtype):
    y, grads = check(*inputs(rows, k, n, dtype, cuda_device), p=0.2)
    assert y.shape == (rows, n) and grads["x"].shape == (rows, k) and grads["w"].shape == (2 * n, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_gated_strides_offsets_and_leading_shapes(cuda_device, dtype):
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=gen).to(dtype).to(cuda_device)  # noqa: E731
    wide = rand(70, 300)
    layouts = {
        "column slice": (wide[:, 5:105], rand(60, 100)),
        "every other row": (wide[::2, :100], rand(60, 100)),
        "transposed": (rand(100, 35).T, rand(100, 60).T),
        "broadcast rows": (rand(1, 100).expand(35, 100), rand(60, 100)),
        "weight rows off 16 bytes": (rand(35, 100), rand(61, 101)[1:, 1:]),
        "odd base": (rand(35 * 100 + 1)[1:].view(35, 100), rand(64, 100)),
    }
    for x, w in layouts.values():
        n = w.size(0) // 2
        check(x, w, rand(2 * n), rand(n, x.size(0)).T, "gelu", 0.2)
        check(x, w, rand(2 * n + 1)[1:], rand(1, n).expand(x.size(0), n), "gelu")
    x, w, b = rand(3, 4, 5, 100), rand(48, 100), rand(48)
    y = gated_linear(x, w, b, dropout=0.1, seed=3)
    assert y.shape == (3, 4, 5, 24)
    assert torch.equal(y.view(-1, 24), gated_linear(x.reshape(-1, 100), w, b, dropout=0.1, seed=3))
    assert torch.equal(gated_linear(x[0, 0, 0], w, b), gated_linear(x[0, 0, :1], w, b)[0])
    turned = x.permute(2, 0, 1, 3)
    assert torch.equal(gated_linear(turned, w, b), gated_linear(turned.contiguous(), w, b))


@pytest.mark.gpu
@pytest.mark.parametrize("need", ["x", "w", "b", "xw", "xb", "wb"])
def test_gated_some_gradients(cuda_device, need):
    for dtype in (BF16, F32):
        check(*inputs(100, 64, 48, dtype, cuda_device), need=need, p=0.1)
        check(*inputs(3, 64, 47, dtype, cuda_device), need=need)


@pytest.mark.gpu
def test_gated_float16(cuda_device):
    x, w, b, g = inputs(60, 40, 24, F16, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = gated_linear(*leaves)
    z = x.detach().double() @ w.detach().double().T + b.detach().double()
    # float16's smallest step is 2^-24: half of it, whatever the number
    near(y.detach(), act64("silu", z[:, :24]) * z[:, 24:], 10 * z.abs().amax() ** 2 + 2.0 ** -25 / SUM, F16)
    assert {t.dtype for t in torch.autograd.grad(y, leaves, g)} == {F16}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(150, 72, 200), (2, 72, 200), (40, 640, 96)])
def test_gated_infinities_and_nans_stay_in_their_rows(cuda_device, dtype, rows, k, n):
    x, w, b, _ = inputs(rows, k, n, dtype, cuda_device)
    clean = gated_linear(x, w, b)
    bad = x.clone()
    bad[1, 5] = float("nan")
    y = gated_linear(bad, w, b)
    assert bool(y[1].isnan().all()) and torch.equal(y[2:], clean[2:]) and torch.equal(y[0], clean[0])
    wide = w.clone()
    wide[n + 2, 1] = math.inf  # one row of up
    y = gated_linear(x, wide, b)
    keep = [i for i in range(n) if i != 2]
    assert torch.equal(y[:, keep], clean[:, keep]) and not bool(y[:, 2].isfinite().any())
    f = factors(rows, n, 0.5, 3, 0).to(cuda_device)
    y = gated_linear(bad, w, b, dropout=0.5, seed=3)  # what is dropped is 0
    assert torch.equal(y[1].isnan(), f[1] > 0) and not bool(y[1][f[1] == 0].any())


@pytest.mark.gpu
def test_gated_gradient_against_differences(cuda_device):
    """Central differences of the forward in float32 along random directions; step 2^-6
    of directions of unit size in a pre-activation: its square times third derivatives
    of order ten is below 2^-8 of the result's size."""
    x, w, b, g = inputs(33, 64, 40, F32, cuda_device)
    run = lambda a: gated_linear(*a, activation="gelu", dropout=0.2, seed=7)  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(run(leaves), leaves, g)
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(i)).to(cuda_device)
        step = 2.0 ** -6 / (8 if i == 1 else 1)
        up, down = ([t.detach() + s * step * v if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1))
        loss = [float((run(a).double() * g.double()).sum()) for a in (up, down)]
        along = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double().square().sum() * v.double().square().sum()).sqrt())
        assert abs((loss[0] - loss[1]) / (2 * step) - along) <= 2.0 ** -8 * size


@pytest.mark.gpu
def test_gated_repeats_its_bits(cuda_device):
    for dtype in (BF16, F32):
        for rows, k, n in ((4000, 256, 512), (33, 2048, 96), (2, 4096, 256)):
            args = inputs(rows, k, n, dtype, cuda_device)
            first, second = (check(*args, p=0.1) for _ in range(2))
            assert torch.equal(first[0], second[0])
            assert all(torch.equal(first[1][m], second[1][m]) for m in first[1])


@pytest.mark.gpu
def test_gated_past_two_to_the_31_elements(cuda_device):
    """Rows whose offsets need 64 bits equal the same rows of a small call, forward and backward."""
    rows, n = 132000, 8200  # 2.16e9 factors
    x = torch.randn(rows, 32, device=cuda_device, dtype=BF16)
    w = torch.randn(2 * n, 32, device=cuda_device, dtype=BF16) / 4
    tail = slice(rows - 300, rows)
    leaf = x.clone().requires_grad_(True)
    y = gated_linear(leaf, w)
    (d,) = torch.autograd.grad(y, [leaf], y.detach())
    small = x[tail].clone().requires_grad_(True)
    part = gated_linear(small, w)
    assert torch.equal(y[tail].detach(), part.detach())
    (e,) = torch.autograd.grad(part, [small], part.detach())
    assert torch.allclose(d[tail].double(), e.double(), rtol=2.0 ** -7, atol=2.0 ** -7 * float(e.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_gated_on_a_side_stream_and_in_a_graph(cuda_device, dtype):
    """Two products at once on two streams; a captured training step with its seed on the device."""
    x, w, b, g = inputs(700, 256, 96, dtype, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def step(seed):
        y = gated_linear(*leaves, dropout=0.3, seed=seed)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    expected = step(5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            results.append([step(5) for _ in range(3)])
    for stream in streams:
        torch.cuda.current_stream().wait_stream(stream)
    for group in results:
        for got in group:
            assert all(torch.equal(a, e) for a, e in zip(got, expected))
    seed = torch.zeros((), dtype=torch.int64, device=cuda_device)
    with torch.cuda.stream(streams[0]):
        step(seed)
    torch.cuda.current_stream().wait_stream(streams[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(seed)
    for value in (5, 6):
        seed.fill_(value)
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip([t.clone() for t in captured], step(value)))


@pytest.mark.gpu
def test_gated_feed_forward_block(cuda_device):
    """The whole block with its product onto the residual, against autograd in 64 bits."""
    x, w, b, _ = inputs(500, 64, 96, F32, cuda_device)
    down, shift, g = (torch.randn(s, generator=torch.Generator().manual_seed(1)).to(cuda_device)
                      for s in ((64, 96), (64,), (500, 64)))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, down, shift)]
    y = linear_act(gated_linear(*leaves[:3], activation="gelu"), leaves[3], leaves[4], leaves[0])
    grads = torch.autograd.grad(y, leaves, g)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    gate, up = torch.nn.functional.linear(wide[0], wide[1], wide[2]).chunk(2, -1)
    z = torch.nn.functional.linear(torch.nn.functional.gelu(gate) * up, wide[3], wide[4]) + wide[0]
    for a, e in zip((y, *grads), (z, *torch.autograd.grad(z, wide, g.double()))):
        assert float((a.double() - e).norm()) <= 2.0 ** -20 * float(e.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [64, 67])
def test_gated_dropped_elements_pass_no_infinity_on(cuda_device, n, dtype):
    x, w, b, g = inputs(50, 32, n, dtype, cuda_device)
    f = factors(50, n, 0.5, SEED, 0).to(cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    run = lambda grad: torch.autograd.grad(gated_linear(*leaves, dropout=0.5, seed=SEED), leaves, grad)  # noqa: E731
    clean = run(torch.where(f > 0, g, torch.zeros_like(g)))
    for value in (math.inf, math.nan):
        for a, e in zip(run(torch.where(f > 0, g, torch.full_like(g, value))), clean):
            assert torch.equal(a, e)


@pytest.mark.gpu
def test_gated_is_differentiable_once(cuda_device):
    from torch.autograd import forward_ad

    x, w, b, _ = inputs(6, 16, 8, F32, cuda_device)
    x.requires_grad_(True)
    (d,) = torch.autograd.grad(gated_linear(x, w, b).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        gated_linear(forward_ad.make_dual(x.detach(), torch.ones_like(x)), w, b)


def test_gated_refusals():
    x, w, b = torch.randn(4, 8), torch.randn(12, 8), torch.randn(12)
    for error, args, how in (
            (TypeError, (1.0, w), {}), (TypeError, (x, w.bfloat16()), {}), (TypeError, (x, w, b.bfloat16()), {}),
            (TypeError, (x.double(), w.double()), {}), (ValueError, (x, w[:11]), {}), (ValueError, (x, w[:, :7]), {}),
            (ValueError, (x, w, b[:6]), {}), (ValueError, (x[0, 0], w), {}), (ValueError, (x, w[0]), {}),
            (ValueError, (x, w), dict(activation="sigmoid")), (ValueError, (x, w), dict(dropout=0.1)),
            (ValueError, (x, w), dict(dropout=2, seed=1)), (TypeError, (x, w), dict(dropout=0.1, seed=0.5)),
            (RuntimeError, (x, w, b), {}), (RuntimeError, (x, w, b), dict(backend="nothing"))):
        with pytest.raises(error):
            gated_linear(*args, **how)
    clear_dispatch_report()
    with pytest.raises(RuntimeError, match="gated linear kernels need CUDA tensors"):
        gated_linear(x, w)
    assert get_last_dispatch_report().operator == "gated_linear"


@pytest.mark.parametrize("dtype", [0, 1])
def test_gated_workspace_holds_the_sums(dtype):
    """Rows off 16 bytes are finished from float32 sums of both halves, read eight at a time."""
    lib = native.load_native_module().lib
    query = lib.msda_gated_linear_forward_workspace
    query.restype, query.argtypes = ctypes.c_int, [ctypes.POINTER(native.GatedLinearArgs), ctypes.POINTER(ctypes.c_size_t)]
    size, p = ctypes.c_size_t(), 4096  # aligned, never dereferenced
    for rows in (2000, 40000):
        for n in (1, 3, 7, 9, 33, 257):
            args = native.GatedLinearArgs(dtype=dtype, rows=rows, in_features=256, out_features=n, input_stride=256,
                                          weight_stride=256, output_stride=n, input=p, weight=p, output=p)
            assert query(args, size) == 0
            assert size.value >= rows * -(-2 * n // 8) * 8 * 4 or (dtype == 0 and rows * 256 * 2 * n <= 2 ** 26)


def test_gated_c_entry_refusals():
    module = native.load_native_module()
    p = 4096

    def fails(name, message, **fields):
        entry = getattr(module.lib, name)
        entry.restype, entry.argtypes = ctypes.c_int, [ctypes.POINTER(native.GatedLinearArgs), ctypes.c_void_p]
        assert entry(native.GatedLinearArgs(**fields), None) == 1 and message in module.last_error()

    good = dict(rows=4, in_features=8, out_features=8, input_stride=8, weight_stride=8, output_stride=8, input=p, weight=p,
                output=p)
    fails("msda_gated_linear_forward", "dtype must be", **{**good, "dtype": 2})
    fails("msda_gated_linear_forward", "activation must be", **{**good, "activation": 4})
    fails("msda_gated_linear_forward", "out_features exceeds", **{**good, "out_features": 2 ** 30})
    fails("msda_gated_linear_forward", "weight is null", **{**good, "weight": None})
    fails("msda_gated_linear_forward", "output rows", **{**good, "output_stride": 4})
    fails("msda_gated_linear_forward", "threshold must be", **{**good, "threshold": -1})
    back = dict(rows=4, in_features=8, out_features=8, grad_output=p, factors=p, grad_bias=p)
    fails("msda_gated_linear_backward", "factors is null", **{**back, "factors": None})
    fails("msda_gated_linear_backward", "input is null", **{**back, "grad_weight": p})
    fails("msda_gated_linear_backward", "workspace has 0 bytes", **back)


# ---- factors of one eight that are far apart ----------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(40, 64), (40, 67), (3000, 512), (3000, 520)])
@pytest.mark.parametrize("spread", [2.0 ** -10, 2.0 ** -18, 2.0 ** -25])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -10, 1.0, 2.0 ** 20])
def test_gated_factors_beside_larger_ones(cuda_device, rows, n, spread, size):
    """One column in eight far smaller than its neighbours keeps its gradients' digits: with the
    eight's largest brought to 2^14, factors down to 2^-28 of it are normal halves. Up's column makes
    its P small, and without an activation the gate's makes its Q small."""
    x, w, b, g = inputs(rows, 64, n, BF16, cuda_device, seed=3)
    up, gate = w.clone(), w.clone()
    up[n:] *= size
    up[n + 3::8] *= spread
    b_up = b.clone()
    b_up[n:] *= size
    b_up[n + 3::8] *= spread
    check(x, up, b_up, g, "silu", 0.1)
    gate[:n] *= size
    gate[3:n:8] *= spread
    b_gate = b.clone()
    b_gate[:n] *= size
    b_gate[3:n:8] *= spread
    check(x, gate, b_gate, g, "none", 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(40, 64), (40, 67), (3000, 512)])
def test_gated_factors_far_below_their_neighbours(cuda_device, rows, n):
    """Below 2^-28 of the eight's largest a factor is off by up to 2^-39 of that one: half of float16's
    smallest step, 2^-24, beside a largest of at least 2^14."""
    x, w, b, g = inputs(rows, 64, n, BF16, cuda_device, seed=4)
    w[n + 3::8] *= 2.0 ** -45
    b[n + 3::8] *= 2.0 ** -45
    leaf = b.clone().requires_grad_(True)
    (db,) = torch.autograd.grad(gated_linear(x, w, leaf), [leaf], g)
    x6, w6, b6, g6 = (t.double() for t in (x, w, b, g.abs()))
    z, size = x6 @ w6.T + b6, x6.abs() @ w6.abs().T + b6.abs()
    zu, slope = z[:, n:], slope64("silu", z[:, :n])
    p = slope * zu
    most = torch.nn.functional.pad(p.abs(), (0, -n % 8)).view(rows, -1, 8).amax(-1).repeat_interleave(8, 1)[:, :n]
    loose = SUM * ((size[:, :n] + 1.2 * FAST[BF16] / SUM) * zu.abs() + slope.abs() * size[:, n:]) + FACTOR[BF16] * p.abs()
    loose = loose + 2 * 2.0 ** -39 * most  # twice, as the largest itself is off by a little
    expected, terms = (g.double() * p).sum(0), (g6 * (p.abs() + loose / SUM)).sum(0)
    near(db[3:n:8], expected[3::8], terms[3::8], BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("rows,n", [(3, 64), (50, 64), (50, 67), (2000, 512), (2000, 516)])
def test_gated_zero_factors_hide_no_gradient(cuda_device, rows, n, p, dtype):
    """Where relu is off both factors are 0, of either sign; a gradient there that is not finite gives
    NaN, as 0 times it is. Dropped elements alone pass nothing on."""
    gen = torch.Generator().manual_seed(3)
    x, w, b, g = (torch.randint(-2, 3, s, generator=gen).to(dtype).to(cuda_device)
                  for s in ((rows, 64), (2 * n, 64), (2 * n,), (rows, n)))
    f = factors(rows, n, p, SEED, SEQUENCE).to(cuda_device) if p else torch.ones(rows, n, device=cuda_device)
    off = (x.double() @ w[:n].double().T + b[:n].double()) <= 0
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    run = lambda grad: torch.autograd.grad(  # noqa: E731
        gated_linear(*leaves, activation="relu", dropout=p, seed=SEED, sequence=SEQUENCE), leaves, grad)
    clean = run(g)
    columns, lines = [2, n - 1], []
    for c in columns:
        kept = (off[:, c] & (f[:, c] > 0)).nonzero()
        assert len(kept)
        lines.append(int(kept[0]))
    for value in (math.inf, math.nan):
        bad = torch.where(f > 0, g, torch.full_like(g, value))  # every dropped element too
        for r, c in zip(lines, columns):
            bad[r, c] = value
        dx, dw, db = run(bad)
        hit = torch.zeros(2 * n, dtype=torch.bool, device=cuda_device)
        hit[columns + [n + c for c in columns]] = True
        assert torch.equal(db.isnan(), hit) and bool(dw[hit].isnan().all()) and torch.equal(db[~hit], clean[2][~hit])
        assert torch.equal(dw[~hit], clean[1][~hit])
        rest = [r for r in range(rows) if r not in lines]
        assert bool(dx[lines].isnan().all()) and torch.equal(dx[rest], clean[0][rest])


def test_gated_float32_workspace_holds_planes_and_sums():
    """The three bfloat16 planes of x and of the weight, and behind them the sums, rows padded to eight."""
    lib = native.load_native_module().lib
    query = lib.msda_gated_linear_forward_workspace
    query.restype, query.argtypes = ctypes.c_int, [ctypes.POINTER(native.GatedLinearArgs), ctypes.POINTER(ctypes.c_size_t)]
    size, p = ctypes.c_size_t(), 4096  # aligned, never dereferenced
    for rows in (2000, 40000):
        for n in (1, 3, 7, 9, 33, 257):
            args = native.GatedLinearArgs(dtype=0, rows=rows, in_features=256, out_features=n, input_stride=256,
                                          weight_stride=256, output_stride=n, input=p, weight=p, output=p)
            assert query(args, size) == 0
            assert size.value >= 3 * 2 * 256 * (rows + 2 * n) + rows * -(-2 * n // 8) * 8 * 4


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(40, 64), (40, 67), (3000, 512)])
@pytest.mark.parametrize("activation,bias", [("silu", -18.0), ("silu", -20.0), ("gelu", -5.5), ("gelu", -6.0)])
def test_gated_closed_gates_keep_the_digits_of_up_gradients(cuda_device, rows, n, activation, bias):
    """Gates of one column in eight far on the flat side: Q is 1e-7 of its neighbours' and less. An error of the
    pre-activation counts relatively, by |act'(z) / act(z)| <= |z| + 1 there."""
    x, w, b, g = inputs(rows, 64, n, BF16, cuda_device, seed=6)
    w[3:n:8] /= 64
    b[3:n:8] = bias
    leaf = b.clone().requires_grad_(True)
    (db,) = torch.autograd.grad(gated_linear(x, w, leaf, activation=activation), [leaf], g)
    x6, w6, b6 = x.double(), w[3:n:8].double(), b[3:n:8].double()
    z, size = x6 @ w6.T + b6, x6.abs() @ w6.abs().T + b6.abs()
    terms = (g[:, 3::8].double() * act64(activation, z)).abs()
    loose = terms * (SUM * size * (z.abs() + 1) + FACTOR[BF16] + 2 * FAST[BF16])
    near(db[n + 3::8], (g[:, 3::8].double() * act64(activation, z)).sum(0), (terms + loose / SUM).sum(0), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32, F16], ids=["bf16", "f32", "f16"])
@pytest.mark.parametrize("rows,n", [(2, 64), (300, 64), (300, 67)])
def test_gated_everything_dropped(cuda_device, rows, n, dtype):
    x, w, b, g = inputs(rows, 32, n, dtype, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = gated_linear(*leaves, dropout=1.0, seed=1)
    assert not bool(y.any())
    for d in torch.autograd.grad(y, leaves, torch.full_like(g, math.inf)):
        assert not bool(d.any())


def test_gated_few_rows_of_large_weights_run_in_tiles():
    """One row, and few rows of a weight that is not large, need no workspace: a warp takes a column. More
    work than that runs in tiles, whose ranges of k leave partial sums."""
    lib = native.load_native_module().lib
    query = lib.msda_gated_linear_forward_workspace
    query.restype, query.argtypes = ctypes.c_int, [ctypes.POINTER(native.GatedLinearArgs), ctypes.POINTER(ctypes.c_size_t)]
    size, p = ctypes.c_size_t(), 4096  # aligned, never dereferenced
    for rows, k, n, tiles in ((1, 8192, 8192, False), (2, 4096, 4096, False), (3, 4096, 4096, False), (4, 4096, 2048, False),
                              (4, 4096, 4096, True), (2, 4096, 11008, True), (4, 256, 512, False), (9, 4096, 1024, True)):
        args = native.GatedLinearArgs(dtype=1, rows=rows, in_features=k, out_features=n, input_stride=k, weight_stride=k,
                                      output_stride=n, input=p, weight=p, output=p)
        assert query(args, size) == 0 and (size.value > 0) == tiles


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(2, 4096, 8200), (3, 4096, 5600), (4, 4096, 4096), (4, 4104, 4099)])
def test_gated_few_rows_of_large_weights(cuda_device, rows, k, n):
    x, w, b, _ = inputs(rows, k, n, BF16, cuda_device, seed=9)
    y = gated_linear(x, w, b, dropout=0.2, seed=SEED, sequence=SEQUENCE)
    f = factors(rows, n, 0.2, SEED, SEQUENCE).to(cuda_device)
    z, size = x.double() @ w.double().T + b.double(), x.double().abs() @ w.double().abs().T + b.double().abs()
    act, zu = act64("silu", z[:, :n]), z[:, n:]
    off = 1.2 * size[:, :n] + FAST[BF16] / SUM * act.abs()
    near(y, f * act * zu, f * (off * zu.abs() + act.abs() * size[:, n:] + (act * zu).abs()), BF16)

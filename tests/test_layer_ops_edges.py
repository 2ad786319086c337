"""Edges of linear_act, layer_norm and 8-bit checkpoints: the ends of the
workspace, what is not finite, forward mode and tracing, waits.

Tolerances as in test_layer_ops.py, from which the formulas come, unless a test
says otherwise.
"""

from __future__ import annotations

import ctypes
import importlib
import math
import warnings

import pytest
import torch
from torch.autograd import forward_ad

from muspace_b200.ops import checkpoint_pack, checkpoint_unpack, layer_norm, linear_act
from muspace_b200.runtime import native
from test_layer_ops import (
    BF16, F16, F32, SUM, check_linear, check_norm, held64, linear_inputs, near, norm_inputs, slope64)


def workspace_of(name: str, **fields) -> int:
    """What the entry point's query asks for; nothing is launched."""
    lib = native.load_native_module().lib
    query = getattr(lib, name + "_workspace")
    query.restype = ctypes.c_int
    query.argtypes = [ctypes.POINTER(native.LinearArgs), ctypes.POINTER(ctypes.c_size_t)]
    args, size = native.LinearArgs(**fields), ctypes.c_size_t()
    assert query(args, size) == 0
    return size.value


@pytest.mark.parametrize("rows", [64, 40000, 262144])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 6, 7, 9, 10, 12, 33, 91, 257, 260])
def test_workspace_holds_the_last_vector_of_partial_sums(n, rows):
    """Bfloat16 rows that are no multiple of 16 bytes are finished from float32 sums
    in the workspace, which are read eight at a time to the end of the last row."""
    p = 4096  # aligned, never dereferenced
    common = dict(dtype=1, rows=rows, in_features=256, out_features=n, input_stride=256, weight_stride=256,
                  input=p, weight=p)
    assert workspace_of("msda_linear_act_forward", output_stride=n, output=p, **common) >= rows * -(-n // 8) * 8 * 4
    # dx of n input features: the sums come last there too
    needed = workspace_of("msda_linear_act_backward", dtype=1, rows=rows, in_features=n, out_features=256,
                          weight_stride=n, grad_output_stride=256, weight=p, grad_output=p, grad_input=p)
    assert needed >= rows * -(-n // 8) * 8 * 4


# ---- what is not finite in float32 (more rows than the kernel for few rows takes) ---------


def same_where_not_finite(got, expected):
    """The same infinities and NaNs; returns the rest of both, zeros elsewhere."""
    assert torch.equal(got.isnan(), expected.isnan())
    assert torch.equal(got.isinf(), expected.isinf())
    inf = expected.isinf()
    assert torch.equal(got[inf].double(), expected[inf])
    zero = expected.isfinite()
    return torch.where(zero, got, 0), torch.where(zero, expected, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1100, 64, 96), (1100, 640, 40), (1100, 67, 33), (5000, 2100, 256)])
def test_float32_products_that_overflow_are_infinities(cuda_device, rows, k, n):
    """One product of some 1e30 * 1e30 to an output: an infinity of its sign, beside finite sums."""
    gen = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=gen, dtype=torch.float64).clamp(-3, 3)
    w = torch.randn(n, k, generator=gen, dtype=torch.float64).clamp(-3, 3)
    sizes = lambda count: 1 + torch.rand(count, generator=gen, dtype=torch.float64)  # noqa: E731
    x[::3, 5] = 1e30 * (sizes(rows) * torch.randn(rows, generator=gen, dtype=torch.float64).sign())[::3]
    w[::2, 5] = 1e30 * (sizes(n) * torch.randn(n, generator=gen, dtype=torch.float64).sign())[::2]
    x, w = x.float().to(cuda_device), w.float().to(cuda_device)
    exact = x.double() @ w.double().T
    terms = x.double().abs() @ w.double().abs().T
    exact = torch.where(exact.abs() > 3.5e38, torch.copysign(torch.full_like(exact, float("inf")), exact), exact)
    got, expected = same_where_not_finite(linear_act(x, w), exact)
    near(got, expected, torch.where(exact.isfinite(), terms, 0), F32)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("rows,k,n", [(1200, 256, 520), (1300, 300, 259)])
def test_float32_infinities_in_most_rows_and_columns(cuda_device, rows, k, n, checkpoint):
    x, w, b, r, g = linear_inputs(rows, k, n, F32, cuda_device, seed=k)
    gen = torch.Generator().manual_seed(1)
    pick = lambda t, part: (torch.rand(t.shape, generator=gen) < part).to(t.device)  # noqa: E731
    g = torch.where(pick(g, 0.5 / n), torch.copysign(torch.full_like(g, float("inf")), g), g)
    g = torch.where(pick(g, 0.05 / n), torch.full_like(g, float("nan")), g)
    bad_x = torch.where(pick(x, 0.5 / k), torch.copysign(torch.full_like(x, float("inf")), x), x)
    bad_w = w.clone()
    bad_w[3, 7], bad_w[11, 2] = -float("inf"), float("nan")
    exact = bad_x.double() @ bad_w.double().T + b.double() + r.double()
    size = torch.nan_to_num(bad_x, 0, 0, 0).double().abs() @ torch.nan_to_num(bad_w, 0, 0, 0).double().abs().T
    got, expected = same_where_not_finite(linear_act(bad_x, bad_w, b, r), exact)
    near(got, expected, 2 * size + r.double().abs() + 1, F32)
    # backward: the gradients of finite inputs for a gradient with infinities and NaNs
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(linear_act(*leaves, activation="silu", checkpoint=checkpoint), leaves, g)
    x6 = held64(x) if checkpoint else x.double()
    z = x6 @ w.double().T + b.double()
    slope, clean = slope64("silu", z), torch.nan_to_num(g, 0, 0, 0).double()
    dz, part = g.double() * slope, (clean * slope).abs()
    loose = clean.abs() * 2 * SUM * (x6.abs() @ w.double().abs().T + b.double().abs())
    for value, exact, terms in zip(
            grads, (dz @ w.double(), dz.T @ x6, dz.sum(0)),
            (part @ w.double().abs() + loose @ w.double().abs() / SUM, part.T @ x6.abs() + loose.T @ x6.abs() / SUM,
             part.sum(0) + loose.sum(0) / SUM)):
        got, expected = same_where_not_finite(value, exact)
        near(got, expected, terms, F32)


@pytest.mark.gpu
def test_float32_infinities_cost_no_time(cuda_device):
    """A gradient that overflowed everywhere takes the time of a finite one (within a factor of three)."""
    x, w, b, _, g = linear_inputs(1200, 256, 256, F32, cuda_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear_act(*leaves)
    took = []
    for gradient in (g, torch.full_like(g, float("inf"))):
        times = []
        for _ in range(9):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(1000000)  # the launches wait here, so that the host's part is not timed
            start.record()
            torch.autograd.grad(y, leaves, gradient, retain_graph=True)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        took.append(sorted(times)[4])
    assert took[1] <= 3 * took[0], took


# ---- sums before their rounding ---------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("rows,k,n", [(300, 72, 200), (300, 72, 77), (2000, 2048, 33), (300, 0, 77)])
def test_bias_gradient_is_rounded_once(cuda_device, rows, k, n, checkpoint):
    """Equal rows, so that a rounding of dz before its sum would be the same one in
    every term: db is within half a unit of its last place (2^-8 of its power of
    two), and the error of a float32 sum, of the exact sum."""
    x, w, b, _, g = linear_inputs(1, k, n, BF16, cuda_device, seed=k)
    x, g = x.expand(rows, k), g.expand(rows, n)
    bias = b.clone().requires_grad_(True)
    (db,) = torch.autograd.grad(linear_act(x, w, bias, activation="silu", checkpoint=checkpoint), [bias], g)
    x6 = held64(x) if checkpoint else x.double()
    z = x6 @ w.double().T + b.double()
    dz = g.double() * slope64("silu", z)
    # the slope: 2^-11 of it where the forward kept it in float16, and what z's error moves it by
    loose = dz.abs() * (0 if checkpoint else 2.0 ** -11) + 2 * SUM * g.double().abs() * (
        x6.abs() @ w.double().abs().T + b.double().abs())
    exact = dz.sum(0)
    bound = torch.exp2(exact.abs().log2().floor() - 8) + SUM * dz.abs().sum(0) + loose.sum(0)
    assert bool(((db.double() - exact).abs() <= bound).all()), float(((db.double() - exact).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [250, 255, 129])
def test_bias_gradient_of_rows_that_end_with_their_storage(cuda_device, n):
    """A gradient whose rows are 256 apart and whose last one ends the tensor's memory; what lies between rows is NaN."""
    rows = 700
    gen = torch.Generator().manual_seed(n)
    held = torch.full((256 * (rows - 1) + n,), float("nan"), dtype=BF16, device=cuda_device)
    g = torch.as_strided(held, (rows, n), (256, 1))
    g.copy_(torch.randn(rows, n, generator=gen).to(BF16))
    x, w = torch.ones(rows, 16, device=cuda_device, dtype=BF16), torch.ones(n, 16, device=cuda_device, dtype=BF16)
    bias = torch.zeros(n, device=cuda_device, dtype=BF16, requires_grad=True)
    (db,) = torch.autograd.grad(linear_act(x, w, bias), [bias], g)
    near(db, g.double().sum(0), g.double().abs().sum(0), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(4, 16), (1300, 64), (1300, 33)])
def test_gelu_of_large_negative_numbers_in_bfloat16(cuda_device, rows, n):
    """One term to a sum, so that z is exact: y is within half a unit in its last
    place, and 2^-12 of it, of z * Phi(z) down to z = -12.5. The approximation of
    Phi is within 2^-13 of it, its exponential's argument of at most 113 within 2^-17."""
    z = torch.linspace(-12.5, 12.5, rows * n, dtype=torch.float64).view(rows, n).to(BF16)
    x = torch.zeros(rows, 8 * n, dtype=BF16)
    x[:, ::8] = z
    w = torch.zeros(n, 8 * n, dtype=BF16)
    w[torch.arange(n), 8 * torch.arange(n)] = 1
    x, w, z = x.to(cuda_device), w.to(cuda_device), z.to(cuda_device).double()
    exact = z * 0.5 * torch.erfc(-z / math.sqrt(2))
    y = linear_act(x, w, activation="gelu").double()
    bound = torch.exp2(exact.abs().log2().floor().clamp(min=-126) - 8) + 2.0 ** -12 * exact.abs()
    assert bool(((y - exact).abs() <= bound)[z != 0].all()), float(((y - exact).abs() / bound)[z != 0].max())
    assert bool((y[z == 0] == 0).all())


# ---- calls that autograd or a tracer has to see ---------------------------------------------


class FakeModule:
    """A library whose calls write 1 into the outputs' memory, unseen by torch, as kernels do."""

    def plain_call(self, name):
        def call(device, *args):
            if name.startswith("msda_checkpoint"):
                out, count = (args[5], args[2] * args[3]) if name.endswith("_pack") else (args[5], 4 * args[3] * args[4])
            else:
                a = args[0]
                out, count = a.output, 4 * a.rows * (a.out_features if "linear" in name else a.cols)
            ctypes.memset(out, 1, count)
        return call


OPERATORS = {
    "linear_act": lambda x: linear_act(x, torch.ones(8, 8, device=x.device), activation="gelu"),
    "layer_norm": lambda x: layer_norm(x, torch.ones(8, device=x.device)),
    "checkpoint_pack": lambda x: checkpoint_pack(x).codes,
    "checkpoint_unpack": lambda x: checkpoint_unpack(checkpoint_pack(x)),
}


@pytest.fixture
def fake_library(monkeypatch):
    """The operators on CPU tensors, with their kernels replaced."""
    for name in ("linear_act", "layer_norm", "checkpoint8"):
        module = importlib.import_module("muspace_b200.ops." + name)
        monkeypatch.setattr(module, "decide", lambda *args: (FakeModule(), None))
        monkeypatch.setattr(module, "record_dispatch_report", lambda report: report)
        if hasattr(module, "failed"):
            monkeypatch.setattr(module, "failed", lambda report, reason: RuntimeError(reason))
        if hasattr(module, "native_module"):
            monkeypatch.setattr(module, "native_module", lambda: FakeModule())


@pytest.mark.parametrize("name", ["linear_act", "layer_norm"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(fake_library, name, grad):
    """A tangent that the kernels would drop: an error, as from any operator without a forward-mode formula."""
    x = torch.ones(3, 8)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward AD|jvp"):
            OPERATORS[name](forward_ad.make_dual(x, torch.ones(3, 8)))
        assert OPERATORS[name](x).shape == (3, 8)  # no tangent: as outside


def traced(name, x):
    with warnings.catch_warnings(), torch.no_grad():
        warnings.simplefilter("ignore")  # sizes become constants
        return torch.jit.trace(OPERATORS[name], (x,), check_trace=False)


@pytest.mark.parametrize("name", sorted(OPERATORS))
def test_a_trace_has_the_call(fake_library, name):
    kinds = [node.kind() for node in traced(name, torch.ones(3, 8)).graph.nodes()]
    assert "prim::PythonOp" in kinds and not any("empty" in kind for kind in kinds)


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(OPERATORS))
def test_a_trace_computes_again(cuda_device, name):
    x, y = torch.randn(3, 8, device=cuda_device), torch.randn(3, 8, device=cuda_device)
    call = traced(name, x)
    for t in (x, y):
        assert torch.equal(call(t), OPERATORS[name](t))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear_act", "layer_norm"])
def test_forward_mode_is_refused_on_the_gpu(cuda_device, name):
    x = torch.randn(3, 8, device=cuda_device)
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward AD|jvp"):
            OPERATORS[name](forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", ["linear_act", "layer_norm"])
def test_errors_keep_their_type(fake_library, monkeypatch, name):
    """A caller that frees memory and tries again looks for torch's own class."""
    def full(*args):
        raise torch.OutOfMemoryError("no memory left")

    monkeypatch.setattr(importlib.import_module("muspace_b200.ops." + name), "_forward", full)
    with pytest.raises(torch.OutOfMemoryError, match="no memory left"):
        OPERATORS[name](torch.ones(3, 8))


# ---- float16 ------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("rows,k,n", [(3, 72, 40), (1100, 72, 200), (1100, 67, 77)])
def test_linear_in_float16(cuda_device, rows, k, n, activation, checkpoint):
    check_linear(*linear_inputs(rows, k, n, F16, cuda_device, seed=n), activation, checkpoint)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("rows,n", [(1, 4096), (700, 256), (700, 33), (160, 5000)])
def test_layer_norm_in_float16(cuda_device, rows, n, checkpoint):
    x, w, b, g = norm_inputs(rows, n, F16, cuda_device, seed=n)
    check_norm(x, w, b, g, checkpoint)
    check_norm(x, w.float(), b.float(), g, checkpoint)
    check_norm(x, None, None, g, checkpoint)

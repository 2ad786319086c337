"""The encoder layer with dropout, a gated feed-forward and norms of its branches: the
operators between the blocks together, against the same layer in 64-bit torch with the
masks of the generator."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from muspace_b200.encoder import DeformableEncoderLayer, example_inputs
from oracle.msda_torch import msda_grid_sample
from test_residual_ops import factors

SHAPES = ((12, 18), (6, 9), (3, 5), (2, 3))


def _plain(layer, seed, queries, features, reference_points, spatial_shapes, level_start_index):
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}

    def linear(name, x):
        return F.linear(x, p[name + ".weight"], p[name + ".bias"])

    def drop(x, place):
        if not layer.dropout or not layer.training:
            return x
        mask = factors(x.numel() // x.size(-1), x.size(-1), layer.dropout, seed, 3 * layer.index + place)
        return x * mask.to(x.device).view(x.shape)

    def join(name, x, residual, place):
        norm = lambda v: F.layer_norm(v, v.shape[-1:], p[name + ".weight"], p[name + ".bias"])  # noqa: E731
        if layer.branch:
            return residual + p[name + ".gate"] * drop(norm(x), place)
        return norm(residual + drop(x, place))

    b, count, width = queries.shape
    value = linear("value", features).view(b, -1, layer.heads, width // layer.heads)
    shape = (b, count, layer.heads, layer.levels, layer.points)
    offsets = linear("offsets", queries).view(*shape, 2)
    weights = linear("weights", queries).view(*shape[:3], -1).softmax(-1).view(shape)
    locations = reference_points[:, :, None, :, None, :] + offsets / spatial_shapes.flip(-1)[None, None, None, :, None, :]
    x = join("norm1", linear("output", msda_grid_sample(value, spatial_shapes, locations, weights)), queries, 0)
    hidden = linear("up", x)
    if layer.gated:
        gate, up = hidden.chunk(2, -1)
        hidden = F.gelu(gate) * up
    else:
        hidden = F.gelu(hidden)
    return join("norm2", linear("down", drop(hidden, 1)), x, 2), p


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [None, 1, 37])
@pytest.mark.parametrize("norms", ["sum", "branch"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_layer_matches_torch(cuda_device, queries, norms, gated, dropout):
    """float32: the attention's bilinear geometry carries 1e-4 (its own tolerance)."""
    torch.manual_seed(1)
    layer = DeformableEncoderLayer(width=64, hidden=96, heads=4, activation="gelu", device=cuda_device, dropout=dropout,
                                   gated=gated, norms=norms, index=2)
    for parameter in layer.parameters():
        with torch.no_grad():
            parameter.add_(0.05 * torch.randn_like(parameter))
    inputs = example_inputs(layer, 2, SHAPES, queries)
    seed = 1 << 40
    out = layer(**inputs, seed=seed)
    expected, p = _plain(layer, seed, **{k: v.double() if v.is_floating_point() else v for k, v in inputs.items()})
    torch.testing.assert_close(out.double(), expected, rtol=1e-4, atol=1e-4)
    g = torch.randn_like(out)
    out.backward(g)
    expected.backward(g.double())
    for name, parameter in layer.named_parameters():
        got, e = parameter.grad.double(), p[name].grad
        assert float((got - e).norm()) <= 1e-3 * float(e.norm()) + 1e-9, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_draws_another_mask_for_each_seed_and_none_in_evaluation(cuda_device, dtype):
    layer = DeformableEncoderLayer(activation="gelu", device=cuda_device, dtype=dtype, dropout=0.1, gated=True)
    inputs = example_inputs(layer, 1, SHAPES)
    seed = torch.zeros((), dtype=torch.int64, device=cuda_device)
    one, again, two = layer(**inputs, seed=seed), layer(**inputs, seed=0), layer(**inputs, seed=seed + 1)
    assert torch.equal(one, again) and not torch.equal(one, two)
    one.backward(torch.ones_like(one))
    assert all(bool(t.grad.isfinite().all()) for t in layer.parameters())
    layer.eval()
    assert torch.equal(layer(**inputs), layer(**inputs, seed=seed))


def test_layer_refusals():
    for how in (dict(norms="both"), dict(checkpoint="int8", dropout=0.1), dict(checkpoint="int8", gated=True),
                dict(checkpoint="int8", norms="branch")):
        with pytest.raises(ValueError):
            DeformableEncoderLayer(width=32, hidden=48, heads=4, **how)

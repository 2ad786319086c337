"""The encoder layer: its operators together against the same layer in 64-bit torch."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from muspace_b200.encoder import DeformableEncoderLayer, example_inputs
from oracle.msda_torch import msda_grid_sample

SHAPES = ((12, 18), (6, 9), (3, 5), (2, 3))


def _plain(layer, queries, features, reference_points, spatial_shapes, level_start_index):
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}

    def linear(name, x):
        return F.linear(x, p[name + ".weight"], p[name + ".bias"])

    def norm(name, x):
        return F.layer_norm(x, x.shape[-1:], p[name + ".weight"], p[name + ".bias"])

    b, count, width = queries.shape
    value = linear("value", features).view(b, -1, layer.heads, width // layer.heads)
    shape = (b, count, layer.heads, layer.levels, layer.points)
    offsets = linear("offsets", queries).view(*shape, 2)
    weights = linear("weights", queries).view(*shape[:3], -1).softmax(-1).view(shape)
    locations = reference_points[:, :, None, :, None, :] + offsets / spatial_shapes.flip(-1)[None, None, None, :, None, :]
    x = norm("norm1", linear("output", msda_grid_sample(value, spatial_shapes, locations, weights)) + queries)
    return norm("norm2", linear("down", F.gelu(linear("up", x))) + x), p


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [None, 1, 37])
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_layer_matches_torch(cuda_device, queries, checkpoint):
    """float32: the attention's bilinear geometry carries 1e-4 (its own tolerance);
    an 8-bit checkpoint moves an input by at most 1/127 of a block's largest value,
    and the gradients by less than 2% of their norm."""
    torch.manual_seed(1)
    layer = DeformableEncoderLayer(width=64, hidden=96, heads=4, activation="gelu", checkpoint=checkpoint,
                                   device=cuda_device)
    for _, parameter in layer.named_parameters():
        with torch.no_grad():
            parameter.add_(0.05 * torch.randn_like(parameter))
    inputs = example_inputs(layer, 2, SHAPES, queries)
    out = layer(**inputs)
    expected, p = _plain(layer, **{k: v.double() if v.is_floating_point() else v for k, v in inputs.items()})
    torch.testing.assert_close(out.double(), expected, rtol=1e-4, atol=1e-4)
    g = torch.randn_like(out)
    out.backward(g)
    expected.backward(g.double())
    tolerance = 1e-3 if checkpoint is None else 2e-2
    for name, parameter in layer.named_parameters():
        got, e = parameter.grad.double(), p[name].grad
        assert float((got - e).norm()) <= tolerance * float(e.norm()) + 1e-9, name


@pytest.mark.gpu
def test_layer_in_bfloat16_holds_less_with_checkpoints(cuda_device):
    held = {}
    for checkpoint in (None, "int8"):
        layer = DeformableEncoderLayer(activation="gelu", checkpoint=checkpoint, device=cuda_device,
                                       dtype=torch.bfloat16)
        inputs = example_inputs(layer, 1, ((40, 60), (20, 30), (10, 15), (5, 8)))
        before = torch.cuda.memory_allocated()
        out = layer(**inputs)
        held[checkpoint] = torch.cuda.memory_allocated() - before
        out.backward(torch.ones_like(out))
        assert all(bool(t.grad.isfinite().all()) for t in layer.parameters())
    assert held["int8"] < 0.8 * held[None]


def test_layer_checks_its_sizes_and_runs_on_cuda_only():
    with pytest.raises(ValueError, match="divisible"):
        DeformableEncoderLayer(width=30, heads=8)
    layer = DeformableEncoderLayer(width=32, hidden=48, heads=4)
    with pytest.raises(RuntimeError, match="need CUDA tensors"):
        layer(**example_inputs(layer, 1, SHAPES))

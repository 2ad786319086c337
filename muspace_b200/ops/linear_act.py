"""Linear layer with bias, activation and residual in one kernel, forward and backward.

The projections and feed-forward products of the layer around a deformable
attention: ``y = act(x W^T + b) + r``. The product runs on the tensor cores,
bias, activation and residual on its float32 sums before the one rounding.

Backward: ``dz = g * act'(z)``, ``dx = dz W``, ``dW = dz^T x``, ``db`` the sum of
``dz`` over rows, and ``g`` itself for the residual. In bfloat16 ``dz`` is rounded
to bfloat16 before the two products, as a tensor core takes it. ``act'(z)`` comes
from the forward (in float16 beside bfloat16: 11 bits of a number in [-0.2, 1.2],
and 2^-25 where it is below 2^-14), which holds as much between the passes as ``z``
itself would, or, with a checkpoint, from computing ``z`` again in the epilogue
that makes ``dz``. Forward and backward, kept and computed again, on a B200: 40000
x 256 x 512 bfloat16 108 and 125 us, 40000 x 2048 x 512 260 and 321; 22223 x 256 x
1024 float32 359 and 418. Kept was the faster one at every size from 64 input
features on, in both types.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import LinearArgs, NativeModule
from ._layer_common import (
    DTYPE_CODES, autograd_sees, check_checkpoint, check_tensor, decide, failed, native_module, pointer, rows_of)
from .checkpoint8 import pack_rows

OPERATOR_NAME = "linear_act"
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _forward(module: NativeModule, x, weight, bias, residual, activation: str, keep_slope: bool):
    """``(output, slope)``; every tensor float32 or bfloat16."""
    rows, x_stride = rows_of(x)
    weight, w_stride = rows_of(weight)
    out = x.new_empty((*x.shape[:-1], weight.size(0)))
    slope = None
    if keep_slope:
        slope = torch.empty(rows.size(0), weight.size(0), device=x.device,
                            dtype=torch.float16 if x.dtype == torch.bfloat16 else torch.float32)
    r_stride = 0
    if residual is not None:
        residual, r_stride = rows_of(residual)
    if bias is not None:
        bias = bias.contiguous()
    args = LinearArgs(DTYPE_CODES[x.dtype], ACTIVATIONS[activation], rows.size(0), weight.size(1), weight.size(0),
                      x_stride, w_stride, r_stride, weight.size(0), 0, rows.data_ptr(), weight.data_ptr(), pointer(bias),
                      pointer(residual), out.data_ptr(), pointer(slope))
    module.plain_call("msda_linear_act_forward")(x.device, args)
    return out, slope


class _LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint):
        module = native_module()
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dz_needed = need_x or need_w or need_b
        keep_slope = dz_needed and activation != "none" and checkpoint is None
        out, slope = _forward(module, x, weight, bias, residual, activation, keep_slope)
        recompute = dz_needed and activation != "none" and not keep_slope
        keep_x = need_w or recompute
        codes = exponents = None
        if keep_x and checkpoint == "int8":
            codes, exponents = pack_rows(module, *rows_of(x))
        ctx.save_for_backward(x if keep_x and checkpoint is None else None,
                              weight if need_x or recompute else None, bias if recompute else None, slope, codes,
                              exponents)
        ctx.activation = activation
        ctx.sizes = (x.shape, weight.shape)
        return out

    @staticmethod
    def backward(ctx, grad):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, grad) if torch.is_grad_enabled() else _backward(ctx, grad)


def _backward(ctx, grad):
    x, weight, bias, slope, codes, exponents = ctx.saved_tensors
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    x_shape, w_shape = ctx.sizes
    dx = dw = db = None
    if need_x or need_w or need_b:
        g, g_stride = rows_of(grad)
        if need_x:
            dx = grad.new_empty(x_shape)
        if need_w:
            dw = grad.new_empty(w_shape)
        if need_b:
            db = grad.new_empty(w_shape[:1])
        x_stride = w_stride = 0
        if x is not None:
            x, x_stride = rows_of(x)
        if weight is not None:
            weight, w_stride = rows_of(weight)
        if bias is not None:
            bias = bias.contiguous()
        args = LinearArgs(DTYPE_CODES[grad.dtype], ACTIVATIONS[ctx.activation], g.size(0), w_shape[1], w_shape[0],
                          x_stride, w_stride, 0, 0, g_stride, pointer(x), pointer(weight), pointer(bias), None,
                          None, pointer(slope), g.data_ptr(), pointer(codes), pointer(exponents), pointer(dx),
                          pointer(dw), pointer(db))
        native_module().plain_call("msda_linear_act_backward")(grad.device, args)
    return dx, dw, db, grad if need_r else None, None, None


_backward_once = once_differentiable(_backward)


def linear_act(input: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, *, activation: str = "none", checkpoint: str | None = None,
               backend: str = "auto") -> torch.Tensor:
    """``act(input @ weight.T + bias) + residual`` (differentiable).

    input ``(..., in)``; weight ``(out, in)``; bias ``(out,)`` or None; residual
    broadcastable to the output ``(..., out)``, or None; activation ``"none"``,
    ``"relu"``, ``"gelu"`` (by the normal distribution function) or ``"silu"``. All
    of one dtype: bfloat16, float32 (24-bit products), or float16, which runs as
    float32.

    ``checkpoint="int8"`` keeps ``input`` for the backward pass in 8 bits (see
    ``checkpoint_pack``) and nothing of the output's size: the gradients are those
    at the input that the checkpoint holds.
    """
    check_tensor(input, "input")
    check_tensor(weight, "weight", input)
    for name, tensor in (("bias", bias), ("residual", residual)):
        if tensor is not None:
            check_tensor(tensor, name, input)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    check_checkpoint(checkpoint)
    if input.dim() == 0 or weight.dim() != 2:
        raise ValueError("input must have at least one dimension and weight two")
    out_features, in_features = weight.shape
    if input.size(-1) != in_features:
        raise ValueError(f"input has {input.size(-1)} features, weight takes {in_features}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must have shape ({out_features},), got {tuple(bias.shape)}")
    if residual is not None:
        shape = (*input.shape[:-1], out_features)
        if residual.shape != shape:
            try:
                residual = residual.expand(shape)
            except RuntimeError as exc:
                raise ValueError(f"residual {tuple(residual.shape)} cannot be broadcast to {tuple(shape)}") from exc
    module, report = decide(OPERATOR_NAME, backend, input, weight, bias, residual)
    dtype = input.dtype
    if dtype == torch.float16:
        input, weight, bias, residual = (t if t is None else t.float() for t in (input, weight, bias, residual))
    tensors = (input, weight, bias, residual)
    try:
        if autograd_sees(*tensors):
            output = _LinearActFunction.apply(*tensors, activation, checkpoint)
        else:
            output, _ = _forward(module, *tensors, activation, False)
    except RuntimeError as exc:
        failed(report, str(exc))
        raise
    record_dispatch_report(report)
    return output if dtype != torch.float16 else output.to(dtype)


__all__ = ["linear_act"]

"""Layer norm over the last dimension, forward and backward.

``y = (x - mean) / sqrt(var + eps) * weight + bias``. The forward reads a row
once, the backward reads row and gradient once and sums the weight's and the
bias' gradients on the way, in an order that does not depend on scheduling.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import LayerNormArgs, NativeModule
from ._layer_common import (
    DTYPE_CODES, autograd_sees, check_checkpoint, check_tensor, decide, failed, native_module, pointer, rows_of)
from .checkpoint8 import BLOCK

OPERATOR_NAME = "layer_norm"


def _forward(module: NativeModule, x, weight, bias, eps: float, keep: str | None):
    """``(output, statistics, codes, exponents)``; ``keep``: "statistics", "int8" or None."""
    rows, stride = rows_of(x)
    count, width = map(int, rows.shape)  # tensors while tracing
    out = x.new_empty(x.shape)
    statistics = codes = exponents = None
    mean = rstd = None
    if keep == "statistics":
        statistics = torch.empty((2, count), dtype=torch.float32, device=x.device)
        mean = statistics.data_ptr()
        rstd = mean + 4 * count
    elif keep == "int8":
        codes = torch.empty((count, width), dtype=torch.int8, device=x.device)
        exponents = torch.empty((count, -(-width // BLOCK)), dtype=torch.uint8, device=x.device)
    kind = weight if weight is not None else bias
    args = LayerNormArgs(DTYPE_CODES[x.dtype], DTYPE_CODES[x.dtype if kind is None else kind.dtype], count, width,
                         stride, 0, eps, rows.data_ptr(), pointer(weight), pointer(bias), out.data_ptr(), mean, rstd,
                         pointer(codes), pointer(exponents))
    module.plain_call("msda_layer_norm_forward")(x.device, args)
    return out, statistics, codes, exponents


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        module = native_module()
        out, statistics, codes, exponents = _forward(module, x, weight, bias, eps, checkpoint or "statistics")
        ctx.save_for_backward(x if checkpoint is None else None, weight, statistics, codes, exponents)
        ctx.eps = eps
        ctx.kind = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
        return out

    @staticmethod
    def backward(ctx, grad):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, grad) if torch.is_grad_enabled() else _backward(ctx, grad)


def _backward(ctx, grad):
    x, weight, statistics, codes, exponents = ctx.saved_tensors
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    g, g_stride = rows_of(grad)
    count, width = g.shape
    dx = grad.new_empty(grad.shape) if need_x else None
    dw, db = (torch.empty(width, dtype=ctx.kind, device=grad.device) if need else None for need in (need_w, need_b))
    stride, mean, rstd = 0, None, None
    if x is not None:
        x, stride = rows_of(x)
        mean = statistics.data_ptr()
        rstd = mean + 4 * count
    args = LayerNormArgs(DTYPE_CODES[grad.dtype], DTYPE_CODES[ctx.kind], count, width, stride, g_stride, ctx.eps,
                         pointer(x), pointer(weight), None, None, mean, rstd, pointer(codes), pointer(exponents),
                         g.data_ptr(), pointer(dx), pointer(dw), pointer(db))
    native_module().plain_call("msda_layer_norm_backward")(grad.device, args)
    return dx, dw, db, None, None


_backward_once = once_differentiable(_backward)


def layer_norm(input: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, *, checkpoint: str | None = None, backend: str = "auto") -> torch.Tensor:
    """``(input - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (differentiable).

    input ``(..., n)`` in bfloat16, float32, or float16, which runs as float32;
    weight and bias ``(n,)`` or None, both of input's dtype or both float32.
    ``checkpoint="int8"`` keeps ``input`` for the backward pass in 8 bits (see
    ``checkpoint_pack``) and no statistics: the gradients are those at the input
    that the checkpoint holds.
    """
    check_tensor(input, "input")
    check_checkpoint(checkpoint)
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor is None:
            continue
        if not isinstance(tensor, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if tensor.dtype not in (input.dtype, torch.float32):
            raise TypeError(f"{name} must have the dtype of input ({input.dtype}) or float32")
        if tensor.shape != input.shape[-1:]:
            raise ValueError(f"{name} must have shape ({input.size(-1)},), got {tuple(tensor.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one dtype")
    module, report = decide(OPERATOR_NAME, backend, input, weight, bias)
    dtype = input.dtype
    if dtype == torch.float16:
        input, weight, bias = (t if t is None else t.float() for t in (input, weight, bias))
    weight, bias = (t if t is None else t.contiguous() for t in (weight, bias))
    tensors = (input, weight, bias)
    try:
        if autograd_sees(*tensors):
            output = _LayerNormFunction.apply(*tensors, float(eps), checkpoint)
        else:
            output = _forward(module, *tensors, float(eps), None)[0]
    except RuntimeError as exc:
        failed(report, str(exc))
        raise
    record_dispatch_report(report)
    return output if dtype != torch.float16 else output.to(dtype)


__all__ = ["layer_norm"]

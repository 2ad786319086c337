"""Dropout from a counter-based generator, whose mask is never stored.

An element's random number follows from the seed, the sequence and the element's
row and column (Philox-4x32, ten rounds; 16 bits an element), so the backward pass
makes the mask again, and so do the operators that have dropout inside them
(``add_norm``, ``norm_add``, ``gated_linear``): with the same seed, sequence, rows
and columns they drop the same elements.
"""

from __future__ import annotations

from numbers import Integral, Real

import torch
from torch.autograd.function import once_differentiable

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import NativeModule
from ._layer_common import WIDE_DTYPE_CODES, autograd_sees, check_tensor, decide, failed, native_module, pointer, rows_of

OPERATOR_NAME = "dropout"


def check_rule(p, seed, sequence, needed: bool = False) -> tuple[int, int, int, torch.Tensor | None]:
    """``(threshold, seed, sequence, seed tensor)`` of a dropout; the seed is needed
    where something is dropped, or always."""
    if p.__class__ is not float and (isinstance(p, bool) or not isinstance(p, Real)):
        raise TypeError("the dropout probability must be a number")
    if not 0.0 <= p <= 1.0:  # NaN is outside too
        raise ValueError(f"the dropout probability must be between 0 and 1, got {p}")
    threshold = round(65536 * float(p))
    if seed is None:
        if threshold or needed:
            raise ValueError("dropout needs a seed")
        return 0, 0, 0, None
    if sequence.__class__ is not int and (isinstance(sequence, bool) or not isinstance(sequence, Integral)):
        raise TypeError("sequence must be an integer")
    if not 0 <= sequence < 2 ** 63:
        raise ValueError(f"sequence must be between 0 and 2^63 - 1, got {sequence}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64:
            raise TypeError("a seed tensor must be int64")
        if seed.numel() != 1:
            raise ValueError(f"a seed tensor must have one element, got shape {tuple(seed.shape)}")
        return threshold, 0, int(sequence), seed
    if seed.__class__ is not int and (isinstance(seed, bool) or not isinstance(seed, Integral)):
        raise TypeError("seed must be an integer or an int64 tensor")
    if not 0 <= seed < 2 ** 63:
        raise ValueError(f"seed must be between 0 and 2^63 - 1, got {seed}")
    return threshold, int(seed), int(sequence), None


def _apply(module: NativeModule, x, threshold, seed, sequence, seed_tensor):
    rows, stride = rows_of(x)
    count, width = map(int, rows.shape)  # tensors while tracing
    out = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    module.plain_call("msda_dropout")(x.device, WIDE_DTYPE_CODES[x.dtype], rows.data_ptr(), count, width, stride,
                                      threshold, seed, sequence, pointer(seed_tensor), out.data_ptr())
    return out


class _DropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, seed_tensor, threshold, seed, sequence):
        ctx.save_for_backward(seed_tensor)
        ctx.rule = (threshold, seed, sequence)
        return _apply(native_module(), x, threshold, seed, sequence, seed_tensor)

    @staticmethod
    def backward(ctx, grad):
        # the wrapper costs 3 us; it is needed where a graph of this pass is asked for
        return _backward_once(ctx, grad) if torch.is_grad_enabled() else _backward(ctx, grad)


def _backward(ctx, grad):
    (seed_tensor,) = ctx.saved_tensors
    return _apply(native_module(), grad, *ctx.rule, seed_tensor), None, None, None, None


_backward_once = once_differentiable(_backward)


def dropout(input: torch.Tensor, p: float = 0.5, *, seed, sequence: int = 0, backend: str = "auto") -> torch.Tensor:
    """``input`` with each element set to 0 with probability ``p``, the others
    multiplied by ``1 / (1 - p)`` (differentiable).

    input ``(..., n)`` in bfloat16, float16 or float32. ``p`` is taken to the nearest
    multiple of 2^-16. ``seed``: an integer, or an int64 tensor of one element on
    input's device, which the kernel reads: a captured graph drops other elements
    whenever the tensor has changed between two replays (it must not change between a
    forward pass and its backward pass). ``sequence``: an integer that tells a
    program's dropouts apart. What is dropped is 0 also where it was not finite.
    """
    check_tensor(input, "input")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    threshold, number, sequence, seed_tensor = check_rule(p, seed, sequence, needed=True)
    module, report = decide(OPERATOR_NAME, backend, input, seed_tensor)
    try:
        if autograd_sees(input):
            output = _DropoutFunction.apply(input, seed_tensor, threshold, number, sequence)
        else:
            output = _apply(module, input, threshold, number, sequence, seed_tensor)
    except RuntimeError as exc:
        failed(report, str(exc))
        raise
    record_dispatch_report(report)
    return output


__all__ = ["dropout"]

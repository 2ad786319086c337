"""Activations kept in 8 bits for the backward pass.

A tensor is cut into blocks of 32 elements along its last dimension (the last
block may be short). A block is held as integers ``q = rint(x / 2^e)``, ties to
even, and one byte ``e + 127``, with ``e`` the smallest integer >= -126 that
gives ``max|x| <= 127 * 2^e``: 8.25 bits per element. The scale is a power of
two, so ``q`` is the only rounding (at most 1/127 of the block's largest value,
half of that where it is rounded to nearest), and what comes back is exact in
float32 and bfloat16. A block with an infinity or a NaN comes back as NaNs.

``linear_act`` and ``layer_norm`` keep their input this way with
``checkpoint="int8"``; their backward passes compute at the values that the
checkpoint holds.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ..runtime.kernel_dispatch import record_dispatch_report
from ..runtime.native import NativeModule
from ._layer_common import DTYPE_CODES, STORAGE, check_tensor, decide, native_module, rows_of

BLOCK = 32


class Checkpoint8(NamedTuple):
    """A tensor in 8 bits: ``codes`` int8 of its shape, ``exponents`` uint8 of its
    leading shape and ``ceil(last / 32)``, and its dtype."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


def pack_rows(module: NativeModule, rows: torch.Tensor, stride: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and exponents of a float32 / bfloat16 matrix."""
    count, width = rows.shape
    codes = torch.empty((count, width), dtype=torch.int8, device=rows.device)
    exponents = torch.empty((count, -(-width // BLOCK)), dtype=torch.uint8, device=rows.device)
    module.plain_call("msda_checkpoint_pack")(rows.device, DTYPE_CODES[rows.dtype], rows.data_ptr(), count, width,
                                              stride, codes.data_ptr(), exponents.data_ptr())
    return codes, exponents


def _unpack(module: NativeModule, codes: torch.Tensor, exponents: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What contiguous codes and exponents hold, in float32 or bfloat16."""
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    width = codes.size(-1)
    module.plain_call("msda_checkpoint_unpack")(codes.device, DTYPE_CODES[dtype], codes.data_ptr(),
                                                exponents.data_ptr(), codes.numel() // max(width, 1), width,
                                                out.data_ptr())
    return out


# Only for tracing, which records a function's call and nothing of what a kernel does.


class _PackFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows):
        outputs = pack_rows(native_module(), *rows_of(rows))
        ctx.mark_non_differentiable(*outputs)
        return outputs

    @staticmethod
    def backward(ctx, *grads):
        return None


class _UnpackFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, codes, exponents, dtype):
        output = _unpack(native_module(), codes, exponents, dtype)
        ctx.mark_non_differentiable(output)
        return output

    @staticmethod
    def backward(ctx, grad):
        return None, None, None


def checkpoint_pack(input: torch.Tensor, *, backend: str = "auto") -> Checkpoint8:
    """The 8-bit checkpoint of a float16, bfloat16 or float32 CUDA tensor."""
    check_tensor(input, "input")
    if input.dim() == 0:
        raise ValueError("input must have at least one dimension")
    module, report = decide("checkpoint_pack", backend, input)
    source = input.detach()
    rows, stride = rows_of(source.float() if source.dtype == torch.float16 else source)
    if torch.jit.is_tracing():
        codes, exponents = _PackFunction.apply(rows)
    else:
        codes, exponents = pack_rows(module, rows, stride)
    record_dispatch_report(report)
    return Checkpoint8(codes.view(input.shape), exponents.view(*input.shape[:-1], exponents.size(1)), input.dtype)


def checkpoint_unpack(checkpoint: Checkpoint8, dtype: torch.dtype | None = None, *,
                      backend: str = "auto") -> torch.Tensor:
    """The tensor that a checkpoint holds, in its own dtype or in ``dtype``."""
    codes, exponents, kept = checkpoint
    dtype = kept if dtype is None else dtype
    if not isinstance(codes, torch.Tensor) or not isinstance(exponents, torch.Tensor):
        raise TypeError("codes and exponents must be tensors")
    if codes.dtype != torch.int8 or exponents.dtype != torch.uint8:
        raise TypeError("codes must be int8 and exponents uint8")
    if dtype not in STORAGE:
        raise TypeError("dtype must be float16, bfloat16 or float32")
    if codes.dim() == 0 or tuple(exponents.shape) != (*codes.shape[:-1], -(-codes.size(-1) // BLOCK)):
        raise ValueError("exponents must have the leading shape of codes and one byte for each block of 32")
    module, report = decide("checkpoint_unpack", backend, codes, exponents)
    codes, exponents = codes.contiguous(), exponents.contiguous()
    stored = torch.float32 if dtype == torch.float16 else dtype
    if torch.jit.is_tracing():
        out = _UnpackFunction.apply(codes, exponents, stored)
    else:
        out = _unpack(module, codes, exponents, stored)
    record_dispatch_report(report)
    return out.to(dtype)


__all__ = ["Checkpoint8", "checkpoint_pack", "checkpoint_unpack"]

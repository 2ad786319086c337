"""What the layer operators (``linear_act``, ``layer_norm``, 8-bit checkpoints)
share: storage types, rows of a tensor, dispatch reports."""

from __future__ import annotations

from functools import lru_cache

import torch

from ..runtime.kernel_dispatch import (
    DispatchDecision,
    DispatchReport,
    explain_dispatch as _explain_dispatch,
    record_dispatch_report,
)
from ..runtime.native import NativeModule, NativeModuleUnavailable, load_native_module

DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1}  # msda_dtype_t
STORAGE = (torch.float16, torch.bfloat16, torch.float32)
CHECKPOINTS = (None, "int8")


def native_module() -> NativeModule | None:
    try:
        return load_native_module()
    except NativeModuleUnavailable:
        return None


def check_tensor(tensor, name: str, like: torch.Tensor | None = None) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if like is None:
        if tensor.dtype not in STORAGE:
            raise TypeError(f"{name} must be float16, bfloat16 or float32")
    elif tensor.dtype != like.dtype:
        raise TypeError(f"{name} must have the dtype of input ({like.dtype})")


def check_checkpoint(checkpoint) -> None:
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be None or 'int8', got {checkpoint!r}")


@lru_cache(maxsize=256)
def _report_of(operator: str, requested: str, selected: str, device: str, reason: str,
               native_available: bool) -> DispatchReport:
    return DispatchReport(operator=operator, requested_backend=requested, selected_backend=selected, device=device,
                          reason=reason, native_available=native_available)


def report(operator: str, backend: str, decision: DispatchDecision, selected: str, reason: str,
           native_available: bool) -> None:
    record_dispatch_report(_report_of(operator, backend, selected, decision.device, reason, native_available))


# the decisions for CUDA tensors with the native library at hand, which depend on nothing else
_CUDA_DECISIONS: dict[tuple[str, str], DispatchDecision] = {}


def decide(operator: str, backend: str, tensor: torch.Tensor, *others: torch.Tensor | None):
    """``(native module, decision)`` of a call whose tensors share a device, or RuntimeError with its report."""
    module = native_module()
    usual = module is not None and tensor.is_cuda
    decision = _CUDA_DECISIONS.get((operator, backend)) if usual else None
    if decision is None:
        decision = _explain_dispatch(tensor, backend=backend, native_available=module is not None, operator=operator)
        if usual:
            _CUDA_DECISIONS[operator, backend] = decision
    reason = decision.reason if decision.backend == "error" else None
    if reason is None:
        device = tensor.device
        for other in others:
            if other is not None and other.device != device:
                reason = f"a tensor is on {other.device}, input is on {device}"
                break
    if reason is not None:
        report(operator, backend, decision, "error", reason, module is not None)
        raise RuntimeError(reason)
    return module, decision


def rows_of(tensor: torch.Tensor) -> tuple[torch.Tensor, int]:
    """The tensor as rows of its last dimension, whose elements are adjacent, and
    the rows' distance: a view where the strides allow it, else a copy."""
    if tensor.dim() != 2:
        tensor = tensor.reshape(-1, tensor.size(-1)) if tensor.numel() else tensor.new_empty(
            (tensor.shape[:-1].numel(), tensor.size(-1)))
    stride, inner = tensor.stride()
    if inner != 1 and tensor.size(1) > 1:
        tensor = tensor.contiguous()
        stride = tensor.stride(0)
    return tensor, stride


def pointer(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()

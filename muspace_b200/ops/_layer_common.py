"""What the layer operators (``linear_act``, ``layer_norm``, 8-bit checkpoints)
share: storage types, rows of a tensor, dispatch reports."""

from __future__ import annotations

from dataclasses import replace

import torch
from torch.autograd import forward_ad

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


# What a call with CUDA tensors and the native library at hand is decided and
# reported as depends on the operator and the requested backend alone.
_USUAL: dict[tuple[str, str], DispatchReport] = {}


def _report_of(operator: str, backend: str, decision: DispatchDecision, selected: str, reason: str,
               native_available: bool) -> DispatchReport:
    return DispatchReport(operator=operator, requested_backend=backend, selected_backend=selected,
                          device=decision.device, reason=reason, native_available=native_available)


def decide(operator: str, backend: str, tensor: torch.Tensor, *others: torch.Tensor | None):
    """``(native module, report of success)`` of a call whose tensors share a
    device. Otherwise RuntimeError, and the report that says so."""
    module = native_module()
    report = _USUAL.get((operator, backend)) if module is not None and tensor.is_cuda else None
    decision = None
    if report is None:
        decision = _explain_dispatch(tensor, backend=backend, native_available=module is not None, operator=operator)
        if decision.backend == "error":
            record_dispatch_report(_report_of(operator, backend, decision, "error", decision.reason,
                                              module is not None))
            raise RuntimeError(decision.reason)
        report = _report_of(operator, backend, decision, "cuda", decision.reason, True)
        _USUAL[operator, backend] = report
    device = tensor.device
    for other in others:
        if other is not None and other.device != device:
            raise failed(report, f"a tensor is on {other.device}, input is on {device}")
    return module, report


def failed(report: DispatchReport, reason: str) -> RuntimeError:
    """The error of a call that would have been reported as ``report``, after reporting it."""
    record_dispatch_report(replace(report, selected_backend="error", reason=reason))
    return RuntimeError(reason)


_is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)  # without the Python around it


def autograd_sees(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these tensors has to go through its autograd function: for
    gradients, within forward mode (where the function refuses a tangent, which the
    kernels would drop), and while tracing (where it is what the trace records).
    Elsewhere a call spares itself the function's 10 us."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0 or _is_tracing())


def rows_of(tensor: torch.Tensor) -> tuple[torch.Tensor, int]:
    """The tensor as rows of its last dimension, whose elements are adjacent, and
    the rows' distance: a view where the strides allow it, else a copy."""
    strides = tensor.stride()
    if len(strides) != 2:
        tensor = tensor.reshape(-1, tensor.size(-1)) if tensor.numel() else tensor.new_empty(
            (tensor.shape[:-1].numel(), tensor.size(-1)))
        strides = tensor.stride()
    if strides[1] != 1 and tensor.size(1) > 1:
        tensor = tensor.contiguous()
        strides = tensor.stride()
    return tensor, strides[0]


def pointer(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()

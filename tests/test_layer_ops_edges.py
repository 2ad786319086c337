"""Edges of linear_act, layer_norm and 8-bit checkpoints: the ends of the
workspace, what is not finite, forward mode and tracing, waits.

Tolerances as in test_layer_ops.py, from which the formulas come, unless a test
says otherwise.
"""

from __future__ import annotations

import ctypes

import pytest

from muspace_b200.runtime import native


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

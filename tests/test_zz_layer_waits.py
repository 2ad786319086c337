"""The bounded waits of the linear and layer-norm kernels: none ran out in the
tests before these, and one that does is counted and ends."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

from muspace_b200.runtime import native

ONE_WAIT = """
import ctypes, torch
from muspace_b200.ops import linear_act
from muspace_b200.runtime import native
x, w = torch.randn(200, 64, device="cuda"), torch.randn(40, 64, device="cuda")
before, counts = linear_act(x, w), [native.layer_wait_timeouts()]
probe = native.load_native_module().lib.msda_layer_wait_probe
probe.argtypes = [ctypes.c_int64, ctypes.c_void_p]
assert probe(1000000, torch.cuda.current_stream().cuda_stream) == 0
counts.append(native.layer_wait_timeouts())
assert torch.equal(linear_act(x, w), before)
print(counts, native.layer_wait_timeouts(0))
"""


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_counted_and_ends(cuda_device):
    """In a process of its own, whose count it raises."""
    run = subprocess.run([sys.executable, "-c", ONE_WAIT], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert run.stdout.split("\n")[0] == "[0, 1] 1"


@pytest.mark.gpu
def test_no_wait_of_the_layer_kernels_ran_out(cuda_device):
    assert native.layer_wait_timeouts() == 0


def test_wait_probe_refuses_what_would_not_end_soon():
    module = native.load_native_module()
    probe = module.lib.msda_layer_wait_probe
    probe.argtypes = [ctypes.c_int64, ctypes.c_void_p]
    for clocks in (-1, 2 ** 31):
        assert probe(clocks, None) == 1 and "clocks must be" in module.last_error()

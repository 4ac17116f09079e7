"""Two decode stacks on one device share its scratch."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# a process of its own: the scratch has not grown before
SCRIPT = r"""
import numpy as np
from peregrine_b200 import cuda
from peregrine_b200.stack import DeviceStack, synth_stack

assert cuda.init([0]) == 1
L = cuda.lib()
sizes = dict(inter=96, n_experts=8, k=2, n_layers=2, first_dense=1, vocab=512)
narrow = DeviceStack(0, synth_stack(seed=3, hidden=256, dense_inter=384, **sizes), 1, 12)
ids0 = np.array([5], np.int32)
want = narrow.decode(ids0, 12)
assert len(narrow.graphs) == 2
recorded = L.coli_cuda_scratch_generation(0)
assert np.array_equal(narrow.decode(ids0, 12), want) and L.coli_cuda_scratch_generation(0) == recorded
wide = DeviceStack(0, synth_stack(seed=4, hidden=512, dense_inter=8192, attention_heads=(4, 2, 64), **sizes), 1, 12, prefix_cap=64)
wide.prefill(np.arange(64))
assert L.coli_cuda_scratch_generation(0) > recorded
other = wide.decode(ids0, 12)
for _ in range(2):
    assert np.array_equal(narrow.decode(ids0, 12), want)
    assert np.array_equal(wide.decode(ids0, 12), other)
assert len(narrow.graphs) == 2 and cuda.last_device_error(0) == 0
narrow.free()
wide.free()
cuda.shutdown()
print("the same")
"""


def test_recorded_steps_follow_scratch_that_a_wider_stack_has_moved():
    done = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and "the same" in done.stdout, done.stdout + done.stderr

"""Two decode stacks on one device share its scratch."""
import numpy as np
import pytest

from peregrine_b200 import cuda
from peregrine_b200.stack import DeviceStack, synth_stack

pytestmark = pytest.mark.gpu


def test_recorded_steps_follow_scratch_that_a_wider_stack_has_moved(dev):
    L = cuda.lib()
    sizes = dict(inter=96, n_experts=8, k=2, n_layers=2, first_dense=1, vocab=512)
    narrow = DeviceStack(dev, synth_stack(seed=3, hidden=256, dense_inter=384, **sizes), 1, 12)
    ids0 = np.array([5], np.int32)
    want = narrow.decode(ids0, 12)
    assert len(narrow.graphs) == 2
    recorded = L.coli_cuda_scratch_generation(dev)
    assert np.array_equal(narrow.decode(ids0, 12), want) and L.coli_cuda_scratch_generation(dev) == recorded
    # wider in every way than what this device has done before in this process
    wide = DeviceStack(dev, synth_stack(seed=4, hidden=512, dense_inter=1 << 16, attention_heads=(4, 2, 64), **sizes), 1, 12,
                       prefix_cap=64)
    wide.prefill(np.arange(64))
    assert L.coli_cuda_scratch_generation(dev) > recorded
    other = wide.decode(ids0, 12)
    for _ in range(2):
        assert np.array_equal(narrow.decode(ids0, 12), want)
        assert np.array_equal(wide.decode(ids0, 12), other)
    assert len(narrow.graphs) == 2 and cuda.last_device_error(dev) == 0
    narrow.free()
    wide.free()

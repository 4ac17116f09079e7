"""A decode stack with attention and a budget whose experts go through the expert-parallel exchange (one rank)."""
import numpy as np
import pytest

from peregrine_b200 import cuda
from peregrine_b200.ep import EpWorkspace
from peregrine_b200.stack import DeviceStack, synth_stack

pytestmark = pytest.mark.gpu


def test_expert_parallel_steps_with_a_budget_are_the_plain_stack_s(dev):
    st = synth_stack(seed=3, hidden=256, inter=96, dense_inter=384, n_experts=8, k=2, n_layers=3, first_dense=1, vocab=512,
                     attention_heads=(4, 2, 64))
    ids0, steps, kw = np.array([5, 9, 300, 411], np.int32), 24, dict(budget=10, slack=4, recent=5)
    plain = DeviceStack(dev, st, 4, steps, **kw)
    want, slots = plain.decode(ids0, steps), [l.pos.download((4, 2, 14), np.int32) for l in plain.attn]
    plain.free()
    ws = EpWorkspace(dev, 0, 1, 4, 256, 2)
    ds = DeviceStack(dev, st, 4, steps, ep=ws, **kw)
    for _ in range(2):
        assert np.array_equal(ds.decode(ids0, steps), want)
        for l, pos in zip(ds.attn, slots):
            assert np.array_equal(l.pos.download((4, 2, 14), np.int32), pos)
    assert cuda.last_device_error(dev) == 0
    with pytest.raises(ValueError):
        ds.prefill(np.zeros(1, np.int32))
    ds.free()
    ws.free()

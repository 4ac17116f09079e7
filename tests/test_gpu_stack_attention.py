"""The decode stack with attention: norms, projections, caches, the shared prefix and the budget together, against the
oracle's integer matrix products around an attention in 64 bits."""
import numpy as np
import pytest
import torch

from peregrine_b200 import cuda
from peregrine_b200.speculative import stack_forward_rows
from peregrine_b200.stack import DeviceStack, synth_stack
from peregrine_b200.synth import SynthLayer
from tests.refmodel import o_expert, o_weight, oracle_layer_forward

pytestmark = pytest.mark.gpu


def small_stack(seed=3, heads=(4, 2, 64)):
    return synth_stack(seed=seed, hidden=256, inter=96, dense_inter=384, n_experts=8, k=2, n_layers=3, first_dense=1,
                       vocab=512, attention_heads=heads)


class Reference:
    """Token by token with the oracle's functions; q, k, v rounded to the cache's type like the stack's."""

    def __init__(self, st, dtype, prompt):
        self.st, self.dtype = st, dtype
        self.prefix = [([], []) for _ in st.layers]
        for i, t in enumerate(prompt):
            self.rows(np.array([t]), i, [self.prefix])
        self.own = None

    def r16(self, x):
        return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(self.dtype).double().numpy()

    def attend(self, li, x, pos, caches):
        import oracle as po

        st, a = self.st, self.st.attn[li]
        H, Kv, D = a.heads, a.kv_heads, a.head_dim
        b = x.shape[0]
        nrm = np.stack([po.rmsnorm(x[s], a.norm, st.eps) for s in range(b)])
        qkv = o_weight(a.wqkv).apply(nrm, b).reshape(b, H + 2 * Kv, D).astype(np.float64)
        ang = pos * np.float64(st.theta) ** (-2.0 * np.arange(D // 2) / D)

        def turn(t, w):
            t = t / np.sqrt((t * t).mean(-1, keepdims=True) + st.eps) * w
            return np.concatenate([t[..., ::2] * np.cos(ang) - t[..., 1::2] * np.sin(ang),
                                   t[..., 1::2] * np.cos(ang) + t[..., ::2] * np.sin(ang)], -1)

        q, k = self.r16(turn(qkv[:, :H], a.q_norm)), self.r16(turn(qkv[:, H:H + Kv], a.k_norm))
        v = self.r16(qkv[:, H + Kv:])
        ctx = np.zeros((b, H, D), np.float32)
        for s in range(b):
            ks, vs = caches[s][li]
            ks.append(k[s])
            vs.append(v[s])
            pk, pv = self.prefix[li] if caches[s] is not self.prefix else ([], [])
            kk, vv = np.stack(pk + ks), np.stack(pv + vs)
            for h in range(H):
                e = kk[:, h // (H // Kv)] @ q[s, h] / np.sqrt(D)
                w = np.exp(e - e.max())
                ctx[s, h] = (w / w.sum()) @ vv[:, h // (H // Kv)]
        return (x + o_weight(a.wo).apply(ctx.reshape(b, H * D), b)).astype(np.float32)

    def rows(self, ids, pos, caches):
        import oracle as po

        st, x, b = self.st, self.st.embed[ids].astype(np.float32).copy(), len(ids)
        for li, layer in enumerate(st.layers):
            x = self.attend(li, x, pos, caches)
            nrm = np.stack([po.rmsnorm(x[s], st.norms[li], st.eps) for s in range(b)])
            if isinstance(layer, SynthLayer):
                ffn = oracle_layer_forward(layer, nrm)
            else:
                ffn = po.swiglu(*o_expert(layer), nrm, b)
            x = (x + ffn).astype(np.float32)
        nrm = np.stack([po.rmsnorm(x[s], st.final_norm, st.eps) for s in range(b)])
        return o_weight(st.lm_head).apply(nrm, b)


@pytest.mark.parametrize("heads, dtype, prompt", [((4, 2, 64), "bf16", 0), ((6, 2, 64), "f16", 70), ((2, 1, 128), "bf16", 130)])
def test_greedy_steps_follow_the_reference(dev, heads, dtype, prompt):
    """Fed with the stack's own tokens, the reference's logits put every pick at (or within rounding of) the top: a last-bit
    difference before a projection moves an element of its int8 row by one step, 1/127 of the row's largest, so logits
    agree to some percent of their spread."""
    st = small_stack(heads=heads)
    steps, batch = 10, 3
    tokens = np.random.default_rng(1).integers(0, 512, prompt).astype(np.int32)
    ds = DeviceStack(dev, st, batch, steps, prefix_cap=prompt + 5 if prompt else 0, dtype=dtype)
    if prompt:
        ds.prefill(tokens[:33])
        ds.prefill(tokens[33:])
    ids0 = np.array([1, 77, 500], np.int32)
    got = ds.decode(ids0, steps)
    assert np.array_equal(ds.decode(ids0, steps), got)  # recorded and replayed
    ref = Reference(st, torch.bfloat16 if dtype == "bf16" else torch.float16, tokens)
    caches = [[([], []) for _ in st.layers] for _ in range(batch)]
    ids = ids0
    for t in range(steps):
        logits = ref.rows(ids, prompt + t, caches).astype(np.float64)
        top, spread = logits.max(1), logits.std(1)
        picked = logits[np.arange(batch), got[t]]
        assert np.all(top - picked <= 0.1 * spread), (t, (top - picked) / spread)
        ids = got[t]
    assert len(np.unique(got)) > 3
    assert cuda.last_device_error(dev) == 0
    ds.free()


def test_steps_call_by_call_and_as_a_graph_are_the_same(dev, monkeypatch):
    st = small_stack()
    ids0 = np.array([5, 9], np.int32)
    prompt = np.arange(40, dtype=np.int32)
    out = []
    for graph in ("1", "0"):
        monkeypatch.setenv("PEREGRINE_B200_STACK_GRAPH", graph)
        ds = DeviceStack(dev, st, 2, 30, prefix_cap=40, budget=8, slack=4, recent=3)
        ds.prefill(prompt)
        ids = ds.decode(ids0, 30)
        out.append((ids, ds.logits.download((2, 512), np.float32)))
        ds.free()
    assert np.array_equal(out[0][0], out[1][0]) and np.array_equal(out[0][1], out[1][1])


def test_a_budget_that_is_never_spent_changes_nothing_and_a_spent_one_keeps_the_newest(dev):
    st = small_stack()
    ids0, steps = np.array([5, 9, 300], np.int32), 24
    plain = DeviceStack(dev, st, 3, steps)
    want = plain.decode(ids0, steps)
    plain.free()
    roomy = DeviceStack(dev, st, 3, steps, budget=steps, slack=2)
    assert np.array_equal(roomy.decode(ids0, steps), want)
    roomy.free()
    tight = DeviceStack(dev, st, 3, steps, budget=10, slack=4, recent=5)
    got = tight.decode(ids0, steps)
    assert np.array_equal(got[:14], want[:14])  # the first eviction comes before step 14
    used = 12                                   # evictions before steps 14, 18 and 22, then two tokens
    for l in tight.attn:
        pos = l.pos.download((3, 2, 14), np.int32)[:, :, :used]
        for row in pos.reshape(-1, used):
            assert len(set(row.tolist())) == used and set(range(17, 24)) <= set(row.tolist()) <= set(range(24))
    assert np.array_equal(tight.decode(ids0, steps), got)
    tight.free()


def test_refusals(dev):
    bare = synth_stack(seed=3, hidden=256, inter=64, dense_inter=128, n_experts=8, k=2, n_layers=1, first_dense=1, vocab=64)
    for kw in (dict(prefix_cap=4), dict(budget=4)):
        with pytest.raises(ValueError):
            DeviceStack(dev, bare, 1, 4, **kw)
    st = small_stack()
    for kw in (dict(budget=0), dict(budget=4, slack=0), dict(budget=4, recent=5)):
        with pytest.raises(ValueError):
            DeviceStack(dev, st, 1, 4, **kw)
    ds = DeviceStack(dev, st, 1, 4, prefix_cap=10)
    with pytest.raises(ValueError):
        ds.prefill(np.zeros(11, np.int32))
    with pytest.raises(ValueError):
        stack_forward_rows(ds)
    ds.free()
    ds = DeviceStack(dev, bare, 1, 4)
    with pytest.raises(ValueError):
        ds.prefill(np.zeros(1, np.int32))
    ds.free()

"""Synthetic decode stack (the shape family of the benchmark's full-stack config) on one device.

    embed -> [ (attention ->) rmsnorm -> (dense SwiGLU | MoE layer) -> residual add ] x L -> rmsnorm -> lm_head -> argmax

This is the loop shape of the reference's batched decode step
(crates/peregrine-model/src/model.rs:1971-2006 per layer, :4260-4261 final norm + lm_head,
sample.rs:21-43 greedy pick), with attention left out or, for stacks that have it, as grouped-query attention:

    rmsnorm -> merged q/k/v projection -> head norms, rotation, cache store -> attention behind the shared
    prefix -> output projection -> residual add

Everything stays on the device between steps: token ids feed the next step's embedding gather without a host
round trip.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass, field

import numpy as np

from . import attention, cuda
from .resident import upload_expert, upload_layer
from .synth import SynthExpert, SynthLayer, SynthMatrix, synth_attention, synth_expert, synth_layer, synth_matrix


@dataclass
class SynthStack:
    hidden: int
    vocab: int
    eps: float
    embed: np.ndarray                  # fp32 [vocab, hidden]
    norms: list                        # per layer fp32 [hidden]
    final_norm: np.ndarray
    lm_head: SynthMatrix               # int4 [vocab, hidden]
    layers: list = field(default_factory=list)   # SynthExpert (dense) or SynthLayer (MoE)
    attn: list = field(default_factory=list)     # SynthAttention per layer, or empty: no attention
    theta: float = 10000.0                       # base of its rotation


def synth_stack(seed: int, hidden: int, inter: int, dense_inter: int, n_experts: int, k: int, n_layers: int,
                first_dense: int, vocab: int, gs: int = 32, distinct_experts: int | None = None,
                scale_std: float = 0.02, attention_heads: tuple | None = None) -> SynthStack:
    """``attention_heads``: (query heads, kv heads, head width) for a stack with attention.  ``scale_std``: standard deviation of the weight scales.  At hidden sizes in the thousands the
    default 0.02 makes every FFN output dwarf the residual stream and greedy decoding collapses onto
    one token whatever the input; wide stacks pass a smaller value so that the ids keep depending on
    the tokens (the arithmetic under test is the same)."""
    rng = np.random.default_rng(seed)
    embed = rng.standard_normal((vocab, hidden)).astype(np.float32)
    norms = [(1.0 + 0.1 * rng.standard_normal(hidden)).astype(np.float32) for _ in range(n_layers)]
    final_norm = (1.0 + 0.1 * rng.standard_normal(hidden)).astype(np.float32)
    lm_head = synth_matrix(rng, vocab, hidden, gs)
    layers = []
    for li in range(n_layers):
        if li < first_dense:
            layers.append(synth_expert(rng, hidden, dense_inter, gs, scale_std))
        else:
            layers.append(synth_layer(seed * 1000 + li, hidden, inter, n_experts, k, gs, shared=True,
                                      distinct_experts=distinct_experts, scale_std=scale_std))
    attn = []
    if attention_heads is not None:
        attn = [synth_attention(rng, hidden, *attention_heads, gs, scale_std) for _ in range(n_layers)]
    return SynthStack(hidden, vocab, 1e-5, embed, norms, final_norm, lm_head, layers, attn)


CHUNK = 64  # prompt tokens of one pass: the most rows of a sequence that an attention call takes


class _DevBuf:
    def __init__(self, device: int, host: np.ndarray | None = None, nbytes: int | None = None):
        self.device = device
        self.nbytes = host.nbytes if host is not None else nbytes
        self.ptr = cuda.lib().coli_cuda_pipe_alloc(device, self.nbytes)
        if not self.ptr:
            raise cuda.CudaError("device allocation failed")
        if host is not None:
            host = np.ascontiguousarray(host)
            if cuda.lib().coli_cuda_pipe_upload(device, self.ptr, host.ctypes.data, host.nbytes) != 1:
                raise cuda.CudaError("device upload failed")

    def download(self, shape, dtype):
        out = np.empty(shape, dtype)
        if cuda.lib().coli_cuda_pipe_download(self.device, self.ptr, out.ctypes.data, out.nbytes) != 1:
            raise cuda.CudaError("device download failed")
        return out

    def free(self):
        if self.ptr:
            cuda.lib().coli_cuda_pipe_free(self.device, self.ptr)
            self.ptr = None


class _AttnLayer:
    """Projections and caches of one attention layer: the shared prefix, and ``cap`` slots per sequence."""

    def __init__(self, device: int, a, hidden: int, batch: int, cap: int, prefix_cap: int, dtype: str):
        up = cuda.Tensor.upload_grouped
        self.wqkv = up(device, a.wqkv.q, a.wqkv.scale, hidden, a.wqkv.o_n, a.wqkv.gs)
        self.wo = up(device, a.wo.q, a.wo.scale, a.wo.i_n, hidden, a.wo.gs)
        self.norm, self.q_norm, self.k_norm = (_DevBuf(device, w) for w in (a.norm, a.q_norm, a.k_norm))
        slots = batch * a.kv_heads * cap
        self.k, self.v = (_DevBuf(device, nbytes=slots * a.head_dim * 2) for _ in range(2))
        self.pos, self.acc = (_DevBuf(device, nbytes=slots * 4) for _ in range(2))
        self.plain = attention.KvView(self.k.ptr, self.v.ptr, batch, a.kv_heads, cap, a.head_dim, dtype)
        self.counted = attention.KvView(self.k.ptr, self.v.ptr, batch, a.kv_heads, cap, a.head_dim, dtype, self.pos.ptr,
                                        self.acc.ptr)
        self.bufs = [self.norm, self.q_norm, self.k_norm, self.k, self.v, self.pos, self.acc]
        self.prefix = None
        if prefix_cap:
            n = prefix_cap * a.kv_heads * a.head_dim * 2
            pk, pv = _DevBuf(device, nbytes=n), _DevBuf(device, nbytes=n)
            self.bufs += [pk, pv]
            self.prefix = attention.KvView(pk.ptr, pv.ptr, 1, a.kv_heads, prefix_cap, a.head_dim, dtype)

    def free(self):
        self.wqkv.free()
        self.wo.free()
        for b in self.bufs:
            b.free()


class DeviceStack:
    """The stack resident on one device; ``decode`` runs greedy steps without host round trips.

    Expert parallel (``ep`` = an ``EpWorkspace`` connected to the other ranks): this rank holds the
    routed experts it owns of every MoE layer and decodes ``batch`` = its home tokens; everything
    outside the MoE layers is per token, so only those layers exchange.

    A stack with attention keeps its caches in 16 bits (``dtype``).  ``prefill`` stores a prompt that all sequences
    share (up to ``prefix_cap`` tokens); a decode then continues behind it.  ``budget``: once a sequence has
    ``budget + slack`` tokens of its own, the ``budget`` slots stay that received the most attention (the ``recent``
    newest always among them)."""

    def __init__(self, device: int, st: SynthStack, batch: int, max_steps: int, ep=None, repeats: str = "upload",
                 prefix_cap: int = 0, dtype: str = "bf16", budget: int | None = None, slack: int = 16,
                 recent: int = 8):
        if st.attn and len(st.attn) != len(st.layers):
            raise ValueError("stack: attention is needed in every layer or in none")
        if not st.attn and (prefix_cap or budget is not None):
            raise ValueError("stack: a prefix or a budget needs attention layers")
        if budget is not None and (budget < 1 or slack < 1 or not 0 <= recent <= budget):
            raise ValueError("stack: budget and slack must be positive, and hold the recent slots")
        L = cuda.lib()
        self.device, self.st, self.batch, self.max_steps, self.ep = device, st, batch, max_steps, ep
        self.embed = _DevBuf(device, st.embed)
        self.norms = [_DevBuf(device, w) for w in st.norms]
        self.final_norm = _DevBuf(device, st.final_norm)
        self.lm_head = cuda.Tensor.upload_grouped(device, st.lm_head.q, st.lm_head.scale, st.hidden, st.vocab,
                                                  st.lm_head.gs)
        self.layers = []
        for layer in st.layers:
            if isinstance(layer, SynthLayer):
                if ep is not None:
                    from .ep import owned_range

                    self.layers.append(upload_layer(device, layer, owned_range(layer.n_experts, ep.rank, ep.world),
                                                    ep.rank, ep.world, repeats))
                else:
                    self.layers.append(upload_layer(device, layer, repeats=repeats))
            else:
                self.layers.append(upload_expert(device, layer, st.hidden, layer.gate.o_n))
        self.budget, self.slack, self.recent, self.prefix_cap, self.prefix_len = budget, slack, recent, prefix_cap, 0
        d, b = st.hidden, max(batch, CHUNK if prefix_cap else 0)  # rows of the widest pass
        widest = max([l.gate.o_n for l in st.layers if isinstance(l, SynthExpert)] + [1])
        self.x = _DevBuf(device, nbytes=b * d * 4)
        self.nrm = _DevBuf(device, nbytes=b * d * 4)
        self.ffn = _DevBuf(device, nbytes=b * d * 4)
        self.g = _DevBuf(device, nbytes=b * widest * 4)
        self.u = _DevBuf(device, nbytes=b * widest * 4)
        self.logits = _DevBuf(device, nbytes=batch * st.vocab * 4)
        self.ids = _DevBuf(device, nbytes=(max_steps + 1) * batch * 4)
        self.attn, self._attn_bufs, self._evict_at = [], [], set()
        if st.attn:
            cap = max_steps + 1 if budget is None else min(max_steps + 1, budget + slack)
            self.attn = [_AttnLayer(device, a, d, batch, cap, prefix_cap, dtype) for a in st.attn]
            wide = max(a.wqkv.o_n for a in st.attn)
            q = max(a.heads * a.head_dim for a in st.attn)

            def buf(nbytes):
                self._attn_bufs.append(_DevBuf(device, nbytes=max(nbytes, 16)))
                return self._attn_bufs[-1]

            self.qkv, self.q16, self.ctx = buf(b * wide * 4), buf(b * q * 2), buf(b * q * 4)
            self.base, self.pos = buf(max(batch, 1) * 4), buf(b * 4)          # of the step under way
            self.bases, self.poss = buf((max_steps + 1) * batch * 4), buf((max_steps + 1) * batch * 4)  # of every step
            self.kept, self.kept_len = buf(batch * max(a.kv_heads for a in st.attn) * (budget or 1) * 4), buf(batch * 4)
            self.full = _DevBuf(device, np.full(batch, (budget or 0) + slack, np.int32))  # slots in use before an eviction
            self._attn_bufs.append(self.full)
            need = 16
            for a, l in zip(st.attn, self.attn):
                need = max(need, attention.attention_workspace(device, batch, a.heads, self._own(l), prefix_cap))
                if prefix_cap:
                    for rows in range(1, CHUNK + 1):
                        need = max(need, attention.attention_workspace(device, rows, a.heads, l.prefix, 0, rows))
            self.work = buf(need)
        self.graphs = None  # step graphs: None = not tried yet, [] = not available
        self.ping = self.pong = None
        self._L = L

    def _ok(self, rc, what):
        if rc != 1:
            raise cuda.CudaError(f"stack: {what} failed")

    def _own(self, layer: _AttnLayer):
        return layer.plain if self.budget is None else layer.counted

    def _attention(self, li: int, rows: int, own, base_ptr: int, rows_per_seq: int, prefix, prefix_len: int):
        """x += attention(x) of layer ``li`` for ``rows`` rows, their keys and values stored in ``own``."""
        L, dev, d = self._L, self.device, self.st.hidden
        vp, a, l = C.c_void_p, self.st.attn[li], self.attn[li]
        self._ok(L.coli_cuda_pipe_rmsnorm(dev, vp(self.nrm.ptr), vp(self.x.ptr), vp(l.norm.ptr), rows, d,
                                          C.c_float(self.st.eps)), "attention rmsnorm")
        self._ok(L.coli_cuda_pipe_gemm(l.wqkv.handle, vp(self.qkv.ptr), vp(self.nrm.ptr), rows), "q/k/v projection")
        attention.qk_norm_rope(dev, self.q16.ptr, self.qkv.ptr, rows, a.heads, own, base_ptr, self.pos.ptr, self.st.theta,
                               q_weight=l.q_norm.ptr, k_weight=l.k_norm.ptr, eps=self.st.eps, rows_per_seq=rows_per_seq)
        attention.attention(dev, self.ctx.ptr, self.q16.ptr, rows, a.heads, own, base_ptr, a.head_dim ** -0.5,
                            self.work.ptr, self.work.nbytes, rows_per_seq=rows_per_seq,
                            prefix=prefix if prefix_len else None, prefix_len=prefix_len)
        self._ok(L.coli_cuda_pipe_gemm(l.wo.handle, vp(self.nrm.ptr), vp(self.ctx.ptr), rows), "output projection")
        self._ok(L.coli_cuda_pipe_add(dev, vp(self.x.ptr), vp(self.nrm.ptr), rows * d), "attention residual")

    def prefill(self, ids) -> None:
        """Appends prompt tokens to the prefix that all sequences share, in passes of up to 64 tokens."""
        ids = np.ascontiguousarray(ids, np.int32).reshape(-1)
        if not self.attn:
            raise ValueError("stack: a prefix needs attention layers")
        if self.ep is not None:
            raise ValueError("stack: expert-parallel stacks take no shared prefix")
        if self.prefix_len + ids.size > self.prefix_cap:
            raise ValueError("stack: more prompt tokens than the prefix holds")
        self._drop_graphs()  # a recorded step has the prefix's length in it
        L, dev, st = self._L, self.device, self.st
        vp = C.c_void_p
        for at in range(0, ids.size, CHUNK):
            c = ids[at:at + CHUNK]
            n, done = c.size, self.prefix_len
            chunk = _DevBuf(dev, c)
            pos = np.arange(done, done + n, dtype=np.int32)
            self._ok(L.coli_cuda_pipe_upload(dev, vp(self.pos.ptr), pos.ctypes.data, pos.nbytes), "positions upload")
            base = np.array([done], np.int32)
            self._ok(L.coli_cuda_pipe_upload(dev, vp(self.base.ptr), base.ctypes.data, 4), "base upload")
            self._ok(L.coli_cuda_pipe_embed(dev, vp(self.x.ptr), vp(self.embed.ptr), vp(chunk.ptr), n, st.hidden, st.vocab),
                     "embed")
            for li in range(len(self.layers)):
                # the prefix is the only sequence of its cache, and its own slots are all there are
                self._attention(li, n, self.attn[li].prefix, self.base.ptr, n, None, 0)
                self._ffn(li, n)
            chunk.free()
            self.prefix_len += n

    def step(self, t: int):
        """ids[t] -> ids[t+1], all on the device's stream, one call per operation."""
        b = self.batch
        self._place(t)
        self._step_ops(self.ids.ptr + t * b * 4, self.ids.ptr + (t + 1) * b * 4)

    def _place(self, t: int):
        """Positions and slots of step ``t``, after an eviction where the budget is spent."""
        if not self.attn:
            return
        L, dev, b = self._L, self.device, self.batch
        vp = C.c_void_p
        if t in self._evict_at:
            for l in self.attn:
                attention.kv_evict(dev, l.counted, l.counted, self.full.ptr, self.kept_len.ptr, self.kept.ptr, self.budget,
                                   sinks=0, recent=self.recent)
        for now, table in ((self.base, self.bases), (self.pos, self.poss)):
            self._ok(L.coli_cuda_pipe_copy2d(dev, vp(now.ptr), b, vp(table.ptr + t * b * 4), b, b, 1), "places of the step")

    def _step_ops(self, ids_in_ptr: int, ids_out_ptr: int):
        L, dev, st, b, d = self._L, self.device, self.st, self.batch, self.st.hidden
        vp = C.c_void_p
        ids_in = vp(ids_in_ptr)
        ids_out = vp(ids_out_ptr)
        self._ok(L.coli_cuda_pipe_embed(dev, vp(self.x.ptr), vp(self.embed.ptr), ids_in, b, d, st.vocab), "embed")
        for li in range(len(self.layers)):
            if self.attn:
                l = self.attn[li]
                self._attention(li, b, self._own(l), self.base.ptr, 1, l.prefix, self.prefix_len)
            self._ffn(li, b)
        self._ok(L.coli_cuda_pipe_rmsnorm(dev, vp(self.nrm.ptr), vp(self.x.ptr), vp(self.final_norm.ptr), b, d,
                                          C.c_float(st.eps)), "final rmsnorm")
        self._ok(L.coli_cuda_pipe_gemm(self.lm_head.handle, vp(self.logits.ptr), vp(self.nrm.ptr), b), "lm_head")
        self._ok(L.coli_cuda_pipe_argmax(dev, ids_out, vp(self.logits.ptr), b, st.vocab), "argmax")

    def _ffn(self, li: int, b: int):
        """x += ffn(rmsnorm(x)) of layer ``li`` for ``b`` rows."""
        L, dev, st, d, layer = self._L, self.device, self.st, self.st.hidden, self.layers[li]
        vp = C.c_void_p
        self._ok(L.coli_cuda_pipe_rmsnorm(dev, vp(self.nrm.ptr), vp(self.x.ptr), vp(self.norms[li].ptr), b, d,
                                          C.c_float(st.eps)), "rmsnorm")
        if isinstance(layer, cuda.MoeLayer):
            if self.ep is not None:
                self._ok(L.coli_cuda_moe_layer_ep_forward_dev(layer.handle, self.ep.handle, vp(self.ffn.ptr),
                                                              vp(self.nrm.ptr)), "expert-parallel layer")
            else:
                layer.forward_dev(self.ffn.ptr, self.nrm.ptr, b)
        else:
            inter = layer.gate.o_n
            self._ok(L.coli_cuda_pipe_gemm(layer.gate.handle, vp(self.g.ptr), vp(self.nrm.ptr), b), "gate")
            self._ok(L.coli_cuda_pipe_gemm(layer.up.handle, vp(self.u.ptr), vp(self.nrm.ptr), b), "up")
            self._ok(L.coli_cuda_pipe_silu_mul(dev, vp(self.g.ptr), vp(self.u.ptr), b * inter), "silu_mul")
            self._ok(L.coli_cuda_pipe_gemm(layer.down.handle, vp(self.ffn.ptr), vp(self.g.ptr), b), "down")
        self._ok(L.coli_cuda_pipe_add(dev, vp(self.x.ptr), vp(self.ffn.ptr), b * d), "residual")

    def start(self, ids0: np.ndarray):
        ids0 = np.ascontiguousarray(ids0, np.int32)
        self._ok(self._L.coli_cuda_pipe_upload(self.device, C.c_void_p(self.ids.ptr), ids0.ctypes.data, ids0.nbytes),
                 "ids upload")
        if not self.attn:
            return
        # slots in use by the sequences at every step, and the steps that an eviction comes before
        base, at = np.zeros((self.max_steps + 1, self.batch), np.int32), 0
        self._evict_at = set()
        for t in range(self.max_steps + 1):
            if self.budget is not None and at >= self.budget + self.slack:
                self._evict_at.add(t)
                at = self.budget
            base[t] = at
            at += 1
        pos = np.repeat(np.arange(self.max_steps + 1, dtype=np.int32)[:, None] + self.prefix_len, self.batch, 1)
        pos = np.ascontiguousarray(pos, np.int32)
        for buf, host in ((self.bases, base), (self.poss, pos)):
            self._ok(self._L.coli_cuda_pipe_upload(self.device, C.c_void_p(buf.ptr), host.ctypes.data, host.nbytes),
                     "places upload")

    def result(self, steps: int) -> np.ndarray:
        return self.ids.download((steps + 1, self.batch), np.int32)[1:]

    def _record_step_graphs(self) -> bool:
        """Records one decode step twice as a replayable graph (ids: ping -> pong and pong -> ping), in
        the manner of the reference's COLI_CUDA_GRAPH pipe capture (cuda/backend_cuda.h:178-184): a step
        is ~90 launches whose arguments never change, and enqueueing them one by one from the host takes
        longer than the device needs to run them.  Needs one step already run (buffers sized, expert
        tables uploaded).  Expert-parallel stacks keep the call-by-call path: their exchange numbers
        its steps on the host."""
        if self.ep is not None or os.environ.get("PEREGRINE_B200_STACK_GRAPH") == "0":
            return False
        L, dev, b = self._L, self.device, self.batch
        self.ping = _DevBuf(dev, nbytes=b * 4)
        self.pong = _DevBuf(dev, nbytes=b * 4)
        graphs = []
        for src, dst in ((self.ping, self.pong), (self.pong, self.ping)):
            if L.coli_cuda_graph_begin(dev) != 1:
                return False
            try:
                self._step_ops(src.ptr, dst.ptr)
                ok = True
            except cuda.CudaError:
                ok = False
            g = C.c_void_p()
            if L.coli_cuda_graph_end(dev, C.byref(g)) != 1 or not ok:
                for h in graphs:
                    L.coli_cuda_graph_free(h)
                return False
            graphs.append(g)
        self.graphs, self._graphs_gen = graphs, L.coli_cuda_scratch_generation(dev)
        return True

    def run(self, steps: int):
        """Enqueues `steps` greedy steps from ids[0] (see ``start``): ids[t + 1] = step(ids[t])."""
        if steps > self.max_steps:
            raise ValueError("more steps than the id buffer holds")
        if steps < 1:
            return
        L, dev, b = self._L, self.device, self.batch
        vp = C.c_void_p
        if self.graphs and self._graphs_gen != L.coli_cuda_scratch_generation(dev):
            self._drop_graphs()  # a wider call has moved the scratch that they hold the addresses of
        if self.graphs is None:
            self.step(0)  # call by call: sizes every buffer, uploads the expert tables
            self.graphs = [] if not self._record_step_graphs() else self.graphs
            first = 1
        else:
            first = 0
        if not self.graphs:
            for t in range(first, steps):
                self.step(t)
            return
        row = lambda t: vp(self.ids.ptr + t * b * 4)
        self._ok(L.coli_cuda_pipe_copy2d(dev, vp(self.ping.ptr), b, row(first), b, b, 1), "ids to the step graph")
        bufs = (self.ping, self.pong)
        for t in range(first, steps):
            k = (t - first) & 1
            self._place(t)
            self._ok(L.coli_cuda_graph_launch_async(self.graphs[k]), "step graph launch")
            self._ok(L.coli_cuda_pipe_copy2d(dev, row(t + 1), b, vp(bufs[1 - k].ptr), b, b, 1), "ids of the step")

    def decode(self, ids0: np.ndarray, steps: int) -> np.ndarray:
        """Greedy decode: returns int32 ids [steps, batch] (the tokens picked at each step)."""
        self.start(ids0)
        self.run(steps)
        return self.result(steps)

    def _drop_graphs(self):
        for g in self.graphs or []:
            self._L.coli_cuda_graph_free(g)
        self.graphs = None
        for buf in (self.ping, self.pong):
            if buf is not None:
                buf.free()
        self.ping = self.pong = None

    def free(self):
        self._drop_graphs()
        self.graphs = []
        for l in self.layers + self.attn:
            l.free()
        for b in self._attn_bufs:
            b.free()
        self.lm_head.free()
        for b in [self.embed, self.final_norm, self.x, self.nrm, self.ffn, self.g, self.u, self.logits, self.ids] + \
                self.norms:
            b.free()

"""The attention half of a decode layer on device memory: norms, rotation and cache store of a projection's rows
(``qk_norm_rope``), attention behind a shared prefix (``attention``) and the eviction that keeps a cache within a
budget (``kv_evict``).  Pointers are device addresses; every call only enqueues work on the device's stream
(``cuda.lib().coli_cuda_stream``) and raises ``CudaError`` when the backend refuses it.  The C declarations in
``include/peregrine_b200.h`` say what each argument means.  The reference has no counterpart: its attention is
MLA on the CPU lane (crates/peregrine-model/src/attention.rs)."""
from __future__ import annotations

import ctypes as C

from . import cuda

DTYPES = {"bf16": 1, "f16": 2}


class _Kv(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("pos", C.c_void_p), ("acc", C.c_void_p), ("n_seq", C.c_int),
                ("n_kv", C.c_int), ("cap", C.c_int), ("D", C.c_int), ("dtype", C.c_int), ("seq_stride", C.c_longlong),
                ("head_stride", C.c_longlong), ("slot_stride", C.c_longlong)]


class KvView:
    """One layer's cache of keys and values in device memory that the caller owns (``ColiCudaKv``).

    ``strides``: elements between sequences, heads and slots (default: dense ``[n_seq, n_kv, cap, head_dim]``);
    ``pos`` and ``acc``: dense ``[n_seq, n_kv, cap]`` int32 / fp32, or 0."""

    def __init__(self, k: int, v: int, n_seq: int, n_kv: int, cap: int, head_dim: int, dtype: str = "bf16",
                 pos: int = 0, acc: int = 0, strides=None):
        if dtype not in DTYPES:
            raise cuda.CudaError(f"kv view: dtype {dtype!r} is not one of {sorted(DTYPES)}")
        self.n_seq, self.n_kv, self.cap, self.head_dim, self.dtype = n_seq, n_kv, cap, head_dim, dtype
        a, b, c = (0, 0, 0) if strides is None else strides
        self._c = _Kv(k, v, pos or None, acc or None, n_seq, n_kv, cap, head_dim, DTYPES[dtype], a, b, c)
        self._ref = C.byref(self._c)


_norm = _attend = _workspace = _evict = None  # the library's functions, bound at the first call


def _bind():
    """Another thread may find a function as soon as it is bound here: it gets there with its argument types."""
    global _norm, _attend, _workspace, _evict
    L = cuda.lib()
    vp, i, f, ll, sz = C.c_void_p, C.c_int, C.c_float, C.c_longlong, C.c_size_t
    norm, attend = L.coli_cuda_pipe_qk_norm_rope, L.coli_cuda_pipe_attention
    workspace, evict = L.coli_cuda_pipe_attention_workspace, L.coli_cuda_pipe_kv_evict
    norm.argtypes = [i, vp, vp, ll, i, i, vp, vp, vp, f, vp, vp, i, f, i, i]
    workspace.argtypes = [i, i, i, vp, i, i]
    workspace.restype = sz
    evict.argtypes = [i, vp, vp, vp, vp, vp, i, i, i]
    attend.argtypes = [i, vp, i, vp, i, i, vp, i, vp, vp, i, vp, f, vp, sz]
    _norm, _attend, _workspace, _evict = norm, attend, workspace, evict


def qk_norm_rope(device: int, q_out: int, qkv: int, rows: int, heads: int, kv: KvView, base: int, pos: int,
                 theta: float, rotary: int | None = None, style: int = 0, q_weight: int = 0, k_weight: int = 0,
                 eps: float = 1e-6, rows_per_seq: int = 1, row_stride: int | None = None) -> None:
    """Rows of a merged q/k/v projection -> normed, rotated queries in ``q_out`` and keys and values in the cache."""
    if _norm is None:
        _bind()
    if rotary is None:
        rotary = kv.head_dim
    if row_stride is None:
        row_stride = (heads + 2 * kv.n_kv) * kv.head_dim
    if _norm(device, q_out, qkv, row_stride, rows, heads, kv._ref, q_weight, k_weight, eps, pos, base, rows_per_seq,
             theta, rotary, style) != 1:
        raise cuda.CudaError("cuda pipe_qk_norm_rope failed")


def attention_workspace(device: int, rows: int, heads: int, own: KvView, prefix_len: int = 0,
                        rows_per_seq: int = 1) -> int:
    """Bytes of scratch that ``attention`` needs for calls of this shape."""
    if _workspace is None:
        _bind()
    n = _workspace(device, rows, heads, own._ref, prefix_len, rows_per_seq)
    if n == 0:
        raise cuda.CudaError("cuda pipe_attention_workspace: shape refused")
    return int(n)


def attention(device: int, out: int, q: int, rows: int, heads: int, own: KvView, base: int, scale: float, work: int,
              work_bytes: int, rows_per_seq: int = 1, prefix: KvView | None = None, prefix_len: int = 0, mask: int = 0,
              out_f32: bool = True) -> None:
    """Attention of every sequence over the shared prefix and its own slots; adds to ``own``'s acc when it has one."""
    if _attend is None:
        _bind()
    if _attend(device, out, 1 if out_f32 else 0, q, rows, heads, None if prefix is None else prefix._ref, prefix_len,
               own._ref, base, rows_per_seq, mask, scale, work, work_bytes) != 1:
        raise cuda.CudaError("cuda pipe_attention failed")


def kv_evict(device: int, dst: KvView, src: KvView, length: int, new_length: int, index: int, keep: int,
             sinks: int = 0, recent: int = 0) -> None:
    """Keeps the ``keep`` best slots of every sequence and head (``dst`` may be ``src``)."""
    if _evict is None:
        _bind()
    if _evict(device, dst._ref, src._ref, length, new_length, index, keep, sinks, recent) != 1:
        raise cuda.CudaError("cuda pipe_kv_evict failed")

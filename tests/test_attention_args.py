"""Calls that the attention entry points refuse: every check comes before the device is touched, so they run without
one.  A call that passes them all is then refused for the missing context, which is how the base case is known good."""
import ctypes as C

import pytest

from peregrine_b200 import attention as at, cuda

P = 1 << 20  # an aligned address that nothing reads


def view(**kw):
    a = dict(k=P, v=P + 4096, n_seq=2, n_kv=2, cap=16, head_dim=64, dtype="bf16", pos=P, acc=P, strides=None)
    a.update({k: v for k, v in kw.items() if k in a})
    v = at.KvView(**a)
    for k, x in kw.items():
        if k not in a:
            setattr(v._c, k, x)
    return v


def norm(kv=None, **kw):
    a = dict(q_out=2 * P, qkv=P, rows=4, heads=4, base=P, pos=P, theta=1e4, rotary=64, style=0, q_weight=P, k_weight=P,
             eps=1e-6, rows_per_seq=2, row_stride=8 * 64)
    a.update(kw)
    at.qk_norm_rope(0, kv=kv or view(), **a)


def attend(own=None, **kw):
    a = dict(out=P, q=P, rows=4, heads=4, base=P, scale=0.1, work=P, work_bytes=1 << 40, rows_per_seq=2,
             prefix=view(n_seq=1, cap=100), prefix_len=100, mask=P, out_f32=True)
    a.update(kw)
    at.attention(0, own=own or view(), **a)


def evict(dst=None, src=None, **kw):
    a = dict(length=P, new_length=P, index=P, keep=8, sinks=1, recent=2)
    a.update(kw)
    at.kv_evict(0, dst or view(k=2 * P, v=3 * P, pos=2 * P, acc=3 * P, cap=8), src or view(), **a)


@pytest.fixture(autouse=True)
def _no_context():
    assert cuda.device_count() == 0


def said(capfd, call, *a, **kw):
    with pytest.raises(cuda.CudaError):
        call(*a, **kw)
    return capfd.readouterr().err


@pytest.mark.parametrize("call", [norm, attend, evict])
def test_a_good_call_lacks_only_the_device(capfd, call):
    assert "device 0 is not initialised" in said(capfd, call)


KV_BAD = [(dict(k=0), "no cache"), (dict(v=0), "no cache"), (dict(n_seq=0), "empty"), (dict(n_kv=0), "empty"),
          (dict(cap=0), "empty"), (dict(head_dim=96), "head width"), (dict(dtype_=3), "cache type"),
          (dict(k=P + 8), "aligned"), (dict(v=P + 2), "aligned"), (dict(acc=P + 2), "aligned"),
          (dict(strides=(2048, 1024, 4)), "multiples of 8"), (dict(strides=(2048, 1024, 56)), "overlap"),
          (dict(strides=(2048, 0, 64)), "overlap"), (dict(strides=(-2048, 1024, 64)), "multiples"),
          (dict(strides=(1 << 50, 1024, 64)), "multiples")]


@pytest.mark.parametrize("bad, why", KV_BAD)
@pytest.mark.parametrize("call", [norm, attend])
def test_caches_that_do_not_hold_together(capfd, call, bad, why):
    bad = dict(bad)
    kv = view(**{k: v for k, v in bad.items() if k != "dtype_"})
    if "dtype_" in bad:
        kv._c.dtype = bad["dtype_"]
    err = said(capfd, call, kv)
    assert why in err and "not initialised" not in err


@pytest.mark.parametrize("bad, why", [
    (dict(rows=5), "sequences"), (dict(rows=0), "empty"), (dict(heads=0), "empty"), (dict(rows_per_seq=0), "empty"),
    (dict(q_out=0), "null"), (dict(qkv=0), "null"), (dict(base=0), "null"), (dict(pos=0), "null"),
    (dict(q_out=P + 4), "aligned"), (dict(qkv=P + 4), "aligned"), (dict(row_stride=8 * 64 + 2), "aligned"),
    (dict(row_stride=8 * 64 - 4), "row stride"), (dict(row_stride=1 << 41), "row stride"), (dict(rotary=63), "rotary"),
    (dict(rotary=66), "rotary"), (dict(rotary=-2), "rotary"), (dict(style=2), "style"), (dict(theta=0.0), "theta"),
    (dict(theta=float("inf")), "theta"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(pos=P + 2), "misaligned"), (dict(k_weight=P + 1), "misaligned"), (dict(q_out=P), "overlaps"),
    (dict(q_out=P + 4 * 512 * 4 - 16), "overlaps"), (dict(q_out=P - 4 * 4 * 64 * 2 + 16), "overlaps")])
def test_norm_refusals(capfd, bad, why):
    err = said(capfd, norm, **bad)
    assert why in err and "not initialised" not in err


@pytest.mark.parametrize("bad, why", [
    (dict(rows=5), "sequences"), (dict(heads=3), "multiple"), (dict(rows=130, rows_per_seq=65), "more than 64"),
    (dict(out=0), "null"), (dict(q=0), "null"), (dict(base=0), "null"), (dict(work=0), "null"),
    (dict(q=P + 2), "misaligned"), (dict(out=P + 4), "misaligned"), (dict(work=P + 128), "misaligned"),
    (dict(mask=P + 4), "misaligned"), (dict(prefix=None), "no cache"), (dict(prefix_len=-1), "negative"),
    (dict(prefix_len=101), "prefix of 101"), (dict(prefix=view(n_seq=2, cap=100)), "one sequence"),
    (dict(prefix=view(n_seq=1, cap=100, n_kv=1)), "one sequence"),
    (dict(prefix=view(n_seq=1, cap=100, dtype="f16")), "one sequence"),
    (dict(prefix=view(n_seq=1, cap=100, head_dim=128)), "one sequence"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=3e38), "scale")])
def test_attention_refusals(capfd, bad, why):
    err = said(capfd, attend, **bad)
    assert why in err and "not initialised" not in err


def test_attention_needs_no_prefix(capfd):
    assert "not initialised" in said(capfd, attend, prefix=None, prefix_len=0)


@pytest.mark.parametrize("bad, why", [
    (dict(keep=0), "cannot be kept"), (dict(keep=9), "cannot be kept"), (dict(sinks=-1), "negative"),
    (dict(recent=-1), "negative"), (dict(length=0), "null"), (dict(new_length=0), "null"), (dict(index=0), "null"),
    (dict(index=P + 2), "misaligned"), (dict(src=view(pos=0)), "pos and acc"), (dict(src=view(acc=0)), "pos and acc"),
    (dict(src=view(n_kv=1)), "differ"), (dict(src=view(dtype="f16")), "differ"), (dict(src=view(head_dim=128)), "differ"),
    (dict(src=view(n_seq=1)), "differ"), (dict(dst=view(cap=8)), "share"),
    (dict(dst=view(k=2 * P, v=3 * P, pos=2 * P)), "share"),
    (dict(dst=view(k=2 * P, v=3 * P, pos=P + 4 * 4 * 16 - 4, acc=3 * P, cap=8)), "share"),
    (dict(dst=view(k=2 * P, v=3 * P, pos=2 * P, acc=P - 4 * 4 * 8 + 4, cap=8)), "share"),
    (dict(dst=view(k=P - 4 * 8 * 64 * 2 + 16, v=3 * P, pos=2 * P, acc=3 * P, cap=8)), "share"),
    (dict(dst=view(k=2 * P, v=P + 4096 + 4 * 16 * 64 * 2 - 16, pos=2 * P, acc=3 * P, cap=8)), "share")])
def test_evict_refusals(capfd, bad, why):
    err = said(capfd, evict, **bad)
    assert why in err and "not initialised" not in err


def test_evict_in_place_is_a_good_call(capfd):
    v = view()
    assert "not initialised" in said(capfd, evict, v, v)


def test_workspace_refuses_like_the_call(capfd):
    for kw in (dict(rows=5), dict(heads=3), dict(prefix_len=-1), dict(rows=130, rows_per_seq=65)):
        a = dict(rows=4, heads=4, prefix_len=0, rows_per_seq=2)
        a.update(kw)
        with pytest.raises(cuda.CudaError):
            at.attention_workspace(0, own=view(), **a)
    assert "initialised" not in capfd.readouterr().err


def test_view_names_its_types():
    with pytest.raises(cuda.CudaError):
        view(dtype="f32")
    assert C.sizeof(at._Kv) == 4 * 8 + 5 * 4 + 4 + 3 * 8

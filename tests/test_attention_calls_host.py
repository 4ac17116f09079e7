"""Host side of the attention entry points: the binding, and checks that come before the device is touched."""
import pytest

from peregrine_b200 import attention as at, cuda
from peregrine_b200.stack import DeviceStack, synth_stack

P = 1 << 20  # an aligned address that nothing reads


class Function:
    """A library function before it is bound: nothing may be visible while its types are still being set."""

    def __init__(self, name):
        object.__setattr__(self, "name", name)

    def __setattr__(self, key, value):
        visible = (at._norm, at._attend, at._workspace, at._evict)
        assert visible == (None,) * 4, f"a function is visible before {self.name} has its {key}"
        object.__setattr__(self, key, value)


class Library:
    def __getattr__(self, name):
        f = Function(name)
        self.__dict__[name] = f
        return f


def test_a_bound_function_is_complete_when_it_becomes_visible(monkeypatch):
    for name in ("_norm", "_attend", "_workspace", "_evict"):
        monkeypatch.setattr(at, name, None)
    library = Library()
    monkeypatch.setattr(cuda, "lib", lambda: library)
    at._bind()
    for f, args in ((at._norm, 16), (at._attend, 15), (at._workspace, 6), (at._evict, 9)):
        assert len(f.argtypes) == args
    assert at._workspace.restype is not None


def refused(capfd, call, *a, **kw):
    """What a call says that fails for lack of a device at the latest."""
    assert cuda.device_count() == 0
    with pytest.raises(cuda.CudaError):
        call(*a, **kw)
    return capfd.readouterr().err


# sequences, heads, kv heads, slots, whether weights are kept, prefix
@pytest.mark.parametrize("n, H, Kv, cap, acc, Tp", [
    (20000, 65536, 64, 16, False, 0), (16384, 65536, 64, 16, False, 0),      # row vectors
    (4096, 512, 256, 40000, True, 0),                                          # slots whose weights are added up
    (1, 64, 1, 2147483647, False, 0), (100, 64, 64, 1073741824, False, 100),  # tiles
    (2, 7, 2, 16, False, 0), (2, 8, 2, 16, False, -1),
])
def test_a_refused_shape_has_no_workspace(capfd, n, H, Kv, cap, acc, Tp):
    own = at.KvView(P, 2 * P, n, Kv, cap, 64, acc=P if acc else 0, strides=(64, 64, 64))
    pre = at.KvView(P, 2 * P, 1, Kv, 128, 64)
    call = refused(capfd, at.attention, 0, P, P, n, H, own, P, 0.1, P, 1 << 60, prefix=pre if Tp else None, prefix_len=Tp)
    space = refused(capfd, at.attention_workspace, 0, n, H, own, Tp)
    assert call.split(": ", 1)[1] == space.split(": ", 1)[1]


@pytest.mark.parametrize("rows, stride, at_byte, why", [
    (4, 600, (3 * 600 + 512) * 4, "not initialised"),      # right behind the last row's values, before its stride ends
    (1, 1 << 20, 512 * 4, "not initialised"),
    (4, 600, (3 * 600 + 512) * 4 - 16, "overlaps"), (1, 1 << 20, 512 * 4 - 16, "overlaps"),
    (4, 600, -4 * 4 * 64 * 2, "not initialised"), (4, 600, -4 * 4 * 64 * 2 + 16, "overlaps"),
    (2147483647, 1 << 40, 0, "too large"),                 # (the rows' bytes pass 64 bits)
])
def test_queries_lie_outside_the_rows_and_not_their_padding(capfd, rows, stride, at_byte, why):
    kv = at.KvView(1 << 30, 1 << 31, rows, 2, 16, 64)
    assert why in refused(capfd, at.qk_norm_rope, 0, P + at_byte, P, rows, 4, kv, P, P, 1e4, row_stride=stride)


# One allocation of 2 sequences x 24 slots x 2 layers x 3 heads x 64 values, slots outermost within a sequence: a cache is
# `slots` slots of a layer from slot `at` on.
def pool(at_slot, slots, layer=0, pos=0, heads_first=False):
    n, kv, D, total = 2, 3, 64, 24
    if heads_first:  # [sequence, layer, head, slot, D] instead
        strides, first = (2 * kv * total * D, total * D, D), layer * kv * total * D + at_slot * D
    else:
        strides, first = (total * 2 * kv * D, D, 2 * kv * D), at_slot * 2 * kv * D + layer * kv * D
    k = (1 << 30) + 2 * first
    return at.KvView(k, k + (1 << 26), n, kv, slots, D, pos=(1 << 28) + pos, acc=(1 << 29) + pos, strides=strides)


def evict(capfd, dst, src, keep=8):
    return refused(capfd, at.kv_evict, 0, dst, src, P, P, P, keep)


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("src, dst, shared", [
    ((0, 16), (16, 8), False), ((8, 16), (0, 8), False),  # one behind the other, in every sequence and head
    ((0, 16), (15, 9), True), ((0, 16), (8, 8), True), ((8, 16), (1, 8), True), ((4, 16), (5, 8), True),
    ((0, 16), (0, 16, 1), False), ((0, 16), (8, 16, 1), False),  # another layer, between the same slots
    ((0, 24, 1), (16, 8, 1), True),
])
def test_targets_beside_or_upon_the_source_in_one_allocation(capfd, src, dst, shared, heads_first):
    err = evict(capfd, pool(*dst, pos=1 << 20, heads_first=heads_first), pool(*src, heads_first=heads_first))
    assert ("share" if shared else "not initialised") in err


def view(k, v, pos, acc, cap=16, strides=None, n=2, kv=2, D=64):
    return at.KvView(k, v, n, kv, cap, D, pos=pos, acc=acc, strides=strides)


M = 1 << 24


@pytest.mark.parametrize("dst, shared", [
    (dict(), False),
    (dict(pos=M + 64), True), (dict(acc=2 * M + 8000), True),                # positions and weights upon keys and values
    (dict(k=3 * M - 64), True), (dict(v=4 * M + 240), True),                 # and the other way round
    (dict(k=3 * M - 16 * 64 * 2 * 4), False), (dict(v=4 * M + 256), False),  # just before, just behind
    (dict(k=2 * M - 16, strides=(1 << 12, 1 << 11, 128)), True),             # a row that ends in the source's first
    (dict(k=M + 16 * 64 * 4 * 2, strides=(1 << 12, 1 << 11, 128)), False),
    (dict(k=M + 128, strides=(1 << 12, 1 << 11, 64)), True),
])
def test_targets_whose_arrays_meet_others_of_the_source(capfd, dst, shared):
    src = view(M, 2 * M, 3 * M, 4 * M)
    d = dict(k=5 * M, v=6 * M, pos=7 * M, acc=8 * M)
    d.update(dst)
    assert ("share" if shared else "not initialised") in evict(capfd, view(**d), src)


def test_targets_with_other_strides_between_the_rows_of_the_source(capfd):
    """Source rows of 64 values every 256, target rows every 512 behind the first of every other: they share nothing; moved on
    by 128 values to the source's rows they do."""
    def two(first, step, cap):
        return at.KvView(M + 2 * first, 2 * M + 2 * first, 1, 1, cap, 64, pos=3 * M + first * 1024, acc=4 * M + first * 1024, strides=(0, 0, step))

    src = two(0, 256, 100)
    assert "not initialised" in evict(capfd, two(128, 512, 40), src)
    assert "share" in evict(capfd, two(256, 512, 40), src)
    assert "share" in evict(capfd, two(200, 512, 40), src)
    assert "not initialised" in evict(capfd, two(128 + 512 * 3, 768, 30), src)


def test_many_sequences_in_one_allocation(capfd):
    """Source and target of every sequence behind one another, 100000 times: told apart.  Sequences in turn within every
    slot, 4096 of them: too many pairs to look at, refused."""
    n, one = 100000, 24 * 64
    src, dst = (at.KvView(M + 2 * f, M + (1 << 40) + 2 * f, n, 1, c, 64, pos=(1 << 50) + f * n, acc=(1 << 51) + f * n, strides=(one, 0, 64))
                for f, c in ((0, 16), (16 * 64, 8)))
    assert "not initialised" in evict(capfd, dst, src)
    src, dst = (at.KvView(M + 2 * f, M + (1 << 40) + 2 * f, 4096, 1, 16, 64, pos=(1 << 50) + f * n, acc=(1 << 51) + f * n,
                          strides=(128, 0, 1 << 20)) for f in (0, 64))
    assert "share" in evict(capfd, dst, src)


@pytest.mark.parametrize("kw", [dict(budget=4, recent=-1), dict(budget=4, recent=5), dict(budget=0), dict(budget=4, slack=0)])
def test_a_stack_refuses_a_budget_that_no_eviction_can_keep(kw):
    st = synth_stack(seed=3, hidden=64, inter=32, dense_inter=64, n_experts=2, k=1, n_layers=1, first_dense=1, vocab=32,
                     attention_heads=(2, 1, 64))
    with pytest.raises(ValueError):
        DeviceStack(0, st, 1, 4, **kw)

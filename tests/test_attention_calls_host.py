"""Host side of the attention entry points: the binding, and checks that come before the device is touched."""
import pytest

from peregrine_b200 import attention as at, cuda

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

"""Host side of the attention entry points: the binding, and checks that come before the device is touched."""
from peregrine_b200 import attention as at, cuda


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

"""The build compiles what is out of date, by its files or by the command it was compiled with (a stand-in for the compiler)."""
import importlib
import os
import subprocess
import time

import pytest

b = importlib.import_module("peregrine_b200.build")  # the package has a function of this name


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """Two units, a header of one of them, and a compiler that notes its arguments and writes its output."""
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for f in ("a.cu", "b.cpp", "a.cuh"):
        (csrc / f).write_text("")
        os.utime(csrc / f, (time.time() - 100,) * 2)
    log = tmp_path / "log"
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(f'#!/bin/sh\necho "$@" >> {log}\n[ -e {tmp_path}/broken ] && exit 1\n'
                    'while [ "$1" != "-o" ]; do shift; done\necho made > "$2"\n')
    nvcc.chmod(0o755)
    monkeypatch.setattr(b, "HERE", str(tmp_path))
    monkeypatch.setattr(b, "CSRC", str(csrc))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(b, "SOURCES", {"a.cu": ["a.cuh"], "b.cpp": []})
    monkeypatch.setattr(b, "NVCC_FLAGS", ["-O3", "-fmad=false"])
    monkeypatch.setattr(b, "LINK_FLAGS", ["-shared"])
    monkeypatch.setattr(b, "_nvcc", lambda: str(nvcc))

    def made(**kw):
        """The units that a build compiles, and whether it links."""
        log.write_text("")
        assert b.build(**kw) == str(tmp_path / "lib.so") and (tmp_path / "lib.so").exists()
        lines = log.read_text().split("\n")[:-1]
        return sorted(x.split()[-1] for x in lines if " -c " in x), sum("-shared" in x for x in lines)

    made.csrc, made.root = csrc, tmp_path
    return made


def later(path):
    os.utime(path, (time.time() + 100,) * 2)


def test_what_is_up_to_date_stays(tree):
    assert tree() == (["a.cu", "b.cpp"], 1)
    assert tree() == ([], 0)
    assert tree(force=True) == (["a.cu", "b.cpp"], 1)


def test_a_newer_file_compiles_its_unit(tree):
    tree()
    later(tree.csrc / "a.cuh")
    assert tree() == (["a.cu"], 1)


@pytest.mark.parametrize("then", [None, "b.cpp"])
def test_other_flags_compile_every_unit(tree, monkeypatch, then):
    tree()
    monkeypatch.setattr(b, "NVCC_FLAGS", ["-O3"])
    if then:  # with one of the files edited, too
        later(tree.csrc / then)
    assert tree() == (["a.cu", "b.cpp"], 1)
    if not then:
        assert tree() == ([], 0)
    monkeypatch.setattr(b, "NVCC_FLAGS", ["-O3", "-fmad=false"])
    assert tree()[0] == ["a.cu", "b.cpp"]


def test_other_link_flags_link_anew(tree, monkeypatch):
    tree()
    monkeypatch.setattr(b, "LINK_FLAGS", ["-shared", "-s"])
    assert tree() == ([], 1)


def test_verbose_prints_every_unit_and_leaves_the_others_up_to_date(tree):
    tree()
    assert tree(verbose=True) == (["a.cu", "b.cpp"], 1)
    assert tree() == ([], 0)


def test_a_unit_that_does_not_compile_is_tried_again(tree):
    tree()
    later(tree.csrc / "b.cpp")
    (tree.root / "broken").write_text("")
    with pytest.raises(subprocess.CalledProcessError):
        b.build()
    (tree.root / "broken").unlink()
    os.utime(tree.csrc / "b.cpp", (time.time() - 100,) * 2)
    assert tree() == (["b.cpp"], 1)

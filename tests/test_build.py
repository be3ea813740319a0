"""The build's order and what it needs, with compilers that only touch their outputs."""
import sys

import pytest

from maxsim_amd import _native, build


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    """Paths in a folder of their own, and a switch for sources that do not compile."""
    failing = set()

    def run(cmd):
        if any(source in cmd for source in failing):
            return 1, ["an error"]
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return 0, []

    monkeypatch.setattr(build, "_run", run)
    for name in ("LIB", "RATES_LIB", "BINDING"):
        monkeypatch.setattr(build, name, str(tmp_path / name))
    return tmp_path, failing


def test_all_of_it(compilers):
    path, _ = compilers
    assert build.build() == build.LIB
    assert sorted(p.name for p in path.iterdir()) == ["BINDING", "LIB", "RATES_LIB"]


def test_the_library_needs_no_torch(compilers, monkeypatch, capsys):
    path, _ = compilers
    monkeypatch.setitem(sys.modules, "torch", None)  # importing it raises ImportError
    build.build(verbose=True)
    assert sorted(p.name for p in path.iterdir()) == ["LIB", "RATES_LIB"]
    assert "torch cannot be imported" in capsys.readouterr().out


def test_a_module_that_does_not_compile(compilers):
    path, failing = compilers
    failing.add(build.BINDING_SRC)
    with pytest.raises(RuntimeError, match="tensor_calls.cpp"):
        build.build()
    assert sorted(p.name for p in path.iterdir()) == ["LIB", "RATES_LIB"]


def test_a_source_that_does_not_compile(compilers):
    path, failing = compilers
    failing.add(build.sources()[0])
    with pytest.raises(RuntimeError, match="compiler failed"):
        build.build()
    assert not any(p.name in ("BINDING", "LIB", "RATES_LIB") for p in path.iterdir())


@pytest.mark.parametrize("there,text", [(False, "is not built"), (True, "cannot be loaded beside torch")])
def test_a_module_that_cannot_be_imported(monkeypatch, tmp_path, there, text):
    monkeypatch.setattr(_native, "_calls", None)
    monkeypatch.setattr(_native, "load", lambda: None)
    monkeypatch.setattr(_native, "HERE", str(tmp_path))
    monkeypatch.setitem(sys.modules, "maxsim_amd._tensor_calls", None)
    monkeypatch.delattr("maxsim_amd._tensor_calls", raising=False)
    if there:
        (tmp_path / "_tensor_calls.so").write_bytes(b"")
    with pytest.raises(_native.NativeLibraryMissing, match=text):
        _native.tensor_calls()

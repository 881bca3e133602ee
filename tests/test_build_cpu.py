"""What the build needs: nvcc for the library, and nothing else where tensor_calls.so cannot be built."""
import os
import sys
import types

import pytest

from aljabr_b200 import build


@pytest.fixture
def lib_only(monkeypatch, tmp_path):
    """The library is built; tensor_calls.so would go to a folder of its own and is not there."""
    assert os.path.exists(build.LIB)
    made = []
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "tensor_calls.so"))
    monkeypatch.setattr(build, "_stale", lambda: False)
    monkeypatch.setattr(build, "_build_lib", lambda verbose: made.append("lib"))
    return made


def test_the_library_is_built_without_torch(lib_only, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB and build.build(force=True) == build.LIB
    assert lib_only == ["lib"] and "is not built" in capsys.readouterr().err and not os.path.exists(build.CALLS)


def test_the_library_is_not_stale_for_want_of_tensor_calls(monkeypatch, tmp_path):
    built = tmp_path / "lib.so"
    built.touch()
    monkeypatch.setattr(build, "LIB", str(built))
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "none.so"))
    assert not build._stale()
    os.utime(built, (0, 0))
    assert build._stale()


@pytest.mark.parametrize("name", ["CXX", "headers", "cuda"])
def test_the_library_is_built_without_a_compiler_headers_or_a_torch_for_cuda(lib_only, monkeypatch, capsys, tmp_path, name):
    torch = pytest.importorskip("torch")
    if name == "CXX":
        monkeypatch.setattr(build, "CXX", "no-such-compiler")
    elif name == "headers":
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "__init__.py"))
    else:
        monkeypatch.setattr(torch.version, "cuda", None)
    assert build.build() == build.LIB and "is not built" in capsys.readouterr().err


def test_a_compiler_that_fails_leaves_the_library(lib_only, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(build, "CXX", "false")
    with pytest.warns(RuntimeWarning, match="could not be built"):
        assert build.build() == build.LIB
    assert not os.path.exists(build.CALLS)


def test_tensor_calls_of_another_torch_is_built_again(monkeypatch):
    torch = pytest.importorskip("torch")
    assert os.path.exists(build.CALLS)
    monkeypatch.setattr(build, "_newer", lambda made, deps: False)
    assert not build._calls_stale(torch)
    for other in ("0.0", torch.__version__ + "1", torch.__version__[:-1]):
        assert build._calls_stale(types.SimpleNamespace(__version__=other))

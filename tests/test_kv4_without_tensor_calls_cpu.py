"""The 4-bit cache, the logits step and the decoder where tensor_calls.so is
missing or of another torch: it shortens the host's part of two calls and is
needed for none."""
import os
import subprocess
import sys
import types

import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("first", ["sys.modules['aljabr_b200.tensor_calls'] = None",
                                   "from aljabr_b200 import native; native.LIB_PATH += '.not'; sys.modules['aljabr_b200.tensor_calls'] = None"])
def test_the_modules_load_without_it(first):
    """(kv4 also where nothing is built yet: its calls name what is missing.)"""
    more = "" if "LIB_PATH" in first else "; from aljabr_b200 import logits, decode; from aljabr_b200.native import lib; lib()"
    code = f"import sys; sys.path.insert(0, {ROOT!r}); {first}; from aljabr_b200 import kv4; assert kv4.tensor_calls is None{more}"
    subprocess.run([sys.executable, "-W", "ignore", "-c", code], check=True, timeout=300)


@pytest.mark.parametrize("made", [{"torch": "1.0"}, {}])
def test_one_of_another_torch_is_not_used(monkeypatch, made):
    import aljabr_b200
    other = types.SimpleNamespace(**made)
    monkeypatch.setitem(sys.modules, "aljabr_b200.tensor_calls", other)
    monkeypatch.setattr(aljabr_b200, "tensor_calls", other, raising=False)
    with pytest.warns(RuntimeWarning, match="tensor_calls.so is not used"):
        assert kv4._load_calls() is None

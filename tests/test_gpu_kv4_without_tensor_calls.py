"""The tree operators through ctypes give the bits that they give through tensor_calls.so."""
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4
from tests.test_gpu_kv4_tree import fault_bits, run_step, step_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_without_tensor_calls(monkeypatch, dtype):
    assert kv4.tensor_calls is not None            # built with the rest, so that the step below is the other way
    a = step_case(dtype)
    want = run_step(a)
    monkeypatch.setattr(kv4, "tensor_calls", None)
    b = step_case(dtype)
    got = run_step(b)
    assert all(torch.equal(x, y) for x, y in zip(want[0], got[0])) and all(torch.equal(x, y) for x, y in zip(want[1], got[1]))
    assert all(torch.equal(x.data, y.data) for x, y in zip(a["caches"], b["caches"]))
    assert fault_bits() == 0

"""The tree operators through ctypes give the bits that they give through tensor_calls.so."""
import os
import subprocess
import sys

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


@pytest.mark.parametrize("call", ["cache.append_rotated(q, x[:, :1], x[:, :1], n, n, rope)",
                                  "accept_tree(cache, n, n, d.view(4, 1), d.view(4, 1), torch.zeros(4, 1, dtype=torch.int32, device='cuda'))"])
def test_tensors_without_memory_are_an_error_in_python(call):
    """Inside vmap a tensor has sizes and no address.  In a process of its own: what torch throws must not end it."""
    code = f"""
import torch
from aljabr_b200 import kv4
from aljabr_b200.kv4 import Kv4Cache, accept_tree
assert kv4.tensor_calls is not None
cache, x, rope = Kv4Cache(4, 16, 1, 64), torch.zeros(4, 1, 64, device='cuda'), torch.zeros(4, 32, 2, device='cuda')
n = torch.zeros(4, dtype=torch.int32, device='cuda')
try:
    torch.func.vmap(lambda q, d: {call})(torch.zeros(2, 4, 1, 64, device='cuda'), torch.zeros(2, 4, dtype=torch.int32, device='cuda'))
except RuntimeError as e:
    print('raised', type(e).__name__)
torch.cuda.synchronize()
"""
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert got.returncode == 0 and "raised" in got.stdout, got.stderr[-2000:]

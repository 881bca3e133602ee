"""Where the rotated append may write: into q, k and v themselves and between other rows, over nothing else."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import kv4, native
from tests.test_gpu_kv4 import fault_bits, make
from tests.test_gpu_kv4_tree import cuda, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,hq,hkv,D,rot,inter", [(1, 4, 1, 64, 64, False), (37, 6, 2, 64, 32, False), (300, 8, 4, 128, 128, False),
                                                  (300, 5, 1, 256, 256, False), (100, 4, 2, 256, 128, True)])
def test_outputs_in_place(n, hq, hkv, D, rot, inter, dtype):
    rng = np.random.default_rng(n + D)
    q, k, v = (cuda(rng.normal(size=(n, h, D)).astype(np.float32), dtype) for h in (hq, hkv, hkv))
    pages = -(-n // 16)
    slots = cuda(rng.permutation(pages * 16)[:n].astype(np.int32))
    pos = rng.integers(0, 90, n).astype(np.int32)
    pos[n // 2:n // 2 + 2] = -1
    args = slots, cuda(pos), cuda(table_of(90, rot // 2)), inter
    a, b = make(pages, 16, hkv, D), make(pages, 16, hkv, D)
    back = torch.empty_like(k), torch.empty_like(v)
    want = a.append_rotated(q, k, v, *args, k_back=back[0], v_back=back[1])
    got = b.append_rotated(q, k, v, *args, q_out=q, k_back=k, v_back=v)
    assert got is q and torch.equal(q, want) and torch.equal(k, back[0]) and torch.equal(v, back[1]) and torch.equal(a.data, b.data)
    assert fault_bits() == 0


@pytest.mark.parametrize("calls", [True, False])
def test_the_wrapper_refuses_overlaps(monkeypatch, calls):
    if not calls:
        monkeypatch.setattr(kv4, "tensor_calls", None)
    cache = make(2, 16, 1, 64)
    wide = torch.zeros(9, 3, 64, device="cuda")
    q, k, v = wide[1:5, 0:1], wide[1:5, 1:2], wide[1:5, 2:3]
    slots, table = torch.arange(4, dtype=torch.int32, device="cuda"), cuda(table_of(9, 32))
    for out in (k, v, wide[0:4, 0:1], wide[2:6, 0:1], wide[2:6, 1:2]):
        with pytest.raises(native.ProviderError, match="overlap"):
            cache.append_rotated(q, k, v, slots, slots, table, q_out=out)
    for out in (q, wide[5:9, 0:1], wide[5:9, 1:2]):
        assert cache.append_rotated(q, k, v, slots, slots, table, q_out=out) is out
    dense = torch.zeros(4, 1, 64, device="cuda")
    for kb, vb in ((dense, dense), (wide.view(-1)[64:320].view(4, 1, 64), dense)):
        with pytest.raises(native.ProviderError, match="overlap"):
            cache.append_rotated(q, k, v, slots, slots, table, k_back=kb, v_back=vb)
    assert fault_bits() == 0

"""A prompt in two chunks and the first decoded token over the 4-bit cache: the
chunks' own attention reads what the cache holds (fp32 rows handed back by
append, or read back), the token's attention the cache itself."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from aljabr_b200 import native
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import check, make

pytestmark = pytest.mark.gpu


def prefill(q, k, v):
    """Causal attention of the last len(q) positions over fp32 rows, on the tensors' stream."""
    from aljabr_b200.kv4 import current_stream
    (T, Hq, D), (S, Hkv, _) = q.shape, k.shape
    out = torch.empty_like(q)
    native.call("aljabr_blackwell_prefill_attention_dev", out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, T, S, Hq,
                Hkv, D, Hkv * D, D ** -0.5, 1, 0, 0.0, current_stream(0))
    return out


@pytest.mark.parametrize("D,Hkv,G,chunks", [(128, 2, 4, (70, 45)), (64, 3, 2, (16, 1)), (256, 1, 4, (33, 130))])
def test_prompt_in_chunks_then_a_token(D, Hkv, G, chunks):
    rng = np.random.default_rng(60 + D)
    n = sum(chunks) + 1
    k, v, q = (torch.from_numpy(rng.normal(size=(n, h, D)).astype(np.float32)).cuda() for h in (Hkv, Hkv, Hkv * G))
    cache = make(-(-n // 16), 16, Hkv, D, fill=0xFF)
    slots = torch.from_numpy(rng.permutation(-(-n // 16))[np.arange(n) // 16] * 16 + np.arange(n) % 16).int().cuda()
    a = chunks[0]
    back = torch.empty_like(k[:a]), torch.empty_like(v[:a])
    cache.append(k[:a], v[:a], slots[:a], k_back=back[0], v_back=back[1])
    outs = [prefill(q[:a].contiguous(), *back)]
    cache.append(k[a:n - 1], v[a:n - 1], slots[a:n - 1])
    outs.append(prefill(q[a:n - 1].contiguous(), *cache.read(slots[:n - 1])))
    cache.append(k[n - 1:], v[n - 1:], slots[n - 1:])
    table = (slots[::16] // 16)[None].contiguous()
    last = cache.attend(q[None, n - 1:], torch.tensor([n], dtype=torch.int32, device="cuda"), table)
    k64, v64 = (ref.values(*ref.quantise(t.cpu().numpy())) for t in (k, v))
    check(last, q[None, n - 1:], [k64], [v64], [n])
    # fp32 dots of D products and sums of at most n weights: errors of some 2^-22 a score, 2^-16 of the norm is ample
    want, _, _ = ref.attention(q[:n - 1].cpu().numpy(), k64[:n - 1], v64[:n - 1], n - 1)
    got = torch.cat(outs).double().cpu().numpy()
    assert np.linalg.norm(got - want) <= 2.0 ** -16 * np.linalg.norm(want)

"""How near the fp32 attention over the 4-bit cache comes to 64 bits in norm:
one lost part of P or of q shows here at once, where a bound of every element
by its largest possible error would hide it.

Bound, relative to the norm of a sequence's output: a query element is off by
at most 2^-23 of the largest of its group of 32 (about 5 standard deviations),
so a score by 2^-23 * 5 / sqrt(3) * 1.2 = 4.2e-7 rms for unit K (scale is
1 / sqrt(D)); exp2 and the two parts of P add 2^-22 each.  These errors are
independent over positions and weigh on the output as the positions' own values
do: under 1.3e-6 together, three times that is 2^-18.  tanh adds 2^-23 of the
cap to a score.  bf16: P and P dV rounded once each to fp16 (2^-11 at most,
2^-12 rms), the output to bf16 (2^-9 at most): 2^-8 together."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import kv4_ref as ref
from tests.test_gpu_kv4 import attend_case, check

pytestmark = pytest.mark.gpu


def near(out, q, k64, v64, lens, window=0, cap=0.0):
    qn, on = q.float().cpu().numpy(), out.double().cpu().numpy()
    bound = 2.0 ** -18 + cap * 2.0 ** -23 if q.dtype == torch.float32 else 2.0 ** -8
    for b, n in enumerate(lens):
        want, _, _ = ref.attention(qn[b], k64[b], v64[b], n, window=window, soft_cap=cap)
        err, size = np.linalg.norm(on[b] - want), np.linalg.norm(want)
        assert err <= bound * size, (b, n, err / size)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,hkv,G,T,ps,lens,window,cap", [
    (128, 2, 4, 1, 16, [1], 0, 0.0),
    (128, 8, 4, 1, 64, [0, 1, 15, 16, 17, 127, 128, 129, 257], 0, 0.0),
    (128, 1, 1, 1, 4096, [3000], 0, 0.0),
    (128, 2, 4, 1, 16, [4000, 100, 9000], 0, 0.0),
    (128, 2, 3, 5, 16, [5, 4, 200, 0, 1], 0, 0.0),
    (128, 1, 16, 7, 64, [900, 60], 100, 0.0),
    (64, 4, 2, 1, 16, [77, 1024], 0, 30.0),
    (64, 3, 7, 3, 16, [40, 2, 513], 33, 0.0),
    (256, 2, 4, 1, 16, [19, 640], 0, 0.0),
    (256, 1, 5, 4, 80, [400, 33], 7, 50.0),
])
def test_norm_of_the_error(D, hkv, G, T, ps, lens, window, cap, dtype):
    _, q, _, _, out, k64, v64 = attend_case(40 + D + G + T, D, hkv, G, T, ps, lens, window, cap, dtype)
    near(out, q, k64, v64, lens, window, cap)


def test_a_long_bf16_context():
    """Sums of 40000 positions stay in the tensor cores' accumulators."""
    lens = [40000]
    _, q, _, _, out, k64, v64 = attend_case(50, 128, 1, 8, 1, 64, lens, dtype=torch.bfloat16)
    check(out, q, k64, v64, lens)
    near(out, q, k64, v64, lens)


def test_the_repeated_case_is_right_too():
    lens = [4000, 100, 9000]
    _, q, _, _, out, k64, v64 = attend_case(11, 128, 2, 4, 1, 16, lens)
    check(out, q, k64, v64, lens)
    near(out, q, k64, v64, lens)


@pytest.mark.parametrize("D,batch", [(64, 700), (128, 600), (256, 300)])
def test_batches_beyond_one_cta_s_half_of_an_sm(D, batch):
    """Above about 550 sequences (D 128) the tables of lengths leave an SM one CTA."""
    lens = [int(n) for n in np.random.default_rng(51).integers(0, 40, batch)]
    _, q, _, _, out, k64, v64 = attend_case(51, D, 1, 2, 1, 48, lens)
    check(out, q, k64, v64, lens)


def test_the_most_rows_a_call_takes():
    """1024 rows of a kv head: 64 query tokens of 16 heads."""
    lens = [100, 64]
    for dtype in (torch.float32, torch.bfloat16):
        _, q, _, _, out, k64, v64 = attend_case(52, 64, 1, 16, 64, 16, lens, dtype=dtype)
        near(out, q, k64, v64, lens)

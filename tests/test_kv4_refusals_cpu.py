"""Arguments at the ends of their ranges, refused before the GPU is touched."""
import pytest

from aljabr_b200 import native
from tests.test_kv4_cpu import ARG, P, append, attend, logits, read


@pytest.mark.parametrize("cap", [float("inf"), 2e30, 1e-31, 1e-40])
def test_soft_caps_whose_reciprocal_is_no_use_are_refused(cap):
    """Scores are divided by the cap through its reciprocal: 0 * inf is NaN, and a subnormal one has lost its bits."""
    assert attend(cap=cap) == ARG and native.last_error()


@pytest.mark.parametrize("cap", [0.0, 1e-30, 30.0, 1e30])
def test_soft_caps_in_range_pass_their_check(cap):
    assert attend(cap=cap, out=P + 8) == ARG and "soft_cap" not in native.last_error()


@pytest.mark.parametrize("at", [P + 1, P + 2])
def test_integers_and_floats_off_their_alignment_are_refused(at):
    """The kernels read and write whole elements: an address between two faults the GPU."""
    assert append(slots=at) == ARG and read(slots=at) == ARG
    assert attend(lens=at) == ARG and attend(table=at) == ARG
    for name in ("out", "x", "h", "hl", "pen", "bt", "bv", "bl", "allow", "token"):
        assert logits(**{name: at}) == ARG, name
    assert logits(x=P + 1, dt=native.KV_BF16, xs=100) == ARG

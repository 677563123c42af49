"""The bounds of tests/tree_precision.py on the CPU: what is as good as the kernel says passes, planted mistakes do not."""
import numpy as np
import pytest

from tests.test_gpu_tree_attend import Case
from tests.tree_precision import Sink, bf16_of, check_norm, check_singled_out, emulated, single_out


def as_fp16(x):
    return np.asarray(x, np.float16)


@pytest.fixture(scope="module")
def sink():
    return Sink()


def test_a_long_flat_tail_holds_under_a_reference_that_rises_with_its_length(sink):
    for kept, lift in ((as_fp16, 6), (np.float32, 0)):
        sink.check(bf16_of(sink.exact(kept, lift)[0]))


@pytest.mark.parametrize("lift", [0, 1, 2])
def test_a_tail_below_the_least_weight_is_seen_to_be_lost(sink, lift):
    with pytest.raises(AssertionError):
        sink.check(bf16_of(sink.exact(as_fp16, lift)[0]))


def small_case(**kw):
    return Case(3, [900, 40], [4, 6], 16, **kw)


def to_bits(bits):
    """Rounds to so many bits."""
    def f(x):
        m, e = np.frexp(x)
        return np.ldexp(np.round(m * 2.0 ** bits) / 2.0 ** bits, e)
    return f


def without_sixteen(codes):
    codes = codes.copy()
    codes[32:48] = 0
    return codes


def sixteen_reversed(codes):
    codes = codes.copy()
    codes[32:48] = codes[32:48][::-1]
    return codes


@pytest.mark.parametrize("scale", [None, 0.0, -0.07])
def test_norms_hold_fp16_weights_and_no_less(scale):
    case = small_case()
    case.scale = case.scale if scale is None else scale
    check_norm(case, emulated(case, as_fp16))
    for kept, moved in ((to_bits(7), None), (as_fp16, without_sixteen), (as_fp16, sixteen_reversed)):
        with pytest.raises(AssertionError):
            check_norm(case, emulated(case, kept, moved))


@pytest.mark.parametrize("scale", [None, 0.0])
def test_norms_tell_bf16_weights(scale):
    case = small_case()
    case.scale = case.scale if scale is None else scale
    with pytest.raises(AssertionError):
        check_norm(case, emulated(case, bf16_of))


@pytest.mark.parametrize("growth", ["flat", "grow", "swing"])
def test_a_row_of_its_own_for_every_token_tells_what_scores_hide(growth):
    case = Case(4, [300], [5], 64, masks="chain")
    own = single_out(case, growth)
    assert set(range(300)) <= set(own.reshape(-1).tolist())
    check_singled_out(case, own, emulated(case, as_fp16))
    for moved in (without_sixteen, sixteen_reversed):
        with pytest.raises(AssertionError):
            check_singled_out(case, own, emulated(case, as_fp16, moved))

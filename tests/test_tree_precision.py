"""The bounds of tests/tree_precision.py on the CPU: what is as good as the kernel says passes, planted mistakes do not."""
import numpy as np
import pytest

from tests.tree_precision import Sink, bf16_of


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

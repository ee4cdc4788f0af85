"""The element-by-element comparison of the feed-forward tests finds what it has to."""

import math

import pytest
import torch

from feed_forward_strict import assert_each


def case():
    want = torch.tensor([1.0, math.nan, math.inf, -math.inf, 0.0], dtype=torch.float64)
    return want.float(), want, torch.full((5,), 0.25, dtype=torch.float64)


def test_equal_values_pass():
    got, want, bound = case()
    assert_each("v", got, want, bound)
    got[0], got[4] = 1.25, -0.25
    assert_each("v", got, want, bound)
    bound[1] = math.nan  # beside a value that is not finite a bound says nothing
    assert_each("v", got, want, bound)


@pytest.mark.parametrize("i,v", [(0, 1.2500001), (0, math.nan), (0, math.inf), (1, 0.0), (1, math.inf), (2, math.nan),
                                 (2, -math.inf), (2, 3e38), (3, math.inf), (4, math.nan), (4, 0.3)])
def test_each_element_counts(i, v):
    got, want, bound = case()
    got[i] = v
    with pytest.raises(AssertionError, match="1 of 5"):
        assert_each("v", got, want, bound)


def test_bounds_and_shapes():
    got, want, bound = case()
    bound[0] = math.inf
    with pytest.raises(AssertionError, match="not finite"):
        assert_each("v", got, want, bound)
    with pytest.raises(AssertionError):
        assert_each("v", got[:4], want, bound)

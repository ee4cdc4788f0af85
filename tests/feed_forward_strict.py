"""Comparison of results with 64-bit values and bounds, element by element:
an element that is not finite on either side hides no other."""

import torch


def assert_each(name, got, want, bound):
    """`got` within `bound` of `want` wherever `want` is finite (`bound` has to
    be finite there); the same infinity, or NaN, wherever it is not."""
    assert tuple(got.shape) == tuple(want.shape) == tuple(bound.shape), (name, got.shape, want.shape, bound.shape)
    got, finite = got.double(), torch.isfinite(want)
    assert bool(torch.isfinite(bound[finite]).all()), f"{name}: a bound is not finite"
    bad = torch.where(finite, ~((got - want).abs() <= bound),
                      ~((got == want) | (torch.isnan(got) & torch.isnan(want))))
    if bool(bad.any()):
        at = [tuple(i.tolist()) for i in bad.nonzero()[:4]]
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} elements out of bounds; " + "; ".join(
            f"{i}: got {got[i].item()!r}, want {want[i].item()!r} +- {bound[i].item():.3g}" for i in at))

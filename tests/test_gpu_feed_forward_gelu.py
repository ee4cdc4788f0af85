"""gelu's left tail, where the value is a small difference: relative to the
value itself, not to 1."""

import math

import pytest
import torch

import feed_forward_ref as R
from feed_forward_strict import assert_each
from test_gpu_feed_forward import BF16, F16

pytestmark = pytest.mark.gpu


def every_value(dtype, lo, hi):
    """All numbers of the type in [lo, hi]."""
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype).double()
    return v[torch.isfinite(v) & (v >= lo) & (v <= hi)].sort().values.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("few", [True, False])
def test_gelu_relative_to_itself(dtype, few):
    """Every 16-bit argument from -12.5 to 12.5 through each of the products:
    fp32 evaluation within 2^-14 of the value, then one rounding."""
    import dsv4_b200 as D
    v = every_value(dtype, -12.5, 12.5)
    z = v.double()
    want = R.act("gelu", z)
    w = torch.zeros(8, 16, device="cuda", dtype=dtype)
    w[:, 0] = 1
    x = torch.zeros(v.numel(), 16, device="cuda", dtype=dtype)
    x[:, 0] = v
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -14) * want.abs() + R.tiny_of(dtype)
    if few:  # up to 8 tokens at a time: the values as weights
        x, w = w[:1], torch.zeros(v.numel(), 16, device="cuda", dtype=dtype)
        w[:, 0] = v
        assert_each("y", D.dense_forward(x, w, activation="gelu")[0], want, bound)
        ones = torch.ones(100, 16, device="cuda", dtype=dtype) * (torch.arange(16, device="cuda") == 0)
        y = D.dense_forward(ones, w, activation="gelu")
        assert_each("y", y[99], want, bound)
    else:
        y, saved = D.dense_forward_save(x, w, activation="gelu")
        assert_each("y", y, want[:, None].expand(-1, 8), bound[:, None].expand(-1, 8))
        # the slope Phi + z phi: each term within 2^-14, at an argument kept within a 32767th of itself
        dy = torch.zeros(v.numel(), 8, device="cuda", dtype=dtype)
        dy[:, 0] = 1
        phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        slope = R.slope("gelu", z)
        e = 2.0 ** -14 * (R.act("gelu", z.abs().neg()).div(z.abs().clamp(min=2.0 ** -40)).abs().clamp(max=0.5)
                          + (z > 0) * 0.5 + z.abs() * phi)
        e = e + 1.1 * phi * (z * z + 2) * z.abs() / 32767
        bound = e + (torch.finfo(dtype).eps / 2) * (slope.abs() + e) + R.tiny_of(dtype)
        assert_each("slope", D.dense_backward(dy, saved)[0][:, 0], slope, bound)

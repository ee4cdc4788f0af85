"""Values before an activation as the backward pass reads them: their side of
the clamp limit and of zero."""

import math

import pytest
import torch

import feed_forward_ref as R
from feed_forward_strict import assert_each
from test_gpu_feed_forward import BF16, F16

pytestmark = pytest.mark.gpu


def bits16(dtype):
    return torch.finfo(dtype).eps / 2


def parts(t, dtype):
    """fp32 numbers as exact sums of three products of `dtype` numbers, the
    second factor 2^0, 2^-8 and 2^-16: bits 1-8, 9-16 and 17-24 of each."""
    out, rest = [], t.double()
    e = torch.floor(torch.log2(rest.abs()))
    for i in range(3):
        step = torch.exp2(e - 7 - 8 * i)
        p = torch.trunc(rest / step) * step
        out.append((p * 2.0 ** (8 * i)).to(dtype))
        assert torch.equal(out[-1].double(), p * 2.0 ** (8 * i))
        rest = rest - p
    assert bool((rest == 0).all())
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("limit", [0.37, 0.75, 1.3, 7.0, 7.7, 9.9, 12.3])
def test_values_a_step_from_the_limit(limit, dtype):
    """Sums that are the limit, or one to three fp32 steps off it, as all
    values of their group: masked exactly where they pass it, and read back
    with their own sign and size."""
    import dsv4_b200 as D
    lim = torch.tensor(limit, dtype=torch.float32)
    near = [lim]
    for way in (math.inf, -math.inf):
        t = lim
        for _ in range(3):
            t = torch.nextafter(t, torch.tensor(way))
            near.append(t)
    near = torch.stack(near)
    near = torch.cat((near, -near)).cuda()
    m, inter, hidden = near.numel(), 32, 64
    x = torch.zeros(m, hidden, device="cuda", dtype=dtype)
    for i, p in enumerate(parts(near, dtype)):
        x[:, 16 * i] = p
    x[:, 1] = 0.25
    factors = torch.zeros(hidden, device="cuda", dtype=dtype)
    factors[0], factors[16], factors[32] = 1, 2.0 ** -8, 2.0 ** -16
    half = torch.zeros(hidden, device="cuda", dtype=dtype)
    half[1] = 1
    w2 = torch.full((8, inter), 0.125, device="cuda", dtype=dtype)
    dy = torch.ones(m, 8, device="cuda", dtype=dtype)  # dh = 1
    z, lim = near.double(), lim.double().cuda()
    h16 = bits16(dtype)
    for kind in ("silu", "relu", None):
        a = lambda v: R.act(kind, v)  # noqa: E731
        s = lambda v: R.slope(kind, v)  # noqa: E731
        c = torch.full_like(z, 0.25)
        # kept within a 32767th; then dz rounded, 32 equal values added and the sum rounded
        off = lambda v, e: 2.1 * h16 * v.abs() + 40 * e  # noqa: E731
        ae = lambda v: 1.15 * v.abs() / 32767 + 2.0 ** -18 * (v.abs() + 1)  # noqa: E731
        se = lambda v: 0.82 * v.abs() / 32767 + 2.0 ** -17 * (v.abs() + 1)  # noqa: E731
        # gates near the limit, ups 1/4
        w13 = torch.cat((factors.expand(inter, -1), half.expand(inter, -1))).contiguous()
        _, saved = D.gated_feed_forward_save(x, w13, w2, activation=kind, clamp_limit=limit)
        gx = D.gated_feed_forward_backward(dy, saved)[0]
        dg = torch.where(z <= lim, 32 * 0.25 * s(z.clamp(max=lim)), torch.zeros_like(z))
        du = 32 * a(z.clamp(max=lim))
        assert_each(f"{kind} dg", gx[:, 0], dg, torch.where(z <= lim, off(dg, se(z)), torch.zeros_like(z)))
        assert_each(f"{kind} du", gx[:, 1], du, off(du, ae(z)))
        # ups near the limit, gates 1/4
        w13 = torch.cat((half.expand(inter, -1), factors.expand(inter, -1))).contiguous()
        _, saved = D.gated_feed_forward_save(x, w13, w2, activation=kind, clamp_limit=limit)
        gx = D.gated_feed_forward_backward(dy, saved)[0]
        du = torch.where(z.abs() <= lim, 32 * a(c), torch.zeros_like(z))
        dg = 32 * z.clamp(-lim, lim) * s(c)
        assert_each(f"{kind} du", gx[:, 0], du, torch.where(z.abs() <= lim, off(du, ae(c)), torch.zeros_like(z)))
        assert_each(f"{kind} dg", gx[:, 1], dg, off(dg, 1.15 * z.abs() / 32767 + se(c) * z.abs()))


@pytest.mark.parametrize("beside", [0.0, 1.0, -1.0, 2.0 ** -101, 2.0 ** 40])
@pytest.mark.parametrize("e", [45, 52, 55, 61, 62])
def test_relu_keeps_the_sign_of_tiny_values(e, beside):
    """2^-90 to 2^-124, alone in their group or beside another value: relu's
    slope is 1 above zero and 0 below it."""
    import dsv4_b200 as D
    m, n, k = 4, 64, 16
    x = torch.zeros(m, k, device="cuda", dtype=BF16)
    x[:, 0] = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda") * 2.0 ** -e
    x[:, 1] = 1
    w = torch.zeros(n, k, device="cuda", dtype=BF16)
    w[:, 0] = 2.0 ** -e
    w[n // 2:, 0] *= -1
    w[5, 0], w[n - 1, 0] = 0, 0
    w[7, 1], w[n - 3, 1] = beside, beside
    z = x.double() @ w.double().T
    dy = torch.full((m, n), 0.5, device="cuda", dtype=BF16)
    bias = torch.zeros(n, device="cuda", dtype=BF16)
    y, saved = D.dense_forward_save(x, w, bias, activation="relu")
    dz = 0.5 * (z > 0).double()
    _, gw, gb = D.dense_backward(dy, saved)
    want = dz.T @ x.double()
    assert_each("grad_weight", gw, want, 2.0 ** -8 * want.abs())
    assert_each("grad_bias", gb, dz.sum(0), torch.zeros(n, device="cuda", dtype=torch.float64))
    # as the gate of a block, ups 1
    one = torch.zeros(n, k, device="cuda", dtype=BF16)
    one[:, 1] = 1
    w2 = torch.full((8, n), 0.125, device="cuda", dtype=BF16)
    _, saved = D.gated_feed_forward_save(x, torch.cat((w, one)), w2, activation="relu")
    _, g13, _ = D.gated_feed_forward_backward(torch.full((m, 8), 0.5, device="cuda", dtype=BF16), saved)
    assert_each("grad_w1", g13[:n], want, 2.0 ** -8 * want.abs())

"""Values before an activation as the backward pass reads them: their side of
the clamp limit and of zero, and how exact they are beside much larger ones."""

import math

import pytest
import torch

import feed_forward_ref as R
from feed_forward_strict import assert_each
from test_gpu_feed_forward import BF16, F16, rand

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


def spread(t, dtype, at, x):
    """Columns `at`, at + 16 and at + 32 of x: numbers as the products with `factors` give them exactly."""
    for i, p in enumerate(parts(t, dtype)):
        x[:, at + 16 * i] = p


def factors(dtype, at, hidden=64):
    f = torch.zeros(hidden, device="cuda", dtype=dtype)
    f[at], f[at + 16], f[at + 32] = 1, 2.0 ** -8, 2.0 ** -16
    return f


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_limit_below_a_larger_value(dtype):
    """Sums up to three fp32 steps from the limit in a group with a larger
    value, which is chosen so that the limit lies where one code ends and the
    next begins, at the ends of their powers of two among them."""
    import dsv4_b200 as D
    digits, steps = (9, 16894) if dtype == BF16 else (10, 17406)
    g = torch.Generator().manual_seed(7)
    w2 = torch.full((8, 32), 0.125, device="cuda", dtype=dtype)
    for limit in (1.3, 0.37, 7.0, *(0.5 + 9.5 * torch.rand(40, generator=g)).tolist()):
        lim = torch.tensor(limit, dtype=torch.float32)
        near = [lim]
        for way in (math.inf, -math.inf):
            t = lim
            for _ in range(3):
                t = torch.nextafter(t, torch.tensor(way))
                near.append(t)
        # the limit in steps of the largest value: borders of codes, and powers of two cut half a step below
        at = [2.0 ** e / (1 + 2.0 ** -(digits + 1)) for e in range(3, digits + 1)]
        at += [2.0 ** e * (1 + (0.5 + i) / 2 ** digits) for e in (3, 6, digits - 1) for i in (-1, 0, 1, 77)]
        at += [2.0 ** digits + 0.5, 2.0 ** digits - 0.5, 3000.5, 9000.0, 12345.5]
        big = torch.tensor([steps * float(lim) / a for a in at], dtype=torch.float64).float()
        big = torch.cat([torch.nextafter(big, torch.zeros_like(big)), big, torch.nextafter(big, big * 2)])
        t = torch.stack(near).repeat(big.numel()).cuda()
        big = big.repeat_interleave(len(near)).cuda()
        x = torch.zeros(t.numel(), 64, device="cuda", dtype=dtype)
        spread(t, dtype, 0, x), spread(big, dtype, 4, x)
        x[:, 1] = 0.25
        one = torch.zeros(64, device="cuda", dtype=dtype)
        one[1] = 1
        row = factors(dtype, 0).expand(32, -1).clone()
        row[9] = factors(dtype, 4)
        dy = torch.ones(t.numel(), 8, device="cuda", dtype=dtype)
        inside = t <= lim.cuda()
        for gate in (True, False):
            w13 = torch.cat((row, one.expand(32, -1)) if gate else (one.expand(32, -1), row))
            _, saved = D.gated_feed_forward_save(x, w13, w2, activation=None, clamp_limit=limit)
            got = D.gated_feed_forward_backward(dy, saved)[0][:, 0].double()
            want = torch.where(inside, 31 * 0.25, 0.0).double()  # dz = 1/4 (the constant is not its group's limit)
            assert_each(f"{limit} {gate}", got, want, 3 * bits16(dtype) * want)


def read_back(g, u, dtype, limit=None):
    """Gate and up values (exact 16-bit numbers), kept in 16-bit groups and read again by the gate's backward
    pass: without an activation and with dh = 1 it writes them as the gradients of up and gate."""
    from dsv4_b200 import _native as N
    m, inter = g.shape
    dt, st = (2 if dtype == BF16 else 1), torch.cuda.current_stream().cuda_stream
    k = -(-m // 8) * 8
    x = torch.eye(m, k, device="cuda", dtype=dtype)  # row i picks column i of w13
    w13 = torch.zeros(2 * inter, k, device="cuda", dtype=dtype)
    w13[:inter, :m], w13[inter:, :m] = g.T, u.T
    n32 = -(-inter // 32) * 32
    ld = -(-inter // 8) * 8
    h = torch.empty(m, ld, device="cuda", dtype=dtype)
    codes = torch.empty(m, 2 * n32, device="cuda", dtype=torch.int16)
    scales = torch.empty(2 * n32 // 32, m, device="cuda")
    clamp = (0, 0.0) if limit is None else (1, limit)
    N.call("dsv4_b200_gated_gemm", x.data_ptr(), k, 0, w13.data_ptr(), k, 0, m, inter, k, dt, 0, *clamp, h.data_ptr(), ld,
           codes.data_ptr(), 16, scales.data_ptr(), st)
    dy = torch.zeros(m, 8, device="cuda", dtype=dtype)
    dy[:, 0] = 1
    w2 = torch.zeros(inter, 8, device="cuda", dtype=dtype)  # by rows: dh = 1
    w2[:, 0] = 1
    dz = torch.empty(m, 2 * ld, device="cuda", dtype=dtype)
    N.call("dsv4_b200_gated_backward_gemm", dy.data_ptr(), 8, 0, w2.data_ptr(), 8, 0, m, inter, 8, dt, 0, *clamp,
           codes.data_ptr(), 16, scales.data_ptr(), dz.data_ptr(), 2 * ld, None, 0, st)
    return dz[:, inter:2 * inter], dz[:, :inter]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("inter", [32, 64, 1, 3, 8, 33, 40, 61, 200])
def test_every_value_beside_larger_ones(inter, dtype):
    """0 to 31 large values in a group, 2^4 to 2^28 (fp16: 2^13) times the
    others: each value as exact as storing it in 16 bits, and the whole group
    within half a 32767th of its largest."""
    m = 192
    base = rand(m, inter, dtype=dtype, seed=inter).double()
    order = torch.rand(m, inter, device="cuda", generator=torch.Generator("cuda").manual_seed(inter)).argsort(1)
    row = torch.arange(m, device="cuda")[:, None]
    big = torch.tensor([0, 1, 2, 3, 4, 6, 7, 8, 12, 16, 24, 28, 30, 31], device="cuda")
    # within each group of 32 the first `count` of a random order
    group = torch.arange(inter, device="cuda")[None] // 32
    rank = ((order[:, :, None] > order[:, None, :]) & (group[:, :, None] == group[:, None, :])).sum(2)
    large = rank < big[row % big.numel()]
    top = 28 if dtype == BF16 else 13
    by = 2.0 ** (4 + (row // big.numel()) * (top - 4) // (m // big.numel()))
    g = torch.where(large, by * base, base).to(dtype)
    u = torch.where(large, by * base.flip(0), base.flip(0)).to(dtype)
    for v, got in zip((g, u), read_back(g, u, dtype)):
        v = v.double()
        pad = torch.nn.functional.pad(v.abs(), (0, -inter % 32)).reshape(m, -1, 32)
        amax = pad.amax(2, keepdim=True).expand_as(pad).reshape(m, -1)[:, :inter]
        h16 = bits16(dtype)
        kept = torch.minimum(1.01 * h16 * v.abs() + (2.0 ** -40 if dtype == BF16 else 2.0 ** -29) * amax, amax / 32767)
        assert_each("kept", got, v, kept + h16 * (v.abs() + kept) + R.tiny_of(dtype))


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("count,n", [(2, 96), (4, 96), (8, 96), (16, 96), (31, 96), (1, 40), (2, 40), (1, 33)])
def test_gradients_beside_large_channels(kind, dtype, count, n):
    """`count` channels of each group (of a ragged last one too) at 4000: the
    gradients of the others are those of values stored in 16 bits."""
    import dsv4_b200 as D
    m, k = 3, 64
    x, w = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, std=1.0 / 8, seed=2)
    b = rand(n, dtype=dtype, std=0.3, seed=3)
    for first in range(0, n, 32):
        b[first:min(first + count, n)] = 4000
    dy = rand(m, n, dtype=dtype, std=0.1, seed=4)
    h16, tiny = bits16(dtype), R.tiny_of(dtype)
    X, W = R.Bounded(x.double()), R.Bounded(w.double())
    z = R.product(X, W)
    z = R.Bounded(z.v + b.double(), z.e + 2.0 ** -23 * (z.v.abs() + b.double().abs()))
    z = R.Bounded(z.v, z.e + h16 * z.v.abs() + 2.0 ** -29 * 4010)
    slope = R.slope_bounded(kind, z)
    far = z.v > 3000  # their slope is 1, whatever their last bits
    slope = R.Bounded(slope.v, torch.where(far, torch.full_like(slope.e, 2.0 ** -20), slope.e))
    exact = R.times(R.Bounded(dy.double()), slope)
    dz = R.rounded(exact, h16, tiny)
    want = {"grad_x": R.rounded(R.product(dz, R.Bounded(W.v.T)), h16, tiny),
            "grad_weight": R.rounded(R.product(R.Bounded(dz.v.T, dz.e.T), R.Bounded(X.v.T)), h16, tiny),
            "grad_bias": R.rounded(R.Bounded(exact.v.sum(0), exact.e.sum(0) + (m + 8) * 2.0 ** -23 * exact.v.abs().sum(0)),
                                   h16, tiny)}
    _, saved = D.dense_forward_save(x, w, b, activation=kind)
    for got, key in zip(D.dense_backward(dy, saved), ("grad_x", "grad_weight", "grad_bias")):
        assert_each(key, got, want[key].v, want[key].e)


def decoded(codes, scales, dtype):
    """Values of 16-bit groups, as the C header writes them down."""
    edge, digits = (512, 9) if dtype == BF16 else (1024, 10)
    c = codes.long() & 0x7fff
    e, f = c >> digits, c & (edge - 1)
    bias = 32 if dtype == BF16 else 16
    fine = torch.where(e > 0, edge * torch.exp2(e.double() - bias) * (1 + f / edge), edge * 2.0 ** (1 - bias) * f / edge)
    t = torch.where(c >= 16384, (c - 16384 + edge).double(), fine)
    scale = scales.double().T.repeat_interleave(32, 1)
    half = (codes.view(torch.float16).double() * -scale) if bool((scale < 0).any()) else t
    return torch.where(scale < 0, half, torch.where(codes < 0, -t, t) * scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_documented_format(dtype):
    """Codes and scales of a product against the values they stand for, in
    groups of all sizes, with an infinity and a NaN in some."""
    from dsv4_b200 import _native as N
    m, n, k = 100, 72, 104
    v = rand(m, n, dtype=dtype, seed=5) * torch.exp2(rand(m, n, dtype=dtype, std=3, seed=6).round())
    v = v.to(dtype)
    v[3, 4], v[5, 40], v[6, 71], v[7] = math.inf, math.nan, -math.inf, 0
    w = torch.zeros(n, k, device="cuda", dtype=dtype)
    x = torch.zeros(m, k, device="cuda", dtype=dtype)
    x[:, :m] = torch.eye(m, device="cuda", dtype=dtype)
    finite = torch.isfinite(v)
    w[:, :m] = torch.where(finite, v, torch.zeros_like(v)).T
    bias = torch.zeros(n, device="cuda", dtype=dtype)
    out = torch.empty(m, n, device="cuda", dtype=dtype)
    n32 = 96
    codes, scales = torch.empty(m, n32, device="cuda", dtype=torch.int16), torch.empty(3, m, device="cuda")
    dt, st = (2 if dtype == BF16 else 1), torch.cuda.current_stream().cuda_stream

    def run():
        N.call("dsv4_b200_dense_gemm", x.data_ptr(), k, 0, w.data_ptr(), k, 0, m, n, k, dt, bias.data_ptr(), 0, None, 0,
               out.data_ptr(), n, codes.data_ptr(), 16, scales.data_ptr(), st)
        return decoded(codes, scales, dtype)[:, :n]

    z = w[:, :m].T.double()
    amax = torch.nn.functional.pad(z.abs(), (0, n32 - n)).reshape(m, 3, 32).amax(2).repeat_interleave(32, 1)[:, :n]
    h16, floor = (2.0 ** -10, 2.0 ** -45) if dtype == BF16 else (2.0 ** -11, 2.0 ** -29)
    bound = torch.minimum(h16 * z.abs(), 2.0 ** -15 * amax) * 1.01 + floor * amax
    assert_each("finite", run(), z, bound)
    assert bool((scales > 0).all())
    for column, value in ((4, math.inf), (40, math.nan), (71, -math.inf)):
        bias[column] = value  # their groups: everything but the column to 2^-11
        z[:, column] = value
    bound = torch.where(torch.isfinite(z), 2.0 ** -11 * z.abs() + 2.0 ** -38 * amax, torch.zeros_like(z))
    assert_each("with infinities", run(), z, bound)
    assert bool((scales < 0).all())

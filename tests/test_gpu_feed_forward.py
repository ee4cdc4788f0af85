"""The 16-bit feed-forward operators against their formulas in 64 bits
(``feed_forward_ref``: every element within a bound derived from the formats)."""

import math

import pytest
import torch

import feed_forward_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rand(*shape, dtype=BF16, std=1.0, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def dense_case(m, k, n, dtype, bias=True, residual=True, seed=1):
    return (rand(m, k, dtype=dtype, seed=seed), rand(n, k, dtype=dtype, std=k ** -0.5, seed=seed + 1),
            rand(n, dtype=dtype, std=0.3, seed=seed + 2) if bias else None,
            rand(m, n, dtype=dtype, seed=seed + 3) if residual else None)


def ffn_case(m, hidden, inter, out, dtype, residual=True, seed=1, std=1.0):
    return (rand(m, hidden, dtype=dtype, std=std, seed=seed),
            rand(2 * inter, hidden, dtype=dtype, std=hidden ** -0.5, seed=seed + 1),
            rand(out, inter, dtype=dtype, std=inter ** -0.5, seed=seed + 2),
            rand(m, out, dtype=dtype, seed=seed + 3) if residual else None)


# one token to a few row tiles; sizes at, next to and off the tiles' multiples
DENSE = [
    (1, 64, 64), (1, 7168, 256), (2, 72, 40), (7, 1000, 333), (16, 512, 1024), (17, 136, 129),
    (33, 1024, 31), (63, 264, 65), (64, 2048, 512), (65, 8, 7), (100, 1, 1), (127, 321, 255),
    (128, 256, 257), (129, 1024, 96), (255, 640, 224), (256, 256, 256), (257, 1032, 264), (513, 192, 1000),
    (1000, 333, 1777),
]


@pytest.mark.parametrize("m,k,n", DENSE)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_dense_forward(m, k, n, dtype):
    import dsv4_b200 as D
    kind = R.ACTS[(m + n) % len(R.ACTS)]
    x, w, b, r = dense_case(m, k, n, dtype, bias=n % 2 == 0 or m % 3 == 0, residual=m % 2 == 1 or n % 3 == 0)
    y = D.dense_forward(x, w, b, activation=kind, residual=r)
    R.assert_within("y", y, R.dense(x, w, b, r, kind, dtype)["y"])


@pytest.mark.parametrize("kind", R.ACTS)
@pytest.mark.parametrize("mode", [None, "int8"])
@pytest.mark.parametrize("m,k,n,dtype", [(5, 40, 24, F16), (70, 257, 129, BF16), (300, 512, 333, F16),
                                         (1, 1024, 512, BF16), (1030, 264, 72, BF16)])
def test_dense_gradients(kind, mode, m, k, n, dtype):
    import dsv4_b200 as D
    x, w, b, r = dense_case(m, k, n, dtype)
    dy = rand(m, n, dtype=dtype, std=0.1, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = D.dense_forward(x, w, b, activation=kind, residual=r, checkpoint=mode)
    grads = torch.autograd.grad(y, leaves, dy)
    want = R.dense(x.detach(), w.detach(), b.detach(), r.detach(), kind, dtype, dy, mode)
    R.assert_within("y", y.detach(), want["y"])
    for name, got in zip(("grad_x", "grad_weight", "grad_bias"), grads):
        R.assert_within(name, got, want[name])
    assert torch.equal(grads[3], dy)


@pytest.mark.parametrize("k", [1, 7, 8, 9, 31, 63, 64, 65, 127, 1001, 2050])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_tokens_at_any_alignment(k, dtype):
    """1 to 9 tokens, rows that begin at every even address of 16 bytes, the
    matrices inside buffers of NaN: nothing beside them is read into a sum."""
    import dsv4_b200 as D

    def inside(t, lead, gap):
        rows, cols = t.shape
        buf = torch.full((lead + rows * (cols + gap) + 8,), math.nan, dtype=dtype, device="cuda")
        view = buf[lead:lead + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
        view.copy_(t)
        return view

    for i, (m, n) in enumerate([(1, 1), (1, 40), (2, 17), (3, 8), (5, 33), (8, 16), (8, 100), (9, 24)]):
        x, w, b, r = dense_case(m, k, n, dtype, seed=k + i)
        want = R.dense(x, w, b, r, "silu", dtype)["y"]
        for lead in range(8):
            xv, wv = inside(x, lead, (i + lead) % 5), inside(w, (3 * lead + i) % 8, lead % 3)
            R.assert_within(f"y {m} {n} {lead}", D.dense_forward(xv, wv, b, activation="silu", residual=r), want)
        x, w13, w2, r = ffn_case(m, k, n, 24, dtype, seed=k + i)
        want = R.ffn(x, w13, w2, r, "gelu", 1.5, dtype)["y"]
        for lead in range(0, 8, 3):
            args = inside(x, lead, 1), inside(w13, lead + 1, lead), inside(w2, 7 - lead, 1)
            y = D.gated_feed_forward(*args, activation="gelu", clamp_limit=1.5, residual=r)
            R.assert_within(f"block {m} {n} {lead}", y, want)


def test_few_tokens_at_the_ends_of_a_buffer():
    """Matrices that begin and end with their buffers, of one and of few values."""
    import dsv4_b200 as D
    for m, k, n in ((1, 1, 1), (1, 3, 1), (2, 5, 3), (1, 17, 2), (8, 23, 5)):
        x, w, _, _ = dense_case(m, k, n, BF16, False, False)
        for cut in range(4):
            xb, wb = torch.empty(m * k + cut, device="cuda", dtype=BF16), torch.empty(n * k + cut, device="cuda", dtype=BF16)
            xv, wv = xb[cut:].view(m, k), wb[cut:].view(n, k)
            xv.copy_(x), wv.copy_(w)
            R.assert_within("y", D.dense_forward(xv, wv), R.dense(x, w, None, None, None, BF16)["y"])


FFN = [
    (1, 64, 32, 64), (1, 1024, 512, 1024), (3, 72, 17, 40), (16, 256, 128, 256), (31, 1000, 77, 1000),
    (64, 512, 509, 512), (65, 136, 64, 129), (128, 1024, 512, 1024), (130, 264, 100, 264),
    (257, 512, 256, 512), (600, 200, 333, 201),
]


@pytest.mark.parametrize("m,hidden,inter,out", FFN)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_feed_forward(m, hidden, inter, out, dtype):
    import dsv4_b200 as D
    kind = R.ACTS[(m + inter) % len(R.ACTS)]
    limit = (None, 1.5, 7.0)[m % 3]
    x, w13, w2, r = ffn_case(m, hidden, inter, out, dtype, residual=inter % 2 == 0)
    y = D.gated_feed_forward(x, w13, w2, activation=kind, clamp_limit=limit, residual=r)
    R.assert_within("y", y, R.ffn(x, w13, w2, r, kind, limit, dtype)["y"])


@pytest.mark.parametrize("mode", [None, "int8"])
@pytest.mark.parametrize("kind,limit", [("silu", None), ("silu", 0.75), ("gelu", 1.0), ("gelu_tanh", None),
                                        ("relu", None), (None, 1.5)])
@pytest.mark.parametrize("m,hidden,inter,out,dtype", [(4, 40, 24, 48, F16), (70, 257, 65, 129, BF16),
                                                      (300, 512, 160, 512, BF16), (1, 512, 256, 512, BF16),
                                                      (520, 136, 100, 72, F16)])
def test_gated_feed_forward_gradients(mode, kind, limit, m, hidden, inter, out, dtype):
    import dsv4_b200 as D
    x, w13, w2, r = ffn_case(m, hidden, inter, out, dtype)
    dy = rand(m, out, dtype=dtype, std=0.1, seed=9)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2, r)]
    y = D.gated_feed_forward(x, w13, w2, activation=kind, clamp_limit=limit, residual=r, checkpoint=mode)
    grads = torch.autograd.grad(y, leaves, dy)
    want = R.ffn(x.detach(), w13.detach(), w2.detach(), r.detach(), kind, limit, dtype, dy, mode)
    R.assert_within("y", y.detach(), want["y"])
    for name, got in zip(("grad_x", "grad_w13", "grad_w2"), grads):
        R.assert_within(name, got, want[name])
    assert torch.equal(grads[3], dy)


@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (16, 1024), (33, 31), (31, 257), (100, 1000), (5, 8193),
                                 (8192, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
def test_checkpoint_round_trip(m, k, dtype):
    import dsv4_b200 as D
    x = rand(m, k, dtype=dtype, seed=k) * rand(1, k, dtype=dtype, seed=k + 1).exp()
    c = D.checkpoint_int8(x)
    back, step, _ = R.eight(x.double())
    # the codes are those of the exact quotient, ties to even
    k32 = -(-k // 32) * 32
    top = torch.nn.functional.pad(x.double(), (0, k32 - k)).reshape(m, -1, 32).abs().amax(2, keepdim=True)
    q = 127 * torch.nn.functional.pad(x.double(), (0, k32 - k)).reshape(m, -1, 32) / torch.where(
        top > 0, top, torch.ones_like(top))
    assert torch.equal(c.codes.double(), torch.round(q).reshape(m, k32))
    step64 = top[:, :, 0] / 127
    step32 = step64.float()  # rounded toward zero: 127 steps never pass the largest value
    step32 = torch.where(step32.double() > step64, torch.nextafter(step32, torch.zeros_like(step32)), step32)
    assert bool((c.scales == step32.T).all())
    got = D.restore_int8(c)
    h = torch.finfo(dtype).eps / 2
    R.assert_within("restored", got, R.Bounded(back, back.abs() * (h + 2.0 ** -22) + R.tiny_of(dtype)))
    assert got.dtype == dtype


def test_checkpoint_ties_and_extremes():
    """Halves of the largest value are exact ties (63.5): they go to even.
    Infinities and NaN spoil their group only; tiny groups are zeros; the
    largest finite values survive."""
    import dsv4_b200 as D
    for dtype in (BF16, F16, torch.float32):
        x = torch.zeros(8, 96, device="cuda", dtype=dtype)
        for i, top in enumerate((1.0, 1.0078125, 1.3125, 1.9921875, 3.328125, 250.0, 0.4375)):
            x[i, 0] = top
            x[i, 1:16] = top / 2
            x[i, 16:31] = -top / 2
        x[7, 0], x[7, 32], x[7, 70] = math.inf, math.nan, torch.finfo(dtype).max
        x[7, 71] = -torch.finfo(dtype).max / 2
        c = D.checkpoint_int8(x)
        assert (c.codes[:7, 1:16] == 64).all() and (c.codes[:7, 16:31] == -64).all()
        got = D.restore_int8(c)
        assert torch.isnan(got[7, :64]).all() and torch.isfinite(got[7, 64:]).all()
        assert got[7, 70] >= torch.finfo(dtype).max * (1 - torch.finfo(dtype).eps)
        assert c.codes[7, 71] == -64
    x = torch.full((1, 64), 2.0 ** -101, device="cuda")
    x[0, 40] = 2.0 ** -100
    c = D.checkpoint_int8(x)
    assert (c.codes[0, :32] == 0).all() and c.codes[0, 40] == 127 and c.codes[0, 41] == 64
    assert (D.restore_int8(c)[0, :32] == 0).all()


def test_checkpoint_near_ties_in_fp32():
    """fp32 values one step to each side of every half code: the code of the
    exact quotient, where a quotient rounded in fp32 would be a tie."""
    import dsv4_b200 as D
    top = torch.tensor([1.0, 1.7320508, 3.0000002, 0.1], device="cuda")
    half = (torch.arange(127, device="cuda").double() + 0.5)[None, :] * top.double()[:, None] / 127
    mid = half.float()
    rows = []
    for t, v in zip(top, mid):
        for near in (v, torch.nextafter(v, torch.full_like(v, 9e9)), torch.nextafter(v, torch.zeros_like(v))):
            for part in near.split(31):
                row = torch.zeros(32, device="cuda")
                row[0] = t
                row[1:1 + part.numel()] = part
                rows.append(row)
    x = torch.stack(rows)
    q = 127 * x.double() / x.double().abs().amax(1, keepdim=True)
    assert torch.equal(D.checkpoint_int8(x).codes.double(), torch.round(q))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_checkpoint_codes_of_every_pair(dtype):
    """The code of every value below every largest value of one binade (all
    16-bit significands): exactly the rounded exact quotient, ties to even."""
    import dsv4_b200 as D
    bits = 7 if dtype == BF16 else 10
    top = (1 + torch.arange(2 ** bits, device="cuda").double() / 2 ** bits)
    for scale in (1.0, 2.0 ** -6, 2.0 ** 9):
        part = torch.cat([top * 2.0 ** -e for e in range(1, 8)]) if bits == 7 else \
            torch.cat([top * 2.0 ** -e for e in (1, 2, 3)])
        sign = torch.where(torch.arange(part.numel(), device="cuda") % 2 == 0, 1.0, -1.0)
        cols = -(-part.numel() // 31) * 31
        part = torch.nn.functional.pad(part * sign, (0, cols - part.numel())).reshape(-1, 31)
        x = torch.cat((top[:, None, None].expand(-1, part.shape[0], 1),
                       part[None].expand(top.numel(), -1, -1)), 2).reshape(top.numel(), -1) * scale
        assert torch.equal(x.to(dtype).double(), x)
        g = x.reshape(x.shape[0], -1, 32)
        want = torch.round(127 * g / g.abs().amax(2, keepdim=True)).reshape(x.shape)
        assert torch.equal(D.checkpoint_int8(x.to(dtype)).codes.double(), want)

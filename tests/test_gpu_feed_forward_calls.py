"""How the 16-bit feed-forward operators may be called: strides, alignment,
broadcast rows, empty batches, values that are not finite, streams, CUDA
graphs, autograd's corners, the C entry points' refusals, and a run of them
together with the routed experts."""

import math

import pytest
import torch

import feed_forward_ref as R
from test_gpu_feed_forward import BF16, F16, dense_case, ffn_case, rand

pytestmark = pytest.mark.gpu


def bits(t):
    return t.view(torch.int16)


def same(a, b):
    return torch.equal(bits(a.contiguous()), bits(b.contiguous()))


# ---- layouts ----

def layouts(t):
    """The same values with other strides and alignments."""
    rows, cols = t.shape
    wide = torch.full((rows, cols + 11), math.nan, dtype=t.dtype, device=t.device)
    wide[:, 3:3 + cols] = t
    flat = torch.full((rows * cols + 1,), math.nan, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    apart = torch.full((rows, 2 * cols), math.nan, dtype=t.dtype, device=t.device)
    apart[:, ::2] = t
    padded = torch.full((rows, -(-cols // 8) * 8 + 8), math.nan, dtype=t.dtype, device=t.device)
    padded[:, :cols] = t
    return {"odd rows": wide[:, 3:3 + cols], "odd address": flat[1:].view(rows, cols),
            "columns apart": apart[:, ::2], "by columns": t.t().contiguous().t(),
            "padded rows": padded[:, :cols]}


@pytest.mark.parametrize("m,k,n", [(5, 136, 72), (40, 100, 50), (300, 264, 136)])
def test_layouts_give_the_same_bits(m, k, n):
    """x, weight and residual of any strides: the results of contiguous ones.
    (The one product that takes tokens by columns sums in the same order.)"""
    import dsv4_b200 as D
    x, w, b, r = dense_case(m, k, n, BF16)
    want = R.dense(x, w, b, r, "gelu", BF16)["y"]
    base = D.dense_forward(x, w, b, activation="gelu", residual=r)
    for name, xv in layouts(x).items():
        y = D.dense_forward(xv, w, b, activation="gelu", residual=r)
        R.assert_within("x " + name, y, want)
    for name, wv in layouts(w).items():
        R.assert_within("weight " + name, D.dense_forward(x, wv, b, activation="gelu", residual=r), want)
    for name, rv in layouts(r).items():
        assert same(base, D.dense_forward(x, w, b, activation="gelu", residual=rv)), name
    apart = torch.empty(2 * n, device="cuda", dtype=BF16)[::2].copy_(b)
    assert same(base, D.dense_forward(x, w, apart, activation="gelu", residual=r))


@pytest.mark.parametrize("mode", [None, "int8"])
@pytest.mark.parametrize("inter", [40, 33])
def test_gradients_of_any_layout(mode, inter):
    import dsv4_b200 as D
    m, hidden, out = 70, 72, 56
    x, w13, w2, _ = ffn_case(m, hidden, inter, out, F16, residual=False)
    dy = rand(m, out, dtype=F16, std=0.1, seed=5)
    want = R.ffn(x, w13, w2, None, "silu", 1.5, F16, dy, mode)
    for name in layouts(x):
        args = [layouts(t)[name] for t in (x, w13, w2)]
        y, saved = D.gated_feed_forward_save(*args, clamp_limit=1.5, checkpoint=mode)
        R.assert_within(name, y, want["y"])
        for g, key in zip(D.gated_feed_forward_backward(layouts(dy)[name], saved), ("grad_x", "grad_w13", "grad_w2")):
            R.assert_within(name + " " + key, g, want[key])
    dz = rand(m, 2 * inter, dtype=F16, seed=6)
    wantd = R.dense(x, w13, None, None, "silu", F16, dz, mode)
    for name in layouts(x):
        y, saved = D.dense_forward_save(layouts(x)[name], layouts(w13)[name], activation="silu", checkpoint=mode)
        gx, gw, gb = D.dense_backward(layouts(dz)[name], saved)
        R.assert_within(name, gx, wantd["grad_x"])
        R.assert_within(name, gw, wantd["grad_weight"])
        assert gb is None


def test_broadcast_rows():
    """Expanded tensors: rows that are one row in memory, forward and backward
    (a gradient of a sum is one too)."""
    import dsv4_b200 as D
    m, k, n = 37, 64, 48
    x, w, b, r = dense_case(m, k, n, BF16)
    one, rrow = x[:1].clone().requires_grad_(True), r[:1].clone().requires_grad_(True)
    bias = b.clone().requires_grad_(True)
    y = D.dense_forward(one.expand(m, k), w, bias, activation="silu", residual=rrow.expand(m, n))
    want = R.dense(x[:1].expand(m, k), w, b, r[:1].expand(m, n), "silu", BF16, torch.ones(m, n, device="cuda", dtype=BF16))
    R.assert_within("y", y.detach(), want["y"])
    y.sum().backward()  # dy is one number, expanded
    h16 = torch.finfo(BF16).eps / 2
    gx = want["grad_x"]
    total = R.Bounded(gx.v.sum(0, keepdim=True), gx.e.sum(0, keepdim=True) + h16 * gx.v.sum(0, keepdim=True).abs()
                      + m * 2.0 ** -23 * gx.v.abs().sum(0, keepdim=True))
    R.assert_within("grad x", one.grad, total)
    R.assert_within("grad bias", bias.grad, want["grad_bias"])
    assert (rrow.grad == m).all()
    for ck in (None, "int8"):
        y, saved = D.dense_forward_save(x[:1].expand(m, k), w, activation="relu", checkpoint=ck)
        D.dense_backward(torch.ones(1, 1, device="cuda", dtype=BF16).expand(m, n), saved)


@pytest.mark.parametrize("mode", [None, "int8"])
def test_empty_batch(mode):
    import dsv4_b200 as D
    x, w, b, r = dense_case(0, 40, 24, BF16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = D.dense_forward(x, w, b, activation="gelu", residual=r, checkpoint=mode)
    assert y.shape == (0, 24)
    grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert grads[0].shape == x.shape and all((g == 0).all() for g in grads)
    x, w13, w2, r = ffn_case(0, 40, 16, 24, BF16)
    leaves = [t.requires_grad_(True) for t in (x, w13, w2)]
    y = D.gated_feed_forward(x, w13, w2, residual=r, checkpoint=mode)
    grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert y.shape == (0, 24) and [g.shape for g in grads] == [t.shape for t in leaves]
    assert all((g == 0).all() for g in grads)
    c = D.checkpoint_int8(torch.empty(0, 40, device="cuda"))
    assert D.restore_int8(c).shape == (0, 40)


@pytest.mark.parametrize("m", [3, 200])
def test_results_stay_inside_their_rows(m):
    """Behind the last row and column nothing is written: the C entry points
    with results inside larger buffers."""
    from dsv4_b200 import _native as N
    k, n = 72, 45
    x, w, _, _ = dense_case(m, k, n, BF16, False, False)
    big = torch.full((m + 4, n + 19), 7.0, device="cuda", dtype=BF16)
    st = torch.cuda.current_stream().cuda_stream
    N.call("dsv4_b200_dense_gemm", x.data_ptr(), k, 0, w.data_ptr(), k, 0, m, n, k, N.DTYPE_BF16, None, 0,
           None, 0, big.data_ptr(), n + 19, None, 0, None, st)
    R.assert_within("y", big[:m, :n], R.dense(x, w, None, None, None, BF16)["y"])
    assert (big[m:] == 7).all() and (big[:, n:] == 7).all()
    codes = torch.full((m + 1, 96), 9, device="cuda", dtype=torch.int8)
    scales = torch.full((3 * m + 5,), 9.0, device="cuda")
    N.call("dsv4_b200_checkpoint_int8", x.data_ptr(), N.DTYPE_BF16, m, k, k, codes.data_ptr(), scales.data_ptr(), st)
    assert (codes[m:] == 9).all() and (scales[3 * m:] == 9).all() and (codes[:m, k:] == 0).all()
    N.call("dsv4_b200_restore_int8", codes.data_ptr(), scales.data_ptr(), m, 37, big.data_ptr(), N.DTYPE_BF16, n + 19, st)
    assert (big[m:] == 7).all() and (big[:, n:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
def test_checkpoints_at_any_alignment(dtype):
    """Rows that begin at every element of 16 bytes, inside a buffer: the codes
    and values of aligned rows, and nothing beside them read or written."""
    import dsv4_b200 as D
    from dsv4_b200 import _native as N
    st = torch.cuda.current_stream().cuda_stream
    dt = {BF16: N.DTYPE_BF16, F16: N.DTYPE_F16, torch.float32: N.DTYPE_F32}[dtype]
    m = 37
    for k in (1, 5, 7, 8, 9, 31, 250, 255, 256, 257, 263, 264, 520, 1001):
        x = rand(m, k, dtype=dtype, seed=k)
        want = D.checkpoint_int8(x)
        back = D.restore_int8(want)
        for lead in range(8):
            ld = k + (lead + k) % 3
            buf = torch.full((lead + m * ld + 9,), math.nan, dtype=dtype, device="cuda")
            view = buf[lead:lead + m * ld].view(m, ld)[:, :k]
            view.copy_(x)
            got = D.checkpoint_int8(view)
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales), (k, lead)
            buf.fill_(7)
            N.call("dsv4_b200_restore_int8", got.codes.data_ptr(), got.scales.data_ptr(), m, k, view.data_ptr(), dt,
                   ld, st)
            assert torch.equal(view, back), (k, lead)
            view.fill_(7)
            assert (buf == 7).all(), (k, lead)


# ---- values ----

@pytest.mark.parametrize("m", [4, 300])
def test_not_finite_values_stay_in_their_rows(m):
    import dsv4_b200 as D
    k, n = 96, 80
    x, w, b, r = dense_case(m, k, n, BF16)
    clean = D.dense_forward(x, w, b, activation="silu", residual=r)
    x2 = x.clone()
    x2[1, 5], x2[2, 7] = math.nan, math.inf
    y = D.dense_forward(x2, w, b, activation="silu", residual=r)
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[1] = keep[2] = False
    assert same(y[keep], clean[keep]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    r2 = r.clone()
    r2[0, 3] = math.inf
    y = D.dense_forward(x, w, b, activation="silu", residual=r2)
    assert y[0, 3] == math.inf and same(y[1:], clean[1:])
    # a weight row that is not finite spoils its column only, at a tile's ragged end too
    w2 = w.clone()
    w2[n - 1, 0] = math.nan
    y = D.dense_forward(x, w2, b, activation="silu", residual=r)
    assert torch.isnan(y[:, n - 1]).all() and same(y[:, :n - 1], clean[:, :n - 1])


@pytest.mark.parametrize("mode", [None, "int8"])
def test_not_finite_gradients(mode):
    """A token that is not finite: its own gradient and the weights' are not,
    the other tokens' gradients are untouched."""
    import dsv4_b200 as D
    x, w13, w2, _ = ffn_case(40, 64, 48, 64, BF16, residual=False)
    dy = rand(40, 64, seed=3)
    y, saved = D.gated_feed_forward_save(x, w13, w2, checkpoint=mode)
    clean = D.gated_feed_forward_backward(dy, saved)
    x2 = x.clone()
    x2[7, 3] = math.nan
    y, saved = D.gated_feed_forward_save(x2, w13, w2, checkpoint=mode)
    gx, g13, g2 = D.gated_feed_forward_backward(dy, saved)
    keep = torch.arange(40, device="cuda") != 7
    assert same(gx[keep], clean[0][keep]) and torch.isnan(gx[7]).all()
    assert torch.isnan(g13).all() and torch.isnan(g2).all()


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_beside_an_outlier(kind, dtype):
    """One column in 32 far above the rest: its neighbours' gradients are as
    exact as elsewhere."""
    import dsv4_b200 as D
    m, k, n = 70, 64, 200
    x, w, b, _ = dense_case(m, k, n, dtype)
    w, b = w / 16, b / 16
    b[5::32] = 4000
    dy = rand(m, n, dtype=dtype, std=0.1, seed=3)
    want = R.dense(x, w, b, None, kind, dtype, dy)
    y, saved = D.dense_forward_save(x, w, b, activation=kind)
    R.assert_within("y", y, want["y"])
    for g, key in zip(D.dense_backward(dy, saved), ("grad_x", "grad_weight", "grad_bias")):
        R.assert_within(key, g, want[key])
    # the block: gates far above in one column of each group (every token), limits inside the others
    x, w13, w2, _ = ffn_case(m, k, 96, 72, dtype, residual=False)
    x[:, 0], w13[5:96:32, 0] = 8, 128
    dy = rand(m, 72, dtype=dtype, std=0.1, seed=4)
    for limit in (None, 0.37):
        want = R.ffn(x, w13, w2, None, kind, limit, dtype, dy)
        y, saved = D.gated_feed_forward_save(x, w13, w2, activation=kind, clamp_limit=limit)
        R.assert_within("y", y, want["y"])
        for g, key in zip(D.gated_feed_forward_backward(dy, saved), ("grad_x", "grad_w13", "grad_w2")):
            R.assert_within(key, g, want[key])


def test_infinities_that_the_formula_masks():
    """A value before the activation that is infinite, with a slope of zero
    there: its neighbours' gradients are those of a large finite value."""
    import dsv4_b200 as D
    m, k, n = 70, 64, 80
    x, w, b, _ = dense_case(m, k, n, BF16)
    dy = rand(m, n, std=0.1, seed=3)
    b[7] = -1000
    want = R.dense(x, w, b, None, "relu", BF16, dy)
    b[7] = -math.inf
    y, saved = D.dense_forward_save(x, w, b, activation="relu")
    R.assert_within("y", y, want["y"])
    for g, key in zip(D.dense_backward(dy, saved), ("grad_x", "grad_weight", "grad_bias")):
        R.assert_within(key, g, want[key])
    # gate and up past the limit by an infinite weight (column 0 of dx is 0 times infinity)
    x, w13, w2, _ = ffn_case(m, k, 48, 72, BF16, residual=False)
    x[:, 0] = 1
    dy = rand(m, 72, std=0.1, seed=4)
    w13[9, 0], w13[48 + 20, 0] = 1000, -1000
    want = R.ffn(x, w13, w2, None, "silu", 1.5, BF16, dy)
    w13[9, 0], w13[48 + 20, 0] = math.inf, -math.inf
    y, saved = D.gated_feed_forward_save(x, w13, w2, clamp_limit=1.5)
    R.assert_within("y", y, want["y"])
    gx, g13, g2 = D.gated_feed_forward_backward(dy, saved)
    R.assert_within("grad_w13", g13, want["grad_w13"])
    R.assert_within("grad_w2", g2, want["grad_w2"])
    assert torch.isnan(gx[:, 0]).all()
    R.assert_within("grad_x", gx[:, 1:], R.Bounded(want["grad_x"].v[:, 1:], want["grad_x"].e[:, 1:]))
    # NaN in one column stays there
    x, w, b, _ = dense_case(m, k, n, BF16)
    dy = rand(m, n, std=0.1, seed=5)
    b[7] = 1000
    want = R.dense(x, w, b, None, "silu", BF16, dy)
    b[7] = math.nan
    y, saved = D.dense_forward_save(x, w, b, activation="silu")
    gx, gw, gb = D.dense_backward(dy, saved)
    keep = torch.arange(n, device="cuda") != 7
    for key in ("grad_weight", "grad_bias"):
        got = {"grad_weight": gw, "grad_bias": gb}[key]
        R.assert_within(key, got[keep], R.Bounded(want[key].v[keep], want[key].e[keep]))
        assert torch.isnan(got[7]).all()
    assert torch.isnan(gx).all()


def test_extreme_activation_arguments():
    """Values far out: no activation or slope makes NaN of a finite number."""
    import dsv4_b200 as D
    v = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 80.0, -80.0, 1e4, -1e4, 1e18, -1e18, 3e38, -3e38], device="cuda")
    x = torch.zeros(12, 16, device="cuda", dtype=BF16)
    x[:, 0] = v.to(BF16)
    w = torch.zeros(8, 16, device="cuda", dtype=BF16)
    w[:, 0] = 1
    dy = torch.ones(12, 8, device="cuda", dtype=BF16)
    for kind in R.ACTS:
        for ck in (None, "int8"):
            y, saved = D.dense_forward_save(x, w, activation=kind, checkpoint=ck)
            gx, gw, _ = D.dense_backward(dy, saved)
            assert torch.isfinite(y).all() and torch.isfinite(gx).all(), (kind, ck)
            assert torch.equal(D.dense_forward(x, w, activation=kind), y)
            if kind is not None:
                assert (y[5].abs() < 1e-32).all() and (y[4] == 80).all()  # silu(-80) = -1.44e-33


def test_clamp_keeps_its_side():
    """Gate and up values at, just inside and just outside the limit: the
    gradient passes exactly where the unrounded value is inside."""
    import dsv4_b200 as D
    limit = 1.3  # not a 16-bit value
    hidden = 16
    x = torch.zeros(64, hidden, device="cuda", dtype=F16)
    x[:, 0] = 1.25 + torch.arange(64, device="cuda") / 512  # crosses 1.3 between whole values
    x[:, 1] = 1
    w13 = torch.zeros(2 * 32, hidden, device="cuda", dtype=F16)
    w13[:32, 0] = 1   # gate = x0
    w13[32:, 0] = -1  # up = -x0
    w2 = torch.ones(8, 32, device="cuda", dtype=F16) / 16
    y, saved = D.gated_feed_forward_save(x, w13, w2, clamp_limit=limit)
    gx, g13, _ = D.gated_feed_forward_backward(torch.ones(64, 8, device="cuda", dtype=F16), saved)
    inside = x[:, 0].double() <= torch.tensor(limit, dtype=torch.float32).double()
    assert (gx[inside, 0] != 0).all() and (gx[~inside, 0] == 0).all()


# ---- streams, graphs, repeatability ----

def test_same_bits_every_time():
    import dsv4_b200 as D
    for m in (1, 64, 333):
        x, w13, w2, r = ffn_case(m, 512, 333, 512, BF16)
        dy = rand(m, 512, seed=2)
        first = None
        for _ in range(5):
            y, saved = D.gated_feed_forward_save(x, w13, w2, residual=r, checkpoint="int8")
            got = (D.gated_feed_forward(x, w13, w2, residual=r), y, *D.gated_feed_forward_backward(dy, saved))
            first = first or got
            assert all(same(a, b) for a, b in zip(first, got))


def test_side_streams():
    """Calls on streams of their own, at the same time."""
    import dsv4_b200 as D
    cases = [ffn_case(m, 512, 256, 512, BF16, seed=m) for m in (1, 48, 300, 700)]
    want = [D.gated_feed_forward(a, b, c, residual=r) for a, b, c, r in cases]
    dys = [rand(*a.shape, seed=9) for a, *_ in cases]

    def train(i):
        a, b, c, r = cases[i]
        y, saved = D.gated_feed_forward_save(a, b, c, residual=r)
        return (y, *D.gated_feed_forward_backward(dys[i], saved))

    trained = [train(i) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got, got_t = [], []
        for i, (s, (a, b, c, r)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got.append(D.gated_feed_forward(a, b, c, residual=r))
                got_t.append(train(i))
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(got, want))
        assert all(same(x, y) for a, b in zip(got_t, trained) for x, y in zip(a, b))


@pytest.mark.parametrize("m", [1, 64, 300])
def test_a_thread_that_has_used_no_cuda_yet(m):
    """Calls from a new thread whose memory all comes from the allocator's
    cache, so that no other call has set the thread up: both directions."""
    import threading

    import dsv4_b200 as D
    x, w13, w2, r = ffn_case(m, 512, 256, 512, BF16)
    dy = rand(m, 512, seed=2)

    def step():
        y, saved = D.gated_feed_forward_save(x, w13, w2, residual=r)
        return (y, D.gated_feed_forward(x, w13, w2), D.dense_forward(x, w13),
                *D.gated_feed_forward_backward(dy, saved))

    def forget(f):  # leaves its memory in the cache
        f()
        torch.cuda.synchronize()

    want = step()
    forget(step)
    got, failed = [], []

    def run(f):
        try:
            got.append(f())
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)

    for f in (lambda: D.gated_feed_forward_backward(dy, saved), lambda: D.dense_forward(x, w13),
              lambda: D.gated_feed_forward(x, w13, w2), step):
        y, saved = D.gated_feed_forward_save(x, w13, w2, residual=r)
        t = threading.Thread(target=run, args=(f,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    g, d, y, all_of_it = got
    assert all(same(a, b) for a, b in zip(g, want[3:])) and same(d, want[2]) and same(y, want[1])
    assert all(same(a, b) for a, b in zip(all_of_it, want))


def test_cuda_graphs():
    """Captured forward and training steps, replayed with other inputs, two
    graphs in turn: the results of eager calls."""
    import dsv4_b200 as D

    def make(m, mode):
        x, w13, w2, r = ffn_case(m, 256, 136, 256, BF16, seed=m)
        dy = rand(m, 256, seed=4)

        def step():
            y = D.gated_feed_forward(x, w13, w2, residual=r)
            z, saved = D.gated_feed_forward_save(x, w13, w2, residual=r, checkpoint=mode)
            return (y, z, *D.gated_feed_forward_backward(dy, saved),
                    D.dense_forward(x, w13, activation="gelu"))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return x, step, graph, out

    made = [make(2, None), make(200, "int8")]
    for turn in range(3):
        for x, step, graph, out in made:
            x.copy_(rand(*x.shape, seed=50 + turn))
        for x, step, graph, out in made:
            graph.replay()
        for x, step, graph, out in made:
            assert all(same(a, b) for a, b in zip(out, step()))


def test_first_call_inside_a_capture():
    """A process whose first call of all is captured."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    code = """
import torch, dsv4_b200 as D
x = torch.randn(300, 72, device="cuda").bfloat16()
w13, w2 = torch.randn(2 * 33, 72, device="cuda").bfloat16(), torch.randn(72, 33, device="cuda").bfloat16()
b, dy = torch.zeros(66, device="cuda").bfloat16(), torch.randn(300, 72, device="cuda").bfloat16()
torch.cuda.synchronize()
def step():
    y, saved = D.gated_feed_forward_save(x, w13, w2, checkpoint="int8")
    z, kept = D.dense_forward_save(x, w13, b, activation="gelu")
    return (y, D.gated_feed_forward(x[:3], w13, w2), D.gated_feed_forward(x[:40], w13, w2),
            *D.gated_feed_forward_backward(dy, saved), *D.dense_backward(z, kept),
            D.restore_int8(D.checkpoint_int8(x)))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
assert all(torch.equal(a, c) for a, c in zip(out, step()))
print("captured")
"""
    env = {**__import__("os").environ, "PYTHONPATH": str(root / "deepseek-v4-a100-sglang_b200")}
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=300)
    assert "captured" in r.stdout, r.stderr[-2000:]


def test_backward_on_another_stream():
    import dsv4_b200 as D
    x, w13, w2, r = ffn_case(300, 512, 256, 512, BF16)
    dy = rand(300, 512, seed=9)
    y, saved = D.gated_feed_forward_save(x, w13, w2, residual=r)
    want = D.gated_feed_forward_backward(dy, saved)
    torch.cuda.synchronize()
    for _ in range(5):
        y, saved = D.gated_feed_forward_save(x, w13, w2, residual=r)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = D.gated_feed_forward_backward(dy, saved)
        del saved
        junk = [torch.full((300, 2048), 7.0, device="cuda") for _ in range(4)]  # takes freed memory
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))
        del junk


def test_autograd_under_capture_is_refused():
    import dsv4_b200 as D
    x, w, _, _ = dense_case(4, 32, 32, BF16, False, False)
    w.requires_grad_(True)
    D.dense_forward(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            D.dense_forward(x, w)
        with torch.no_grad():
            y = D.dense_forward(x, w)
    graph.replay()
    assert same(y, D.dense_forward(x, w).detach())


# ---- autograd ----

@pytest.mark.parametrize("mode", [None, "int8"])
def test_any_subset_of_gradients(mode):
    import dsv4_b200 as D
    x, w13, w2, r = ffn_case(50, 64, 40, 48, BF16)
    dy = rand(50, 48, seed=3)
    full = None
    for mask in range(15, 0, -1):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w13, w2, r))]
        y = D.gated_feed_forward(*leaves[:3], residual=leaves[3], checkpoint=mode)
        y.backward(dy)
        full = full or [t.grad for t in leaves]
        for i, (t, want) in enumerate(zip(leaves, full)):
            if not mask >> i & 1:
                assert t.grad is None
            elif i == 2 and mode and not mask & 3:  # w2 alone keeps the product itself
                R.assert_within("w2", t.grad, R.ffn(x, w13, w2, r, "silu", None, BF16, dy)["grad_w2"])
            else:
                assert same(t.grad, want), (mask, i)
    x, w, b, r = dense_case(50, 64, 40, BF16)
    dy = rand(50, 40, seed=3)
    full = None
    for mask in range(15, 0, -1):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b, r))]
        D.dense_forward(*leaves[:3], residual=leaves[3], activation="gelu", checkpoint=mode).backward(dy)
        full = full or [t.grad for t in leaves]
        for i, (t, want) in enumerate(zip(leaves, full)):
            assert t.grad is None if not mask >> i & 1 else same(t.grad, want)


def test_autograd_corners():
    import dsv4_b200 as D
    x, w, b, _ = dense_case(20, 32, 24, BF16, residual=False)
    w.requires_grad_(True)
    x.requires_grad_(True)
    y = D.dense_forward(x, w, b, activation="silu")
    a = torch.autograd.grad(y, [x, w], torch.ones_like(y), retain_graph=True)
    c = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert all(same(p, q) for p, q in zip(a, c))
    y = D.dense_forward(x, w, b, activation="silu")  # a second derivative is refused
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|twice"):
        torch.autograd.grad(g.sum(), w)
    y = D.dense_forward(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    # the same tensor twice: its gradients add up
    s = rand(32, 32, seed=1).requires_grad_(True)
    D.dense_forward(s, s, residual=s).backward(torch.ones(32, 32, device="cuda", dtype=BF16))
    one = torch.ones(32, 32, device="cuda", dtype=torch.float64)
    want = one @ s.detach().double() + one.T @ s.detach().double() + one
    assert (s.grad.double() - want).abs().max() <= 4 * torch.finfo(BF16).eps * want.abs().max()
    with torch.no_grad():
        assert not D.dense_forward(x, w).requires_grad
    with torch.inference_mode():
        D.gated_feed_forward(*ffn_case(3, 16, 8, 16, BF16)[:3])


def test_wrong_gradient_shape_is_refused():
    import dsv4_b200 as D
    x, w, _, _ = dense_case(8, 32, 24, BF16, False, False)
    y, saved = D.dense_forward_save(x, w)
    with pytest.raises(ValueError, match="grad_out"):
        D.dense_backward(torch.zeros(8, 23, device="cuda", dtype=BF16), saved)
    with pytest.raises(TypeError, match="grad_out"):
        D.dense_backward(torch.zeros(8, 24, device="cuda"), saved)
    with pytest.raises(RuntimeError, match="cpu"):
        D.dense_forward(x, w.cpu())


# ---- C entry points ----

def test_c_refusals():
    """Arguments that the host must turn into errors, before any launch."""
    from dsv4_b200 import _native as N
    x, w, _, _ = dense_case(16, 64, 32, BF16, False, False)
    out = torch.zeros(16, 32, device="cuda", dtype=BF16)
    st = torch.cuda.current_stream().cuda_stream
    base = dict(a=x.data_ptr(), lda=64, a_mn=0, b=w.data_ptr(), ldb=64, b_mn=0, m=16, n=32, k=64, dtype=2, bias=None,
                act=0, res=None, ldr=0, out=out.data_ptr(), ldo=32, z=None, zb=0, zs=None, st=st)

    def call(**new):
        N.call("dsv4_b200_dense_gemm", *dict(base, **new).values())

    call()
    for new, text in (({"a": x.data_ptr() + 2}, "aligned"), ({"lda": 63}, "aligned"), ({"lda": 60}, "aligned"),
                      ({"lda": 56}, "row stride"), ({"b": None}, "null"), ({"out": None}, "null"), ({"n": 0}, "shape"),
                      ({"k": 0}, "shape"), ({"m": -1}, "shape"), ({"dtype": 0}, "dtype"), ({"act": 5}, "activation"),
                      ({"ldo": 31}, "row stride"), ({"zb": 8}, "go together"), ({"zb": 4}, "z_bits"),
                      ({"m": 1 << 40}, "shape")):
        with pytest.raises(RuntimeError, match=text):
            call(**new)
    call(m=0, a=None, b=None, out=None)
    h = torch.zeros(16, 24, device="cuda", dtype=BF16)
    w13 = torch.zeros(64, 40, device="cuda", dtype=BF16)  # by columns: 2 * 20 rows of 64
    with pytest.raises(RuntimeError, match="multiple of 8"):
        N.call("dsv4_b200_gated_gemm", x.data_ptr(), 64, 0, w13.data_ptr(), 40, 1, 16, 20, 64, 2, 2, 0, 0.0, h.data_ptr(),
               24, None, 0, None, st)
    for limit in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="limit"):
            N.call("dsv4_b200_gated_gemm", x.data_ptr(), 64, 0, w13.data_ptr(), 64, 0, 16, 20, 64, 2, 2, 1, limit,
                   h.data_ptr(), 24, None, 0, None, st)
    with pytest.raises(RuntimeError, match="kept"):
        N.call("dsv4_b200_gated_backward_gemm", x.data_ptr(), 64, 0, w13.data_ptr(), 64, 0, 16, 20, 64, 2, 2, 0, 0.0,
               None, 0, None, h.data_ptr(), 40, None, 0, st)
    codes, scales = torch.zeros(16, 64, device="cuda", dtype=torch.int8), torch.zeros(2, 16, device="cuda")
    with pytest.raises(RuntimeError, match="aligned"):
        N.call("dsv4_b200_checkpoint_int8", x.data_ptr(), 2, 15, 64, 64, codes.data_ptr() + 8, scales.data_ptr(), st)
    with pytest.raises(RuntimeError, match="shape"):
        N.call("dsv4_b200_checkpoint_int8", x.data_ptr(), 2, 16, 64, 63, codes.data_ptr(), scales.data_ptr(), st)
    with pytest.raises(RuntimeError, match="dtype"):
        N.call("dsv4_b200_restore_int8", codes.data_ptr(), scales.data_ptr(), 16, 64, out.data_ptr(), 7, 64, st)
    with pytest.raises(RuntimeError, match="slabs"):
        N.call("dsv4_b200_act_backward", x.data_ptr(), 64, None, 0, None, 16, 64, 2, 0, None, 64, scales.data_ptr(), 0,
               out.data_ptr(), st)
    N.check_device_status()


def test_c_refuses_addresses_between_elements():
    from dsv4_b200 import _native as N
    x, w, _, _ = dense_case(16, 64, 32, BF16, False, False)
    st = torch.cuda.current_stream().cuda_stream
    p, q = x.data_ptr(), w.data_ptr()
    out, codes = torch.zeros(16, 64, device="cuda", dtype=BF16), torch.zeros(16, 64, device="cuda", dtype=torch.int8)
    scales = torch.zeros(64, device="cuda")
    o, c, s = out.data_ptr(), codes.data_ptr(), scales.data_ptr()
    for name, *args in (
            ("dense_gemm", p, 64, 0, q, 64, 0, 16, 32, 64, 2, o + 1, 0, None, 0, o, 32, None, 0, None),
            ("dense_gemm", p, 64, 0, q, 64, 0, 16, 32, 64, 2, None, 0, o + 1, 32, o, 32, None, 0, None),
            ("dense_gemm", p, 64, 0, q, 64, 0, 16, 32, 64, 2, None, 0, None, 0, o + 1, 32, None, 0, None),
            ("dense_gemm", p + 1, 64, 0, q, 64, 0, 1, 32, 64, 2, None, 0, None, 0, o, 32, None, 0, None),
            ("dense_gemm", p, 64, 0, q, 64, 0, 16, 32, 64, 2, None, 2, None, 0, o, 32, c, 8, s + 2),
            ("gated_gemm", p, 64, 0, q, 64, 0, 16, 16, 64, 2, 2, 0, 0.0, o + 1, 16, None, 0, None),
            ("gated_backward_gemm", p, 64, 0, q, 64, 0, 16, 16, 64, 2, 2, 0, 0.0, c, 8, s, o + 1, 32, None, 0),
            ("checkpoint_int8", p + 1, 2, 16, 63, 64, c, s), ("checkpoint_int8", p, 2, 16, 64, 64, c, s + 1),
            ("checkpoint_int8", p + 2, 0, 8, 31, 32, c, s), ("restore_int8", c, s, 16, 64, o + 1, 2, 64),
            ("restore_int8", c, s, 8, 32, o + 2, 0, 32), ("restore_int8", c, s + 2, 16, 64, o, 2, 64),
            ("pack_rows", p + 1, 64, 1, 16, 63, o, 64), ("pack_rows", p, 64, 1, 16, 63, o + 1, 64),
            ("act_backward", p + 1, 64, None, 0, None, 16, 63, 2, 0, None, 64, s, 600, o)):
        with pytest.raises(RuntimeError, match="aligned to"):
            N.call("dsv4_b200_" + name, *args, st)
    N.check_device_status()


# ---- long ----

def test_more_than_two_to_the_31_values():
    """Offsets past 32 bits: 300,000 rows of 8,192, every 997th row checked."""
    import dsv4_b200 as D
    m, k = 300_000, 8192
    x = torch.empty(m, k, device="cuda", dtype=BF16)
    for part in x.split(20_000):
        part.normal_()
    c = D.checkpoint_int8(x)
    rows = torch.arange(0, m, 997, device="cuda")
    back, _, _ = R.eight(x[rows].double())
    got = D.restore_int8(c)
    h = torch.finfo(BF16).eps / 2
    R.assert_within("restored", got[rows], R.Bounded(back, back.abs() * (h + 2.0 ** -22) + R.tiny_of(BF16)))
    del got, c
    w = rand(16, k, std=k ** -0.5, seed=3)
    y = D.dense_forward(x, w, activation="relu")
    R.assert_within("y", y[rows], R.dense(x[rows], w, None, None, "relu", BF16)["y"])
    del x
    wide = rand(16, 8, seed=1)
    x = rand(m, 8, seed=2)
    y = D.dense_forward(x, rand(8192, 8, seed=4))  # a result of 2.5e9 values
    R.assert_within("wide", y[rows], R.dense(x[rows], rand(8192, 8, seed=4), None, None, None, BF16)["y"])
    assert wide is not None


# ---- together ----

def test_moe_layer_with_shared_expert_and_its_training():
    """Routed MXFP4 experts, the shared expert added to them in its own down
    projection, a projection behind it; then the backward pass through the
    16-bit part, in 16 and in 8 kept bits."""
    import dsv4_b200 as D
    import gen_inputs as G
    e, t, h, i, topk = 8, 48, 256, 128, 2
    w13, s13 = G.make_random_packed_mxfp4(e, 2 * i, h, 11, exp_range=(-8, -4))
    w2, s2 = G.make_random_packed_mxfp4(e, h, i, 12, exp_range=(-8, -4))
    ids, tw = G.routing_softmax_topk(t, e, topk, 13)
    x = G.randn_bf16((t, h), 14).cuda()
    experts = D.Mxfp4Int8MoeWeights(*D.remap_mxfp4_weight_for_int8(w13.cuda(), s13.cuda()),
                                    *D.remap_mxfp4_weight_for_int8(w2.cuda(), s2.cuda()), 3)
    routed = D.mxfp4_int8_moe_forward(x, experts, ids.cuda(), tw.cuda(), hidden_size=h, intermediate_size=i)
    _, sw13, sw2, _ = ffn_case(t, h, i, h, BF16, residual=False, seed=21)
    head, bias = rand(96, h, std=h ** -0.5, seed=31), rand(96, std=0.1, seed=32)
    dy = rand(t, 96, std=0.1, seed=33)
    for mode in (None, "int8"):
        leaves = [v.clone().requires_grad_(True) for v in (x, sw13, sw2, head, bias)]
        layer = D.gated_feed_forward(leaves[0], leaves[1], leaves[2], clamp_limit=7.0, residual=routed, checkpoint=mode)
        y = D.dense_forward(layer, leaves[3], leaves[4], activation="gelu", checkpoint=mode)
        grads = torch.autograd.grad(y, leaves, dy)
        first = R.ffn(x, sw13, sw2, routed, "silu", 7.0, BF16)["y"]
        R.assert_within("layer", layer.detach(), first)
        second = R.dense(layer.detach(), head, bias, None, "gelu", BF16, dy, mode)
        R.assert_within("y", y.detach(), second["y"])
        R.assert_within("grad head", grads[3], second["grad_weight"])
        R.assert_within("grad bias", grads[4], second["grad_bias"])
        back, saved = D.dense_forward_save(layer.detach(), head, bias, activation="gelu", checkpoint=mode)
        dlayer = D.dense_backward(dy, saved)[0]
        R.assert_within("grad layer", dlayer, second["grad_x"])
        third = R.ffn(x, sw13, sw2, routed, "silu", 7.0, BF16, dlayer, mode)
        for g, key in zip(grads, ("grad_x", "grad_w13", "grad_w2")):
            R.assert_within(key, g, third[key])

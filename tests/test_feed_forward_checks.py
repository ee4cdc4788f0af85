"""The 16-bit feed-forward operators without a GPU: refusals of their
arguments, and the 64-bit formulas of their tests against differences."""

import math

import pytest
import torch

import feed_forward_ref as R

BF16 = torch.bfloat16


def z(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def test_dense_refusals():
    import dsv4_b200 as D
    x, w = z(4, 16), z(8, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.dense_forward(x, w)
    with pytest.raises(ValueError, match="2-D"):
        D.dense_forward(z(16), w)
    with pytest.raises(ValueError, match=r"weight must have shape \[\*, 16\]"):
        D.dense_forward(x, z(8, 15))
    with pytest.raises(TypeError, match="fp16 or bf16"):
        D.dense_forward(z(4, 16, dtype=torch.float32), w)
    with pytest.raises(TypeError, match="weight must be torch.bfloat16"):
        D.dense_forward(x, z(8, 16, dtype=torch.float16))
    with pytest.raises(ValueError, match="empty"):
        D.dense_forward(z(4, 0), z(8, 0))
    with pytest.raises(ValueError, match="empty"):
        D.dense_forward(x, z(0, 16))
    with pytest.raises(ValueError, match=r"bias must have shape \[8\]"):
        D.dense_forward(x, w, z(7))
    with pytest.raises(ValueError, match=r"bias must have shape \[8\]"):
        D.dense_forward(x, w, z(1, 8))
    with pytest.raises(TypeError, match="bias"):
        D.dense_forward(x, w, z(8, dtype=torch.float32))
    with pytest.raises(ValueError, match="residual"):
        D.dense_forward(x, w, residual=z(4, 7))
    with pytest.raises(TypeError, match="residual"):
        D.dense_forward(x, w, residual=z(4, 8, dtype=torch.float16))
    for activation in ("swish", "GELU", 1, ["silu"]):
        with pytest.raises(ValueError, match="activation"):
            D.dense_forward(x, w, activation=activation)
    with pytest.raises(ValueError, match="checkpoint"):
        D.dense_forward(x, w, checkpoint="int4")
    with pytest.raises(TypeError, match="tensor"):
        D.dense_forward(None, w)


def test_gated_refusals():
    import dsv4_b200 as D
    x, w13, w2 = z(4, 16), z(12, 16), z(20, 6)
    with pytest.raises(RuntimeError, match="CUDA"):
        D.gated_feed_forward(x, w13, w2)
    with pytest.raises(ValueError, match="as many up rows"):
        D.gated_feed_forward(x, z(11, 16), w2)
    with pytest.raises(ValueError, match="w2 must have shape"):
        D.gated_feed_forward(x, w13, z(20, 7))
    with pytest.raises(ValueError, match="w13 must have shape"):
        D.gated_feed_forward(x, z(12, 17), w2)
    with pytest.raises(ValueError, match="residual"):
        D.gated_feed_forward(x, w13, w2, residual=z(4, 16))
    with pytest.raises(ValueError, match="w2 must not be empty"):
        D.gated_feed_forward(x, w13, z(0, 6))
    for limit in (0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="clamp_limit"):
            D.gated_feed_forward(x, w13, w2, clamp_limit=limit)
    with pytest.raises(TypeError, match="w2 must be"):
        D.gated_feed_forward(x, w13, z(20, 6, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="CUDA"):
        D.gated_feed_forward_save(x, w13, w2)


def test_checkpoint_refusals():
    import dsv4_b200 as D
    with pytest.raises(ValueError, match="2-D"):
        D.checkpoint_int8(z(4))
    with pytest.raises(TypeError, match="fp32, fp16 or bf16"):
        D.checkpoint_int8(torch.zeros((4, 4), dtype=torch.float64))
    with pytest.raises(ValueError, match="no columns"):
        D.checkpoint_int8(z(4, 0))
    with pytest.raises(RuntimeError, match="CUDA"):
        D.checkpoint_int8(z(4, 4))
    good = D.Int8Checkpoint(torch.zeros((4, 32), dtype=torch.int8), torch.zeros((1, 4)), (4, 20), BF16)
    with pytest.raises(TypeError, match="tensor"):
        D.checkpoint_int8([[1.0]])
    with pytest.raises(TypeError, match="Int8Checkpoint"):
        D.restore_int8(z(4, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        D.restore_int8(good)
    with pytest.raises(TypeError, match="dtype"):
        D.restore_int8(good, torch.int8)
    for codes, scales in ((torch.zeros((4, 20), dtype=torch.int8), good.scales),
                          (good.codes, torch.zeros((4, 1))),
                          (good.codes.to(torch.uint8), good.scales),
                          (torch.zeros((32, 4), dtype=torch.int8).t(), good.scales)):
        with pytest.raises(ValueError, match="codes must be"):
            D.restore_int8(D.Int8Checkpoint(codes, scales, (4, 20), BF16))


def rand(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def differences(f, x, v, h=1e-5):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("kind", R.ACTS)
def test_slopes_against_differences(kind):
    x = torch.linspace(-6, 6, 2001, dtype=torch.float64) + 1e-3  # no point at relu's corner
    d = differences(lambda t: R.act(kind, t), x, torch.ones_like(x))
    assert (d - R.slope(kind, x)).abs().max() < 1e-8


@pytest.mark.parametrize("kind", ["silu", "gelu", "gelu_tanh", None])
@pytest.mark.parametrize("limit", [None, 0.8])
def test_block_gradients_against_differences(kind, limit):
    """The gradients that the GPU tests take as exact, along random directions."""
    m, hidden, inter, out = 5, 12, 7, 9
    x, w13, w2, dy = rand(m, hidden), rand(2 * inter, hidden, seed=1) / 3, rand(out, inter, seed=2), rand(m, out, seed=3)
    args = {"grad_x": x, "grad_w13": w13, "grad_w2": w2}

    def loss(**new):
        a = dict(args, **new)
        y = R.ffn(a["grad_x"], a["grad_w13"], a["grad_w2"], None, kind, limit, torch.bfloat16)["y"].v
        return (dy * y).sum()

    got = R.ffn(x, w13, w2, None, kind, limit, torch.bfloat16, dy)
    for name, t in args.items():
        v = rand(*t.shape, seed=7)
        d = differences(lambda s: loss(**{name: s}), t, v, 1e-6)
        assert abs(float(d - (got[name].v * v).sum())) < 1e-6 * (1 + abs(float(d))), name


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu", None])
def test_dense_gradients_against_differences(kind):
    m, k, n = 6, 11, 5
    x, w, b, dy = rand(m, k), rand(n, k, seed=1) / 3, rand(n, seed=2), rand(m, n, seed=3)
    args = {"grad_x": x, "grad_weight": w, "grad_bias": b}

    def loss(**new):
        a = dict(args, **new)
        return (dy * R.dense(a["grad_x"], a["grad_weight"], a["grad_bias"], None, kind, torch.bfloat16)["y"].v).sum()

    got = R.dense(x, w, b, None, kind, torch.bfloat16, dy)
    for name, t in args.items():
        v = rand(*t.shape, seed=7)
        d = differences(lambda s: loss(**{name: s}), t, v, 1e-6)
        assert abs(float(d - (got[name].v * v).sum())) < 1e-6 * (1 + abs(float(d))), name


def test_operand_layouts():
    """Which tensors a product reads where they lie (no copy, no kernel)."""
    from dsv4_b200 import feed_forward as F
    t = torch.empty(64, 64, dtype=BF16)
    assert F._operand(t)[2:] == (64, 0)
    assert F._operand(t[:, :40])[2:] == (64, 0)
    assert F._operand(t.t())[2:] == (64, 1)
    assert F._operand(t[:, :40].t())[2:] == (64, 1)
    assert F._operand(t[:1, :5])[2:] == (8, 0)
    assert F._operand(t[::2])[2:] == (128, 0)
    assert F._operand(t[:, :1].t())[2:] in ((8, 0), (64, 1))

"""Products whose operands lie by columns, of up to 1,024 rows: the
weight-streaming product takes them as a backward pass hands them over
(gradient of the input, of the weight), in every combination of orders, with
tiles below and above 64 tokens, one and several blocks of the contraction a
stage, short and long contractions; rows and columns beside the matrices are
NaN."""

import math

import pytest
import torch

import feed_forward_ref as R
from feed_forward_strict import assert_each
from test_gpu_feed_forward import BF16, F16, ffn_case, rand

pytestmark = pytest.mark.gpu


def by_columns(t):
    """The same values with contiguous, 16-byte aligned columns, NaN between them and around."""
    rows, cols = t.shape
    buf = torch.full((cols + 2, -(-rows // 8) * 8 + 8), math.nan, dtype=t.dtype, device=t.device)
    view = buf[1:1 + cols, :rows].t()
    view.copy_(t)
    return view


def by_rows(t):
    return by_columns(t.t()).t()


@pytest.mark.parametrize("x_order,w_order", [(by_rows, by_columns), (by_columns, by_rows), (by_columns, by_columns)])
@pytest.mark.parametrize("m", [9, 16, 40, 64, 72, 128, 136, 200, 520, 1000])
@pytest.mark.parametrize("n", [8, 72, 136, 264, 1000])
def test_dense_orders(x_order, w_order, m, n):
    import dsv4_b200 as D
    for i, k in enumerate((1, 40, 64, 65, 130, 520, 1024, 4104)):
        dtype = (BF16, F16)[i & 1]
        x, w = rand(m, k, dtype=dtype, seed=k), rand(n, k, dtype=dtype, std=k ** -0.5, seed=k + 1)
        want = R.dense(x, w, None, None, "silu", dtype)["y"]
        assert_each(f"k {k}", D.dense_forward(x_order(x), w_order(w), activation="silu"), want.v, want.e)


@pytest.mark.parametrize("x_order,w_order", [(by_rows, by_columns), (by_columns, by_rows), (by_columns, by_columns)])
@pytest.mark.parametrize("m", [9, 64, 72, 136, 520])
@pytest.mark.parametrize("inter", [8, 40, 72, 264])
def test_block_orders(x_order, w_order, m, inter):
    import dsv4_b200 as D
    for i, hidden in enumerate((8, 64, 200, 1024, 2056)):
        dtype = (BF16, F16)[i & 1]
        x, w13, w2, r = ffn_case(m, hidden, inter, 136, dtype, seed=hidden)
        want = R.ffn(x, w13, w2, r, "gelu_tanh", 1.5, dtype)["y"]
        y = D.gated_feed_forward(x_order(x), w_order(w13), w_order(w2), activation="gelu_tanh", clamp_limit=1.5, residual=r)
        assert_each(f"hidden {hidden}", y, want.v, want.e)


@pytest.mark.parametrize("mode", [None, "int8"])
@pytest.mark.parametrize("m,k,n", [(16, 264, 72), (64, 1024, 128), (129, 136, 1000), (1000, 512, 136), (2048, 96, 256),
                                   (4000, 72, 64)])
def test_gradients_through_the_streamed_products(mode, m, k, n):
    """dx of few tokens and dW of few rows (a long contraction over the tokens)."""
    import dsv4_b200 as D
    x, w = rand(m, k, seed=1), rand(n, k, std=k ** -0.5, seed=2)
    b, dy = rand(n, std=0.3, seed=3), rand(m, n, std=0.1, seed=4)
    want = R.dense(x, w, b, None, "gelu", BF16, dy, mode)
    y, saved = D.dense_forward_save(x, w, b, activation="gelu", checkpoint=mode)
    for got, key in zip(D.dense_backward(dy, saved), ("grad_x", "grad_weight", "grad_bias")):
        assert_each(key, got, want[key].v, want[key].e)

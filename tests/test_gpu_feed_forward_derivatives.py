"""Forward-mode derivatives of the feed-forward operators are refused on the
GPU too, a tangent that arrives through a backward pass among them."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_feed_forward import BF16, dense_case, ffn_case

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    import dsv4_b200 as D
    x, w, b, _ = dense_case(12, 32, 24, BF16, residual=False)
    y = D.dense_forward(x, w, b)
    with fwd.dual_level():
        for i in range(3):
            args = [x, w, b]
            args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                D.dense_forward(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            D.checkpoint_int8(fwd.make_dual(x.float(), x.float()))
        assert torch.equal(D.dense_forward(x, w, b), y)  # a level alone changes nothing


@pytest.mark.parametrize("mode", [None, "int8"])
def test_tangents_of_output_gradients_are_refused(mode):
    import dsv4_b200 as D
    x, w, b, _ = dense_case(12, 32, 24, BF16, residual=False)
    x.requires_grad_(True)
    y = D.dense_forward(x, w, b, activation="silu", checkpoint=mode)
    fx, w13, w2, _ = ffn_case(12, 32, 24, 40, BF16, residual=False)
    w2.requires_grad_(True)
    z = D.gated_feed_forward(fx, w13, w2, checkpoint=mode)
    with fwd.dual_level():
        for out, leaf in ((y, x), (z, w2)):
            dy = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, dy)

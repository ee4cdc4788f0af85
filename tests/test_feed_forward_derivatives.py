"""Derivatives that the feed-forward operators do not give are refused, not
dropped (without a GPU: the checks come before any launch)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

BF16 = torch.bfloat16


def z(*shape):
    return torch.zeros(shape, dtype=BF16)


def calls():
    import dsv4_b200 as D
    x, w, b, r = z(4, 16), z(8, 16), z(8), z(4, 8)
    w13, w2, r2 = z(12, 16), z(20, 6), z(4, 20)
    dense, block = (D.dense_forward, D.dense_forward_save), (D.gated_feed_forward, D.gated_feed_forward_save)
    for i in range(4):
        for f in dense:
            yield f, (x, w, b, r), i, lambda f, t: f(*t[:3], residual=t[3])
        for f in block:
            yield f, (x, w13, w2, r2), i, lambda f, t: f(*t[:3], residual=t[3])
    yield D.checkpoint_int8, (x,), 0, lambda f, t: f(t[0])


def test_forward_mode_is_refused():
    for f, tensors, i, go in calls():
        with fwd.dual_level():
            dual = list(tensors)
            dual[i] = fwd.make_dual(tensors[i], torch.ones_like(tensors[i]))
            for tracked in (torch.enable_grad, torch.no_grad):  # no_grad does not switch tangents off
                with tracked(), pytest.raises(NotImplementedError, match="forward-mode"):
                    go(f, dual)
            with torch.autograd.forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA"):
                go(f, dual)  # tangents switched off: an ordinary call
            with pytest.raises(RuntimeError, match="CUDA"):  # a level without tangents
                go(f, tensors)
        with pytest.raises(RuntimeError, match="CUDA"):
            go(f, tensors)


def test_forward_mode_of_the_gradients_is_refused():
    import dsv4_b200 as D
    saved = D.SavedDense(z(4, 16), z(8, 16), z(4, 8), None, (4, 8, 16), False, 16, 0)
    block = D.SavedFeedForward(z(4, 16), z(12, 16), z(20, 6), z(4, 8), "silu", None, (4, 16, 6, 20), 16, 0)
    for f, s, cols in ((D.dense_backward, saved, 8), (D.gated_feed_forward_backward, block, 20)):
        with fwd.dual_level():
            dy = fwd.make_dual(z(4, cols), z(4, cols))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(dy, s)

"""The 16-bit feed-forward operators in 64 bits, each result with a bound on
what a kernel with fp32 sums and 16-bit stored values may differ from it.

Bounds, per element, from the formats alone:
  h16    half a step of the 16-bit type, relative: finfo.eps / 2
  sum    an fp32 sum of K products, in any order and with truncated additions:
         (K + 8) 2^-23 sum |a b|
  act    the activations' slopes are below 1.13 and their second derivatives
         below 0.8 (gelu: 2 phi(0) = 0.798; silu: 1/2); evaluated in fp32 with
         a relative error below 2^-18 of |z| + 1
and first-order propagation, the second order covered by 2 %.
"""

import math

import torch

ACTS = (None, "relu", "silu", "gelu", "gelu_tanh")
GROUP = 32


def act(kind, z):
    if kind == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def eight(v):
    """(what 8-bit groups give back, the step of each value, the distance of
    each quotient to the nearest half)."""
    m, k = v.shape
    g = torch.nn.functional.pad(v, (0, -k % GROUP)).reshape(m, -1, GROUP)
    top = g.abs().amax(2, keepdim=True)
    live = top >= 2.0 ** -100
    bad = ~torch.isfinite(g).all(2, keepdim=True)
    q = 127 * g / torch.where(live, top, torch.ones_like(top))
    code = torch.round(q) * live
    step = (top / 127).expand_as(g)
    back = torch.where(bad, torch.full_like(g, math.nan), torch.where(live, code * step, torch.zeros_like(g)))
    edge = ((q.abs() - q.abs().floor()) - 0.5).abs() / 127 * top
    cut = lambda t: t.reshape(m, -1)[:, :k]  # noqa: E731
    return cut(back), cut(step), cut(edge)


class Bounded:
    """A value and how far it may be off."""

    def __init__(self, v, e=None):
        self.v = v
        self.e = torch.zeros_like(v) if e is None else e


def product(a, b, h16=None):
    """a @ b.T of Bounded operands, in an fp32 sum, rounded if h16 is given."""
    v = a.v @ b.v.T
    size = a.v.abs() @ b.v.abs().T
    e = 1.02 * (a.e @ b.v.abs().T + a.v.abs() @ b.e.T) + (a.v.shape[1] + 8) * 2.0 ** -23 * size
    return rounded(Bounded(v, e), h16)


def rounded(x, h16, tiny=0.0):
    return x if h16 is None else Bounded(x.v, x.e + h16 * (x.v.abs() + x.e) + tiny)


def tiny_of(dtype):
    """Half a step of the smallest values of the 16-bit type (subnormals)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def kept(z, mode):
    """z as the backward pass reads it: groups of 32, off by half a step of
    amax / 32767, or a whole one to stay on its side of a limit or of zero (a
    group whose largest value is over 4 times its root mean square: fp16
    multiples of a power of two up to amax / 2^14, off by at most a step of those); or in 8 bits."""
    if mode is None:
        k = z.v.shape[1]
        g = torch.nn.functional.pad(z.v.abs() + z.e, (0, -k % GROUP)).reshape(z.v.shape[0], -1, GROUP)
        top = g.amax(2, keepdim=True).expand_as(g)
        live = (k - GROUP * torch.arange(g.shape[1], device=g.device)).clamp(max=GROUP).view(1, -1, 1)
        ratio = top.square() * live / g.square().sum(2, keepdim=True).clamp(min=1e-300)
        even, wide = 1.001 * top / 32767, 2.0 ** -10 * g + 2.0 ** -38 * top
        e = torch.where(ratio < 15, even, torch.where(ratio > 17, wide, torch.maximum(even, wide)))
        return Bounded(z.v, z.e + e.reshape(z.v.shape[0], -1)[:, :k])
    back, step, edge = eight(z.v)
    # the largest value of a group may be off as well: the step with it
    top_e = torch.nn.functional.pad(z.e, (0, -z.e.shape[1] % GROUP)).reshape(z.e.shape[0], -1, GROUP)
    top_e = top_e.amax(2, keepdim=True).expand_as(top_e).reshape(z.e.shape[0], -1)[:, :z.e.shape[1]]
    flip = edge <= z.e + 2 * top_e + 2.0 ** -20 * z.v.abs()
    e = 2 * top_e + 2.0 ** -22 * back.abs() + torch.where(flip, step, torch.zeros_like(step))
    return Bounded(back, e)


def act_bounded(kind, z):
    v = act(kind, z.v)
    if kind is None:
        return Bounded(v, z.e)
    return Bounded(v, 1.15 * z.e + 2.0 ** -18 * (z.v.abs() + 1))


def slope_bounded(kind, z):
    v = slope(kind, z.v)
    if kind is None:
        return Bounded(v)
    if kind == "relu":
        return Bounded(v, (z.v.abs() <= z.e).to(v.dtype))
    return Bounded(v, 0.82 * z.e + 2.0 ** -17 * (z.v.abs() + 1))


def times(a, b):
    return Bounded(a.v * b.v, a.e * b.v.abs() + a.v.abs() * b.e + a.e * b.e + 2.0 ** -22 * (a.v * b.v).abs())


def dense(x, w, bias, residual, kind, dtype, dy=None, mode=None):
    """{name: Bounded} of y and, with dy, the gradients."""
    h16, tiny = torch.finfo(dtype).eps / 2, tiny_of(dtype)
    X, W = Bounded(x.double()), Bounded(w.double())
    z = product(X, W)
    if bias is not None:
        z = Bounded(z.v + bias.double(), z.e + 2.0 ** -23 * (z.v.abs() + bias.double().abs()))
    y = act_bounded(kind, z)
    if residual is not None:
        r = residual.double()
        y = Bounded(y.v + r, y.e + 2.0 ** -23 * (y.v.abs() + r.abs()))
    out = {"y": rounded(y, h16, tiny)}
    if dy is None:
        return out
    dz = Bounded(dy.double())
    if kind is not None:
        zk = kept(z, mode)
        if kind == "relu" and mode is None:
            zk = z  # kept with its sign
        unrounded = times(dz, slope_bounded(kind, zk))
        dz = rounded(unrounded, h16, tiny)
    else:
        unrounded = dz
    xk = X if mode is None else rounded(Bounded(eight(X.v)[0]), 2 * h16, tiny)
    out["grad_x"] = rounded(product(dz, Bounded(W.v.T)), h16, tiny)
    out["grad_weight"] = rounded(product(Bounded(dz.v.T, dz.e.T), Bounded(xk.v.T, xk.e.T)), h16, tiny)
    if bias is not None:
        m = x.shape[0]
        e = unrounded.e.sum(0) + (m + 8) * 2.0 ** -24 * unrounded.v.abs().sum(0)
        out["grad_bias"] = rounded(Bounded(unrounded.v.sum(0), e), h16, tiny)
    return out


def ffn(x, w13, w2, residual, kind, limit, dtype, dy=None, mode=None):
    h16, tiny = torch.finfo(dtype).eps / 2, tiny_of(dtype)
    lim = math.inf if limit is None else limit
    X, W13, W2 = Bounded(x.double()), Bounded(w13.double()), Bounded(w2.double())
    inter = w2.shape[1]
    z = product(X, W13)
    g, u = Bounded(z.v[:, :inter], z.e[:, :inter]), Bounded(z.v[:, inter:], z.e[:, inter:])

    def gate(g, u, sign_e=None):
        gc, uc = Bounded(g.v.clamp(max=lim), g.e), Bounded(u.v.clamp(-lim, lim), u.e)
        gs = gc if sign_e is None else Bounded(gc.v, sign_e)
        return act_bounded(kind, gc), slope_bounded(kind, gs), uc

    a, _, uc = gate(g, u)
    h = rounded(times(a, uc), h16, tiny)
    y = product(h, W2)
    if residual is not None:
        r = residual.double()
        y = Bounded(y.v + r, y.e + 2.0 ** -23 * (y.v.abs() + r.abs()))
    out = {"y": rounded(y, h16, tiny)}
    if dy is None:
        return out
    gk, uk = kept(g, mode), kept(u, mode)
    # relu keeps the sign: its slope is as sure as the sum itself
    a, s, uc = gate(gk, uk, g.e if kind == "relu" and mode is None else None)
    DY = Bounded(dy.double())
    dh = product(DY, Bounded(W2.v.T))

    def masked(d, inside, near):
        e = torch.where(near, d.e + d.v.abs(), torch.where(inside, d.e, torch.zeros_like(d.e)))
        return Bounded(torch.where(inside, d.v, torch.zeros_like(d.v)), e)

    # a value may cross the limit by its error before it is kept; 8-bit values also by their own
    gate_e, up_e = (g.e, u.e) if mode is None else (gk.e, uk.e)
    dg = masked(times(times(dh, uc), s), gk.v <= lim, (gk.v - lim).abs() <= gate_e)
    du = masked(times(dh, a), uk.v.abs() <= lim, (uk.v.abs() - lim).abs() <= up_e)
    dz = rounded(Bounded(torch.cat((dg.v, du.v), 1), torch.cat((dg.e, du.e), 1)), h16, tiny)
    hk = h if mode is None else rounded(times(a, uc), h16, tiny)
    xk = X if mode is None else rounded(Bounded(eight(X.v)[0]), 2 * h16, tiny)
    out["grad_x"] = rounded(product(dz, Bounded(W13.v.T)), h16, tiny)
    out["grad_w13"] = rounded(product(Bounded(dz.v.T, dz.e.T), Bounded(xk.v.T, xk.e.T)), h16, tiny)
    out["grad_w2"] = rounded(product(Bounded(DY.v.T), Bounded(hk.v.T, hk.e.T)), h16, tiny)
    return out


def assert_within(name, got, want):
    """Every element within its bound; the message names the worst."""
    assert tuple(got.shape) == tuple(want.v.shape), (name, got.shape, want.v.shape)
    off = (got.double() - want.v).abs()
    assert torch.isfinite(got).all() or not torch.isfinite(want.v).all(), f"{name}: not finite"
    over = off - want.e
    if over.numel() and float(over.max()) > 0:
        i = int(over.argmax())
        raise AssertionError(f"{name}: element {i} of {off.numel()}: got {got.flatten()[i].item()!r}, "
                             f"want {want.v.flatten()[i].item()!r} +- {want.e.flatten()[i].item():.3g}; "
                             f"{int((over > 0).sum())} elements out of bounds")

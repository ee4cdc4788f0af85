"""The bf16/fp16 feed-forward operators, as they are measured.

Three operators that a DeepSeek-style layer needs next to its routed experts
(its shared expert, its dense first layers, the projections around them, and
their fine-tuning):

``dense``       ``act(x @ weight.T + bias) + residual``, and its gradients
``ffn``         ``(act(x @ w1.T) * (x @ w3.T)) @ w2.T + residual`` with ``w13 = [w1; w3]``, and its gradients
``checkpoint``  activations kept in 8 bits (one scale for each 32 values of a row) and restored

With ``own`` false, :func:`run` computes the plain form: elementary torch
operations in fp32, rounded once at the end.  With ``own`` true it makes the
calls of the framework's users.
"""

import math

import numpy as np  # noqa: F401  (the measuring programs hand cases of plain Python and numpy values)
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_GROUP = 32  # values of a row that share one scale of an 8-bit checkpoint
_TINY = 2.0 ** -100  # a group below this is kept as zeros


def _dense(name, m, k, n, dtype, bias, activation, residual, train=False, checkpoint=""):
    return {"name": name, "op": "dense", "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias,
            "activation": activation, "residual": residual, "train": train, "checkpoint": checkpoint}


def _ffn(name, m, hidden, inter, dtype, activation="silu", limit=0.0, residual=True, train=False, checkpoint=""):
    return {"name": name, "op": "ffn", "m": m, "hidden": hidden, "inter": inter, "dtype": dtype,
            "activation": activation, "limit": limit, "residual": residual, "train": train,
            "checkpoint": checkpoint}


def listed():
    return [
        # one token's projection, its residual added: the latency of a decode step
        _dense("dense_decode_1", 1, 7168, 4096, "bf16", False, "none", True),
        # a small decode batch through a projection with bias and activation
        _dense("dense_decode_16", 16, 7168, 4096, "bf16", True, "gelu_tanh", False),
        # sizes that fit no tile, as a converted vision or draft head has them
        _dense("dense_ragged", 509, 1000, 1777, "fp16", True, "gelu", True),
        # a prefill chunk through a projection
        _dense("dense_prefill", 4096, 7168, 4096, "bf16", True, "silu", True),
        # fine-tuning a projection: forward, and the gradients of all that takes part
        _dense("dense_train", 2048, 2048, 7168, "bf16", True, "gelu", True, train=True),
        # the shared expert for one token; the residual is the routed experts' output
        _ffn("ffn_decode_1", 1, 7168, 2048, "bf16"),
        # the shared expert for a decode batch of 64
        _ffn("ffn_decode_64", 64, 7168, 2048, "bf16", limit=10.0),
        # the shared expert over a whole prefill
        _ffn("ffn_prefill", 8192, 7168, 2048, "bf16", limit=10.0),
        # fine-tuning the shared expert: forward and all gradients
        _ffn("ffn_train", 4096, 7168, 2048, "bf16", train=True),
        # the same for a small layer with ragged sizes, its activations kept in 8 bits
        _ffn("ffn_train_int8", 1531, 1024, 509, "fp16", limit=7.0, train=True, checkpoint="int8"),
        # a few tokens' activations kept in 8 bits and restored: latency
        {"name": "checkpoint_small", "op": "checkpoint", "m": 16, "k": 1024, "dtype": "bf16"},
        # a prefill's activations kept in 8 bits and restored
        {"name": "checkpoint_large", "op": "checkpoint", "m": 8192, "k": 7168, "dtype": "bf16"},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def size(lo, hi):  # a third of the sizes are odd or ragged, the others multiples of 64 or 8
        v = log(lo, hi)
        step = rng.choice((1, 8, 64))
        return max(step, v // step * step)

    dtype = rng.choice(("bf16", "bf16", "fp16"))
    op = rng.choice(("dense", "dense", "ffn", "ffn", "checkpoint"))
    if op == "checkpoint":
        return {"op": op, "m": log(1, 8192), "k": size(32, 7168), "dtype": dtype}
    train = rng.random() < 0.4
    m = log(1, 4096 if train else 8192)
    checkpoint = rng.choice(("", "int8")) if train else ""
    if op == "dense":
        c = _dense("", m, size(64, 7168), size(64, 4096), dtype, rng.random() < 0.5,
                   rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")), rng.random() < 0.5, train, checkpoint)
    else:
        c = _ffn("", m, size(64, 7168), size(32, 2048), dtype, rng.choice(("silu", "silu", "gelu", "gelu_tanh")),
                 rng.choice((0.0, 7.0, 10.0)), rng.random() < 0.5, train, checkpoint)
    del c["name"]
    return c


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    m = case["m"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(std).to(dt)

    def hidden(rows, cols):  # a hidden state: some channels are much larger than others
        x = torch.randn(rows, cols, device="cuda", generator=gen)
        return x.mul_(torch.randn(cols, device="cuda", generator=gen).mul_(0.5).exp_()).to(dt)

    state = {"case": dict(case)}
    if case["op"] == "checkpoint":
        state["x"] = hidden(m, case["k"])
        return state
    if case["op"] == "dense":
        k, n = case["k"], case["n"]
        state["x"] = hidden(m, k)
        state["weight"] = normal(n, k, std=1.0 / math.sqrt(k))
        state["bias"] = normal(n, std=0.1) if case["bias"] else None
        out = n
        wanted = ("x", "weight", "bias", "residual")
    else:
        h, i = case["hidden"], case["inter"]
        state["x"] = hidden(m, h)
        state["w13"] = normal(2 * i, h, std=1.0 / math.sqrt(h))
        state["w2"] = normal(h, i, std=1.0 / math.sqrt(i))
        out = h
        wanted = ("x", "w13", "w2", "residual")
    state["residual"] = normal(m, out) if case["residual"] else None
    if case["train"]:
        state["grad"] = normal(m, out, std=0.02)
        state["wanted"] = [w for w in wanted if state[w] is not None]
        for w in state["wanted"]:
            state[w].requires_grad_(True)
    return state


# ---- the framework's calls ----

def _run_own(s):
    import sys
    if "deepseek-v4-a100-sglang_b200" not in sys.path:
        sys.path.insert(0, "deepseek-v4-a100-sglang_b200")
    import dsv4_b200 as D

    c = s["case"]
    if c["op"] == "checkpoint":
        return D.restore_int8(D.checkpoint_int8(s["x"]))
    kw = {"residual": s["residual"], "activation": None if c["activation"] == "none" else c["activation"],
          "checkpoint": c["checkpoint"] or None}
    if c["op"] == "dense":
        y = D.dense_forward(s["x"], s["weight"], s["bias"], **kw)
    else:
        y = D.gated_feed_forward(s["x"], s["w13"], s["w2"], clamp_limit=c["limit"] or None, **kw)
    if not c["train"]:
        return y
    grads = torch.autograd.grad(y, [s[w] for w in s["wanted"]], s["grad"])
    return {"y": y, **{"grad_" + w: g for w, g in zip(s["wanted"], grads)}}


# ---- the plain form: fp32, rounded once at the end ----

def _act(kind, z):
    if kind == "relu":
        return z * (z > 0)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _kept(v):
    """What an 8-bit checkpoint of the rows of `v` gives back."""
    m, k = v.shape
    pad = -k % _GROUP
    g = torch.cat((v, v.new_zeros(m, pad)), 1) if pad else v
    g = g.reshape(m, -1, _GROUP)
    top = g.abs().amax(2, keepdim=True)
    live = top >= _TINY
    # in 64 bits: values next to the border of two codes
    codes = torch.round(127.0 * g.double() / torch.where(live, top, 1.0).double()).float() * live
    return (codes * (top / 127.0)).reshape(m, -1)[:, :k]


def _run_plain(s):
    c = s["case"]
    dt = _DTYPES[c["dtype"]]
    if c["op"] == "checkpoint":
        return _kept(s["x"].float()).to(dt)
    keep = _kept if c["checkpoint"] else (lambda v: v)
    x = s["x"].detach().float()
    res = None if s["residual"] is None else s["residual"].detach().float()
    dy = s["grad"].float() if c["train"] else None
    out = {}
    if c["op"] == "dense":
        w = s["weight"].detach().float()
        z = x @ w.T
        if s["bias"] is not None:
            z = z + s["bias"].detach().float()
        y = _act(c["activation"], z)
        if c["train"]:
            dz = dy if c["activation"] == "none" else dy * _act_slope(c["activation"], keep(z))
            out["grad_x"] = (dz @ w).to(dt)
            out["grad_weight"] = (dz.T @ keep(x)).to(dt)
            if s["bias"] is not None:
                out["grad_bias"] = dz.sum(0).to(dt)
    else:
        i, lim = c["inter"], c["limit"] or math.inf
        w13, w2 = s["w13"].detach().float(), s["w2"].detach().float()
        z = x @ w13.T
        g, u = z[:, :i], z[:, i:]
        y = (_act(c["activation"], g.clamp(max=lim)) * u.clamp(-lim, lim)) @ w2.T
        if c["train"]:
            g, u = keep(g), keep(u)
            gc, uc = g.clamp(max=lim), u.clamp(-lim, lim)
            a, dh = _act(c["activation"], gc), dy @ w2
            dg = dh * uc * _act_slope(c["activation"], gc) * (g <= lim)
            du = dh * a * (u.abs() <= lim)
            dz = torch.cat((dg, du), 1)
            out["grad_x"] = (dz @ w13).to(dt)
            out["grad_w13"] = (dz.T @ keep(x)).to(dt)
            out["grad_w2"] = (dy.T @ (a * uc)).to(dt)
    if res is not None:
        y = y + res
    y = y.to(dt)
    if not c["train"]:
        return y
    if res is not None:
        out["grad_residual"] = s["grad"]
    return {"y": y, **out}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- the definition in 64 bits, row blocks at a time ----

def exact(case, seed):
    s = prepare(case, seed)
    t = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    act = case.get("activation")

    def phi(v):  # the normal distribution's function
        return 0.5 * torch.special.erfc(-v / math.sqrt(2.0))

    def f(v):
        if act == "relu":
            return torch.where(v > 0, v, torch.zeros_like(v))
        if act == "silu":
            return v * torch.sigmoid(v)
        if act == "gelu":
            return v * phi(v)
        if act == "gelu_tanh":  # (1 + tanh a) / 2 = sigmoid(2 a)
            return v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
        return v

    def df(v):
        with torch.enable_grad():
            v = v.detach().requires_grad_(True)
            return torch.autograd.grad(f(v).sum(), v)[0]

    def eight(v):
        rows = []
        for r in v.split(1024):
            parts = []
            for p in r.split(_GROUP, dim=1):
                top = p.abs().max(dim=1, keepdim=True).values
                step = top / 127
                q = torch.round(torch.div(p * 127, torch.where(top > 0, top, torch.ones_like(top))))
                parts.append(torch.where(top < _TINY, torch.zeros_like(p), q * step))
            rows.append(torch.cat(parts, 1))
        return torch.cat(rows)

    if case["op"] == "checkpoint":
        return eight(t["x"])
    keep = eight if case["checkpoint"] else (lambda v: v)
    x = t["x"]
    if case["op"] == "dense":
        z = torch.einsum("mk,nk->mn", x, t["weight"])
        if "bias" in t:
            z += t["bias"]
        y = f(z)
        if case["train"]:
            dz = t["grad"] * df(keep(z) if act != "none" else z)
            grads = {"grad_x": torch.einsum("mn,nk->mk", dz, t["weight"]),
                     "grad_weight": torch.einsum("mn,mk->nk", dz, keep(x))}
            if "bias" in t:
                grads["grad_bias"] = torch.einsum("mn->n", dz)
    else:
        lim = case["limit"] or math.inf
        w1, w3 = t["w13"].chunk(2)
        gate, up = torch.einsum("mk,nk->mn", x, w1), torch.einsum("mk,nk->mn", x, w3)
        y = torch.einsum("mi,hi->mh", f(gate.clamp(max=lim)) * up.clamp(-lim, lim), t["w2"])
        if case["train"]:
            gate, up = keep(gate), keep(up)
            lo, mid = gate.clamp(max=lim), up.clamp(-lim, lim)
            dh = torch.einsum("mh,hi->mi", t["grad"], t["w2"])
            dgate = torch.where(gate <= lim, dh * mid * df(lo), torch.zeros_like(dh))
            dup = torch.where((up <= lim) & (up >= -lim), dh * f(lo), torch.zeros_like(dh))
            kept = keep(x)
            grads = {"grad_x": torch.einsum("mi,ih->mh", dgate, w1) + torch.einsum("mi,ih->mh", dup, w3),
                     "grad_w13": torch.cat((torch.einsum("mi,mh->ih", dgate, kept),
                                            torch.einsum("mi,mh->ih", dup, kept))),
                     "grad_w2": torch.einsum("mh,mi->hi", t["grad"], f(lo) * mid)}
    if "residual" in t:
        y = y + t["residual"]
    if not case["train"]:
        return y
    if "residual" in t:
        grads["grad_residual"] = t["grad"]
    return {"y": y, **grads}


def work(case):
    m, train = case["m"], case.get("train", False)
    if case["op"] == "checkpoint":  # the activations in; codes and scales out and in; the activations out
        kept = m * case["k"] + 4 * m * -(-case["k"] // _GROUP)
        return {"bytes": 2 * (2 * m * case["k"] + kept), "flops": 4 * m * case["k"]}
    if case["op"] == "dense":
        k, n = case["k"], case["n"]
        weights, rows_in, rows_out = n * k, m * k, m * n
        other = n if case["bias"] else 0
    else:
        k, n = case["hidden"], case["hidden"]
        weights, rows_in, rows_out = 3 * case["inter"] * k, m * k, m * n
        other = 0
    elements = weights + rows_in + rows_out * (2 if case["residual"] else 1) + other
    flops = 2 * m * weights
    if train:  # the output's gradient in; a gradient of each input out
        elements += rows_out + rows_in + weights + other
        flops *= 3
    return {"bytes": 2 * elements, "flops": flops}

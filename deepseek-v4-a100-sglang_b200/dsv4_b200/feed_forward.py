"""16-bit feed-forward operators for B200 (sm_100a): what stands next to the
routed MXFP4 experts in a DeepSeek-style layer (shared expert, dense layers,
projections), forward and backward.

    dense_forward          y = act(x @ weight.T + bias) + residual
    gated_feed_forward     y = (act(x @ w1.T) * (x @ w3.T)) @ w2.T + residual,  w13 = [w1; w3]
    checkpoint_int8 / restore_int8    activations kept in 8 bits

bf16 and fp16; sums, activations and their slopes in fp32, one rounding where
a value is stored.  The values before an activation are kept for the backward
pass as groups of 32 with a shared scale, in 16 bits: each to 2^-15 of the
group's largest value and to 2^-10 (fp16: 2^-11) of itself.  ``dense_forward`` and
``gated_feed_forward`` are differentiable; their ``*_save`` / ``*_backward``
forms give the same steps without autograd (and are the ones to capture into a
CUDA graph).  With ``checkpoint="int8"`` what the backward pass needs is kept
in 8 bits.  Every call is asynchronous on the current stream of the tensors'
device; there is no CPU path.

Results follow the inputs' values: NaN and infinities propagate as the
formulas say (kept in 8 bits they make their whole group of 32 NaN in the
backward pass).  All results are the same bits from call to call.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _native as N

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_CHECKPOINTS = (None, "int8")
_DTYPES = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_CHECKPOINT_DTYPES = {torch.float32: N.DTYPE_F32, **_DTYPES}
_GROUP = 32
_FEW = 8  # tokens up to which a product without kept values reads rows of any alignment


class _Functions(dict):
    """C entry points by name without the ``dsv4_b200_`` prefix."""

    def __missing__(self, name):
        self[name] = fn = getattr(N.load(), "dsv4_b200_" + name)
        return fn


_functions = _Functions()


def _call(name: str, *args) -> None:
    rc = _functions[name](*args)
    if rc:
        N.check(rc, "dsv4_b200_" + name)


# ---- argument checks ----
# The checks that a call in a decode loop pays for are one expression over
# plain attributes; the functions that name the fault run only when it fails.

def _explain_matrix(t, name: str, rows=None, cols=None, like=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    if like is None:
        if t.dtype not in _DTYPES:
            raise TypeError(f"{name} must be fp16 or bf16, got {t.dtype}")
    elif t.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype} like the input, got {t.dtype}")
    if (rows is not None and t.shape[0] != rows) or (cols is not None and t.shape[1] != cols):
        want = ("*" if rows is None else rows, "*" if cols is None else cols)
        raise ValueError(f"{name} must have shape [{want[0]}, {want[1]}], got {tuple(t.shape)}")


def _explain_device(first: torch.Tensor, **others) -> None:
    if not first.is_cuda:
        raise RuntimeError("the feed-forward operators need CUDA tensors on an sm_100a device "
                           "(no CPU path)")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{name} is on {t.device}, expected {first.device}")


def _explain_options(activation, checkpoint, clamp_limit=None) -> None:
    if not isinstance(activation, (str, type(None))) or activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if checkpoint not in _CHECKPOINTS:
        raise ValueError(f'checkpoint must be None or "int8", got {checkpoint!r}')
    if clamp_limit is not None and not (0 < float(clamp_limit) < math.inf):
        raise ValueError(f"clamp_limit must be positive and finite, got {clamp_limit}")


def _refuse_tangents(*tensors) -> None:
    """A tensor of forward-mode autograd carries a tangent that a kernel does not see."""
    if _forward_ad._current_level < 0 or not torch._C._is_fwd_grad_enabled():
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the feed-forward operators have no forward-mode derivative")


def _is_matrix(t, rows, cols, dtype, dev) -> bool:
    return t.shape == (rows, cols) and t.dtype is dtype and t.get_device() == dev


def _on(dev: int):
    """Launches go to the tensors' device, whichever is current."""
    if torch._C._cuda_getDevice() == dev:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") \
    else lambda dev: torch.cuda.current_stream(dev).cuda_stream


# ---- operands ----

def _up(v: int, to: int) -> int:
    return -(-v // to) * to


def _operand(t: torch.Tensor, columns: bool = True):
    """A 2-D tensor as a product reads it: ``(tensor, address, stride, mn)``
    with rows (mn 0) or columns (mn 1) contiguous and 16-byte aligned.
    Others are laid out anew (one pass over them).  ``columns`` False: only
    contiguous rows will do."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    ptr = t.data_ptr()
    if ptr & 15 == 0:
        if s1 == 1 or cols == 1:
            if rows == 1:
                return t, ptr, _up(cols, 8), 0
            if s1 == 1 and s0 & 7 == 0 and s0 >= cols:
                return t, ptr, s0, 0
        if columns and s0 == 1:
            if cols == 1:
                return t, ptr, _up(rows, 8), 1
            if s1 & 7 == 0 and s1 >= rows:
                return t, ptr, s1, 1
    ld = _up(cols, 8)
    out = t.new_empty((rows, ld))
    ptr2 = out.data_ptr()
    _call("pack_rows", ptr, s0, s1, rows, cols, ptr2, ld, _stream(t.get_device()))
    return out, ptr2, ld, 0


def _laid_out(operand, t: torch.Tensor) -> torch.Tensor:
    """t, or the copy of it that a product reads, to be kept for the backward pass."""
    return t if operand[0] is t else operand[0][:, :t.shape[1]]


def _row_operands(x: torch.Tensor, w: torch.Tensor, columns: bool = True):
    """:func:`_operand` of both for a product of few tokens: where both lie by
    rows, any alignment will do."""
    if x.shape[0] <= _FEW and w.stride(1) == 1 and x.stride(1) == 1:
        m, k = x.shape
        ldx, ldw = x.stride(0) if m > 1 else _up(k, 8), w.stride(0)
        if ldx >= k and ldw >= k:
            return (x, x.data_ptr(), ldx, 0), (w, w.data_ptr(), ldw, 0)
    return _operand(x), _operand(w, columns)


def _plain_rows(t: torch.Tensor) -> torch.Tensor:
    """A tensor whose rows are contiguous (any alignment; row stride 0 allowed)."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    if (s1 == 1 or cols == 1) and (rows <= 1 or s0 >= cols or s0 == 0):
        return t
    return t.contiguous()


def _distinct_rows(t: torch.Tensor) -> torch.Tensor:
    """:func:`_plain_rows` without a row stride of 0."""
    t = _plain_rows(t)
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) == 0 else t


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


# ---- what a training step keeps, and the backward pass's workspace ----
# One allocation each, in the inputs' 16-bit type: parts at multiples of 256
# bytes, passed by address.  The layouts are functions of the sizes alone.

@functools.lru_cache(maxsize=4096)
def _layout(*sizes):
    """(elements of 2 bytes, byte offset of each part, None for a size of None)."""
    total, at = 0, []
    for size in sizes:
        at.append(None if size is None else total)
        total += 0 if size is None else _up(size, 256)
    return total // 2, tuple(at)


def _group_bytes(rows: int, cols: int, bits: int):
    """Bytes of the codes and of the scales of [rows, cols] kept in groups."""
    k32 = _up(cols, _GROUP)
    return rows * k32 * bits // 8, rows * (k32 // _GROUP) * 4


def _at(base: int, offsets):
    return [None if o is None else base + o for o in offsets]


def _on_stream(saved, *tensors) -> None:
    """What a forward call kept is in use on the current stream too: its memory
    must not go to others while this stream reads it."""
    dev = saved.kept.get_device()
    if _stream(dev) != saved.stream:
        now = torch.cuda.current_stream(dev)
        for t in (saved.kept, *tensors):
            if t is not None:
                t.record_stream(now)


# ---- 8-bit checkpoints ----

@dataclass(slots=True)
class Int8Checkpoint:
    """Rows of activations in 8 bits: ``codes`` int8 [M, K up to 32], ``scales``
    fp32 [groups, M].  32 consecutive values of a row share a scale
    ``amax / 127`` (rounded toward zero); a code is ``127 v / amax`` rounded to
    the nearest whole number, ties to even.  A group that holds an infinity or
    a NaN is restored as NaN, one whose largest magnitude is below 2^-100 as
    zeros."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    dtype: torch.dtype


def _empty_codes(rows: int, cols: int, like: torch.Tensor):
    groups = -(-cols // _GROUP)
    return (like.new_empty((rows, groups * _GROUP), dtype=torch.int8),
            like.new_empty((groups, rows), dtype=torch.float32))


def checkpoint_int8(x: torch.Tensor) -> Int8Checkpoint:
    """Keep the rows of ``x`` [M, K] (fp32, fp16 or bf16) in 8 bits: 1.125
    bytes per value.  ``restore_int8(checkpoint_int8(x))`` differs from x by at
    most half a step, ``amax / 254`` of its group, and the rounding to x's type.
    Codes have no gradient: for autograd a graph ends here."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a tensor, got {type(x).__name__}")
    _refuse_tangents(x)
    shape, dtype = x.shape, x.dtype
    if len(shape) != 2:
        raise ValueError(f"x must be 2-D, got shape {tuple(shape)}")
    if dtype not in _CHECKPOINT_DTYPES:
        raise TypeError(f"x must be fp32, fp16 or bf16, got {dtype}")
    m, k = shape
    if k == 0:
        raise ValueError("x has no columns")
    dev = x.get_device()
    if dev < 0:
        _explain_device(x)
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return checkpoint_int8(x)
    ld, s1 = x.stride()
    if m == 1 and (s1 == 1 or k == 1):
        ld = k
    elif (s1 != 1 and k > 1) or ld < k:
        x = x.detach().contiguous()
        ld = k
    codes, scales = _empty_codes(m, k, x)
    _call("checkpoint_int8", x.data_ptr(), _CHECKPOINT_DTYPES[dtype], m, k, ld, codes.data_ptr(),
          scales.data_ptr(), _stream(dev))
    return Int8Checkpoint(codes, scales, (m, k), dtype)


def restore_int8(checkpoint: Int8Checkpoint, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The kept rows, in their own type or in ``dtype``."""
    if not isinstance(checkpoint, Int8Checkpoint):
        raise TypeError(f"checkpoint must be an Int8Checkpoint, got {type(checkpoint).__name__}")
    dtype = checkpoint.dtype if dtype is None else dtype
    if dtype not in _CHECKPOINT_DTYPES:
        raise TypeError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
    m, k = checkpoint.shape
    k32 = _up(k, _GROUP)
    c, s = checkpoint.codes, checkpoint.scales
    if (c.dtype != torch.int8 or c.shape != (m, k32) or not c.is_contiguous()
            or s.dtype != torch.float32 or s.shape != (k32 // _GROUP, m)
            or not s.is_contiguous()):
        raise ValueError(f"codes must be contiguous int8 [{m}, {k32}] and scales contiguous fp32 "
                         f"[{k32 // _GROUP}, {m}]")
    dev = c.get_device()
    if dev < 0 or s.get_device() != dev:
        _explain_device(c, scales=s)
    if torch._C._cuda_getDevice() != dev:
        with torch.cuda.device(dev):
            return restore_int8(checkpoint, dtype)
    out = c.new_empty((m, k), dtype=dtype)
    _call("restore_int8", c.data_ptr(), s.data_ptr(), m, k, out.data_ptr(), _CHECKPOINT_DTYPES[dtype], k,
          _stream(dev))
    return out


# ---- dense product ----

@dataclass
class SavedDense:
    """What :func:`dense_backward` needs of a :func:`dense_forward_save` call."""
    x: Optional[torch.Tensor]  # None: in 8 bits among `kept`
    weight: torch.Tensor
    kept: torch.Tensor         # the value before the activation, and x in 8 bits
    activation: Optional[str]
    shape: tuple
    has_bias: bool
    bits: int
    stream: int


def _check_dense(x, weight, bias, activation, residual, checkpoint):
    """(m, n, k) of a call whose arguments go together; raises otherwise."""
    _refuse_tangents(x, weight, bias, residual)
    try:
        (m, k), n, dt, dev = x.shape, weight.shape[0], x.dtype, x.get_device()
        if (n and k and dev >= 0 and dt in _DTYPES and _is_matrix(weight, n, k, dt, dev)
                and activation in ACTIVATIONS and checkpoint in _CHECKPOINTS
                and (bias is None or (bias.shape == (n,) and bias.dtype is dt
                                      and bias.get_device() == dev))
                and (residual is None or _is_matrix(residual, m, n, dt, dev))):
            return m, n, k
    except (AttributeError, IndexError, TypeError, ValueError):
        pass
    _explain_options(activation, checkpoint)
    _explain_matrix(x, "x")
    _explain_matrix(weight, "weight", cols=x.shape[1], like=x)
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError(f"weight must not be empty, got shape {tuple(weight.shape)}")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"bias must have shape [{n}]")
        if bias.dtype != x.dtype:
            raise TypeError(f"bias must be {x.dtype} like the input, got {bias.dtype}")
    if residual is not None:
        _explain_matrix(residual, "residual", x.shape[0], n, like=x)
    _explain_device(x, weight=weight, bias=bias, residual=residual)
    raise RuntimeError("unsupported arguments")


@functools.lru_cache(maxsize=4096)
def _dense_kept(m, n, k, act, bits, keep_x, keep_z):
    """Layout of z codes, z scales, x codes, x scales."""
    z = _group_bytes(m, n, bits) if keep_z and act else (None, None)
    xs = _group_bytes(m, k, 8) if keep_x and bits == 8 else (None, None)
    return _layout(*z, *xs)


@functools.lru_cache(maxsize=4096)
def _dense_workspace(m, n, k, act, bias, restore):
    """Slabs of the bias gradient, and the layout of dz, their partial sums and
    the restored x."""
    slabs = 0
    if bias:
        count = ctypes.c_int64(0)
        _call("act_backward_slabs", m, n, ctypes.byref(count))
        slabs = count.value
    return slabs, _layout(m * _up(n, 8) * 2 if act else None, slabs * n * 4 if bias else None,
                          m * _up(k, 8) * 2 if restore else None)


def _dense(x, weight, bias, activation, residual, m, n, k, bits=0, keep_x=False, keep_z=False):
    """(y, x and weight as laid out, kept buffer); launches on the current device."""
    dt, st = _DTYPES[x.dtype], _stream(x.get_device())
    out = x.new_empty((m, n))
    kept = zc = zs = xc = None
    if keep_x or keep_z:
        size, offsets = _dense_kept(m, n, k, activation is not None, bits, keep_x, keep_z)
        kept = x.new_empty(size)
        zc, zs, xc, xs = _at(kept.data_ptr(), offsets)
    if m == 0:
        return out, x, weight, kept
    if kept is None:
        a, b = _row_operands(x, weight)
    else:
        a, b = _operand(x), _operand(weight)
    if xc is not None:
        rows = a if a[3] == 0 else _operand(x, False)
        _call("checkpoint_int8", rows[1], dt, m, k, rows[2], xc, xs, st)
    if bias is not None and bias.stride(0) != 1:
        bias = bias.contiguous()
    r = None if residual is None else _plain_rows(residual)
    _call("dense_gemm", a[1], a[2], a[3], b[1], b[2], b[3], m, n, k, dt,
          None if bias is None else bias.data_ptr(), ACTIVATIONS[activation],
          None if r is None else r.data_ptr(), 0 if r is None else _row_stride(r), out.data_ptr(), n,
          zc, 0 if zc is None else bits, zs, st)
    if kept is None:
        return out, x, weight, None
    return out, _laid_out(a, x), _laid_out(b, weight), kept


def dense_forward(x, weight, bias=None, *, activation=None, residual=None, checkpoint=None):
    """``act(x @ weight.T + bias) + residual`` in one kernel.

    x [M, K], weight [N, K], bias [N], residual [M, N], all fp16 or all bf16;
    activation None, "relu", "silu", "gelu" (erf) or "gelu_tanh".
    Differentiable in all four.  ``checkpoint="int8"`` keeps x and the value
    before the activation in 8 bits for the backward pass (:class:`Int8Checkpoint`);
    y does not change.  x, weight and residual may have any strides; rows (or
    columns) that are not 16-byte aligned cost one more pass over them."""
    m, n, k = _check_dense(x, weight, bias, activation, residual, checkpoint)
    if _recorded(x, weight, bias, residual):
        return _DenseFunction.apply(x, weight, bias, residual, activation, checkpoint, m, n, k)
    if torch._C._cuda_getDevice() == x.get_device():  # a decode step: no context to enter
        return _dense(x, weight, bias, activation, residual, m, n, k)[0]
    with torch.cuda.device(x.device):
        return _dense(x, weight, bias, activation, residual, m, n, k)[0]


def dense_forward_save(x, weight, bias=None, *, activation=None, residual=None, checkpoint=None):
    """:func:`dense_forward` that also returns what :func:`dense_backward`
    needs: ``(y, saved)``.  ``saved`` refers to x (unless kept in 8 bits) and
    weight; they must not change before the backward call."""
    m, n, k = _check_dense(x, weight, bias, activation, residual, checkpoint)
    bits = 16 if checkpoint is None else 8
    with torch.no_grad(), _on(x.get_device()):
        y, xk, wk, kept = _dense(x, weight, bias, activation, residual, m, n, k, bits, True, True)
    return y, SavedDense(xk if bits == 16 else None, wk, kept, activation, (m, n, k),
                         bias is not None, bits, _stream(x.get_device()))


def dense_backward(grad_out, saved: SavedDense, *, need_x=True, need_weight=True, need_bias=True):
    """Gradients of ``y = act(x @ weight.T + bias) + residual`` given dy:
    ``(grad_x, grad_weight, grad_bias)``, None where not needed.  (The
    residual's gradient is dy.)"""
    m, n, k = saved.shape
    _refuse_tangents(grad_out)
    _explain_matrix(grad_out, "grad_out", m, n, like=saved.weight)
    _explain_device(grad_out, weight=saved.weight)
    _on_stream(saved, saved.x, saved.weight)
    with torch.no_grad(), _on(grad_out.get_device()):
        return _dense_backward(grad_out, saved.x, saved.weight, saved.kept, True, True,
                               saved.activation, m, n, k, saved.bits, need_x, need_weight,
                               need_bias and saved.has_bias)


def _dense_backward(dy, x, weight, kept, kept_x, kept_z, activation, m, n, k, bits, need_x, need_weight,
                    need_bias):
    dt, st = _DTYPES[dy.dtype], _stream(dy.get_device())
    gx = dy.new_empty((m, k)) if need_x else None
    gw = dy.new_empty((n, k)) if need_weight else None
    gb = dy.new_empty((n,)) if need_bias else None
    if m == 0:
        return gx, None if gw is None else gw.zero_(), None if gb is None else gb.zero_()
    if not (need_x or need_weight or need_bias):
        return None, None, None
    act = activation is not None
    zc, zs, xc, xsc = _at(kept.data_ptr(), _dense_kept(m, n, k, act, bits, kept_x, kept_z)[1])
    rows, d, ld, ldx = dy, (None, None, 0, 0), _up(n, 8), _up(k, 8)
    if act or need_bias:
        rows = _distinct_rows(dy)
    slabs, (size, offsets) = _dense_workspace(m, n, k, act, need_bias, need_weight and xc is not None)
    ws = dy.new_empty(size)
    dz, partial, xr = _at(ws.data_ptr(), offsets)
    if act:
        d = (ws, dz, ld, 0)
    elif need_x or need_weight:
        d = _operand(dy)
    xo = _operand(x) if need_weight and xc is None else (None, None, 0, 0)
    w = _operand(weight) if need_x else (None, None, 0, 0)
    _call("dense_backward", rows.data_ptr(), _row_stride(rows), *d[1:], *xo[1:], xc, xsc, xr, ldx, *w[1:],
          m, n, k, dt, ACTIVATIONS[activation], zc, 0 if zc is None else bits, zs, partial, slabs,
          N.ptr(gx), N.ptr(gw), N.ptr(gb), st)
    return gx, gw, gb


def _recorded(*tensors) -> bool:
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            break
    else:
        return False
    if torch.cuda.is_current_stream_capturing():
        # a backward pass that is captured while an eager graph of the same
        # leaves lives accumulates on that graph's stream and ends the process
        raise RuntimeError(
            "autograd under CUDA graph capture is not supported: capture the *_save and "
            "*_backward forms (or call under torch.no_grad())")
    return True


class _DenseFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, checkpoint, m, n, k):
        need = ctx.needs_input_grad
        bits = 16 if checkpoint is None else 8
        keep_z = need[0] or need[1] or need[2]
        args = (x, weight, bias, activation, residual, m, n, k, bits, need[1], keep_z)
        if torch._C._cuda_getDevice() == x.get_device():
            y, xk, wk, kept = _dense(*args)
        else:
            with torch.cuda.device(x.device):
                y, xk, wk, kept = _dense(*args)
        ctx.save_for_backward(wk, kept, xk if need[1] and bits == 16 else None)
        ctx.args = (need[1], keep_z, activation, m, n, k, bits)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        _refuse_tangents(grad_out)
        need = ctx.needs_input_grad
        gx = gw = gb = None
        if need[0] or need[1] or need[2]:
            w, kept, x = ctx.saved_tensors  # (the engine has made their device current)
            gx, gw, gb = _dense_backward(grad_out, x, w, kept, *ctx.args, *need[:3])
        return gx, gw, gb, grad_out if need[3] else None, None, None, None, None, None


# ---- gated feed-forward block ----

@dataclass
class SavedFeedForward:
    """What :func:`gated_feed_forward_backward` needs of a
    :func:`gated_feed_forward_save` call."""
    x: Optional[torch.Tensor]  # None: in 8 bits among `kept`
    w13: torch.Tensor
    w2: torch.Tensor
    kept: torch.Tensor         # gate and up, and their product or x in 8 bits
    activation: Optional[str]
    clamp_limit: Optional[float]
    shape: tuple
    bits: int
    stream: int


def _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint):
    """(m, hidden, inter, out) of a call whose arguments go together; raises otherwise."""
    _refuse_tangents(x, w13, w2, residual)
    try:
        (m, hidden), (out, inter), dt, dev = x.shape, w2.shape, x.dtype, x.get_device()
        if (hidden and out and inter and dev >= 0 and dt in _DTYPES
                and _is_matrix(w13, 2 * inter, hidden, dt, dev)
                and w2.dtype is dt and w2.get_device() == dev
                and activation in ACTIVATIONS and checkpoint in _CHECKPOINTS
                and (clamp_limit is None or 0 < float(clamp_limit) < math.inf)
                and (residual is None or _is_matrix(residual, m, out, dt, dev))):
            return m, hidden, inter, out
    except (AttributeError, IndexError, TypeError, ValueError):
        pass
    _explain_options(activation, checkpoint, clamp_limit)
    _explain_matrix(x, "x")
    m, hidden = x.shape
    _explain_matrix(w13, "w13", cols=hidden, like=x)
    if w13.shape[0] == 0 or hidden == 0 or w13.shape[0] % 2:
        raise ValueError("w13 must hold gate rows and as many up rows, [2 * intermediate, hidden], "
                         f"got {tuple(w13.shape)}")
    _explain_matrix(w2, "w2", cols=w13.shape[0] // 2, like=x)
    if w2.shape[0] == 0:
        raise ValueError("w2 must not be empty")
    if residual is not None:
        _explain_matrix(residual, "residual", m, w2.shape[0], like=x)
    _explain_device(x, w13=w13, w2=w2, residual=residual)
    raise RuntimeError("unsupported arguments")


def _limit_args(clamp_limit):
    return (0, 0.0) if clamp_limit is None else (1, float(clamp_limit))


@functools.lru_cache(maxsize=4096)
def _ffn_kept(m, hidden, inter, bits, keep_x, keep_z, keep_h):
    """Layout of z codes, z scales, x codes, x scales, h."""
    z = _group_bytes(m, 2 * _up(inter, _GROUP), bits) if keep_z else (None, None)
    xs = _group_bytes(m, hidden, 8) if keep_x and bits == 8 else (None, None)
    return _layout(*z, *xs, m * _up(inter, 8) * 2 if keep_h else None)


def _ffn(x, w13, w2, activation, clamp_limit, residual, m, hidden, inter, n, bits=0, keep_x=False,
         keep_z=False, keep_h=False):
    """(y, x, w13 and w2 as laid out, kept buffer); launches on the current device."""
    out = x.new_empty((m, n))
    ldh = _up(inter, 8)
    kept = zc = zs = xc = xs = h = None
    if keep_x or keep_z or keep_h:
        size, offsets = _ffn_kept(m, hidden, inter, bits, keep_x, keep_z, keep_h)
        kept = x.new_empty(size)
        zc, zs, xc, xs, h = _at(kept.data_ptr(), offsets)
    if h is None:
        ws = x.new_empty((m, ldh))
        h = ws.data_ptr()
    if m == 0:
        return out, x, w13, w2, kept
    # w13 stored by columns: its up rows begin `inter` elements into a row;
    # x to be kept in 8 bits is read by rows
    if zc is None and xc is None:
        a, b = _row_operands(x, w13, inter & 7 == 0)
    else:
        a, b = _operand(x, xc is None), _operand(w13, inter & 7 == 0)
    c = (w2, w2.data_ptr(), w2.stride(0), 0) if m <= _FEW and w2.stride(1) == 1 and w2.stride(0) >= inter \
        else _operand(w2)
    r = None if residual is None else _plain_rows(residual)
    _call("gated_feed_forward", a[1], a[2], a[3], b[1], b[2], b[3], c[1], c[2], c[3], m, hidden, inter,
          n, _DTYPES[x.dtype], ACTIVATIONS[activation], *_limit_args(clamp_limit),
          None if r is None else r.data_ptr(), 0 if r is None else _row_stride(r), h, ldh,
          out.data_ptr(), n, zc, 0 if zc is None else bits, zs, xc, xs, _stream(x.get_device()))
    if kept is None:
        return out, x, w13, w2, None
    return out, _laid_out(a, x), _laid_out(b, w13), _laid_out(c, w2), kept


def gated_feed_forward(x, w13, w2, *, activation="silu", clamp_limit=None, residual=None,
                       checkpoint=None):
    """``(act(min(g, L)) * clamp(u, -L, L)) @ w2.T + residual`` with ``g, u`` the
    halves of ``x @ w13.T``: a shared expert or dense feed-forward layer in two
    kernels (both projections, the activation and the product in one, the
    down projection with the residual in the other).

    x [M, hidden], w13 [2 * intermediate, hidden] (gate rows, then up rows,
    as the routed experts' W13), w2 [out, intermediate], residual [M, out];
    all fp16 or all bf16.  ``clamp_limit`` is L (none: no clamp).
    With the routed experts' output as ``residual`` the result is the whole
    MoE layer's.  Differentiable in x, w13, w2 and residual (the routed experts
    have no backward pass: what x contributes through them is not in its
    gradient).  The product between the two kernels is rounded to 16 bits; in
    fp16 without a clamp it is infinite past 65,504.
    ``checkpoint="int8"`` keeps x, g and u in 8 bits for the backward pass and
    forms the product again there; y does not change."""
    shape = _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint)
    if _recorded(x, w13, w2, residual):
        return _FeedForwardFunction.apply(x, w13, w2, residual, activation, clamp_limit, checkpoint,
                                          shape)
    if torch._C._cuda_getDevice() == x.get_device():
        return _ffn(x, w13, w2, activation, clamp_limit, residual, *shape)[0]
    with torch.cuda.device(x.device):
        return _ffn(x, w13, w2, activation, clamp_limit, residual, *shape)[0]


def gated_feed_forward_save(x, w13, w2, *, activation="silu", clamp_limit=None, residual=None,
                            checkpoint=None):
    """:func:`gated_feed_forward` that also returns what
    :func:`gated_feed_forward_backward` needs: ``(y, saved)``.  ``saved``
    refers to x (unless kept in 8 bits), w13 and w2; they must not change
    before the backward call."""
    shape = _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint)
    bits = 16 if checkpoint is None else 8
    with torch.no_grad(), _on(x.get_device()):
        y, xk, w13k, w2k, kept = _ffn(x, w13, w2, activation, clamp_limit, residual, *shape, bits, True,
                                      True, bits == 16)
    return y, SavedFeedForward(xk if bits == 16 else None, w13k, w2k, kept, activation, clamp_limit,
                               shape, bits, _stream(x.get_device()))


def gated_feed_forward_backward(grad_out, saved: SavedFeedForward, *, need_x=True, need_w13=True,
                                need_w2=True):
    """Gradients of the block given dy: ``(grad_x, grad_w13, grad_w2)``, None
    where not needed.  (The residual's gradient is dy.)

    The gradient of the gated product, ``dh = dy @ w2``, stays in the
    registers of the kernel that turns it into the gradients of gate and up."""
    m, hidden, inter, n = saved.shape
    _refuse_tangents(grad_out)
    _explain_matrix(grad_out, "grad_out", m, n, like=saved.w2)
    _explain_device(grad_out, w2=saved.w2)
    _on_stream(saved, saved.x, saved.w13, saved.w2)
    with torch.no_grad(), _on(grad_out.get_device()):
        return _ffn_backward(grad_out, saved.x, saved.w13, saved.w2, saved.kept, True, True,
                             saved.bits == 16, saved.activation, saved.clamp_limit, *saved.shape,
                             saved.bits, need_x, need_w13, need_w2)


def _ffn_backward(grad_out, x, w13, w2, kept, kept_x, kept_z, kept_h, activation, clamp_limit, m,
                  hidden, inter, n, bits, need_x, need_w13, need_w2):
    gx = grad_out.new_empty((m, hidden)) if need_x else None
    g13 = grad_out.new_empty((2 * inter, hidden)) if need_w13 else None
    g2 = grad_out.new_empty((n, inter)) if need_w2 else None
    if m == 0:
        return gx, None if g13 is None else g13.zero_(), None if g2 is None else g2.zero_()
    if not (need_x or need_w13 or need_w2):
        return None, None, None
    zc, zs, xc, xs, h = _at(kept.data_ptr(),
                            _ffn_kept(m, hidden, inter, bits, kept_x, kept_z, kept_h)[1])
    form_h = need_w2 and not kept_h
    ldh, lddz, ldx = _up(inter, 8), _up(2 * inter, 8), _up(hidden, 8)
    size, offsets = _layout(m * lddz * 2 if need_x or need_w13 or form_h else None,
                            m * ldh * 2 if form_h else None,
                            m * ldx * 2 if need_w13 and xc is not None else None)
    ws = grad_out.new_empty(size)
    dz, hw, xr = _at(ws.data_ptr(), offsets)
    none = (None, None, 0, 0)
    dy, w = _operand(grad_out), _operand(w2)
    u = _operand(w13) if need_x else none
    xo = _operand(x) if need_w13 and xc is None else none
    _call("gated_feed_forward_backward", *dy[1:], *xo[1:], xc, xs, xr, ldx, *u[1:], *w[1:], m, hidden, inter,
          n, _DTYPES[grad_out.dtype], ACTIVATIONS[activation], *_limit_args(clamp_limit), zc,
          0 if zc is None else bits, zs, hw if form_h else h, ldh, int(form_h), dz, lddz, N.ptr(gx),
          N.ptr(g13), N.ptr(g2), _stream(grad_out.get_device()))
    return gx, g13, g2


class _FeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, residual, activation, clamp_limit, checkpoint, shape):
        need = ctx.needs_input_grad
        bits = 16 if checkpoint is None else 8
        inner = need[0] or need[1]
        # w2's gradient alone needs h only, which is no larger than z in 8 bits
        keep_h = need[2] and (bits == 16 or not inner)
        args = (x, w13, w2, activation, clamp_limit, residual, *shape, bits, need[1], inner, keep_h)
        if torch._C._cuda_getDevice() == x.get_device():
            y, xk, w13k, w2k, kept = _ffn(*args)
        else:
            with torch.cuda.device(x.device):
                y, xk, w13k, w2k, kept = _ffn(*args)
        ctx.save_for_backward(w13k, w2k, kept, xk if need[1] and bits == 16 else None)
        ctx.args = (need[1], inner, keep_h, activation, clamp_limit, *shape, bits)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        _refuse_tangents(grad_out)
        need = ctx.needs_input_grad
        gx = g13 = g2 = None
        if need[0] or need[1] or need[2]:
            w13, w2, kept, x = ctx.saved_tensors  # (the engine has made their device current)
            gx, g13, g2 = _ffn_backward(grad_out, x, w13, w2, kept, *ctx.args, *need[:3])
        return gx, g13, g2, grad_out if need[3] else None, None, None, None, None

"""16-bit feed-forward operators for B200 (sm_100a): what stands next to the
routed MXFP4 experts in a DeepSeek-style layer (shared expert, dense layers,
projections), forward and backward.

    dense_forward          y = act(x @ weight.T + bias) + residual
    gated_feed_forward     y = (act(x @ w1.T) * (x @ w3.T)) @ w2.T + residual,  w13 = [w1; w3]
    checkpoint_int8 / restore_int8    activations kept in 8 bits

bf16 and fp16; sums, activations and their slopes in fp32, one rounding where
a value is stored.  ``dense_forward`` and ``gated_feed_forward`` are
differentiable; their ``*_save`` / ``*_backward`` forms give the same steps
without autograd (and are the ones to capture into a CUDA graph).  With
``checkpoint="int8"`` what the backward pass needs is kept in 8 bits.  Every
call is asynchronous on the current stream of the tensors' device; there is
no CPU path.

Results follow the inputs' values: NaN and infinities propagate as the
formulas say.  All results are the same bits from call to call.
"""

from __future__ import annotations

import contextlib
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _native as N

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_DTYPES = {torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_CHECKPOINT_DTYPES = {torch.float32: N.DTYPE_F32, **_DTYPES}
_GROUP = 32


# ---- argument checks ----

def _check_matrix(t, name: str, rows=None, cols=None, like=None) -> None:
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


def _check_device(first: torch.Tensor, **others) -> None:
    if not first.is_cuda:
        raise RuntimeError("the feed-forward operators need CUDA tensors on an sm_100a device "
                           "(no CPU path)")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{name} is on {t.device}, expected {first.device}")


def _check_options(activation, checkpoint, clamp_limit=None) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if checkpoint not in (None, "int8"):
        raise ValueError(f'checkpoint must be None or "int8", got {checkpoint!r}')
    if clamp_limit is not None and not (0 < float(clamp_limit) < math.inf):
        raise ValueError(f"clamp_limit must be positive and finite, got {clamp_limit}")


def _on(device: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    if torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


# ---- operands ----

def _up(v: int, to: int) -> int:
    return -(-v // to) * to


def _rows_buffer(rows: int, cols: int, like: torch.Tensor) -> torch.Tensor:
    """[rows, cols] with rows at multiples of 16 bytes."""
    return torch.empty((rows, _up(cols, 8)), dtype=like.dtype, device=like.device)[:, :cols]


class _Operand:
    """A 2-D tensor as a product reads it: rows or columns contiguous and
    16-byte aligned.  Others are laid out anew (one pass over them).
    ``columns`` False: only contiguous rows will do."""

    __slots__ = ("t", "ptr", "ld", "mn")

    def __init__(self, t: torch.Tensor, columns: bool = True):
        rows, cols = t.shape
        s0, s1 = t.stride()
        ptr = t.data_ptr()
        self.t, self.ptr = t, ptr
        if ptr % 16 == 0:
            if (s1 == 1 or cols == 1) and rows == 1:
                self.ld, self.mn = _up(cols, 8), 0
                return
            if s1 == 1 and s0 % 8 == 0 and s0 >= cols:
                self.ld, self.mn = s0, 0
                return
            if columns and s0 == 1 and cols == 1:
                self.ld, self.mn = _up(rows, 8), 1
                return
            if columns and s0 == 1 and s1 % 8 == 0 and s1 >= rows:
                self.ld, self.mn = s1, 1
                return
        self.t = _rows_buffer(rows, cols, t)
        self.ptr, self.ld, self.mn = self.t.data_ptr(), self.t.stride(0), 0
        N.call("dsv4_b200_pack_rows", ptr, s0, s1, rows, cols, self.ptr, self.ld, _stream(t))


def _plain_rows(t: torch.Tensor) -> torch.Tensor:
    """A tensor whose rows are contiguous (any alignment; row stride 0 allowed)."""
    if t.stride(1) == 1 or t.shape[1] == 1:
        if t.shape[0] <= 1 or t.stride(0) >= t.shape[1] or t.stride(0) == 0:
            return t
    return t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _gemm(a: _Operand, a_mn: int, b: _Operand, b_mn: int, m: int, n: int, k: int, dtype, out, *,
          bias=None, activation=None, residual=None, z=None, codes=None, scales=None) -> None:
    N.call("dsv4_b200_dense_gemm", a.ptr, a.ld, a_mn, b.ptr, b.ld, b_mn, m, n, k, _DTYPES[dtype],
           N.ptr(bias), ACTIVATIONS[activation], N.ptr(residual),
           0 if residual is None else _row_stride(residual), out.data_ptr(), _row_stride(out),
           N.ptr(z), 0 if z is None else z.stride(0), N.ptr(codes), N.ptr(scales),
           _stream(out))


# ---- 8-bit checkpoints ----

@dataclass
class Int8Checkpoint:
    """Rows of activations in 8 bits: ``codes`` int8 [M, K up to 32], ``scales``
    fp32 [groups, M].  32 consecutive values of a row share a scale
    ``amax / 127`` (rounded toward zero); a code is ``127 v / amax`` rounded to the nearest whole
    number, ties to even.  A group that holds an infinity or a NaN is restored
    as NaN, one whose largest magnitude is below 2^-100 as zeros."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    dtype: torch.dtype


def _empty_codes(rows: int, cols: int, device):
    k32 = _up(cols, _GROUP)
    return (torch.empty((rows, k32), dtype=torch.int8, device=device),
            torch.empty((k32 // _GROUP, rows), dtype=torch.float32, device=device))


def checkpoint_int8(x: torch.Tensor) -> Int8Checkpoint:
    """Keep the rows of ``x`` [M, K] (fp32, fp16 or bf16) in 8 bits: 1.125
    bytes per value.  ``restore_int8(checkpoint_int8(x))`` differs from x by at
    most half a step, ``amax / 254`` of its group, and the rounding to x's type."""
    if x.dim() != 2:
        raise ValueError(f"x must be 2-D, got shape {tuple(x.shape)}")
    if x.dtype not in _CHECKPOINT_DTYPES:
        raise TypeError(f"x must be fp32, fp16 or bf16, got {x.dtype}")
    if x.shape[1] == 0:
        raise ValueError("x has no columns")
    _check_device(x)
    x = _plain_rows(x.detach())
    m, k = x.shape
    if m > 1 and x.stride(0) == 0:
        x = x.contiguous()
    with _on(x.device):
        codes, scales = _empty_codes(m, k, x.device)
        N.call("dsv4_b200_checkpoint_int8", x.data_ptr(), _CHECKPOINT_DTYPES[x.dtype], m, k,
               _row_stride(x), codes.data_ptr(), scales.data_ptr(), _stream(x))
    return Int8Checkpoint(codes, scales, (m, k), x.dtype)


def restore_int8(checkpoint: Int8Checkpoint, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The kept rows, in their own type or in ``dtype``."""
    dtype = checkpoint.dtype if dtype is None else dtype
    if dtype not in _CHECKPOINT_DTYPES:
        raise TypeError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
    m, k = checkpoint.shape
    k32 = _up(k, _GROUP)
    c, s = checkpoint.codes, checkpoint.scales
    if (c.dtype != torch.int8 or tuple(c.shape) != (m, k32) or not c.is_contiguous()
            or s.dtype != torch.float32 or tuple(s.shape) != (k32 // _GROUP, m)
            or not s.is_contiguous()):
        raise ValueError(f"codes must be contiguous int8 [{m}, {k32}] and scales contiguous fp32 "
                         f"[{k32 // _GROUP}, {m}]")
    _check_device(c, scales=s)
    with _on(c.device):
        return _restore(c, s, m, k, torch.empty((m, k), dtype=dtype, device=c.device))


def _restore(codes, scales, m, k, out):
    N.call("dsv4_b200_restore_int8", codes.data_ptr(), scales.data_ptr(), m, k, out.data_ptr(),
           _CHECKPOINT_DTYPES[out.dtype], _row_stride(out), _stream(out))
    return out


class _Kept:
    """An input as the backward pass gets it back: itself, or its 8-bit codes."""

    __slots__ = ("tensors", "shape", "dtype")

    def __init__(self, x: torch.Tensor, checkpoint):
        self.shape, self.dtype = tuple(x.shape), x.dtype
        if checkpoint is None:
            self.tensors = (x,)
        else:
            c = checkpoint_int8(x)
            self.tensors = (c.codes, c.scales)

    def operand(self) -> _Operand:
        if len(self.tensors) == 1:
            return _Operand(self.tensors[0])
        m, k = self.shape
        out = torch.empty((m, _up(k, 8)), dtype=self.dtype, device=self.tensors[0].device)[:, :k]
        return _Operand(_restore(*self.tensors, m, k, out))


# ---- dense product ----

@dataclass
class SavedDense:
    """What :func:`dense_backward` needs of a :func:`dense_forward_save` call."""
    x: Optional[_Kept]
    weight: torch.Tensor
    z: Optional[tuple]  # (z,) in 16 bits, (codes, scales), or None without an activation
    activation: Optional[str]
    shape: tuple
    has_bias: bool


def _check_dense(x, weight, bias, activation, residual, checkpoint):
    _check_options(activation, checkpoint)
    _check_matrix(x, "x")
    _check_matrix(weight, "weight", cols=x.shape[1], like=x)
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError(f"weight must not be empty, got shape {tuple(weight.shape)}")
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"bias must have shape [{n}], got {tuple(bias.shape)}")
        if bias.dtype != x.dtype:
            raise TypeError(f"bias must be {x.dtype} like the input, got {bias.dtype}")
    if residual is not None:
        _check_matrix(residual, "residual", x.shape[0], n, like=x)
    _check_device(x, weight=weight, bias=bias, residual=residual)


def _dense(x, weight, bias, activation, residual, checkpoint, save, keep_x):
    m, k = x.shape
    n = weight.shape[0]
    with _on(x.device):
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
        z = kept = None
        codes = scales = None
        if save:
            if keep_x:
                kept = _Kept(x, checkpoint)
            if activation is not None:
                if checkpoint is None:
                    z = _rows_buffer(m, n, x)
                else:
                    codes, scales = _empty_codes(m, n, x.device)
        if m:
            a, b = _Operand(x), _Operand(weight)
            _gemm(a, a.mn, b, b.mn, m, n, k, x.dtype, out,
                  bias=None if bias is None else bias.contiguous(), activation=activation,
                  residual=None if residual is None else _plain_rows(residual), z=z, codes=codes,
                  scales=scales)
    if not save:
        return out, None
    zs = (z,) if z is not None else None if codes is None else (codes, scales)
    return out, SavedDense(kept, weight, zs, activation, (m, n, k), bias is not None)


def dense_forward_save(x, weight, bias=None, *, activation=None, residual=None, checkpoint=None):
    """:func:`dense_forward` that also returns what :func:`dense_backward`
    needs: ``(y, saved)``.  ``saved`` refers to x (unless kept in 8 bits) and
    weight; they must not change before the backward call."""
    _check_dense(x, weight, bias, activation, residual, checkpoint)
    with torch.no_grad():
        return _dense(x, weight, bias, activation, residual, checkpoint, True, True)


def dense_backward(grad_out, saved: SavedDense, *, need_x=True, need_weight=True, need_bias=True):
    """Gradients of ``y = act(x @ weight.T + bias) + residual`` given dy:
    ``(grad_x, grad_weight, grad_bias)``, None where not needed.  (The
    residual's gradient is dy.)"""
    m, n, k = saved.shape
    _check_matrix(grad_out, "grad_out", m, n, like=saved.weight)
    _check_device(grad_out, weight=saved.weight)
    need_bias = need_bias and saved.has_bias
    dev, dt = grad_out.device, grad_out.dtype
    gx = gw = gb = None
    with torch.no_grad(), _on(dev):
        if need_x:
            gx = torch.empty((m, k), dtype=dt, device=dev)
        if need_weight:
            if saved.x is None:
                raise RuntimeError("the forward call did not keep x")
            gw = torch.empty((n, k), dtype=dt, device=dev)
        if need_bias:
            gb = torch.empty((n,), dtype=dt, device=dev)
        if m == 0:
            return gx, None if gw is None else gw.zero_(), None if gb is None else gb.zero_()
        if not (need_x or need_weight or need_bias):
            return None, None, None
        act = saved.activation
        dy = grad_out
        dz = dy if act is None else _rows_buffer(m, n, dy)
        if act is not None or need_bias:
            if dy.stride(1) != 1 or (m > 1 and dy.stride(0) < n):
                dy = dy.contiguous()
            partial, slabs = None, 0
            if need_bias:
                slabs = _slabs(m, n)
                partial = torch.empty((slabs, n), dtype=torch.float32, device=dev)
            z, codes, scales = _z_parts(saved.z)
            N.call("dsv4_b200_act_backward", dy.data_ptr(), _row_stride(dy), N.ptr(z),
                   0 if z is None else z.stride(0), N.ptr(codes), N.ptr(scales), m, n, _DTYPES[dt],
                   ACTIVATIONS[act], None if act is None else dz.data_ptr(),
                   n if act is None else dz.stride(0), N.ptr(partial), slabs, N.ptr(gb),
                   _stream(dy))
            if act is None:
                dz = dy
        if need_x or need_weight:
            d = _Operand(dz)
        if need_x:
            w = _Operand(saved.weight)
            _gemm(d, d.mn, w, 1 - w.mn, m, k, n, dt, gx)
        if need_weight:
            xo = saved.x.operand()
            _gemm(d, 1 - d.mn, xo, 1 - xo.mn, n, k, m, dt, gw)
    return gx, gw, gb


def _z_parts(kept):
    if kept is None:
        return None, None, None
    return (kept[0], None, None) if len(kept) == 1 else (None, *kept)


def _slabs(m: int, n: int) -> int:
    import ctypes
    v = ctypes.c_int64(0)
    N.call("dsv4_b200_act_backward_slabs", m, n, ctypes.byref(v))
    return v.value


def dense_forward(x, weight, bias=None, *, activation=None, residual=None, checkpoint=None):
    """``act(x @ weight.T + bias) + residual`` in one kernel.

    x [M, K], weight [N, K], bias [N], residual [M, N], all fp16 or all bf16;
    activation None, "relu", "silu", "gelu" (erf) or "gelu_tanh".
    Differentiable in all four.  ``checkpoint="int8"`` keeps x and the value
    before the activation in 8 bits for the backward pass (:class:`Int8Checkpoint`);
    y does not change.  x, weight and residual may have any strides; rows (or
    columns) that are not 16-byte aligned cost one more pass over them."""
    _check_dense(x, weight, bias, activation, residual, checkpoint)
    if not _recorded(x, weight, bias, residual):
        return _dense(x, weight, bias, activation, residual, None, False, False)[0]
    return _DenseFunction.apply(x, weight, bias, residual, activation, checkpoint)


def _recorded(*tensors) -> bool:
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)):
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
    def forward(ctx, x, weight, bias, residual, activation, checkpoint):
        need = ctx.needs_input_grad
        y, saved = _dense(x, weight, bias, activation, residual, checkpoint, any(need[:3]), need[1])
        if saved is not None:
            xs = () if saved.x is None else saved.x.tensors
            zs = saved.z or ()
            ctx.save_for_backward(weight, *xs, *zs)
            ctx.counts = (len(xs), len(zs))
            saved.weight = None
            saved.z = None
            if saved.x is not None:
                saved.x.tensors = ()
            ctx.saved = saved
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        need = ctx.needs_input_grad
        gx = gw = gb = None
        if any(need[:3]):
            gx, gw, gb = dense_backward(grad_out, _unpack(ctx), need_x=need[0], need_weight=need[1],
                                        need_bias=need[2])
        return gx, gw, gb, grad_out if need[3] else None, None, None


def _unpack(ctx):
    """The saved object of a context, its tensors taken from autograd (which
    checks that they were not changed in place)."""
    import copy
    nx, nz = ctx.counts
    weight, *rest = ctx.saved_tensors
    s = copy.copy(ctx.saved)
    s.weight = weight
    if nx:
        s.x = copy.copy(s.x)
        s.x.tensors = tuple(rest[:nx])
    s.z = tuple(rest[nx:nx + nz]) or None
    return s


# ---- gated feed-forward block ----

@dataclass
class SavedFeedForward:
    """What :func:`gated_feed_forward_backward` needs of a
    :func:`gated_feed_forward_save` call."""
    x: Optional[_Kept]
    weight: torch.Tensor  # w13
    w2: torch.Tensor
    z: Optional[tuple]    # (z,) [M, 2I] in 16 bits, or (codes, scales)
    h: Optional[torch.Tensor]  # the gated product; formed again from z when kept in 8 bits
    activation: Optional[str]
    clamp_limit: Optional[float]
    shape: tuple


def _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint):
    _check_options(activation, checkpoint, clamp_limit)
    _check_matrix(x, "x")
    m, hidden = x.shape
    _check_matrix(w13, "w13", cols=hidden, like=x)
    if w13.shape[0] == 0 or hidden == 0 or w13.shape[0] % 2:
        raise ValueError("w13 must hold gate rows and as many up rows, [2 * intermediate, hidden], "
                         f"got {tuple(w13.shape)}")
    inter = w13.shape[0] // 2
    _check_matrix(w2, "w2", cols=inter, like=x)
    if w2.shape[0] == 0:
        raise ValueError("w2 must not be empty")
    if residual is not None:
        _check_matrix(residual, "residual", m, w2.shape[0], like=x)
    _check_device(x, w13=w13, w2=w2, residual=residual)


def _limit_args(clamp_limit):
    return (0, 0.0) if clamp_limit is None else (1, float(clamp_limit))


def _ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint, keep_x, keep_z, keep_h):
    m, hidden = x.shape
    inter, n = w2.shape[1], w2.shape[0]
    kept = z = codes = scales = None
    with _on(x.device):
        out = torch.empty((m, n), dtype=x.dtype, device=x.device)
        h = _rows_buffer(m, inter, x)
        if keep_x:
            kept = _Kept(x, checkpoint)
        if keep_z and checkpoint is None:
            z = _rows_buffer(m, 2 * inter, x)
        elif keep_z:
            i32 = _up(inter, _GROUP)
            codes, scales = _empty_codes(m, 2 * i32, x.device)
        if m:
            # stored by columns, the up rows begin `inter` elements into a row
            a, b = _Operand(x), _Operand(w13, columns=inter % 8 == 0)
            N.call("dsv4_b200_gated_gemm", a.ptr, a.ld, a.mn, b.ptr, b.ld, b.mn, m, inter, hidden,
                   _DTYPES[x.dtype], ACTIVATIONS[activation], *_limit_args(clamp_limit),
                   h.data_ptr(), h.stride(0), N.ptr(z),
                   0 if z is None else z.stride(0), N.ptr(codes), N.ptr(scales), _stream(x))
            a, b = _Operand(h), _Operand(w2)
            _gemm(a, a.mn, b, b.mn, m, n, inter, x.dtype, out,
                  residual=None if residual is None else _plain_rows(residual))
    zs = (z,) if z is not None else None if codes is None else (codes, scales)
    return out, SavedFeedForward(kept, w13, w2, zs, h if keep_h else None, activation, clamp_limit,
                                 (m, hidden, inter, n))


def gated_feed_forward_save(x, w13, w2, *, activation="silu", clamp_limit=None, residual=None,
                            checkpoint=None):
    """:func:`gated_feed_forward` that also returns what
    :func:`gated_feed_forward_backward` needs: ``(y, saved)``.  ``saved``
    refers to x (unless kept in 8 bits), w13 and w2; they must not change
    before the backward call."""
    _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint)
    with torch.no_grad():
        return _ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint, True, True,
                    checkpoint is None)


def gated_feed_forward_backward(grad_out, saved: SavedFeedForward, *, need_x=True, need_w13=True,
                                need_w2=True):
    """Gradients of the block given dy: ``(grad_x, grad_w13, grad_w2)``, None
    where not needed.  (The residual's gradient is dy.)

    The gradient of the gated product, ``dh = dy @ w2``, stays in the
    registers of the kernel that turns it into the gradients of gate and up."""
    m, hidden, inter, n = saved.shape
    _check_matrix(grad_out, "grad_out", m, n, like=saved.w2)
    _check_device(grad_out, w2=saved.w2)
    dev, dt = grad_out.device, grad_out.dtype
    gx = g13 = g2 = None
    with torch.no_grad(), _on(dev):
        if need_x:
            gx = torch.empty((m, hidden), dtype=dt, device=dev)
        if need_w13:
            g13 = torch.empty((2 * inter, hidden), dtype=dt, device=dev)
        if need_w2:
            g2 = torch.empty((n, inter), dtype=dt, device=dev)
        if m == 0:
            return gx, None if g13 is None else g13.zero_(), None if g2 is None else g2.zero_()
        if (need_w13 and saved.x is None) or ((need_x or need_w13) and saved.z is None):
            raise RuntimeError("the forward call did not keep what this gradient needs")
        if not (need_x or need_w13 or need_w2):
            return None, None, None
        dy = _Operand(grad_out)
        h = saved.h
        dz = None
        form_h = need_w2 and h is None
        if need_x or need_w13 or form_h:
            w2 = _Operand(saved.w2)
            dz = _rows_buffer(m, 2 * inter, grad_out)
            if form_h:
                h = _rows_buffer(m, inter, grad_out)
            z, codes, scales = _z_parts(saved.z)
            N.call("dsv4_b200_gated_backward_gemm", dy.ptr, dy.ld, dy.mn, w2.ptr, w2.ld, 1 - w2.mn,
                   m, inter, n, _DTYPES[dt], ACTIVATIONS[saved.activation],
                   *_limit_args(saved.clamp_limit), N.ptr(z), 0 if z is None else z.stride(0),
                   N.ptr(codes), N.ptr(scales), dz.data_ptr(), dz.stride(0),
                   h.data_ptr() if form_h else None, h.stride(0) if form_h else 0,
                   _stream(grad_out))
        if need_w2:
            ho = _Operand(h)
            _gemm(dy, 1 - dy.mn, ho, 1 - ho.mn, n, inter, m, dt, g2)
        if need_x or need_w13:
            d = _Operand(dz)
        if need_x:
            w = _Operand(saved.weight)
            _gemm(d, d.mn, w, 1 - w.mn, m, hidden, 2 * inter, dt, gx)
        if need_w13:
            xo = saved.x.operand()
            _gemm(d, 1 - d.mn, xo, 1 - xo.mn, 2 * inter, hidden, m, dt, g13)
    return gx, g13, g2


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
    MoE layer's.  Differentiable in x, w13, w2 and residual;
    ``checkpoint="int8"`` keeps x, g and u in 8 bits for the backward pass and
    forms the product again there; y does not change."""
    _check_ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint)
    if not _recorded(x, w13, w2, residual):
        return _ffn(x, w13, w2, activation, clamp_limit, residual, None, False, False, False)[0]
    return _FeedForwardFunction.apply(x, w13, w2, residual, activation, clamp_limit, checkpoint)


class _FeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2, residual, activation, clamp_limit, checkpoint):
        need = ctx.needs_input_grad
        inner = need[0] or need[1]
        # w2's gradient alone needs h only, which is no larger than z in 8 bits
        keep_h = need[2] and (checkpoint is None or not inner)
        y, saved = _ffn(x, w13, w2, activation, clamp_limit, residual, checkpoint, need[1], inner,
                        keep_h)
        xs = () if saved.x is None else saved.x.tensors
        zs = saved.z or ()
        hs = () if saved.h is None else (saved.h,)
        ctx.save_for_backward(w13, *xs, *zs, w2, *hs)
        ctx.counts = (len(xs), len(zs))
        saved.weight = saved.w2 = saved.z = saved.h = None
        if saved.x is not None:
            saved.x.tensors = ()
        ctx.saved = saved
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        need = ctx.needs_input_grad
        gx = g13 = g2 = None
        if any(need[:3]):
            s = _unpack(ctx)
            s.w2, *hs = ctx.saved_tensors[1 + sum(ctx.counts):]
            s.h = hs[0] if hs else None
            gx, g13, g2 = gated_feed_forward_backward(grad_out, s, need_x=need[0], need_w13=need[1],
                                                      need_w2=need[2])
        return gx, g13, g2, grad_out if need[3] else None, None, None, None

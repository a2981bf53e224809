"""Activation checkpoints in 8 bits and their use in the backward pass.

What a backward pass needs of an activation is kept as e4m3 values with one power-of-two scale
per 32 columns (csrc/kernels/ckpt8.hip): 1.03 bytes per value instead of 2.  The forward result is
that of the plain layer; only the saved copy is rounded (half an e4m3 step, 2^-4 relative):

* ``bias_gelu(x, b)``   GELU whose backward takes the derivative at the kept x + b;
* ``linear(x, w, b)``   a linear layer whose weight gradient reads the kept x;
* ``ffn(x, w1, b1, w2)``  both layers of the transformer FFN: x and the GELU's input in 8 bits, the
  GELU's output not kept at all (recomputed from its input in the backward): 5.2 bytes per token and
  hidden unit (intermediate = 4 x hidden) instead of 18;
* ``pack`` / ``unpack`` for any activation.

CPU: the same rounding in plain torch.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

from .. import _native
from . import dense as dops
from . import grad_sink
from . import transformer as tops
from ._common import P, check, lib, on_device, refuse_held_capture, stream, use_hip

BLOCK = 32
FP8_MAX = 448.0
_K, _C = math.sqrt(2.0 / math.pi), 0.044715


class Packed(NamedTuple):
    """A checkpoint: ``q`` (..., D) uint8 e4m3 bytes, ``s`` (..., ceil(D / 32)) uint8 exponents + 127 (255: the
    block is not finite), ``dtype`` of the activation."""

    q: torch.Tensor
    s: torch.Tensor
    dtype: torch.dtype


def _blocks(D: int) -> int:
    return -(-D // BLOCK)


def _check_x(x: torch.Tensor, name: str) -> None:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{name}: needs at least one column, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: takes bfloat16 or float32, got {x.dtype}")
    if x.numel() // x.shape[-1] >= 1 << 31 or x.shape[-1] > 1 << 24:
        raise ValueError(f"{name}: shape {tuple(x.shape)} is outside the kernels' range")


def _check_packed(p: "Packed", name: str) -> None:
    D = p.q.shape[-1] if p.q.dim() else 0
    if D == 0:
        raise ValueError(f"{name}: needs at least one column, got shape {tuple(p.q.shape)}")
    if p.q.dtype != torch.uint8 or p.s.dtype != torch.uint8 or p.s.shape != (*p.q.shape[:-1], _blocks(D)):
        raise ValueError(f"{name}: {tuple(p.q.shape)} {p.q.dtype} values do not go with {tuple(p.s.shape)} {p.s.dtype} scales")
    if p.q.device != p.s.device:
        raise ValueError(f"{name}: values and scales are on different devices")


def _same_device(x: torch.Tensor, name: str, **others: Optional[torch.Tensor]) -> None:
    for what, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: {what} is on {t.device}, x on {x.device}")


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e (fp32), -126 <= e <= 127, from its bit pattern."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pack_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    D = x.shape[-1]
    nb = _blocks(D)
    b = F.pad(x.float(), (0, nb * BLOCK - D)).reshape(*x.shape[:-1], nb, BLOCK)
    top = b.abs().amax(-1)
    mant, ex = torch.frexp(top)
    e = torch.where(top == 0, -126, ex - 9 + (mant > 0.875).int()).clamp(-126, 126)
    fine = torch.isfinite(top)
    e = torch.where(fine, e, torch.zeros_like(e))
    q = (b * _pow2(-e).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    q = torch.where(fine.unsqueeze(-1), q, torch.full_like(q, 0x7F))
    s = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return q.reshape(*x.shape[:-1], nb * BLOCK)[..., :D].contiguous(), s


def _unpack_reference(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    r = torch.where(s == 255, torch.full(s.shape, float("nan"), device=s.device), _pow2(s.int().clamp(1, 254) - 127))
    return q.view(torch.float8_e4m3fn).float() * r.repeat_interleave(BLOCK, -1)[..., :q.shape[-1]]


def _alloc(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty(x.shape, dtype=torch.uint8, device=x.device),
            torch.empty(*x.shape[:-1], _blocks(x.shape[-1]), dtype=torch.uint8, device=x.device))


def pack(x: torch.Tensor) -> Packed:
    """The 8-bit checkpoint of x (..., D), bf16 or fp32 (not differentiable)."""
    _check_x(x, "ckpt8.pack")
    x = x.detach()
    if not use_hip(x):
        return Packed(*_pack_reference(x), x.dtype)
    return Packed(*_native.binding().pack(x), x.dtype)


def unpack(p: Packed, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values the checkpoint stands for, in ``dtype`` (bf16 or fp32; default: the activation's)."""
    dtype = p.dtype if dtype is None else dtype
    if dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"ckpt8.unpack: dtype must be bfloat16 or float32, got {dtype}")
    _check_packed(p, "ckpt8.unpack")
    if not use_hip(p.q):
        return _unpack_reference(p.q, p.s).to(dtype)
    return _native.binding().unpack(p.q, p.s, dtype == torch.bfloat16)


# ---- bias + GELU -----------------------------------------------------------------------------------------

def _gelu(u: torch.Tensor) -> torch.Tensor:
    return F.gelu(u, approximate="tanh")


def _gelu_slope(u: torch.Tensor) -> torch.Tensor:
    sg = torch.sigmoid(2 * _K * (u + _C * u ** 3))
    c = u.clamp(-16.0, 16.0)  # sg (1 - sg) is 0 behind
    return sg + c * sg * (1 - sg) * (2 * _K + 6 * _K * _C * c * c)


def gelu_pack(x: torch.Tensor, b: torch.Tensor) -> Tuple[torch.Tensor, Packed]:
    """y = gelu(x + b) and the checkpoint of x + b: x (..., D) (bf16 on the GPU), b (D).  Not differentiable: what
    bias_gelu and ffn are made of."""
    _bias_ok(x, b, "ckpt8.gelu_pack")
    x, b = x.detach().contiguous(), b.detach().float().contiguous()
    if not use_hip(x):
        u = x.float() + b.float()
        return _gelu(u).to(x.dtype), Packed(*_pack_reference(u), x.dtype)
    y = torch.empty_like(x)
    q, s = _alloc(x)
    D = x.shape[-1]
    with on_device(x):
        check(lib().pv_ckpt8_gelu_fwd(P(x), P(b), P(y), P(q), P(s), x.numel() // D, D, stream(x.device)),
              "pv_ckpt8_gelu_fwd")
    return y, Packed(q, s, x.dtype)


def gelu_backward(p: Packed, dy: torch.Tensor, with_y: bool = False, db: Optional[torch.Tensor] = None):
    """(dx, db, y): dx = dy gelu'(u) at the kept u, db (D) fp32 its column sums (added into ``db`` if given: contiguous
    fp32), y = gelu(u) (``with_y``, else None)."""
    _check_packed(p, "ckpt8.gelu_backward")
    D = p.q.shape[-1]
    if dy.shape != p.q.shape or not dy.is_floating_point():
        raise ValueError(f"ckpt8.gelu_backward: dy {tuple(dy.shape)} {dy.dtype} does not go with a checkpoint of {tuple(p.q.shape)}")
    if db is not None and (db.shape != (D,) or db.dtype != torch.float32 or not db.is_contiguous()):
        raise ValueError(f"ckpt8.gelu_backward: db must be {D} contiguous float32 sums, got {tuple(db.shape)} {db.dtype}")
    _same_device(p.q, "ckpt8.gelu_backward", dy=dy, db=db)
    if not use_hip(dy):
        u = _unpack_reference(p.q, p.s)
        du = dy.float() * _gelu_slope(u)
        sums = du.reshape(-1, D).sum(0)
        sums = sums if db is None else db.add_(sums)
        return du.to(dy.dtype), sums, _gelu(u).to(p.dtype) if with_y else None
    q, s = p.q.contiguous(), p.s.contiguous()
    dy = dy.detach().to(torch.bfloat16).contiguous()
    T = dy.numel() // D
    dx = torch.empty_like(dy)
    y = torch.empty_like(dy) if with_y else None
    add = db is not None
    if db is None:
        db = torch.empty(D, dtype=torch.float32, device=dy.device)
    with on_device(dy):
        ws = torch.empty(int(lib().pv_ckpt8_gelu_bwd_ws(T, D)), dtype=torch.float32, device=dy.device)
        check(lib().pv_ckpt8_gelu_bwd(P(q), P(s), P(dy), P(dx), P(y), P(db), int(add), P(ws), T, D,
                                      stream(dy.device)), "pv_ckpt8_gelu_bwd")
    return dx, db, y


def _bias_ok(x: torch.Tensor, b: torch.Tensor, name: str) -> None:
    _check_x(x, name)
    if b.shape != (x.shape[-1],):
        raise ValueError(f"{name}: bias {tuple(b.shape)} does not go with {x.shape[-1]} columns")
    _same_device(x, name, bias=b)
    if use_hip(x) and x.dtype != torch.bfloat16:
        raise TypeError(f"{name}: the GPU kernels take bfloat16, got {x.dtype}")


class _BiasGelu8Fn(torch.autograd.Function):
    """CPU, and biases whose gradient lives in the flat buffer (ops/optim.py::FlatParams): the kernel adds into it.  Other
    biases on the GPU take the C++ node (csrc/binding/autograd.cpp)."""

    @staticmethod
    def forward(ctx, x, b):
        y, p = gelu_pack(x.contiguous(), b.float().contiguous())
        ctx.save_for_backward(p.q, p.s)
        ctx.dtype = x.dtype
        ctx.b = b  # flat-gradient direct-write target (ops/grad_sink.py)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        b = ctx.b
        tb = grad_sink.accum_target(b) if ctx.needs_input_grad[1] and b.dtype == torch.float32 else None
        dx, db, _ = gelu_backward(Packed(*ctx.saved_tensors, ctx.dtype), dy, db=tb)
        if tb is not None:
            grad_sink.done(b)
            return dx, None
        return dx, db.to(b.dtype)


class _GeluAloneFn(torch.autograd.Function):
    """y = gelu(x + b) on the GPU where nothing is kept, in the arithmetic of the differentiable form.  An autograd
    function although it has no backward: torch refuses to lose a forward-mode tangent in it."""

    @staticmethod
    def forward(ctx, x, b):
        x, b = x.contiguous(), b.float().contiguous()
        y = torch.empty_like(x)
        D = x.shape[-1]
        with on_device(x):
            check(lib().pv_ckpt8_gelu_fwd(P(x), P(b), P(y), None, None, x.numel() // D, D, stream(x.device)),
                  "pv_ckpt8_gelu_fwd")
        return y


def _gelu_alone(x: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """gelu(x + b) where no gradient is wanted: the bits of the differentiable form, for the same widths and biases."""
    if use_hip(x):
        return _GeluAloneFn.apply(x, b)
    return _gelu(x.contiguous().float() + b.float()).to(x.dtype)


def bias_gelu(x: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """gelu(x + b), keeping x + b in 8 bits for the backward (transformer.py::bias_gelu keeps x in bf16)."""
    _bias_ok(x, b, "ckpt8.bias_gelu")
    if not (torch.is_grad_enabled() and (x.requires_grad or b.requires_grad)):
        return _gelu_alone(x, b)
    if use_hip(x) and grad_sink.flat_of(b) is None:
        return _native.binding().bias_gelu8(x, b)
    if use_hip(x):
        refuse_held_capture("ckpt8.bias_gelu", x, b)
    return _BiasGelu8Fn.apply(x, b)


# ---- linear layers ---------------------------------------------------------------------------------------

class _Linear8Fn(torch.autograd.Function):
    """transformer.py::_Linear16Fn with its saved input in 8 bits."""

    @staticmethod
    def forward(ctx, x, w, b, w16, res=None):
        x2 = x.to(torch.bfloat16).reshape(-1, x.shape[-1])
        y = torch.addmm(b.to(torch.bfloat16), x2, w16.t()) if b is not None else x2 @ w16.t()
        p = pack(x2)
        ctx.save_for_backward(p.q, p.s, w16)
        ctx.shape = x.shape
        ctx.params = (w, b)
        ctx.res = res
        return y.view(*x.shape[:-1], w16.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, s, w16 = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1]).to(torch.bfloat16)
        dx = tops._dx_residual(ctx.res, dy2, w16, ctx.shape) if ctx.needs_input_grad[0] else None
        w, b = ctx.params
        dw = _weight_grad(w, dy2, unpack(Packed(q, s, torch.bfloat16))) if ctx.needs_input_grad[1] else None
        db = None
        if b is not None and ctx.needs_input_grad[2]:
            tb = grad_sink.write_target(b)
            if dy2.shape[0]:
                db = dops.colsum(dy2, out=tb, accumulate=tb is not None)
            else:  # no rows: nothing to add
                db = torch.zeros(b.shape, dtype=torch.float32, device=dy2.device)
            if tb is not None:
                grad_sink.done(b)
                db = None
        return dx, dw, db, None, None


def _weight_grad(w, dy2, x2):
    tw = grad_sink.write_target(w)
    dw = tops.wgrad_f32(dy2, x2, out=tw)
    if tw is None:
        return dw
    grad_sink.done(w)
    return None


class _RoundSaved(torch.autograd.Function):
    """CPU: y = x W^T whose weight gradient reads the 8-bit x."""

    @staticmethod
    def forward(ctx, x, w):
        p = pack(x)
        ctx.save_for_backward(p.q, p.s, w)
        return F.linear(x, w.to(x.dtype))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, s, w = ctx.saved_tensors
        x = _unpack_reference(q, s)
        dw = dy.reshape(-1, dy.shape[-1]).float().t() @ x.reshape(-1, x.shape[-1])
        return dy @ w.to(dy.dtype), dw.to(w.dtype)


def linear(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None,
           res: Optional[tops.ResidualLink] = None) -> torch.Tensor:
    """x W^T (+ b) like transformer.py::linear, keeping x in 8 bits for the weight gradient."""
    _check_x(x, "ckpt8.linear")
    if w.dim() != 2 or w.shape[1] != x.shape[-1]:
        raise ValueError(f"ckpt8.linear: weight {tuple(w.shape)} does not go with {x.shape[-1]} columns")
    if b is not None and b.shape != w.shape[:1]:
        raise ValueError(f"ckpt8.linear: bias {tuple(b.shape)} does not go with {w.shape[0]} outputs")
    _same_device(x, "ckpt8.linear", weight=w, bias=b)
    if not (torch.is_grad_enabled() and w.requires_grad):
        return tops.linear(x, w, b, res=res)
    if use_hip(x):
        refuse_held_capture("ckpt8.linear", x, w, b)
        return _Linear8Fn.apply(x, w, b, tops.weight_bf16(w), res)
    y = _RoundSaved.apply(x, w)
    return y if b is None else y + b.to(y.dtype)


class _FFN8Fn(torch.autograd.Function):
    """gelu(x W1^T + b1) W2^T; saved: x and x W1^T + b1 in 8 bits.  The backward's GELU kernel gives the
    second layer's input again (for its weight gradient) beside du and the bias gradient."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, w1h, w2h, res=None):
        x2 = x.to(torch.bfloat16).reshape(-1, x.shape[-1])
        y, p = gelu_pack(x2 @ w1h.t(), b1.float().contiguous())
        px = pack(x2)
        ctx.save_for_backward(px.q, px.s, p.q, p.s, w1h, w2h)
        ctx.shape = x.shape
        ctx.params = (w1, b1, w2)
        ctx.res = res
        return (y @ w2h.t()).view(*x.shape[:-1], w2h.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        xq, xs, uq, us, w1h, w2h = ctx.saved_tensors
        w1, b1, w2 = ctx.params
        do2 = do.reshape(-1, do.shape[-1]).to(torch.bfloat16).contiguous()
        tb = grad_sink.accum_target(b1) if ctx.needs_input_grad[2] and b1.dtype == torch.float32 else None
        du, db, y = gelu_backward(Packed(uq, us, torch.bfloat16), do2 @ w2h, with_y=ctx.needs_input_grad[3], db=tb)
        if tb is not None:
            grad_sink.done(b1)
            db = None
        dw2 = _weight_grad(w2, do2, y) if ctx.needs_input_grad[3] else None
        dw1 = _weight_grad(w1, du, unpack(Packed(xq, xs, torch.bfloat16))) if ctx.needs_input_grad[1] else None
        dx = tops._dx_residual(ctx.res, du, w1h, ctx.shape) if ctx.needs_input_grad[0] else None
        return dx, dw1, None if db is None else db.to(b1.dtype), dw2, None, None, None


def ffn(x: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor,
        res: Optional[tops.ResidualLink] = None) -> torch.Tensor:
    """transformer.py::ffn (gelu(x W1^T + b1) W2^T) with its saved activations in 8 bits."""
    _check_x(x, "ckpt8.ffn")
    if w1.dim() != 2 or w2.dim() != 2 or w1.shape[1] != x.shape[-1] or w2.shape[1] != w1.shape[0] or b1.shape != w1.shape[:1]:
        raise ValueError(f"ckpt8.ffn: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, b1 {tuple(b1.shape)}, w2 {tuple(w2.shape)} do not fit")
    _same_device(x, "ckpt8.ffn", w1=w1, b1=b1, w2=w2)
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in (x, w1, b1, w2))):
        return tops.linear(_gelu_alone(tops.linear(x, w1, res=res), b1), w2)
    if use_hip(x):
        refuse_held_capture("ckpt8.ffn", x, w1, b1, w2)
        return _FFN8Fn.apply(x, w1, b1, w2, tops.weight_bf16(w1), tops.weight_bf16(w2), res)
    return _RoundSaved.apply(bias_gelu(_RoundSaved.apply(x, w1), b1), w2)

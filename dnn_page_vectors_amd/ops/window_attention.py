"""Attention with a sliding window and a few first tokens that stay visible, for long pages.

Key ``j`` is visible to query ``i`` when it is not masked, ``j <= i + right``, and either
``j >= i - left`` or ``j < sinks``: the window moves with the query, and the first ``sinks``
tokens stay visible once it has moved past them (the page's [CLS] position is one).
``left`` / ``right`` ``None`` = unbounded on that side, ``right = 0`` = causal.  A query without a
visible key gets zeros and contributes no gradient.

GPU: the HIP kernels of csrc/kernels/window_attention.hip (bf16 operands, fp32 softmax
statistics and accumulators), which read only the key tiles that hold a visible pair.
CPU / ``backend="torch"`` / ``dtype="fp32"``: the same in plain torch (fp32 inside).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from .. import _native
from ._common import P, check, lib, on_device, refuse_held_capture, stream, use_hip

HEAD_DIMS = (32, 64, 128)
MAX_LEN = 1 << 29


def _window(left: Optional[int], right: Optional[int], sinks: int, L: int) -> Tuple[int, int, int]:
    """Clamped to the sequence (L = unbounded)."""
    for name, x in (("left", left), ("right", right)):
        if x is not None and (isinstance(x, bool) or int(x) != x or x < 0):
            raise ValueError(f"window_attention: {name} must be None (unbounded) or an integer >= 0, got {x!r}")
    if isinstance(sinks, bool) or int(sinks) != sinks or sinks < 0:
        raise ValueError(f"window_attention: sinks must be an integer >= 0, got {sinks!r}")
    return (L if left is None else min(int(left), L), L if right is None else min(int(right), L), min(int(sinks), L))


def _scale(scale: Optional[float], d: int) -> float:
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0 ** -126 <= s <= 2.0 ** 120:  # times log2(e) it has to stay a finite, normal fp32 number
        raise ValueError(f"window_attention: scale must be positive and finite (2^-126 to 2^120), got {scale!r}")
    return s


def _key_mask(mask: Optional[torch.Tensor], N: int, L: int, device) -> Optional[torch.Tensor]:
    if mask is None:
        return None
    if mask.shape != (N, L):
        raise ValueError(f"window_attention: mask must be {(N, L)} (batch, keys), got {tuple(mask.shape)}")
    if mask.is_floating_point() or mask.is_complex():
        raise TypeError(f"window_attention: mask must be boolean or integer (non-zero = a real token), got {mask.dtype}")
    if mask.device != device:
        raise ValueError(f"window_attention: mask is on {mask.device}, the operands on {device}")
    if mask.dtype not in (torch.bool, torch.uint8, torch.int32):
        mask = mask != 0
    return mask if L == 1 or mask.stride(1) == 1 else mask.contiguous()


def _check_range(N: int, L: int, H: int, d: int = 0) -> None:
    """A workgroup per 128 queries and head, of 128 threads for up to 64 tokens and 256 above, in a grid of fewer than
    2^32 threads; offsets within a tile of 64 rows in 32 bits."""
    if H * d >= 1 << 24:
        raise ValueError(f"window_attention: {H} heads of {d} columns are outside the kernels' range (2^24 columns)")
    if L > MAX_LEN or N * H * -(-L // 128) * (128 if L <= 64 else 256) >= 1 << 32:
        raise ValueError(f"window_attention: {N} sequences of {L} tokens and {H} heads are outside the kernels' range "
                         f"(length {MAX_LEN}, 2^25 heads of up to 64 tokens, 2^24 blocks of 128 queries of longer ones)")


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("window_attention: q, k, v must be (batch, length, heads, head dim)")
    if k.shape != v.shape:
        raise ValueError(f"window_attention: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"window_attention: q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, length or head dim")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"window_attention: {q.shape[2]} query heads are no multiple of {k.shape[2]} key/value heads")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"window_attention: q, k, v have different types: {q.dtype}, {k.dtype}, {v.dtype}")
    if not (q.device == k.device == v.device):
        raise ValueError("window_attention: q, k, v are on different devices")


def _strides(*ts: torch.Tensor):
    return (ctypes.c_long * (3 * len(ts)))(*[s for t in ts for s in t.stride()[:3]])


def _mask_args(mask: Optional[torch.Tensor]):
    return (None, 0, 1) if mask is None else (mask.data_ptr(), mask.stride(0), mask.element_size())


# the packed form's calls (views of one buffer); the plain form's are in csrc/binding/autograd.cpp

def _forward(q, k, v, out, mask, win, scale: float, lse, rest) -> None:
    N, L, H, d = q.shape
    st = _strides(q, k, v, out)
    with on_device(q):
        check(lib().pv_wattn_fwd(P(q), P(k), P(v), P(out), st, *_mask_args(mask), P(lse), P(rest), N, L, H,
                                 H // k.shape[2], d, *win, scale, stream(q.device)), "pv_wattn_fwd")


def _backward(q, k, v, out, do, dq, dk, dv, mask, win, scale: float, lse, rest) -> None:
    N, L, H, d = q.shape
    G = H // k.shape[2]
    D = torch.empty_like(lse)
    n = lib().pv_wattn_bwd_ws(N, L, H, G, d, win[0], win[2]) if win[2] else 0
    ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
    st = _strides(q, k, v, out, do, dq, dk, dv)
    with on_device(q):
        check(lib().pv_wattn_bwd(P(q), P(k), P(v), P(out), P(do), P(dq), P(dk), P(dv), st, *_mask_args(mask), P(lse),
                                 P(rest), P(D), P(ws), n, N, L, H, G, d, *win, scale, stream(q.device)), "pv_wattn_bwd")


def visible(L: int, left: Optional[int], right: Optional[int], sinks: int, device=None) -> torch.Tensor:
    """(L, L) bool: which key (column) a query (row) sees, the key mask aside."""
    left, right, sinks = _window(left, right, sinks, L)
    i = torch.arange(L, device=device)[:, None]
    j = torch.arange(L, device=device)[None, :]
    return (j <= i + right) & ((j >= i - left) | (j < sinks))


def _reference(q, k, v, mask, left, right, sinks, scale: float):
    """Plain torch in fp32 (fp64 stays fp64); differentiable."""
    N, L, H, d = q.shape
    G = H // k.shape[2]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    see = visible(L, left, right, sinks, q.device)[None, None]
    kk, vv = k.to(wide), v.to(wide)
    if mask is not None:
        m = mask != 0
        see = see & m[:, None, None, :]
        kk = kk.masked_fill(~m[:, :, None, None], 0.0)  # whatever a masked row holds stays out of the products
        vv = vv.masked_fill(~m[:, :, None, None], 0.0)
    qh = q.to(wide).transpose(1, 2)
    kh = kk.transpose(1, 2).repeat_interleave(G, 1)
    vh = vv.transpose(1, 2).repeat_interleave(G, 1)
    s = torch.matmul(qh, kh.transpose(-1, -2)) * scale
    some = see.any(-1, keepdim=True)
    # a row without a visible key: softmax over zeros, then zeroed (no NaN for its gradient)
    p = torch.softmax(s.masked_fill(~see & some, float("-inf")).masked_fill(~some, 0.0), -1)
    p = p.masked_fill(~see, 0.0)
    return torch.matmul(p, vh).transpose(1, 2).to(q.dtype)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: Optional[int] = None,
                     right: Optional[int] = None, sinks: int = 0, mask: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """q (N, L, H, d), k / v (N, L, Hkv, d) with H a multiple of Hkv (query head h reads key/value
    head h // (H / Hkv)), mask (N, L) of the keys (non-zero = a real token; masked keys and values
    may hold anything) -> (N, L, H, d).  ``scale`` defaults to 1 / sqrt(d).

    Differentiable once in q, k and v, on the GPU in reverse mode alone.  On the GPU: bf16, d in (32, 64, 128), any strides (operands
    whose rows are not 16-byte aligned are copied).  A non-finite value at a *visible* key may reach
    queries up to 64 tokens outside its window."""
    _check_qkv(q, k, v)
    N, L, H, d = q.shape
    win = _window(left, right, sinks, L)
    scale = _scale(scale, d)
    mask = _key_mask(mask, N, L, q.device)
    if not use_hip(q):
        return _reference(q, k, v, mask, left, right, sinks, scale)
    if q.dtype != torch.bfloat16:
        raise TypeError(f"window_attention: the GPU kernels take bfloat16, got {q.dtype}")
    if d not in HEAD_DIMS:
        raise ValueError(f"window_attention: head dim must be one of {HEAD_DIMS} on the GPU, got {d}")
    _check_range(N, L, H, d)
    if q.numel() == 0:
        return q * 1.0 + (k.sum() + v.sum())  # nothing to add, but a result of all three
    return _native.binding().window_attention(q, k, v, mask, *win, scale)


class _PackedWindowAttnFn(torch.autograd.Function):
    """window_attention over sequence groups packed token-major (transformer.py::packed_attention):
    the kernels read q / k / v from and write their gradients into the slots of the packed
    projection, so there are no splits, copies or gradient concatenations."""

    @staticmethod
    def forward(ctx, qkv, masks, shapes, heads, win, scale, train):
        qkv = qkv.contiguous()
        C = qkv.shape[1]
        d = C // (3 * heads)
        out = torch.empty(qkv.shape[0], heads * d, dtype=qkv.dtype, device=qkv.device)
        stats = []  # per group: log-sum-exp, and the bits of out below its bf16
        for (q, k, v, o), m, (N, L) in zip(_groups(qkv, out, shapes, heads, d), masks, shapes):
            kept = (torch.empty(N, heads, L, dtype=torch.float32, device=qkv.device),
                    torch.empty(N, heads, (L + 31) // 32 * 32, d, dtype=torch.uint8, device=qkv.device)) if train else (None, None)
            _forward(q, k, v, o, m, _window(*win, L), scale, *kept)
            stats += kept
        ctx.save_for_backward(qkv, out, *masks, *stats)
        ctx.meta = (shapes, heads, d, win, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        shapes, heads, d, win, scale = ctx.meta
        n = len(shapes)
        qkv, out = ctx.saved_tensors[:2]
        masks, stats = ctx.saved_tensors[2:2 + n], ctx.saved_tensors[2 + n:]
        do = do.to(qkv.dtype).contiguous()
        if do.data_ptr() % 16:
            do = do.clone()
        dqkv = torch.empty_like(qkv)
        for (q, k, v, o), (dq, dk, dv, g), m, lse, rest, (N, L) in zip(_groups(qkv, out, shapes, heads, d),
                                                                       _groups(dqkv, do, shapes, heads, d), masks, stats[::2], stats[1::2],
                                                                       shapes):
            _backward(q, k, v, o, g, dq, dk, dv, m, _window(*win, L), scale, lse, rest)
        return dqkv, None, None, None, None, None, None


def _groups(qkv, out, shapes, heads: int, d: int):
    """(q, k, v, out) views (N, L, heads, d) of each packed group."""
    off = 0
    for N, L in shapes:
        x = qkv[off:off + N * L].view(N, L, 3, heads, d)
        yield x[:, :, 0], x[:, :, 1], x[:, :, 2], out[off:off + N * L].view(N, L, heads, d)
        off += N * L


def packed_window_attention(qkv: torch.Tensor, masks: Sequence[Optional[torch.Tensor]],
                            shapes: Sequence[Tuple[int, int]], heads: int, left: Optional[int] = None,
                            right: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """``window_attention`` on a packed projection: qkv (T, 3 * heads * d) holds groups of (N_i, L_i)
    sequences back to back, masks [(N_i, L_i) or None] -> (T, heads * d)."""
    if qkv.dim() != 2 or qkv.shape[1] % (3 * heads):
        raise ValueError(f"packed_window_attention: qkv must be (tokens, 3 * {heads} * d), got {tuple(qkv.shape)}")
    d = qkv.shape[1] // (3 * heads)
    shapes = [(int(N), int(L)) for N, L in shapes]
    if len(masks) != len(shapes) or sum(N * L for N, L in shapes) != qkv.shape[0]:
        raise ValueError("packed_window_attention: the group shapes and masks do not cover the packed tokens")
    _window(left, right, sinks, 1)
    masks = [_key_mask(m, N, L, qkv.device) for m, (N, L) in zip(masks, shapes)]
    if use_hip(qkv) and qkv.dtype == torch.bfloat16 and d in HEAD_DIMS and min((n for s in shapes for n in s), default=0) > 0 \
            and qkv.data_ptr() % 16 == 0 and qkv.shape[1] < 1 << 24:
        for N, L in shapes:
            _check_range(N, L, heads)
        train = torch.is_grad_enabled() and qkv.requires_grad
        if train:
            refuse_held_capture("packed_window_attention", qkv)
        return _PackedWindowAttnFn.apply(qkv, masks, shapes, heads, (left, right, sinks), _scale(None, d), train)
    outs, off = [], 0
    for (N, L), m in zip(shapes, masks):
        x = qkv[off:off + N * L].view(N, L, 3, heads, d)
        outs.append(window_attention(x[:, :, 0], x[:, :, 1], x[:, :, 2], left, right, sinks, m).reshape(N * L, heads * d))
        off += N * L
    return torch.cat(outs, 0)

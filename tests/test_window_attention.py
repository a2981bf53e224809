"""Windowed attention with sinks (ops/window_attention.py) against the formula in 64 bits.

Tolerances follow from the roundings the kernels make, computed per element with the oracle's own
matrices.  One rounding to bf16 is off by at most h = 2^-8 relative.

* forward: every probability and the result are rounded once:  h P|V| + h |o|;
* scores and the exponential are fp32: a product of d terms is off by d 2^-24 of the sum of
  magnitudes, log2e and the subtraction of the maximum add a few 2^-24 of the same size; twice that,
  as a relative error of p, is e = 2^-23 (d + 16) max scale |q||k| + 2^-17 (the 2^-17 covers the
  hardware exponential, the logarithm and the row sum's up to 2^6 half steps);
* D is taken with o before its last rounding (here with it): off by |do| (h P|V| + h |o|) at most;
* dS = p (dP - D) is rounded once: its error E = p (err D + d 2^-23 |do||v|) + (h + e) |dS|;
  dq, dk: E against |k|, |q| and one rounding; dv: (h + e) P^T|do| and one rounding.
"""
import ctypes
import gc
import math

import pytest
import torch

from dnn_page_vectors_amd.ops.window_attention import (packed_window_attention, visible,
                                                       window_attention)

H_ = 2.0 ** -8


def oracle(q, k, v, do, left, right, sinks, mask, scale=None):
    """(o, dq, dk, dv) and their tolerances, fp64, from the definition (explicit index conditions)."""
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    N, L, H, d = q.shape
    Hkv = k.shape[2]
    G = H // Hkv
    scale = 1 / math.sqrt(d) if scale is None else scale
    i = torch.arange(L).view(L, 1)
    j = torch.arange(L).view(1, L)
    see = torch.ones(L, L, dtype=torch.bool)
    if right is not None:
        see &= j - i <= right
    if left is not None:
        see &= (i - j <= left) | (j < sinks)
    see = see.expand(N, 1, L, L).clone()
    if mask is not None:
        m = mask.cpu() != 0
        see &= m[:, None, None, :]
        k = torch.where(m[:, :, None, None], k, torch.zeros_like(k))
        v = torch.where(m[:, :, None, None], v, torch.zeros_like(v))
    hq = lambda t: t.transpose(1, 2)
    hk = lambda t: t.transpose(1, 2).repeat_interleave(G, 1)
    Q, K, V, dO = hq(q), hk(k), hk(v), hq(do)
    S = scale * Q @ K.transpose(-1, -2)
    top = torch.where(see, S, torch.full_like(S, -1e300)).amax(-1, keepdim=True)
    P = torch.where(see, torch.exp(S - top), torch.zeros_like(S))
    P = P / P.sum(-1, keepdim=True).clamp(min=1e-300)
    O = P @ V
    dP = dO @ V.transpose(-1, -2)
    D = (dO * O).sum(-1, keepdim=True)
    dS = P * (dP - D)
    back = lambda t: t.transpose(1, 2)
    group = lambda t: t.reshape(N, Hkv, G, L, d).sum(2).transpose(1, 2)
    res = [back(O), back(scale * dS @ K), group(scale * dS.transpose(-1, -2) @ Q), group(P.transpose(-1, -2) @ dO)]
    smag = float((scale * Q.abs() @ K.abs().transpose(-1, -2)).max()) if L else 0.0
    e = 2.0 ** -23 * (d + 16) * smag + 2.0 ** -17
    eo = (H_ + e) * (P @ V.abs()) + H_ * O.abs()
    E = P * ((dO.abs() * eo).sum(-1, keepdim=True) + d * 2.0 ** -23 * dO.abs() @ V.abs().transpose(-1, -2))
    E = E + (H_ + e) * dS.abs()
    tol = [back(eo), back(scale * E @ K.abs()) + H_ * res[1].abs(),
           group(scale * E.transpose(-1, -2) @ Q.abs()) + H_ * res[2].abs(),
           group((H_ + e) * P.transpose(-1, -2) @ dO.abs()) + H_ * res[3].abs()]
    return res, [t + 1e-30 for t in tol]


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() - tol)
    assert (over <= 0).all(), f"{what}: off by {float((got - want).abs().max()):.3g}, {float(over.max()):.3g} over the bound"


def inputs(N, L, H, Hkv, d, seed, dtype=torch.bfloat16, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h: torch.randn(N, L, h, d, generator=g).to(dtype).to(device)
    return mk(H), mk(Hkv), mk(Hkv), mk(H)


def ragged(N, L, seed, holes=False):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, L + 1, (N,), generator=g)
    n[0] = 0          # a sequence without a real token: every row is empty
    if N > 1:
        n[1] = L
    m = torch.arange(L)[None, :] < n[:, None]
    if holes:
        m &= torch.rand(N, L, generator=g) > 0.4
    return m


def check(q, k, v, do, left, right, sinks, mask, scale=None):
    want, tol = oracle(q, k, v, do, left, right, sinks, mask, scale)
    mask = None if mask is None else mask.to(q.device)
    a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
    o = window_attention(a, b, c, left, right, sinks, mask, scale)
    got = (o,) + torch.autograd.grad(o, (a, b, c), do)
    for x, w, t, n in zip(got, want, tol, ("out", "dq", "dk", "dv")):
        assert x.shape == w.shape
        close(x, w, t, n)
    with torch.no_grad():  # the forward without anything kept
        assert torch.equal(window_attention(q, k, v, left, right, sinks, mask, scale), o)
    return got


# ---------------------------------------------------------------------------------- CPU

@pytest.mark.parametrize("left,right,sinks", [(None, None, 0), (2, 1, 0), (3, 0, 2), (0, 0, 0), (1, 1, 9), (None, 0, 0)])
@pytest.mark.parametrize("L", [1, 2, 7])
def test_cpu_matches_definition_and_gradients(left, right, sinks, L):
    q, k, v, do = inputs(2, L, 4, 2, 8, 3, torch.float64, "cpu")
    mask = ragged(2, L, 5)
    want, _ = oracle(q, k, v, do, left, right, sinks, mask)
    a, b, c = (t.requires_grad_() for t in (q, k, v))
    o = window_attention(a, b, c, left, right, sinks, mask)
    got = (o,) + torch.autograd.grad(o, (a, b, c), do)
    for x, w in zip(got, want):
        assert torch.allclose(x.double(), w, rtol=0, atol=1e-12)
    assert torch.equal(o[0], torch.zeros_like(o[0]))  # no real token
    fn = lambda x, y, z: window_attention(x, y, z, left, right, sinks, mask)
    assert torch.autograd.gradcheck(fn, (a, b, c), eps=1e-6, atol=1e-7)


def test_visible_pairs():
    m = visible(6, 1, 0, 2)
    rows = [[0], [0, 1], [0, 1, 2], [0, 1, 2, 3], [0, 1, 3, 4], [0, 1, 4, 5]]
    assert [torch.nonzero(r).flatten().tolist() for r in m] == rows
    assert visible(5, None, None, 0).all()


@pytest.mark.parametrize("kw,err", [
    (dict(left=-1), ValueError), (dict(right=1.5), ValueError), (dict(sinks=-2), ValueError), (dict(left=True), ValueError),
    (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError), (dict(scale=-1.0), ValueError),
    (dict(scale=float("inf")), ValueError),
    (dict(mask=torch.ones(2, 5)), TypeError), (dict(mask=torch.ones(2, 4).bool()), ValueError),
    (dict(mask=torch.ones(5).bool()), ValueError),
])
def test_refusals(kw, err):
    q, k, v, _ = inputs(2, 5, 4, 2, 8, 0, torch.float32, "cpu")
    with pytest.raises(err):
        window_attention(q, k, v, **kw)


@pytest.mark.parametrize("shapes,err", [
    (((2, 5, 4, 8), (2, 5, 3, 8), (2, 5, 3, 8)), ValueError),   # 4 heads over 3
    (((2, 5, 4, 8), (2, 6, 4, 8), (2, 6, 4, 8)), ValueError),   # lengths differ
    (((2, 5, 4, 8), (2, 5, 4, 8), (2, 5, 2, 8)), ValueError),
    (((2, 5, 4, 8), (2, 5, 4, 16), (2, 5, 4, 16)), ValueError),
    (((5, 4, 8), (5, 4, 8), (5, 4, 8)), ValueError),
])
def test_shape_refusals(shapes, err):
    with pytest.raises(err):
        window_attention(*(torch.zeros(s) for s in shapes))


def test_type_refusals():
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(TypeError):
        window_attention(x, x.double(), x.double())
    with pytest.raises(ValueError):
        packed_window_attention(torch.zeros(4, 24), [None], [(1, 3)], 1)
    with pytest.raises(ValueError):
        packed_window_attention(torch.zeros(4, 25), [None], [(1, 4)], 1)


def test_packed_cpu_equals_separate():
    g = torch.Generator().manual_seed(1)
    shapes, H, d = [(2, 3), (1, 7)], 2, 8
    qkv = torch.randn(13, 3 * H * d, generator=g)
    masks = [torch.tensor([[1, 1, 0], [1, 1, 1]]), None]
    got = packed_window_attention(qkv, masks, shapes, H, 1, 1, 1)
    off = 0
    for (N, L), m in zip(shapes, masks):
        x = qkv[off:off + N * L].view(N, L, 3, H, d)
        want = window_attention(x[:, :, 0], x[:, :, 1], x[:, :, 2], 1, 1, 1, m).reshape(N * L, H * d)
        assert torch.equal(got[off:off + N * L], want)
        off += N * L


# ---------------------------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 300])
@pytest.mark.parametrize("left,right,sinks", [(None, None, 0), (16, 16, 1), (0, 0, 0), (40, 0, 3), (7, 90, 70)])
def test_lengths_and_windows(L, left, right, sinks):
    check(*inputs(2, L, 2, 2, 64, L), left, right, sinks, None)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 2), (6, 1), (3, 3)])
def test_heads_and_dims(d, H, Hkv):
    check(*inputs(3, 150, H, Hkv, d, d + H), 33, 20, 2, ragged(3, 150, d))
    check(*inputs(2, 97, H, Hkv, d, d + H), None, 0, 0, ragged(2, 97, 1, holes=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int32, torch.int64])
@pytest.mark.parametrize("left,right,sinks", [(10, 10, 0), (20, 0, 5), (None, None, 0), (64, 64, 130)])
def test_masks(dtype, left, right, sinks):
    m = ragged(4, 260, 3, holes=True)
    m[2, 64:128] = False         # a whole tile masked
    m[3, :200] = False           # sinks masked, rows whose window is masked
    mm = (m.to(dtype) * (3 if dtype != torch.bool else 1)).to(dtype).cuda()
    got = check(*inputs(4, 260, 2, 1, 64, 8), left, right, sinks, mm)
    empty = ~(visible(260, left, right, sinks)[None] & m[:, None, :]).any(-1)
    assert empty.any()
    assert (got[0].cpu()[empty] == 0).all() and (got[1].cpu()[empty] == 0).all()
    assert (got[2].cpu()[~m] == 0).all() and (got[3].cpu()[~m] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("left", [None, 20])
def test_masked_keys_may_hold_anything(bad, left):
    q, k, v, do = inputs(3, 140, 2, 2, 64, 4)
    m = ragged(3, 140, 9, holes=True)
    clean = check(q, k, v, do, left, 5, 2, m.cuda())
    k2, v2 = k.clone(), v.clone()
    k2[~m] = bad
    v2[~m] = bad
    dirty = check(q, k2, v2, do, left, 5, 2, m.cuda())
    for x, y in zip(clean, dirty):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_long_sinks_and_wide_scores():
    """Scores of some hundreds: the running maximum moves by a lot from tile to tile."""
    q, k, v, do = inputs(1, 700, 2, 1, 64, 5)
    check(q * 8, k * 4, v, do, 100, 0, 65, None)
    check(q, k, v, do, 30, 30, 700, None)      # every key a sink
    check(q, k, v, do, 0, 0, 1, None, scale=2.5)
    check(q, k, v, do, 699, 0, 0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("L,left,right,sinks", [(1100, 20, 20, 1), (1000, 5, 0, 40), (1217, 64, 3, 128), (2300, 10, 10, 33),
                                                (1700, 0, 0, 32), (1000, 20, 20, 129)])
def test_far_queries_of_the_sinks(d, L, left, right, sinks):
    """Sinks seen from far behind their window: summed by workgroups of their own."""
    check(*inputs(1, L, 2, 1, d, L), left, right, sinks, None)
    if d == 64:
        m = ragged(3, L, 2, holes=True)
        m[1, :7] = False                     # a masked sink
        check(*inputs(3, L, 2, 2, d, L + 1), left, right, sinks, m)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("L", [3, 40, 131])
def test_row_sums_of_the_gradient_are_exact_enough_for_values_far_from_zero(d, L):
    """Values around 64: D and do.v_j are large and nearly cancel.  With q = 0 every probability is 1 / keys from
    exponentials that are exactly 1, so D's error is o's alone: kept to 2^-8 of its last bf16 place (off by 2^-15 |o| at
    most), not to bf16 (2^-8).  fp32: the products of d terms and the start value D are off by d 2^-23 of the sum of
    magnitudes each; p and the quotient by 2^-17.  Then dS and dq are rounded once."""
    _, k, v, do = inputs(2, L, 2, 2, d, 11, device="cpu")
    v = (v.float() + 64).bfloat16()
    q = torch.zeros_like(k)
    res, _ = oracle(q, k, v, do, 1, 1, 0, None)
    K, V, dO, O = (t.double().transpose(1, 2) for t in (k, v, do, res[0]))
    see = visible(L, 1, 1, 0)
    P = see.double() / see.double().sum(-1, keepdim=True)
    dP = dO @ V.transpose(-1, -2)
    dS = P * (dP - (dO * O).sum(-1, keepdim=True))
    E = P * (2.0 ** -15 * (dO.abs() * O.abs()).sum(-1, keepdim=True) + 2 * d * 2.0 ** -23 * dO.abs() @ V.abs().transpose(-1, -2))
    E = E + (H_ + 2.0 ** -17) * dS.abs()
    tol = (E @ K.abs()).transpose(1, 2) / math.sqrt(d) + H_ * res[1].abs() + 1e-30
    qg = q.cuda().requires_grad_()
    window_attention(qg, k.cuda(), v.cuda(), 1, 1).backward(do.cuda())
    close(qg.grad, res[1], tol, "dq")


@pytest.mark.gpu
def test_strides():
    N, L, H, d = 2, 130, 3, 64
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(N, L, 3, H, d, generator=g).bfloat16().cuda()
    do = torch.randn(N, L, H, d, generator=g).bfloat16().cuda()
    q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
    base = check(q.contiguous(), k.contiguous(), v.contiguous(), do, 17, 9, 1, None)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(N, L, H, d + 1, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = k
    last = v.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)   # head dim not contiguous
    wide = do.repeat_interleave(2, 1)[:, ::2]
    for qq, kk, vv, dd in ((q, k, v, do), (heads_first(q), heads_first(k), heads_first(v), heads_first(do)),
                           (q, odd[..., 1:], last, wide)):
        got = check(qq, kk, vv, dd, 17, 9, 1, None)
        for x, y in zip(base, got):
            assert torch.equal(x, y)
    one = do[:1, :1, :, :].expand(N, L, H, d)                        # a broadcast gradient: stride 0
    check(q, k, v, one, 17, 9, 1, None)
    shared = k[:1].expand(N, L, H, d)                                # a broadcast input: its gradient is summed
    a = k[:1].clone().requires_grad_()
    o = window_attention(q, a.expand(N, L, H, d), v, 17, 9, 1)
    (ga,) = torch.autograd.grad(o, a, do)
    want, tol = oracle(q, shared, v, do, 17, 9, 1, None)
    close(ga, want[2].sum(0, keepdim=True), tol[2].sum(0, keepdim=True) * (1 + 2 * H_) + 2 * H_ * want[2].abs().sum(0, keepdim=True), "dk")
    mask = ragged(N, 2 * L, 1).cuda()[:, ::2]                        # strided mask
    check(q, k, v, do, 17, 9, 1, mask)
    check(q, k, v, do, 17, 9, 1, torch.tensor([True], device="cuda").expand(N, L))


@pytest.mark.gpu
def test_offsets_past_32_bits_by_strides():
    """Sequences 2^31 + 64 elements apart; rows 2^24 - 8 apart, the widest that is not copied."""
    def spread(t, step, row):
        x = torch.empty((t.shape[0] - 1) * step + (t.shape[1] - 1) * row + t[0, 0].numel(), dtype=t.dtype, device=t.device)
        return x.as_strided(t.shape, (step, row, *t.stride()[2:])).copy_(t)

    for N, L, step, row in ((2, 150, (1 << 31) + 64, 2 * 64), (1, 131, 0, (1 << 24) - 8)):
        q, k, v, do = inputs(N, L, 2, 2, 64, 5)
        base = check(q, k, v, do, 30, 30, 1, None)
        got = check(*(spread(t, step, row) for t in (q, k, v, do)), 30, 30, 1, None)
        for x, y in zip(base, got):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_offsets_past_32_bits_by_length():
    """2^31 and more elements per operand: the last rows equal those of the last tiles alone."""
    L, H, d, tail = (1 << 20) + 300, 16, 128, 300 + 256
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(1, L, H, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    whole = [t.requires_grad_() for t in (q, k, v)]
    o = window_attention(*whole, 9, 5)
    got = (o,) + torch.autograd.grad(o, whole, do)
    part = [t.detach()[:, -tail:].contiguous().requires_grad_() for t in (q, k, v)]
    o2 = window_attention(*part, 9, 5)
    want = (o2,) + torch.autograd.grad(o2, part, do[:, -tail:].contiguous())
    for x, y in zip(got, want):
        assert torch.equal(x[:, -300:], y[:, -300:])


@pytest.mark.gpu
def test_same_bits_every_run_and_on_a_side_stream():
    q, k, v, do = inputs(3, 333, 4, 2, 64, 6)
    m = ragged(3, 333, 2).cuda()
    ref = check(q, k, v, do, 50, 50, 4, m)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:  # two calls in flight at once
        with torch.cuda.stream(s):
            a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
            o = window_attention(a, b, c, 50, 50, 4, m)
            outs.append((o,) + torch.autograd.grad(o, (a, b, c), do))
    torch.cuda.synchronize()
    for got in outs:
        for x, y in zip(ref, got):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_graph_replays_forward_and_backward():
    shapes = [(2, 200), (1, 77)]
    st = []
    for N, L in shapes:  # two captured graphs, each with its own state
        q, k, v, do = inputs(N, L, 2, 2, 64, L)
        m = ragged(N, L, 1).cuda()
        q, k, v = (t.requires_grad_() for t in (q, k, v))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            o = window_attention(q, k, v, 30, 30, 2, m)
            torch.autograd.grad(o, (q, k, v), do)
            del o
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = window_attention(q, k, v, 30, 30, 2, m)
            got = (o,) + torch.autograd.grad(o, (q, k, v), do)
        st.append((graph, got, (q, k, v, do, m)))
    for rep in range(4):
        for graph, got, (q, k, v, do, m) in st:
            with torch.no_grad():
                q.copy_(torch.randn_like(q))
                do.copy_(torch.randn_like(do))
            graph.replay()
        torch.cuda.synchronize()
        for graph, got, (q, k, v, do, m) in st:
            a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
            o = window_attention(a, b, c, 30, 30, 2, m)
            want = (o,) + torch.autograd.grad(o, (a, b, c), do)
            for x, y in zip(got, want):
                assert torch.equal(x, y), rep


@pytest.mark.gpu
def test_packed_gradients_land_in_their_slots():
    H, d = 3, 64
    shapes = [(3, 20), (2, 150), (1, 1)]
    T = sum(a * b for a, b in shapes)
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(T, 3 * H * d, generator=g).bfloat16().cuda().requires_grad_()
    do = torch.randn(T, H * d, generator=g).bfloat16().cuda()
    masks = [ragged(3, 20, 1).cuda(), ragged(2, 150, 2, holes=True).to(torch.int32).cuda(), None]
    o = packed_window_attention(qkv, masks, shapes, H, 25, 10, 1)
    (dqkv,) = torch.autograd.grad(o, qkv, do)
    off = 0
    for (N, L), m in zip(shapes, masks):
        x = qkv.detach()[off:off + N * L].view(N, L, 3, H, d)
        gx = dqkv[off:off + N * L].view(N, L, 3, H, d)
        got = (o[off:off + N * L].view(N, L, H, d), gx[:, :, 0], gx[:, :, 1], gx[:, :, 2])
        want, tol = oracle(x[:, :, 0], x[:, :, 1], x[:, :, 2], do[off:off + N * L].view(N, L, H, d), 25, 10, 1, m)
        for a, b, t, n in zip(got, want, tol, ("out", "dq", "dk", "dv")):
            close(a, b, t, n)
        off += N * L


@pytest.mark.gpu
def test_gradient_against_differences():
    """A directional difference of the GPU forward itself: (f(x + t) - f(x - t)) / 2 against <grad, t>.  A bf16 output
    rounding is h |o| per element, weighted by do, twice over 2 eps; the step is large (eps = 0.25) and the third-order
    term is measured by the fp64 oracle."""
    q, k, v, do = inputs(1, 70, 2, 1, 64, 11)
    dirs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i, t in enumerate((q, k, v))]
    a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
    o = window_attention(a, b, c, 20, 20, 2)
    grads = torch.autograd.grad(o, (a, b, c), do)
    eps = 0.25
    for n in range(3):
        args = [q, k, v]
        vals, exact, room = [], [], 0.0
        for s in (1, -1):
            x = list(args)
            x[n] = (args[n].float() + s * eps * dirs[n].float()).bfloat16()
            y = window_attention(*x, 20, 20, 2).double().cpu()
            (w, *_), (t, *_) = oracle(*x, do, 20, 20, 2, None)
            vals.append(float((y * do.double().cpu()).sum()))
            exact.append(float((w * do.double().cpu()).sum()))
            room += float((t * do.double().cpu().abs()).sum())
        (_, *gw), (_, *gt) = oracle(q, k, v, do, 20, 20, 2, None)
        inner = float((grads[n].double() * dirs[n].double()).sum())
        want = float((gw[n] * dirs[n].double().cpu()).sum())
        curve = abs((exact[0] - exact[1]) / (2 * eps) - want)
        slack = room / (2 * eps) + curve + float((gt[n] * dirs[n].double().cpu().abs()).sum())
        assert abs((vals[0] - vals[1]) / (2 * eps) - inner) <= slack


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_capture_is_refused_while_an_eager_graph_holds_the_operands(packed):
    x = torch.randn(2 * 40, 3 * 2 * 32, device="cuda").bfloat16().requires_grad_()
    do = torch.randn(2 * 40, 2 * 32, device="cuda").bfloat16()

    def call():
        if packed:
            return packed_window_attention(x, [None], [(2, 40)], 2, 8, 8)
        y = x.detach().view(2, 40, 3, 2, 32)
        return window_attention(q, y[:, :, 1], y[:, :, 2], 8, 8).reshape(80, 64)

    q = x.detach().view(2, 40, 3, 2, 32)[:, :, 0].contiguous().requires_grad_()
    leaf = x if packed else q
    out = call()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    (want,) = torch.autograd.grad(out, leaf, do)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(call(), leaf, do)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_nothing_outlives_its_graph():
    q, k, v, do = inputs(1, 70, 2, 2, 64, 3)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    gc.collect()
    gc.disable()
    try:
        used = []
        for _ in range(4):
            torch.autograd.grad(window_attention(q, k, v, 9, 9, 1), (q, k, v), do)
            window_attention(q, k, v, 9, 9, 1)  # a graph without a backward
            used.append(torch.cuda.memory_allocated())
    finally:
        gc.enable()
    assert used[1] == used[-1]


@pytest.mark.gpu
def test_gpu_refusals():
    x = torch.zeros(1, 4, 2, 64, device="cuda")
    with pytest.raises(TypeError):
        window_attention(x, x, x)
    y = torch.zeros(1, 4, 2, 48, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        window_attention(y, y, y)
    z = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        window_attention(z, z, z, mask=torch.ones(1, 4, dtype=torch.bool))
    e = torch.zeros(0, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert window_attention(e, e, e).shape == (0, 4, 2, 64)
    a = z.clone().requires_grad_()
    o = window_attention(a, a, a)
    (ga,) = torch.autograd.grad(o, a, z, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        torch.autograd.grad(ga.sum(), a)


def test_shapes_beyond_the_grid_are_refused_by_every_layer():
    """A launch holds fewer than 2^32 threads: 128 per head up to 64 tokens, 256 per 128 queries above."""
    from dnn_page_vectors_amd import _native
    from dnn_page_vectors_amd.ops.window_attention import _check_range

    fwd = _native.hip(required=True).pv_wattn_fwd
    for N, L, H in ((1 << 25, 1, 1), (1 << 22, 64, 8), (1 << 24, 65, 1), (1 << 20, 200, 8), (1, 1 << 29, 4)):
        with pytest.raises(ValueError):
            _check_range(N, L, H)
        st = (ctypes.c_long * 12)()
        assert fwd(None, None, None, None, st, None, 0, 1, None, None, N, L, H, 1, 32, 1, 1, 0, 0.5, None) == -4
    for N, L, H in (((1 << 25) - 1, 1, 1), ((1 << 24) - 1, 65, 1), (1, 1 << 29, 3)):
        _check_range(N, L, H)


@pytest.mark.gpu
def test_largest_grid_of_short_sequences():
    """2^25 - 1 sequences of one token, the most that a launch holds; one more is refused."""
    N, d = (1 << 25) - 1, 32
    v = torch.randn(1, 1, 1, d, device="cuda").bfloat16()
    one = torch.randn(1, 1, 1, d, device="cuda").bfloat16().expand(N, 1, 1, d)
    out = window_attention(one, one, v.expand(N, 1, 1, d), 0, 0)
    assert torch.equal(out[-3:], v.expand(3, 1, 1, d)) and bool((out == v).all())
    more = one[:1].expand(N + 1, 1, 1, d)
    with pytest.raises(ValueError):
        window_attention(more, more, more, 0, 0)
    packed = torch.zeros(1, 3 * d, device="cuda").bfloat16().expand(N + 1, 3 * d)
    with pytest.raises(ValueError):
        packed_window_attention(packed, [None], [(N + 1, 1)], 1, 0, 0)


def check_empty(device, dtype):
    for N, L in ((0, 5), (3, 0)):
        q, k, v = (torch.zeros(N, L, h, 32, dtype=dtype, device=device).requires_grad_() for h in (4, 2, 2))
        out = window_attention(q, k, v, 3, 3, 1, torch.ones(N, L, dtype=torch.bool, device=device))
        assert out.shape == q.shape and out.dtype == dtype
        for t, g in zip((q, k, v), torch.autograd.grad(out, (q, k, v), torch.zeros_like(out))):
            assert g.shape == t.shape and g.dtype == dtype


def test_empty_results_have_all_gradients_cpu():
    check_empty("cpu", torch.float32)


@pytest.mark.gpu
def test_empty_results_have_all_gradients():
    check_empty("cuda", torch.bfloat16)
    x = torch.zeros(4, 3 * 64, device="cuda").bfloat16().requires_grad_()
    out = packed_window_attention(x, [None, None], [(2, 2), (0, 7)], 2, 1, 1)
    (g,) = torch.autograd.grad(out, x, torch.ones_like(out))
    assert out.shape == (4, 64) and g.shape == x.shape


@pytest.mark.parametrize("scale", [1e-46, 2.0 ** -127, 2.0 ** 121, 1e39, 1e300])
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(ValueError, match="scale"):
        window_attention(q, q, q, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -20, 2.0 ** 40])
def test_extreme_scales(scale):
    """Scores of at most 2^4 whatever the scale: the factor goes into the queries."""
    q, k, v, do = inputs(2, 70, 2, 2, 64, 9)
    big = (q.float() / 16 / scale).clamp(-2.0 ** 100, 2.0 ** 100).bfloat16()
    want, tol = oracle(big, k, v, do, 9, 9, 1, None, scale)
    close(window_attention(big, k, v, 9, 9, 1, None, scale), want[0], tol[0], "out")


def test_rows_too_far_apart_for_32_bit_tile_offsets_are_refused():
    """63 rows of 2^25 columns are 2^32 bytes: the last rows of a tile would be read from its beginning."""
    from dnn_page_vectors_amd import _native
    from dnn_page_vectors_amd.ops.window_attention import _check_range

    with pytest.raises(ValueError):
        _check_range(1, 65, 1 << 18, 64)
    _check_range(1, 65, (1 << 18) - 1, 64)
    lib = _native.hip(required=True)
    for i in (1, 2):
        st = (ctypes.c_long * 12)(*[64] * 12)
        st[3 * i + 1] = 1 << 25
        assert lib.pv_wattn_fwd(None, None, None, None, st, None, 0, 1, None, None, 1, 65, 1, 1, 64, 1, 1, 0, 0.5, None) == -6
    for i in (0, 1, 2, 4):
        st = (ctypes.c_long * 24)(*[64] * 24)
        st[3 * i + 1] = 1 << 25
        assert lib.pv_wattn_bwd(*[None] * 8, st, None, 0, 1, None, None, None, None, 0, 1, 65, 1, 1, 64, 1, 1, 0, 0.5, None) == -6


@pytest.mark.gpu
def test_too_many_columns_are_refused():
    q = torch.zeros(1, 1, 1, 64, device="cuda").bfloat16().expand(1, 65, 1 << 18, 64)
    with pytest.raises(ValueError):
        window_attention(q, q, q, 3, 3)

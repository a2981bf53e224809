"""8-bit activation checkpoints (ops/ckpt8.py).

Packing is exact arithmetic but for one rounding to e4m3, so bytes are compared for equality with an
independent fp64 computation.  GELU: the result is one bf16 rounding (2^-8) of an fp32 value whose sigmoid
is off by a few 2^-24 times the exponent's argument a; |a| sg (1 - sg) stays below 1 where the factor
q = 2k u + 6kc u^3 is below 64, so a slope is off by at most 2^-17 and y by 2^-20 |u|.
"""
import gc
import math

import pytest
import torch

from dnn_page_vectors_amd.ops import ckpt8

K, C = math.sqrt(2 / math.pi), 0.044715


def oracle_pack(x):
    """(kept values, bytes, scale bytes) in fp64: search of the exponent, nearest entry of the e4m3 table."""
    x = x.double().cpu()
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    pos = table[:0x7F]                                   # 0 .. 448, ascending
    flat = x.detach().reshape(-1, x.shape[-1])
    kept, q = torch.empty_like(flat), torch.empty(flat.shape, dtype=torch.uint8)
    nb = -(-x.shape[-1] // 32)
    s = torch.empty(flat.shape[0], nb, dtype=torch.uint8)
    for b in range(nb):
        part = flat[:, 32 * b:32 * b + 32]
        for r in range(flat.shape[0]):
            row = part[r]
            if not torch.isfinite(row).all():
                kept[r, 32 * b:32 * b + 32], q[r, 32 * b:32 * b + 32], s[r, b] = float("nan"), 0x7F, 255
                continue
            top = float(row.abs().max())
            e = -126 if top == 0 else max(-126, math.frexp(top / 448.0)[1] - 1)
            if top > 448.0 * 2.0 ** e:
                e += 1
            u = row.abs() / 2.0 ** e
            hi = torch.searchsorted(pos, u).clamp(max=0x7E)
            lo = (hi - 1).clamp(min=0)
            dl, dh = u - pos[lo], pos[hi] - u
            pick = torch.where(dl < dh, lo, torch.where(dh < dl, hi, torch.where(lo % 2 == 0, lo, hi)))
            kept[r, 32 * b:32 * b + 32] = torch.sign(row) * pos[pick] * 2.0 ** e
            q[r, 32 * b:32 * b + 32] = pick.to(torch.uint8) | (torch.signbit(row).to(torch.uint8) << 7)
            s[r, b] = e + 127
    return kept.view(x.shape), q.view(x.shape), s.view(*x.shape[:-1], nb)


def values(T, D, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, D, generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g)) * torch.exp(torch.randn(D, generator=g))
    return x.to(dtype)


def special(dtype):
    x = values(12, 70, 1, dtype)
    x[0] = 0
    x[1] = 448.0
    x[2, 3] = float("inf")
    x[3, 40] = float("-inf")
    x[4, 69] = float("nan")
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).tiny
    x[7] = 0
    x[7, 33] = -torch.finfo(dtype).tiny / 2             # a subnormal
    x[8] = -0.0
    x[9] *= 1e-36
    x[10, :32] = torch.linspace(-448, 448, 32).to(dtype)
    x[11] = 464.0                                        # between 448 and its next power of two
    return x


def check_pack(x, device):
    p = ckpt8.pack(x.to(device))
    kept, q, s = oracle_pack(x)
    assert p.q.shape == x.shape and p.s.shape == s.shape and p.dtype == x.dtype
    assert torch.equal(p.s.cpu(), s) and torch.equal(p.q.cpu(), q)
    for dt in (torch.bfloat16, torch.float32):
        got = ckpt8.unpack(p, dt)
        assert got.dtype == dt and got.shape == x.shape
        want = kept.to(dt)
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=7e7), torch.nan_to_num(want, nan=7e7))
    fine = torch.isfinite(kept)
    unit = (2.0 ** (p.s.cpu().double() - 127)).repeat_interleave(32, -1)[..., :x.shape[-1]]
    assert ((kept - x.double()).abs()[fine] <= (2.0 ** -4 * x.double().abs() + 2.0 ** -10 * unit)[fine]).all()


def gelu64(u):
    return u * torch.sigmoid(2 * K * (u + C * u ** 3))


def slope64(u):
    s = torch.sigmoid(2 * K * (u + C * u ** 3))
    return s + torch.where(u.abs() < 40, u * s * (1 - s) * 2 * K * (1 + 3 * C * u * u), torch.zeros_like(u))


def check_gelu(x, b, dy, device):
    a, c = x.to(device).requires_grad_(), b.to(device).requires_grad_()
    y = ckpt8.bias_gelu(a, c)
    dx, db = torch.autograd.grad(y, (a, c), dy.to(device))
    u = (x.float() + b.float()).double()                 # the kept sum is that of 32 bits
    h = 2.0 ** -8
    y64 = gelu64(u)
    assert ((y.double().cpu() - y64).abs() <= h * y64.abs() + 2.0 ** -20 * u.abs() + 1e-38).all()
    kept, _, _ = oracle_pack(u.float())
    du = dy.double() * slope64(kept)
    assert ((dx.double().cpu() - du).abs() <= h * du.abs() + (1 + h) * 2.0 ** -17 * dy.double().abs()).all()
    T = max(1, x.numel() // x.shape[-1])
    mag = du.abs().reshape(-1, x.shape[-1]).sum(0)
    room = 2.0 ** -17 * dy.double().abs().reshape(-1, x.shape[-1]).sum(0) + (T + 1) * 2.0 ** -24 * mag
    assert ((db.double().cpu() - du.reshape(-1, x.shape[-1]).sum(0)).abs() <= room + 1e-38).all()
    assert y.dtype == x.dtype and dx.dtype == x.dtype and db.dtype == b.dtype
    return y, dx, db


# ---------------------------------------------------------------------------------- CPU

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cpu_pack(dtype):
    check_pack(special(dtype), "cpu")
    check_pack(values(3, 33, 2, dtype).view(3, 1, 33), "cpu")


def test_cpu_gelu_and_layers():
    g = torch.Generator().manual_seed(0)
    check_gelu(values(5, 40, 3, torch.float32), torch.randn(40, generator=g), torch.randn(5, 40, generator=g), "cpu")
    x, w, b = torch.randn(6, 40, generator=g), torch.randn(8, 40, generator=g), torch.randn(8, generator=g)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    dy = torch.randn(6, 8, generator=g)
    y = ckpt8.linear(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w) + b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    kept = oracle_pack(x.detach())[0].float()
    assert torch.allclose(dx, dy @ w, atol=1e-5) and torch.allclose(dw, dy.t() @ kept, atol=1e-4)
    assert torch.allclose(db, dy.sum(0), atol=1e-5)


@pytest.mark.parametrize("call,err", [
    (lambda: ckpt8.pack(torch.zeros(3, 4, dtype=torch.int32)), TypeError),
    (lambda: ckpt8.pack(torch.zeros(3, 4, dtype=torch.float64)), TypeError),
    (lambda: ckpt8.pack(torch.zeros(())), ValueError), (lambda: ckpt8.pack(torch.zeros(3, 0)), ValueError),
    (lambda: ckpt8.unpack(ckpt8.pack(torch.zeros(3, 4)), torch.float16), TypeError),
    (lambda: ckpt8.unpack(ckpt8.Packed(torch.zeros(3, 40, dtype=torch.uint8), torch.zeros(3, 1, dtype=torch.uint8), torch.float32)), ValueError),
    (lambda: ckpt8.unpack(ckpt8.Packed(torch.zeros(3, 40), torch.zeros(3, 2, dtype=torch.uint8), torch.float32)), ValueError),
    (lambda: ckpt8.bias_gelu(torch.zeros(3, 4), torch.zeros(5)), ValueError),
    (lambda: ckpt8.linear(torch.zeros(3, 4), torch.zeros(2, 5)), ValueError),
    (lambda: ckpt8.ffn(torch.zeros(3, 4), torch.zeros(8, 4), torch.zeros(8), torch.zeros(4, 7)), ValueError),
])
def test_refusals(call, err):
    with pytest.raises(err):
        call()


# ---------------------------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pack_special_values(dtype):
    x = special(dtype)
    check_pack(x, "cuda")
    check_pack(x[:, :64].contiguous(), "cuda")           # the same through the 16-byte kernels
    check_pack(x[:, :8].contiguous(), "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,D", [(1, 1), (1, 8), (3, 31), (5, 32), (2, 33), (7, 40), (4, 300), (9, 768), (2, 2048), (2, 2056),
                                 (1, 4096), (3, 4100), (65, 96)])
def test_pack_shapes(T, D, dtype):
    check_pack(values(T, D, T + D, dtype), "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(5000, 96), (700, 768), (4097, 2048), (100001, 8)])
def test_pack_many_rows_matches_cpu_form(T, D):
    x = values(T, D, 3)
    a, b = ckpt8.pack(x.cuda()), ckpt8.pack(x)           # the CPU form is checked against the oracle above
    assert torch.equal(a.q.cpu(), b.q) and torch.equal(a.s.cpu(), b.s)
    assert torch.equal(ckpt8.unpack(a).cpu(), ckpt8.unpack(b))


@pytest.mark.gpu
def test_pack_strides_alignment_and_empty():
    x = values(20, 128, 1).cuda()
    want = ckpt8.pack(x)
    shifted = torch.empty(20 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(20, 128)
    shifted.copy_(x)
    for v in (x.t().contiguous().t(), shifted, x.repeat_interleave(2, 0)[::2]):
        p = ckpt8.pack(v)
        assert torch.equal(p.q, want.q) and torch.equal(p.s, want.s)
    assert torch.equal(ckpt8.unpack(ckpt8.Packed(want.q.t().contiguous().t(), want.s, want.dtype)), ckpt8.unpack(want))
    e = ckpt8.pack(x[:0])
    assert e.q.shape == (0, 128) and ckpt8.unpack(e).shape == (0, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(1, 1), (1, 32), (3, 7), (45, 300), (128, 64), (129, 64), (200, 40), (600, 768), (33, 2048),
                                 (40, 2056), (17, 4100)])
def test_gelu(T, D):
    g = torch.Generator().manual_seed(T * D)
    check_gelu(values(T, D, T), torch.randn(D, generator=g), torch.randn(T, D, generator=g).bfloat16(), "cuda")


@pytest.mark.gpu
def test_gelu_large_and_small_values():
    x = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 15.9, -15.9, 16.1, -16.1, 100.0, -100.0, 1e20, -1e20, 3e38, -3e38] * 2).bfloat16()
    x = torch.stack([x, x.flip(0) * 0.5])
    rows = torch.cat([x[:, i:i + 1].expand(2, 32) for i in range(32)], 0)      # one magnitude per block
    check_gelu(rows.contiguous(), torch.zeros(32), torch.ones(rows.shape).bfloat16(), "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 33])
def test_gelu_not_finite(D):
    """A NaN makes its whole block's gradient NaN (the kept copy is one scale per block) and no other's."""
    x = values(4, 2 * D, 0)
    x[1, 3] = float("nan")
    a, b = x.cuda().requires_grad_(), torch.zeros(2 * D, device="cuda", requires_grad=True)
    y = ckpt8.bias_gelu(a, b)
    dx, db = torch.autograd.grad(y, (a, b), torch.ones_like(y))
    assert y.isnan().sum() == 1 and y[1, 3].isnan()
    assert dx[1, :32].isnan().all() and dx.isnan().sum() == 32
    assert db[:32].isnan().all() and not db[32:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,D", [(40, 48), (300, 40), (2000, 256)])
def test_gelu_backward_gives_y_again_and_adds(T, D):
    g = torch.Generator().manual_seed(0)
    x, b, dy = values(T, D, 5).cuda(), torch.randn(D, generator=g).cuda(), torch.randn(T, D, generator=g).bfloat16().cuda()
    _, p = ckpt8.gelu_pack(x, b)
    dx, db, none = ckpt8.gelu_backward(p, dy)
    assert none is None
    base = torch.randn(D, device="cuda")
    dx2, db2, y = ckpt8.gelu_backward(p, dy, with_y=True, db=base.clone())
    assert torch.equal(dx, dx2) and torch.equal(db2, base + db)
    u = ckpt8.unpack(p, torch.float32).double()
    y64 = gelu64(u)
    assert ((y.double() - y64).abs() <= 2.0 ** -8 * y64.abs() + 2.0 ** -20 * u.abs()).all()


@pytest.mark.gpu
def test_gelu_same_bits_streams_and_graph():
    x, b = values(700, 512, 2).cuda().requires_grad_(), torch.randn(512, device="cuda", requires_grad=True)
    dy = torch.randn(700, 512, device="cuda").bfloat16()

    def step():
        y = ckpt8.bias_gelu(x, b)
        return (y,) + torch.autograd.grad(y, (x, b), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(side, step()):
        assert torch.equal(p, q)
    del side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(4):
        with torch.no_grad():
            x.copy_(values(700, 512, 20 + rep))
            dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(got, step()):
            assert torch.equal(p, q), rep


def _errors_of_products(a, b):
    """bound of an fp32-accumulated product of bf16 operands: k 2^-24 |a||b| (k terms)."""
    return a.shape[-1] * 2.0 ** -23 * (a.abs() @ b.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("T,I,O", [(10, 64, 32), (300, 768, 256), (33, 100, 20)])
def test_linear(T, I, O):
    g = torch.Generator().manual_seed(T)
    x = values(T, I, 1).cuda().requires_grad_()
    w, b = (0.1 * torch.randn(O, I, generator=g)).cuda().requires_grad_(), torch.randn(O, generator=g).cuda().requires_grad_()
    dy = torch.randn(T, O, generator=g).bfloat16().cuda()
    y = ckpt8.linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    from dnn_page_vectors_amd.ops import transformer as tops
    x2 = x.detach().requires_grad_()
    y2 = tops.linear(x2, w, b)
    dx2, _, db2 = torch.autograd.grad(y2, (x2, w, b), dy)
    assert torch.equal(y, y2) and torch.equal(dx, dx2)     # only the weight gradient differs
    # the column sum of the dense layers splits rows over workgroups that add by atomics: any order of T terms
    assert ((db - db2).abs() <= T * 2.0 ** -23 * dy.float().abs().sum(0)).all()
    kept = oracle_pack(x.detach())[0]
    want = dy.double().cpu().t() @ kept
    assert ((dw.double().cpu() - want).abs() <= _errors_of_products(dy.double().cpu().t(), kept)).all()


@pytest.mark.gpu
def test_ffn_gradients():
    """Against the formula with the kept values: du = (do W2) gelu'(u^), dW2 = do^T gelu(u^), dW1 = du^T x^."""
    T, Hd, I = 96, 64, 128
    g = torch.Generator().manual_seed(3)
    x = torch.randn(T, Hd, generator=g).bfloat16().cuda().requires_grad_()
    w1 = (0.2 * torch.randn(I, Hd, generator=g)).bfloat16().float().cuda().requires_grad_()
    w2 = (0.2 * torch.randn(Hd, I, generator=g)).bfloat16().float().cuda().requires_grad_()
    b1 = (0.1 * torch.randn(I, generator=g)).cuda().requires_grad_()
    do = torch.randn(T, Hd, generator=g).bfloat16().cuda()
    out = ckpt8.ffn(x, w1, b1, w2)
    got = torch.autograd.grad(out, (x, w1, b1, w2), do)
    h = 2.0 ** -8
    D = lambda t: t.detach().double().cpu()
    W1, W2, X, DO = D(w1), D(w2), D(x), D(do)
    pre = (x.detach() @ w1.detach().bfloat16().t())              # the product that the layer rounds to bf16
    u = (pre.float() + b1.detach()).cpu()
    kept = oracle_pack(u)[0]
    dh = D(do @ w2.detach().bfloat16())                           # rounded to bf16 on its way to the GELU
    du = dh * slope64(kept)
    edu = h * du.abs() + 2.0 ** -16 * dh.abs()
    yk, xk = gelu64(kept), oracle_pack(x.detach())[0]
    eyk = h * yk.abs() + 2.0 ** -20 * kept.abs()
    want = (du @ W1, du.t() @ xk, du.sum(0), DO.t() @ yk)
    tol = (edu @ W1.abs() + _errors_of_products(du, W1) + h * (du @ W1).abs() * (1 + h), edu.t() @ xk.abs() + _errors_of_products(du.t(), xk),
           edu.sum(0) + T * 2.0 ** -23 * du.abs().sum(0), DO.t().abs() @ eyk + _errors_of_products(DO.t(), yk))
    for a, w, t, n in zip(got, want, tol, ("dx", "dw1", "db1", "dw2")):
        err = (a.double().cpu() - w).abs()
        assert (err <= t + 1e-30).all(), (n, float((err - t).max()))


@pytest.mark.gpu
def test_gpu_refusals():
    x = torch.zeros(2, 4, device="cuda")
    with pytest.raises(TypeError):
        ckpt8.bias_gelu(x, torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        ckpt8.bias_gelu(x.bfloat16(), torch.zeros(4))
    with pytest.raises(TypeError):
        ckpt8.pack(x.half())


def test_unpack_refuses_no_columns():
    empty = torch.zeros(3, 0, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ckpt8.unpack(ckpt8.Packed(empty, empty, torch.bfloat16))


@pytest.mark.gpu
def test_capture_is_refused_while_an_eager_graph_holds_the_leaves():
    """The refusal leaves the process and the stream usable; once the eager graph is gone the capture works."""
    x = torch.randn(40, 96, device="cuda").bfloat16().requires_grad_()
    b = torch.randn(96, device="cuda", requires_grad=True)
    dy = torch.randn(40, 96, device="cuda").bfloat16()
    y = ckpt8.bias_gelu(x, b)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ckpt8.bias_gelu(x, b)
    want = torch.autograd.grad(y, (x, b), dy)
    del y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ckpt8.bias_gelu(x, b), (x, b), dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_nothing_outlives_its_graph():
    x = torch.randn(64, 128, device="cuda").bfloat16().requires_grad_()
    b = torch.randn(128, device="cuda", requires_grad=True)
    dy = torch.randn(64, 128, device="cuda").bfloat16()
    gc.collect()
    gc.disable()
    try:
        used = []
        for _ in range(4):
            torch.autograd.grad(ckpt8.bias_gelu(x, b), (x, b), dy)
            ckpt8.bias_gelu(x, b)  # a graph without a backward
            used.append(torch.cuda.memory_allocated())
    finally:
        gc.enable()
    assert used[1] == used[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("D", [2048, 2047])
def test_offsets_past_32_bits(D):
    """More than 2^31 elements: the last rows equal those of a call of their own."""
    T, tail = (1 << 31) // D + 40, 40
    x = torch.randn(T, D, device="cuda", dtype=torch.bfloat16)
    b = torch.randn(D, device="cuda")
    p, q = ckpt8.pack(x), ckpt8.pack(x[-tail:].clone())
    assert torch.equal(p.q[-tail:], q.q) and torch.equal(p.s[-tail:], q.s)
    assert torch.equal(ckpt8.unpack(p)[-tail:], ckpt8.unpack(q))
    del p
    both = []
    for t in (x, x[-tail:].clone()):
        t.requires_grad_()
        y = ckpt8.bias_gelu(t, b)
        both.append((y[-tail:].clone(), torch.autograd.grad(y, t, y.detach())[0][-tail:].clone()))
        del y
    for u, w in zip(*both):
        assert torch.equal(u, w)


BIASES = {"fp32": lambda b: b, "bf16": lambda b: b.bfloat16(), "fp64": lambda b: b.double(),
          "strided": lambda b: torch.stack([b, b - 9.0], 1)[:, 0]}


def check_without_gradients(x, b):
    """The result where nothing is kept is the differentiable form's, bit for bit, in its type."""
    want = ckpt8.bias_gelu(x.detach().requires_grad_(), b)
    for got in (ckpt8.bias_gelu(x, b), ckpt8.bias_gelu(x.t().contiguous().t(), b)):
        assert got.dtype == want.dtype == x.dtype and got.shape == x.shape and torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(ckpt8.bias_gelu(x, b.detach().requires_grad_()), want)


def check_ffn_without_gradients(x, w1, b1, w2):
    want = ckpt8.ffn(x.detach().requires_grad_(), w1, b1, w2)
    got = ckpt8.ffn(x, w1, b1, w2)
    assert got.dtype == want.dtype and got.shape == want.shape and torch.equal(got, want)
    c = b1.detach().requires_grad_()                     # the only operand with a gradient
    (db,) = torch.autograd.grad(ckpt8.ffn(x, w1, c, w2).float().sum(), c)
    assert db.dtype == c.dtype and db.shape == c.shape and bool(db.abs().sum() > 0) == (x.shape[0] > 0)


def ffn_operands(T, I, D):
    g = torch.Generator().manual_seed(I)
    return (values(T, D, 8).float(), 0.2 * torch.randn(I, D, generator=g), torch.randn(I, generator=g),
            0.2 * torch.randn(D, I, generator=g))


@pytest.mark.parametrize("bias", BIASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cpu_without_gradients(bias, dtype):
    b = BIASES[bias](torch.randn(33, generator=torch.Generator().manual_seed(1)))
    check_without_gradients(values(5, 33, 4, dtype), b)
    x, w1, b1, w2 = ffn_operands(5, 33, 40)
    check_ffn_without_gradients(x, w1, BIASES[bias](b1), w2)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", BIASES)
@pytest.mark.parametrize("T,D", [(0, 40), (1, 1), (5, 7), (45, 300), (33, 2047), (33, 2048), (700, 2056)])
def test_without_gradients(T, D, bias):
    b = BIASES[bias](torch.randn(D, generator=torch.Generator().manual_seed(D)).cuda())
    check_without_gradients(values(T, D, T).cuda(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", BIASES)
@pytest.mark.parametrize("T,I", [(0, 40), (3, 33), (70, 128)])
def test_ffn_without_gradients(T, I, bias):
    x, w1, b1, w2 = (t.cuda() for t in ffn_operands(T, I, 64))
    check_ffn_without_gradients(x.bfloat16(), w1, BIASES[bias](b1), w2)


def u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


@pytest.mark.parametrize("call,err", [
    (lambda: ckpt8.gelu_pack(torch.zeros(3, 4), torch.zeros(5)), ValueError),
    (lambda: ckpt8.gelu_pack(torch.zeros(3, 4), torch.zeros(4, device="meta")), ValueError),
    (lambda: ckpt8.gelu_pack(torch.zeros(3, 4, dtype=torch.int32), torch.zeros(4)), TypeError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 1), torch.bfloat16), torch.zeros(3, 40)), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(4, 40)), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(3, 40, device="meta")), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(3, 40, dtype=torch.int32)), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(3, 40), db=torch.zeros(39)), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(3, 40), db=torch.zeros(40).double()), ValueError),
    (lambda: ckpt8.gelu_backward(ckpt8.Packed(u8(3, 40), u8(3, 2), torch.bfloat16), torch.zeros(3, 40), db=torch.zeros(80)[::2]), ValueError),
    (lambda: ckpt8.linear(torch.zeros(3, 4), torch.zeros(2, 4), torch.zeros(3)), ValueError),
    (lambda: ckpt8.linear(torch.zeros(3, 4), torch.zeros(2, 4), torch.zeros(2, device="meta")), ValueError),
    (lambda: ckpt8.ffn(torch.zeros(3, 4), torch.zeros(8, 4), torch.zeros(8, device="meta"), torch.zeros(4, 8)), ValueError),
])
def test_refused_operands(call, err):
    with pytest.raises(err):
        call()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [33, 64])
def test_gelu_pack_and_backward_take_any_strides(D):
    g = torch.Generator().manual_seed(D)
    x, b, dy = values(20, D, 6).cuda(), torch.randn(D, generator=g).cuda(), torch.randn(20, D, generator=g).bfloat16().cuda()
    turned = lambda t: t.t().contiguous().t()
    y, p = ckpt8.gelu_pack(x, b)
    for c in (torch.stack([b, b + 1], 1)[:, 0], b.double()):
        y2, p2 = ckpt8.gelu_pack(turned(x), c)
        assert torch.equal(y2, y) and torch.equal(p2.q, p.q) and torch.equal(p2.s, p.s)
    want = ckpt8.gelu_backward(p, dy, with_y=True)
    got = ckpt8.gelu_backward(ckpt8.Packed(turned(p.q), turned(p.s), p.dtype), turned(dy), with_y=True)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    with pytest.raises(ValueError):
        ckpt8.ffn(x[:, :32].contiguous(), torch.randn(64, 32).cuda(), torch.randn(64), torch.randn(32, 64).cuda())
    with pytest.raises(TypeError):
        ckpt8.gelu_pack(x.float(), b)


def check_no_rows(device, dtype):
    x = torch.zeros(0, 32, dtype=dtype, device=device).requires_grad_()
    mk = lambda *s: torch.randn(*s, device=device).requires_grad_()
    w, b, w2 = mk(16, 32), mk(16), mk(32, 16)
    for out, ts in ((ckpt8.linear(x, w, b), (x, w, b)), (ckpt8.linear(x, w), (x, w)), (ckpt8.ffn(x, w, b, w2), (x, w, b, w2)),
                    (ckpt8.bias_gelu(x, torch.zeros(32, device=device)), (x,))):
        assert out.shape[0] == 0
        for t, g in zip(ts, torch.autograd.grad(out, ts, torch.zeros_like(out))):
            assert g.shape == t.shape and not g.any()


def test_layers_of_no_rows_cpu():
    check_no_rows("cpu", torch.float32)


@pytest.mark.gpu
def test_layers_of_no_rows():
    check_no_rows("cuda", torch.bfloat16)

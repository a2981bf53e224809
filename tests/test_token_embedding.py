"""Scaled token lookup and its sorted gradient (ops/embedding.py::scaled_embedding).

The lookup is one fp32 product and one rounding: equal bits.  The gradient of a row adds n terms in fp32, in
any order: off by at most n 2^-24 of the sum of magnitudes, and one more rounding for the scale.
"""
import math

import pytest
import torch

from dnn_page_vectors_amd.ops.embedding import scaled_embedding


def zipf(T, V, seed, pad_share=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.exp(torch.rand(T, generator=g) * math.log(max(V - 1, 2))).long().clamp(0, V - 1)
    ids[torch.rand(T, generator=g) < pad_share] = 0
    return ids


def grad_oracle(ids, g, V, scale, pad):
    """(dW, bound) in fp64, one token after the other."""
    g = g.double().cpu()
    ids = ids.reshape(-1).cpu()
    keep = (ids >= 0) & (ids < V)
    if pad is not None:
        keep &= ids != pad
    want = torch.zeros(V, g.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(want)
    n = torch.zeros(V, 1, dtype=torch.float64)
    at = ids[keep]
    want.index_put_((at,), scale * g[keep], accumulate=True)
    mag.index_put_((at,), abs(scale) * g[keep].abs(), accumulate=True)
    n.index_put_((at,), torch.ones(len(at), 1, dtype=torch.float64), accumulate=True)
    return want, (n + 1) * 2.0 ** -24 * mag + 1e-40


def check(ids, V, E, out_dtype, pad, scale=3.7, wdtype=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    W = torch.randn(V, E, generator=gen).to(wdtype).cuda().requires_grad_()
    g = torch.randn(ids.numel(), E, generator=gen).to(out_dtype).cuda().view(*ids.shape, E)
    dev = ids.cuda()
    out = scaled_embedding(dev, W, scale, pad, out_dtype)
    assert out.shape == (*ids.shape, E) and out.dtype == out_dtype
    assert torch.equal(out, (W.detach().float()[dev.long()] * scale).to(out_dtype))
    (dW,) = torch.autograd.grad(out, W, g)
    want, tol = grad_oracle(ids, g.reshape(-1, E), V, scale, pad)
    if wdtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * want.abs()
    err = (dW.double().cpu() - want).abs()
    assert dW.dtype == wdtype and (err <= tol).all(), float((err - tol).max())
    assert (dW.cpu()[(tol < 1e-39).all(1)] == 0).all()
    (again,) = torch.autograd.grad(scaled_embedding(dev, W, scale, pad, out_dtype), W, g)
    assert torch.equal(dW, again)
    return W, g, dW


# ---------------------------------------------------------------------------------- CPU

def test_cpu_values_and_gradient():
    W = torch.randn(6, 3, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[1, 0, 5], [1, 1, 2]], dtype=torch.int32)
    out = scaled_embedding(ids, W, -0.5, padding_idx=0)
    assert torch.equal(out, W[ids.long()] * -0.5)
    out.sum().backward()
    assert torch.equal(W.grad[:, 0], torch.tensor([0, -1.5, -0.5, 0, 0, -0.5], dtype=torch.float64))
    assert torch.autograd.gradcheck(lambda w: scaled_embedding(ids, w, 2.0), (W,))
    assert scaled_embedding(ids, W.float(), 2.0, out_dtype=torch.bfloat16).dtype == torch.bfloat16


@pytest.mark.parametrize("bad,err", [
    (dict(ids=torch.zeros(2)), TypeError), (dict(ids=torch.zeros(2, dtype=torch.int16)), TypeError),
    (dict(W=torch.zeros(4)), TypeError), (dict(W=torch.zeros(4, 2, dtype=torch.int32)), TypeError),
    (dict(padding_idx=4), ValueError), (dict(padding_idx=-1), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(scale=float("inf")), ValueError), (dict(ids=torch.tensor([4])), IndexError),
])
def test_refusals(bad, err):
    kw = dict(ids=torch.tensor([0, 1]), W=torch.zeros(4, 2))
    kw.update(bad)
    with pytest.raises(err):
        scaled_embedding(**kw)


# ---------------------------------------------------------------------------------- GPU

@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 500, 2047, 2048, 2049, 2080, 2081, 5000, 40000])
@pytest.mark.parametrize("E", [1, 4, 100, 300, 768])
def test_sizes(T, E):
    V = 5000
    check(zipf(T, V, T + E), V, E, torch.bfloat16 if (T + E) % 2 else torch.float32, 0 if T % 3 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 64, 65, 255, 256, 65534, 65535, 65536, 70000])
@pytest.mark.parametrize("T", [300, 3000])
def test_tables(V, T):
    check(zipf(T, V, V), V, 24, torch.float32, None)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,E", [(131072, 200, 8), (131073, 3000, 4), (300001, 70000, 3), (2100, 1 << 24, 1)])
def test_sort_of_many_tokens(T, V, E):
    """Parts of several tiles with a ragged last one; one to four passes over the ids' bits."""
    check(zipf(T, V, 5), V, E, torch.float32, 7)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^31 elements; a gradient that is zero but for the last tokens."""
    V, E, tail = 1000, 768, 500
    T = (1 << 31) // E + tail
    ids = zipf(T, V, 9).int().cuda()
    W = torch.randn(V, E, device="cuda", requires_grad=True)
    out = scaled_embedding(ids, W, 0.5, 0)
    assert torch.equal(out[-tail:], (W.detach()[ids[-tail:].long()] * 0.5).bfloat16())
    g = torch.zeros_like(out)
    g[-tail:] = torch.randn(tail, E, device="cuda").bfloat16()
    (dW,) = torch.autograd.grad(out, W, g)
    want, tol = grad_oracle(ids[-tail:], g[-tail:], V, 0.5, 0)
    assert ((dW.double().cpu() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("E", [1021, 1024, 1028, 2500])
@pytest.mark.parametrize("T", [100, 4000])
def test_wide_rows(E, T):
    check(zipf(T, 50, 1), 50, E, torch.bfloat16, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 64, 65, 255, 256, 65534, 65535, 65536, 70000])
def test_tables_of_sorted_tokens(V):
    check(zipf(4500, V, V), V, 24, torch.float32, None)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4095, 4096, 4097, 4128, 4129, 5121])
def test_sizes_around_the_sort(T):
    check(zipf(T, 700, T), 700, 36, torch.bfloat16, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1500, 2049, 9000, 33 * 64, 4097, 65 * 64])
@pytest.mark.parametrize("kind", ["one id", "all padding", "two ids", "runs of 32", "runs of 64", "sorted down", "one late"])
def test_runs(T, kind):
    """Runs that end on, begin on and span the borders of the sorted chunks."""
    V = 1000
    ids = {"one id": torch.full((T,), 7), "all padding": torch.zeros(T, dtype=torch.long),
           "two ids": (torch.arange(T) % 2) + 3, "runs of 32": torch.arange(T) // 32 % V,
           "runs of 64": torch.arange(T) // 64 % V, "sorted down": (V - 1) - torch.arange(T) % V,
           "one late": torch.where(torch.arange(T) == T - 1, torch.tensor(999), torch.tensor(1))}[kind]
    check(ids, V, 100, torch.bfloat16, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [50, 3000])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_types_shapes_and_strides(T, idt):
    ids = zipf(T, 300, 2).to(idt)
    check(ids.view(T // 2, 2), 300, 64, torch.bfloat16, 0, wdtype=torch.bfloat16)
    check(ids, 300, 64, torch.float32, 0, wdtype=torch.bfloat16)
    check(ids, 300, 64, torch.float32, 5, scale=0.0)
    check(torch.stack([ids, ids], 1)[:, 1], 300, 40, torch.bfloat16, 0, scale=-1.5)      # strided ids
    flat = torch.randn(300 * 64 + 1, device="cuda")
    W = flat[1:].view(300, 64).requires_grad_()                                          # 4-byte aligned table
    out = scaled_embedding(ids.cuda(), W, 2.0)
    assert torch.equal(out, (W.detach()[ids.cuda().long()] * 2.0).bfloat16())
    g = torch.randn(64, T, device="cuda").bfloat16().t()                                 # strided gradient
    (dW,) = torch.autograd.grad(out, W, g)
    want, tol = grad_oracle(ids, g, 300, 2.0, None)
    assert ((dW.double().cpu() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 5000])
def test_ids_outside_the_table_and_nan_gradients(T):
    V, E = 100, 32
    ids = zipf(T, V, 3)
    ids[5], ids[7], ids[9], ids[11] = -1, V, 2 ** 40, -2 ** 40
    W = torch.randn(V, E, device="cuda", requires_grad=True)
    out = scaled_embedding(ids.cuda(), W, 1.0, 0, torch.float32)
    bad = (ids < 0) | (ids >= V)
    assert out[bad.cuda()].isnan().all() and not out[~bad.cuda()].isnan().any()
    g = torch.randn(T, E, device="cuda")
    g[bad.cuda()] = float("nan")
    g[(ids == 0).cuda()] = float("inf")      # padding rows take part in nothing
    (dW,) = torch.autograd.grad(out, W, g)
    want, tol = grad_oracle(ids, torch.nan_to_num(g, posinf=0.0), V, 1.0, 0)
    assert ((dW.double().cpu() - want).abs() <= tol).all()


@pytest.mark.gpu
def test_no_tokens():
    W = torch.randn(10, 8, device="cuda", requires_grad=True)
    out = scaled_embedding(torch.zeros(0, dtype=torch.int32, device="cuda"), W)
    assert out.shape == (0, 8) and out.dtype == torch.bfloat16
    (dW,) = torch.autograd.grad(out, W, torch.zeros(0, 8, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(dW, torch.zeros_like(W))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [700, 6000])
def test_adds_into_the_flat_gradient(T):
    """Under FlatParams the kernel adds into the parameter's flat gradient, rows without a token untouched."""
    from dnn_page_vectors_amd.ops.optim import FlatParams

    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.W = torch.nn.Parameter(torch.randn(200, 64))

    m = M().cuda()
    flat = FlatParams(m.named_parameters())
    flat.zero_grad()
    m.W.grad.fill_(0.5)
    ids = zipf(T, 150, 1)
    g = torch.randn(T, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    scaled_embedding(ids.cuda(), m.W, 2.0, 0).backward(g)
    want, tol = grad_oracle(ids, g, 200, 2.0, 0)
    got = m.W.grad.double().cpu()
    assert ((got - want - 0.5).abs() <= tol + 2.0 ** -24 * (want.abs() + 0.5)).all()
    assert (got[150:] == 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [700, 6000])
@pytest.mark.parametrize("E", [2, 5, 7, 257, 258, 259])
def test_odd_rows_written_and_added_to(T, E):
    """Rows whose last piece overlaps its neighbour's, across a slab's border too: written, and added into."""
    from dnn_page_vectors_amd.ops.embedding import sorted_row_grad

    V = 90
    ids = zipf(T, V - 20, E)
    _, g, _ = check(ids, V, E, torch.float32, 0, scale=1.5, seed=E)
    want, tol = grad_oracle(ids, g, V, 1.5, 0)
    room = torch.full((V * E + 2,), 0.25, device="cuda")
    sorted_row_grad(ids.cuda(), g, room[1:-1].view(V, E), 1.5, 0, accumulate=True)
    got = room[1:-1].view(V, E).double().cpu()
    assert ((got - want - 0.25).abs() <= tol + 2.0 ** -24 * (want.abs() + 0.25)).all()
    assert room[0] == 0.25 and room[-1] == 0.25 and (got[V - 20:] == 0.25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [400, 5000])
def test_graph_replays_and_side_stream(T):
    V, E = 900, 100
    W = torch.randn(V, E, device="cuda", requires_grad=True)
    ids = zipf(T, V, 0).int().cuda()
    g = torch.randn(T, E, device="cuda").bfloat16()

    def step():
        out = scaled_embedding(ids, W, 2.0, 0)
        return (out,) + torch.autograd.grad(out, W, g)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    for x, y in zip(side, step()):
        assert torch.equal(x, y)
    del side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for rep in range(4):
        ids.copy_(zipf(T, V, 10 + rep).int())
        g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, step()):
            assert torch.equal(x, y), rep


@pytest.mark.gpu
def test_capture_is_refused_while_an_eager_graph_holds_the_table():
    W = torch.randn(50, 16, device="cuda", requires_grad=True)
    ids = torch.arange(30, device="cuda")
    g = torch.randn(30, 16, device="cuda")
    out = scaled_embedding(ids, W, out_dtype=torch.float32)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            scaled_embedding(ids, W, out_dtype=torch.float32)
    (want,) = torch.autograd.grad(out, W, g)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(scaled_embedding(ids, W, out_dtype=torch.float32), W, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_gpu_refusals():
    ids = torch.tensor([0], device="cuda")
    with pytest.raises(TypeError):
        scaled_embedding(ids, torch.zeros(4, 2, device="cuda", dtype=torch.float16))
    with pytest.raises(TypeError):
        scaled_embedding(ids, torch.zeros(4, 2, device="cuda"), out_dtype=torch.float16)
    with pytest.raises(ValueError):
        scaled_embedding(ids.cpu(), torch.zeros(4, 2, device="cuda"))


@pytest.mark.gpu
def test_tables_and_token_counts_whose_grid_would_pass_2_to_the_32():
    """2^30 rows of one column: 2^24 groups of 64 rows to zero.  2^30 tokens of one column."""
    V = (1 << 30) + 70
    ids = torch.tensor([3, V - 1, 3, 64, V - 1, 0], device="cuda")
    W = torch.zeros(V, 1, device="cuda", dtype=torch.bfloat16).requires_grad_()
    out = scaled_embedding(ids, W, 2.0, padding_idx=0)
    g = torch.tensor([1.0, 2.0, 4.0, 8.0, 16.0, 32.0], device="cuda").bfloat16().view(6, 1)
    (dW,) = torch.autograd.grad(out, W, g)
    assert int(torch.count_nonzero(dW)) == 3
    assert dW[[3, 64, V - 1], 0].tolist() == [10.0, 16.0, 36.0]
    del W, dW, out
    T = (1 << 30) + 70
    ids = torch.randint(0, 50, (T,), device="cuda", dtype=torch.int32)
    W = torch.randn(50, 1, device="cuda")
    out = scaled_embedding(ids, W, 2.0)
    for part in (slice(0, 1000), slice(T // 2, T // 2 + 1000), slice(T - 1000, T)):
        assert torch.equal(out[part], (W[ids[part].long()] * 2.0).bfloat16())


@pytest.mark.parametrize("T,V,E", [(-1, 5, 4), (5, 0, 4), (5, 5, 0), ((1 << 31) - 128, 5, 4), (5, (1 << 31) - 1, 4), (5, 5, (1 << 20) + 1)])
def test_sizes_beyond_the_kernels_are_refused(T, V, E):
    from dnn_page_vectors_amd import _native

    lib = _native.hip(required=True)
    assert lib.pv_temb_fwd(None, 0, None, 0, None, 0, T, V, E, 1.0, None, None, None, None, 0, None) < 0
    assert lib.pv_temb_grad(None, 0, None, 0, None, T, V, E, -1, 1.0, 0, None, 0, None) < 0


F = lambda *s: torch.zeros(*s)
I = lambda *s: torch.zeros(*s, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda e: e.lookup_rows(F(4), F(9, 8), F(4, 8), 1.0),
    lambda e: e.lookup_rows(I(8)[::2], F(9, 8), F(4, 8), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(5, 8), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8).t(), F(4, 9), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8).double(), F(4, 8), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8).half(), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8, ).to("meta"), 1.0),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8), 1.0, F(6, 8), F(8), [(1, 3)]),
    lambda e: e.lookup_rows(I(5), F(9, 8), F(5, 8), 1.0, F(6, 8), F(8), [(1, 1)] * 5),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8), 1.0, F(1, 8), F(8), [(2, 2)]),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8), 1.0, F(6, 8).bfloat16(), F(8), [(2, 2)]),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8), 1.0, F(6, 8), None, [(2, 2)]),
    lambda e: e.lookup_rows(I(4), F(9, 8), F(4, 8), 1.0, F(6, 8), F(7), [(2, 2)]),
    lambda e: e.sorted_row_grad(I(4), F(5, 8), F(9, 8), 1.0, None, False),
    lambda e: e.sorted_row_grad(I(4), F(4, 7), F(9, 8), 1.0, None, False),
    lambda e: e.sorted_row_grad(I(4), F(4, 8).double(), F(9, 8), 1.0, None, False),
    lambda e: e.sorted_row_grad(I(4), F(4, 8), F(9, 8).bfloat16(), 1.0, None, False),
    lambda e: e.sorted_row_grad(I(4), F(4, 16)[:, ::2], F(9, 8), 1.0, None, False),
])
def test_refused_operands_of_the_row_functions(call):
    from dnn_page_vectors_amd.ops import embedding

    with pytest.raises((TypeError, ValueError)):
        call(embedding)


@pytest.mark.gpu
@pytest.mark.parametrize("E", [5, 64, 770])
@pytest.mark.parametrize("groups", [[(1, 1)], [(3, 7), (2, 40)], [(1, 300), (0, 5), (4, 0), (9, 31)]])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_lookup_with_position_and_type_rows(E, groups, out):
    """round(scale W[id] + pos[l] + typ): three fp32 roundings, each of at most the magnitudes' sum, and the last."""
    from dnn_page_vectors_amd.ops.embedding import lookup_rows

    gen = torch.Generator().manual_seed(E)
    V, T = 60, sum(N * L for N, L in groups)
    W, pos, typ = torch.randn(V, E, generator=gen), torch.randn(300, E, generator=gen), torch.randn(E, generator=gen)
    ids = torch.randint(0, V, (T,), generator=gen)
    where = torch.cat([torch.arange(L).repeat(N) for N, L in groups])
    got = torch.empty(T, E, dtype=out, device="cuda")
    lookup_rows(ids.cuda(), W.cuda(), got, 1.7, pos.cuda(), typ.cuda(), groups)
    scale = float(torch.tensor(1.7))
    parts = (scale * W.double()[ids], pos.double()[where], typ.double().expand(T, E))
    want, mag = sum(parts), sum(p.abs() for p in parts)
    last = 2.0 ** -8 if out == torch.bfloat16 else 0.0
    assert ((got.double().cpu() - want).abs() <= (3 * 2.0 ** -24 * mag) * (1 + last) + last * want.abs()).all()


@pytest.mark.gpu
def test_ids_outside_the_table_without_the_kernels():
    """The plain form on the GPU (dtype="fp32", backend "torch"): a row of NaN, no gradient, no device assertion."""
    from dnn_page_vectors_amd.ops import _common

    W = torch.randn(20, 6, device="cuda").requires_grad_()
    ids = torch.tensor([3, -1, 20, 3, 1 << 40, 0], device="cuda")
    before = _common.get_backend()
    _common.set_backend("torch")
    try:
        out = scaled_embedding(ids, W, 2.0, padding_idx=0)
        (dW,) = torch.autograd.grad(out, W, torch.ones_like(out))
    finally:
        _common.set_backend(before)
    assert out[[1, 2, 4]].isnan().all() and torch.equal(out[[0, 3, 5]], 2 * W[[3, 3, 0]])
    want = torch.zeros_like(W)
    want[3] = 4
    assert torch.equal(dW, want)

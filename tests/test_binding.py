"""The C++ autograd binding (csrc/binding): built, loadable without a GPU, over the launchers of the library in use."""
import ctypes
import threading

import pytest
import torch

from dnn_page_vectors_amd import _build, _native


def test_built_and_loads():
    assert not _build.binding_stale()
    b = _native.binding()
    assert b is _native.binding()
    for name in ("window_attention", "scaled_embedding", "pack", "unpack", "bias_gelu8", "check_capture"):
        assert callable(getattr(b, name))
    assert _build.TORCH_LIB in _native.loaded_libraries()


def test_needs_every_launcher():
    lib = _native.hip(required=True)
    b = _native.binding()
    names = _native._BINDING_NEEDS
    full = {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names}
    with pytest.raises(KeyError):
        b.init({n: full[n] for n in names[1:]})
    b.init(full)


@pytest.mark.gpu
def test_calls_the_debug_library(monkeypatch):
    """The same results from the debug library's launchers; the release library's again afterwards."""
    from dnn_page_vectors_amd.ops import ckpt8

    x = torch.randn(70, 96, device="cuda").bfloat16()
    want = ckpt8.pack(x)
    debug = ctypes.CDLL(_build.HIP_DEBUG_LIB)
    release, b = _native.hip(required=True), _native.binding()
    addresses = lambda lib: {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _native._BINDING_NEEDS}
    assert addresses(debug) != addresses(release)
    b.init(addresses(debug))
    try:
        got = ckpt8.pack(x)
    finally:
        b.init(addresses(release))
    assert torch.equal(got.q, want.q) and torch.equal(got.s, want.s)
    assert _native.binding() is b


@pytest.mark.gpu
def test_two_threads_on_their_own_streams():
    """A run of the three operators from two threads at once equals the same run alone."""
    from dnn_page_vectors_amd.ops import ckpt8
    from dnn_page_vectors_amd.ops.embedding import scaled_embedding
    from dnn_page_vectors_amd.ops.window_attention import window_attention

    N, L, H, d = 3, 150, 2, 64
    gen = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 500, (N, L), generator=gen).cuda()
    W = torch.randn(500, 3 * H * d, generator=gen).cuda()
    b = torch.randn(H * d, generator=gen).cuda()
    do = torch.randn(N, L, H * d, generator=gen).bfloat16().cuda()

    def run():
        w, bias = W.detach().requires_grad_(), b.detach().requires_grad_()
        q, k, v = scaled_embedding(ids, w, 0.5, 0).view(N, L, 3, H, d).unbind(2)
        y = ckpt8.bias_gelu(window_attention(q, k, v, 20, 20, 1, ids != 0).reshape(N, L, H * d), bias)
        return (y,) + torch.autograd.grad(y, (w, bias), do)

    want = run()
    torch.cuda.synchronize()
    failed = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = run()
                s.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want)):
                    failed.append(threading.get_ident())

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def forward_mode_calls(device):
    """The operators as functions of operands that get tangents."""
    from dnn_page_vectors_amd.ops import ckpt8
    from dnn_page_vectors_amd.ops.embedding import scaled_embedding
    from dnn_page_vectors_amd.ops.window_attention import packed_window_attention, window_attention

    gen = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(device)
    q, x, b, w = mk(1, 8, 2, 32), mk(8, 32), mk(32).float(), mk(32, 32).float()
    ids = torch.arange(4, device=device)
    return {
        "q": (lambda t: window_attention(t, q, q, 2, 2), q), "k": (lambda t: window_attention(q, t, q, 2, 2), q),
        "v": (lambda t: window_attention(q, q, t, 2, 2), q),
        "packed": (lambda t: packed_window_attention(t, [None], [(1, 8)], 2, 2, 2), mk(8, 192)),
        "table": (lambda t: scaled_embedding(ids, t, 0.5), w),
        "gelu": (lambda t: ckpt8.bias_gelu(t, b), x), "gelu bias": (lambda t: ckpt8.bias_gelu(x, t), b),
        "linear": (lambda t: ckpt8.linear(t, w), x),
        "ffn": (lambda t: ckpt8.ffn(t, w, b, w), x), "ffn bias": (lambda t: ckpt8.ffn(x, w, t, w), b),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "packed", "table", "gelu", "gelu bias", "linear", "ffn", "ffn bias"])
def test_forward_mode_is_refused(name, grad):
    """A tangent is never lost in silence: the kernels have no forward-mode form."""
    f, t = forward_mode_calls("cuda")[name]
    t = t.requires_grad_(grad)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            f(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
        f(t)  # without a tangent the level does no harm


@pytest.mark.parametrize("name", ["q", "k", "v", "table", "gelu", "gelu bias", "ffn", "ffn bias"])
def test_forward_mode_cpu(name):
    f, t = forward_mode_calls("cpu")[name]
    with torch.autograd.forward_ad.dual_level():
        out = torch.autograd.forward_ad.unpack_dual(f(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))))
        assert out.tangent is not None and out.tangent.abs().max() > 0


def capture_calls():
    """Differentiable calls of the Python nodes: (function, its leaves, which of them a backward can reach)."""
    from dnn_page_vectors_amd.ops import ckpt8
    from dnn_page_vectors_amd.ops import transformer as tops
    from dnn_page_vectors_amd.ops.embedding import scaled_embedding
    from dnn_page_vectors_amd.ops.optim import FlatParams

    mk = lambda *s: torch.nn.Parameter(torch.randn(*s, device="cuda") * 0.1)
    x = torch.randn(40, 64, device="cuda").bfloat16().requires_grad_()
    w1, b1, w2 = mk(96, 64), mk(96), mk(64, 96)
    word, pos, typ = mk(50, 64), mk(20, 64), mk(2, 64)
    flat_word, flat_bias = mk(50, 64), mk(64)
    FlatParams([("w", flat_word), ("b", flat_bias)])
    ids = torch.randint(0, 50, (4, 10), device="cuda")
    return {
        "linear": (lambda: ckpt8.linear(x, w1, b1), (x, w1, b1)),
        "ffn": (lambda: ckpt8.ffn(x, w1, b1, w2), (x, w1, b1, w2)),
        "embed": (lambda: tops.bert_embed(word, pos, typ, [ids], 2.0), (word, pos, typ)),
        "flat table": (lambda: scaled_embedding(ids, flat_word, 2.0), (flat_word,)),
        "flat bias": (lambda: ckpt8.bias_gelu(x, flat_bias), (x, flat_bias)),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear", "ffn", "embed", "flat table", "flat bias"])
def test_python_nodes_refuse_a_capture_over_held_leaves(name):
    """As the C++ nodes do: nothing is captured, and once the eager graph is gone the capture works."""
    f, leaves = capture_calls()[name]
    held = f()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            f()
    del held
    dy = torch.randn_like(f().detach())
    want = torch.autograd.grad(f(), leaves, dy, allow_unused=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(f(), leaves, dy, allow_unused=True)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert (a is None) == (c is None)   # a flat parameter's gradient is written in place
            # a bias of the linear layer is summed by atomics: any order of 40 terms
            assert a is None or torch.allclose(a, c, rtol=1e-4, atol=40 * 2.0 ** -23 * float(dy.float().abs().sum(0).max()))

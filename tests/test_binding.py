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

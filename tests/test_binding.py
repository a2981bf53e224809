"""The C++ autograd binding (csrc/binding): built, loadable without a GPU, over the launchers of the library in use."""
import ctypes

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

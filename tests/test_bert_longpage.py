"""The long-page transformer tower: scaled lookup, windowed attention and 8-bit checkpoints run together, through the
model, the trainer and encode()."""
import ctypes

import pytest
import torch

from dnn_page_vectors_amd.config import Configuration, preset_config
from dnn_page_vectors_amd.data.synthetic import SyntheticPairs, spec_from_config
from dnn_page_vectors_amd.models import build_model
from dnn_page_vectors_amd.train.trainer import Trainer


def config(**kw):
    base = dict(bert_layers=2, bert_hidden=64, bert_heads=2, bert_intermediate=128, vocab_hash_size=400, query_length=8,
                document_length=80, bert_max_len=80, batch_size=8, bert_dropout=0.0, bert_window=12, bert_sinks=1,
                bert_embed_scale=8.0, bert_ckpt8=True)
    base.update(kw)
    return preset_config("bert_longpage").replace(**base)


def pair_batch(cfg, device="cpu", seed=3):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(1, 400, (cfg.batch_size, cfg.query_length), generator=g)
    d = torch.randint(1, 400, (cfg.batch_size, 1, cfg.document_length), generator=g)
    n = torch.randint(5, cfg.document_length + 1, (cfg.batch_size, 1, 1), generator=g)
    d = torch.where(torch.arange(cfg.document_length) < n, d, torch.zeros_like(d))
    d[0] = 0                                       # an empty page
    return q.to(torch.int32).to(device), d.to(torch.int32).to(device)


def loss_of(m, q, d):
    a, b = m(q, d)
    return (torch.nn.functional.normalize(a.float(), dim=-1) @ torch.nn.functional.normalize(b[:, 0].float(), dim=-1).t()).square().sum()


def grads_of(cfg, device, backend=None):
    m = build_model(cfg, 400).to(device)
    m.train()
    q, d = pair_batch(cfg, device)
    loss = loss_of(m, q, d)
    loss.backward()
    return float(loss.detach()), {n: p.grad.detach().double().cpu() for n, p in m.named_parameters()}


def test_window_over_the_page_is_dense_attention_cpu():
    a, ga = grads_of(config(bert_window=80, bert_ckpt8=False, bert_embed_scale=0.0), "cpu")
    b, gb = grads_of(config(bert_window=0, bert_ckpt8=False, bert_embed_scale=0.0), "cpu")
    assert abs(a - b) <= 1e-5 * abs(b)
    for n in ga:
        assert torch.allclose(ga[n], gb[n], rtol=1e-3, atol=1e-6), n


def test_packed_and_separate_towers_agree_cpu():
    cfg = config()
    m = build_model(cfg, 400).eval()
    q, d = pair_batch(cfg)
    with torch.no_grad():
        a, b = m(q, d)
        assert torch.allclose(a, m.tower_forward("query", q, False, 0), atol=1e-5)
        assert torch.allclose(b[:, 0], m.tower_forward("doc", d[:, 0], False, 0), atol=1e-5)


def test_window_limits_what_a_token_sees_cpu():
    """One layer: [CLS] sees the tokens 0 .. window; changing a later one changes nothing."""
    cfg = config(bert_layers=1, bert_window=5)
    m = build_model(cfg, 400).eval()
    ids = torch.randint(1, 400, (1, 40), generator=torch.Generator().manual_seed(0))
    far, near = ids.clone(), ids.clone()
    far[0, 6], near[0, 5] = 7, 7
    with torch.no_grad():
        v, w, x = (m.tower_forward("doc", t, False, 0) for t in (ids, far, near))
    assert torch.equal(v, w) and not torch.equal(v, x)


def test_config_refusals_and_round_trip(tmp_path):
    with pytest.raises(ValueError):
        Configuration(bert_window=-1)
    with pytest.raises(ValueError):
        Configuration(bert_sinks=-1)
    for scale in (-1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            Configuration(bert_embed_scale=scale)
    cfg = config()
    cfg.save_json(str(tmp_path / "c.json"))
    back = Configuration.load_json(str(tmp_path / "c.json"))
    assert (back.bert_window, back.bert_sinks, back.bert_embed_scale, back.bert_ckpt8) == (12, 1, 8.0, True)
    assert cfg.override(["bert_window=7", "bert_ckpt8=false"]).bert_window == 7


def test_trains_and_encodes_cpu():
    cfg = config()
    m = build_model(cfg, 400)
    tr = Trainer(cfg, m)
    before = tr.flat.data.clone()
    out = tr.train_step(*SyntheticPairs(spec_from_config(cfg, 400, num_pages=64)).batch(cfg.batch_size))
    assert float(out["loss"]) == float(out["loss"]) and not torch.equal(before, tr.flat.data)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("kw", [dict(), dict(bert_ckpt8=False), dict(bert_window=0), dict(bert_embed_scale=0.0)])
def test_gradients_against_the_cpu_model(heads, kw):
    """Two layers in bf16 against the same model in fp32.  A layer rounds about 12 times to bf16 in each direction
    (2^-8 each): 2 x 2 x 12 x 2^-8 = 0.19 of a gradient's norm if all added up, and a weight gradient reads
    activations that are off by up to 2^-4 = 0.06."""
    cfg = config(bert_heads=heads, **kw)
    l0, want = grads_of(cfg, "cpu")
    l1, got = grads_of(cfg, "cuda")
    assert abs(l0 - l1) <= 0.19 * abs(l0)
    for n in want:
        if float(want[n].norm()) > 1e-3 * max(float(w.norm()) for w in want.values()):
            off = float((got[n] - want[n]).norm() / want[n].norm())
            assert off <= 0.25, (n, off)


@pytest.mark.gpu
def test_same_bits_in_deterministic_mode():
    # hidden 256: the LayerNorm kernels of 256 / 512 / 768 / 1024 columns have no atomics (others do)
    cfg = config(deterministic=True, loss_mode="in_batch", bert_hidden=256, bert_heads=4, bert_intermediate=512)
    ends = []
    for _ in range(2):
        m = build_model(cfg, 400)
        tr = Trainer(cfg, m, torch.device("cuda:0"))
        data = SyntheticPairs(spec_from_config(cfg, 400, num_pages=64), torch.device("cuda:0"), seed=1)
        for _ in range(3):
            tr.train_step(*data.batch(cfg.batch_size))
        torch.cuda.synchronize()
        ends.append(tr.flat.data.clone())
    assert torch.equal(*ends) and torch.isfinite(ends[0]).all()
    from dnn_page_vectors_amd.ops import determinism
    determinism.ensure(False)


@pytest.mark.gpu
def test_trains_with_dropout_and_encodes():
    cfg = config(bert_dropout=0.1)
    dev = torch.device("cuda:0")
    m = build_model(cfg, 400)
    tr = Trainer(cfg, m, dev)
    data = SyntheticPairs(spec_from_config(cfg, 400, num_pages=64), dev, seed=1)
    before = tr.flat.data.clone()
    for _ in range(3):
        out = tr.train_step(*data.batch(cfg.batch_size))
    assert float(out["loss"]) == float(out["loss"]) and not torch.equal(before, tr.flat.data)
    ids = pair_batch(cfg, dev)[1][:, 0]
    v = m.encode(ids, "doc")
    assert v.shape == (cfg.batch_size, m.out_dim) and torch.isfinite(v).all()
    assert torch.equal(v[2:3], m.encode(ids[2:3], "doc"))        # a page's vector does not depend on its batch


@pytest.mark.gpu
def test_captured_step_replays():
    """Forward and backward of the tower in a hipGraph, replayed with eager steps between, against the eager step."""
    cfg = config(loss_mode="in_batch")
    dev = torch.device("cuda:0")
    m = build_model(cfg, 400).to(dev)
    m.train()
    q, d = pair_batch(cfg, dev)
    ps = [p for p in m.parameters()]

    def step():
        return torch.autograd.grad(loss_of(m, q, d), ps)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    names = [n for n, _ in m.named_parameters()]
    for rep in range(4):
        a, b = pair_batch(cfg, dev, seed=20 + rep)
        q.copy_(a)
        d.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for n, x, y in zip(names, got, step()):
            if n.endswith((".pos", ".typ")):
                continue                             # torch's own sums (see below)
            # bias and LayerNorm sums of the dense layers add by atomics: any order of T terms
            assert torch.allclose(x, y, rtol=1e-3, atol=1e-4 * float(y.abs().max()) + 1e-12), (rep, n)


def node_kinds(graph):
    """How many nodes of each kind a captured graph holds (0 kernel, 1 copy, 2 memset)."""
    hip = ctypes.CDLL("libamdhip64.so")
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    kinds = []
    for x in nodes:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(x), ctypes.byref(t)) == 0
        kinds.append(t.value)
    return {k: kinds.count(k) for k in set(kinds)}


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(bert_window=0, bert_ckpt8=False, bert_embed_scale=0.0)])
def test_captured_step_replays_position_and_type_gradients(kw):
    """Tables of 2000 positions, whose sum into the type row torch would split over workgroups.  At 256 columns nothing
    on the way to these gradients is added by atomics: the same bits in every replay as in the eager step."""
    cfg = config(loss_mode="in_batch", bert_max_len=2000, document_length=300, bert_hidden=256, bert_heads=4, **kw)
    dev = torch.device("cuda:0")
    m = build_model(cfg, 400).to(dev)
    m.train()
    q, d = pair_batch(cfg, dev)
    ps = list(m.parameters())

    def step():
        return torch.autograd.grad(loss_of(m, q, d), ps)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        got = step()
    assert 2 not in node_kinds(graph)
    for rep in range(4):
        a, b = pair_batch(cfg, dev, seed=20 + rep)
        q.copy_(a)
        d.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for (n, _), x, y in zip(m.named_parameters(), got, step()):
            if n.endswith((".pos", ".typ")):
                assert y.abs().max() > 0 and torch.equal(x, y), (rep, n)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(bert_window=0, bert_ckpt8=False, bert_embed_scale=0.0)])
def test_captured_step_of_separate_towers(kw):
    """The same where each tower runs alone, its position and type rows added to the token rows."""
    test_captured_step_replays_position_and_type_gradients(dict(share_doc_tower=False, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [[(1, 1)], [(3, 7), (5, 40)], [(200, 5), (0, 9), (2, 1999)], [(70, 33)]])
def test_position_and_type_gradients(groups):
    """Against 64 bits: a sum of n fp32 terms in any order is off by n 2^-24 of the sum of magnitudes."""
    from dnn_page_vectors_amd.ops import transformer as tops

    H, P = 96, 2000
    T = sum(N * L for N, L in groups)
    g = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).bfloat16()
    want, mag, terms = torch.zeros(P, H).double(), torch.zeros(P, H).double(), 0
    off = 0
    for N, L in groups:
        part = g[off:off + N * L].view(N, L, H).double()
        want[:L] += part.sum(0)
        mag[:L] += part.abs().sum(0)
        terms += N
        off += N * L
    pos, typ = torch.zeros(P, H, device="cuda"), torch.zeros(2, H, device="cuda")
    dpos, dtyp = tops._position_grads(g.cuda(), groups, pos, typ, True, True)
    assert ((dpos.double().cpu() - want).abs() <= (terms + 1) * 2.0 ** -24 * mag).all()
    assert ((dtyp[0].double().cpu() - want.sum(0)).abs() <= (terms + P + 1) * 2.0 ** -24 * mag.sum(0)).all()
    assert not dtyp[1].any()
    again = tops._position_grads(g.cuda(), groups, pos, typ, True, True)
    assert torch.equal(dpos, again[0]) and torch.equal(dtyp, again[1])


def test_head_dims_that_the_gpu_refuses_are_found_before_the_first_step():
    """96 columns in 4 heads of 24: the CPU form takes them, a trainer on the GPU says so when it is made."""
    bad = config(bert_hidden=96, bert_heads=4)
    m = build_model(bad, 400)
    with pytest.raises(ValueError, match="head dims"):
        Trainer(bad, m, torch.device("cuda:0"))
    out = Trainer(bad, m, torch.device("cpu")).train_step(*SyntheticPairs(spec_from_config(bad, 400, num_pages=64)).batch(8))
    assert float(out["loss"]) == float(out["loss"])
    for fine in (bad.replace(bert_window=0), bad.replace(dtype="fp32"), config()):
        build_model(fine, 400).check_device(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,status", [("bf16", "captured"), ("fp32", "eager")])
def test_steps_with_memsets_are_not_replayed(dtype, status):
    """dtype="fp32" runs torch's own sums, whose memsets replays repeat wrongly (bias gradients off by orders of
    magnitude): the trainer keeps such a step eager and says so.  The gradients are then those of a trainer without graphs."""
    kw = dict(dtype=dtype, loss_mode="in_batch", bert_max_len=2000, document_length=300, bert_hidden=256, bert_heads=4)
    dev = torch.device("cuda:0")
    grads = []
    for graph in (True, False):
        cfg = config(lr=0.0, **kw)                   # the weights stay: every step of a batch has the same gradient
        tr = Trainer(cfg, build_model(cfg, 400), dev, graph=graph)
        for seed in range(6):
            q, d = pair_batch(cfg, dev, seed=seed)
            tr.train_step(q, d)
        torch.cuda.synchronize()
        assert tr.graph_status.startswith(status if graph else "off")
        assert (tr._graph is not None) == (graph and status == "captured")
        grads.append(tr.flat.grad.clone())
        tr.close()
    a, b = grads
    assert torch.isfinite(a).all() and b.abs().max() > 0
    # sums of the same terms in another order (atomics)
    assert float((a - b).norm()) <= 1e-3 * float(b.norm())


@pytest.mark.gpu
def test_memset_nodes_are_counted():
    from dnn_page_vectors_amd import _native

    x = torch.randn(4000, 256, device="cuda")
    for f, sets in ((lambda: x * 2, 0), (lambda: x.sum(0), 1)):
        f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            y = f()
        kinds = node_kinds(graph)
        assert _native.binding().graph_memsets(graph.raw_cuda_graph()) == kinds.get(2, 0) == sets
        del y

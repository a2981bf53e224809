"""What the operators of the long-page transformer tower cost: the calls that are timed, over the range of sizes
that training and encoding pages meet, with the same results computed by elementary torch operations in 32 bits.

Three operators, in the order a step runs them:

* ``embed``   scaled token-embedding lookup, its table gradient summed over the sorted tokens (ops/embedding.py)
* ``attn``    attention with a sliding window and a few first tokens that stay visible (ops/window_attention.py)
* ``gelu8`` / ``pack8``  activation checkpoints in 8 bits: the FFN's bias + GELU whose backward reads e4m3 values
  with a power-of-two scale per 32 columns, and the packing of any activation (ops/ckpt8.py)

``own`` False: ``run`` computes the plain form.  True: it calls the framework.
"""
import math

import torch

own = False

DEV = "cuda"
GELU_K, GELU_C = math.sqrt(2.0 / math.pi), 0.044715
BLOCK = 32          # columns that share one scale of the 8-bit checkpoints
E4M3_TOP = 448.0    # the largest e4m3 value, 1.75 * 2^8


# ------------------------------------------------------------------------------------------------ cases
def _attn(name, N, L, H, Hkv, d, left, right, sinks, fill, train):
    c = {"op": "attn", "N": N, "L": L, "H": H, "Hkv": Hkv, "d": d, "left": left, "right": right, "sinks": sinks,
         "fill": fill, "train": train}
    return c if name is None else {"name": name, **c}


def _embed(name, T, V, E, scale, pad, out, train):
    c = {"op": "embed", "T": T, "V": V, "E": E, "scale": scale, "pad": pad, "out": out, "train": train}
    return c if name is None else {"name": name, **c}


def _ckpt(name, op, T, D, dtype):
    c = {"op": op, "T": T, "D": D, "dtype": dtype}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # four queries of 32 words encoded for a search: the smallest call, all latency
        _attn("attn_query_encode", 4, 32, 12, 12, 64, 16, 16, 1, 1.0, False),
        # a training step's ngram pages, 2000 tokens, ragged, the first token stays visible
        _attn("attn_page_train", 32, 2000, 12, 12, 64, 256, 256, 1, 0.75, True),
        # word-level pages of odd length 975, a narrower window and four sinks
        _attn("attn_word_train", 64, 975, 12, 12, 64, 128, 128, 4, 0.6, True),
        # a causal tower with grouped key/value heads and wider heads, chunked-page length 4096
        _attn("attn_causal_grouped_train", 4, 4096, 16, 4, 128, 1023, 0, 4, 1.0, True),
        # one very long page encoded alone
        _attn("attn_long_encode", 1, 16384, 12, 12, 64, 512, 512, 16, 1.0, False),
        # one query's tokens looked up: the smallest lookup
        _embed("embed_query_encode", 45, 30522, 768, 27.712812921102035, 0.0, "bfloat16", False),
        # a small tower's step: 32 queries of 45 trigrams, table of 1024 x 300
        _embed("embed_small_train", 1440, 1024, 300, 17.320508075688775, 0.2, "float32", True),
        # the dual encoder's step: 256 queries of 32 and 256 pages of 256 words
        _embed("embed_step_train", 73728, 30522, 768, 27.712812921102035, 0.3, "bfloat16", True),
        # a step over 128 pages of 2000 tokens
        _embed("embed_pages_train", 256000, 30522, 512, 22.627416997969522, 0.25, "bfloat16", True),
        # the FFN activation of the dual encoder's step
        _ckpt("gelu8_step", "gelu8", 73728, 2048, "bfloat16"),
        # a few queries through a narrow FFN whose width ends inside a block
        _ckpt("gelu8_small_odd", "gelu8", 45, 300, "bfloat16"),
        # the input of a projection, kept for its weight gradient
        _ckpt("pack8_pages", "pack8", 256000, 768, "bfloat16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "embed", "embed", "gelu8", "pack8"])
    if op == "attn":
        train = rng.random() < 0.65
        d = rng.choice([32, 64, 64, 128])
        Hkv = rng.choice([1, 2, 3, 4, 8, 12])
        H = Hkv * rng.choice([g for g in (1, 1, 2, 4) if Hkv * g <= 16])
        L = _log(rng, 8 if train else 1, 8192)   # a lone key has no gradient but its rounding
        left = rng.choice([None, _log(rng, 2, 1024), _log(rng, 2, 1024), _log(rng, 2, 256)])
        right = rng.choice([0, left, left])
        one = {"L": L, "left": left, "right": right, "sinks": 0}
        if H * d * 14 * _pairs(one) > 4e11:
            one["left"] = left = 256
            one["right"] = right = min(right or 0, 256)
        most = min(65536 // L, 1.2e9 / (H * L * L), 64, 4e11 / (H * d * 14 * _pairs(one)))
        N = _log(rng, 1, max(1, int(most)))
        sinks = rng.choice([0, 1, 4, rng.randint(2, 80)])
        fill = rng.choice([1.0, rng.uniform(0.5, 0.95)])
        return _attn(None, N, L, H, Hkv, d, left, right, sinks, round(fill, 3), train)
    if op == "embed":
        E = rng.choice([_log(rng, 1, 1024), 8 * _log(rng, 4, 128), 100, 768])
        V = _log(rng, 16, 60000)
        out = rng.choice(["bfloat16", "float32"])
        T = _log(rng, 1, min(256000, int((1.3e8 if out == "bfloat16" else 6.5e7) / E)))
        return _embed(None, T, V, E, round(math.sqrt(E), 6), round(rng.choice([0.0, rng.uniform(0.05, 0.6)]), 3), out,
                      rng.random() < 0.75)
    D = rng.choice([_log(rng, 1, 4096), 32 * _log(rng, 1, 128), 768])
    dtype = rng.choice(["bfloat16", "float32"]) if op == "pack8" else "bfloat16"
    T = _log(rng, 1, min(80000, int((1.5e8 if dtype == "bfloat16" else 7.5e7) / D)))
    return _ckpt(None, op, T, D, dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _lengths(case, g):
    """Real tokens of each page: the mean share is ``fill``, spread evenly around it; at least one."""
    N, L, f = case["N"], case["L"], case["fill"]
    lo = max(0.0, 2 * f - 1)
    u = lo + (1 - lo) * torch.rand(N, generator=g, device=DEV)
    return (u * L).round().clamp(1, L).long()


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "attn":
        N, L, H, Hkv, d = (case[k] for k in ("N", "L", "H", "Hkv", "d"))
        mk = lambda h: torch.randn(N, L, h, d, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
        q, k, v = mk(H), mk(Hkv), mk(Hkv)
        mask = None
        if case["fill"] < 1.0:
            mask = torch.arange(L, device=DEV)[None, :] < _lengths(case, g)[:, None]
        st = {"case": case, "q": q, "k": k, "v": v, "mask": mask}
        if case["train"]:
            st["do"] = mk(H)
            for n in "qkv":
                st[n].requires_grad_()
        return st
    if op == "embed":
        T, V, E = case["T"], case["V"], case["E"]
        u = torch.rand(T, generator=g, device=DEV)
        ids = torch.exp(u * math.log(max(V - 1, 2))).long().clamp(1, V - 1)   # few ids are frequent, most are rare
        ids = torch.where(torch.rand(T, generator=g, device=DEV) < case["pad"], torch.zeros_like(ids), ids)
        W = torch.randn(V, E, generator=g, device=DEV) * 0.02
        st = {"case": case, "ids": ids.to(torch.int32), "W": W, "out": getattr(torch, case["out"])}
        if case["train"]:
            st["do"] = torch.randn(T, E, generator=g, device=DEV).to(st["out"])
            W.requires_grad_()
        return st
    T, D = case["T"], case["D"]
    # activations of a trained layer: columns of different sizes, a few of them large
    col = torch.exp(0.8 * torch.randn(D, generator=g, device=DEV))
    x = (torch.randn(T, D, generator=g, device=DEV) * col).to(getattr(torch, case["dtype"]))
    st = {"case": case, "x": x}
    if op == "gelu8":
        st["b"] = torch.randn(D, generator=g, device=DEV) * 0.1
        st["dy"] = torch.randn(T, D, generator=g, device=DEV).to(torch.bfloat16)
        st["x"].requires_grad_()
        st["b"].requires_grad_()
    return st


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(st):
    from dnn_page_vectors_amd.ops import ckpt8
    from dnn_page_vectors_amd.ops.embedding import scaled_embedding
    from dnn_page_vectors_amd.ops.window_attention import window_attention

    c = st["case"]
    if c["op"] == "attn":
        def call():
            return window_attention(st["q"], st["k"], st["v"], left=c["left"], right=c["right"], sinks=c["sinks"],
                                    mask=st["mask"])
        if not c["train"]:
            with torch.no_grad():
                return {"out": call()}
        out = call()
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "embed":
        def call():
            return scaled_embedding(st["ids"], st["W"], scale=c["scale"], padding_idx=0, out_dtype=st["out"])
        if not c["train"]:
            with torch.no_grad():
                return {"out": call()}
        out = call()
        (dW,) = torch.autograd.grad(out, st["W"], st["do"])
        return {"out": out.detach(), "dW": dW}
    if c["op"] == "gelu8":
        y = ckpt8.bias_gelu(st["x"], st["b"])
        dx, db = torch.autograd.grad(y, (st["x"], st["b"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "db": db}
    return {"x": ckpt8.unpack(ckpt8.pack(st["x"]))}


# ------------------------------------------------------------------------------------------------ the plain forms
def _visible(c):
    """(L, L) truth values: key j is visible to query i when i - left <= j <= i + right, or when j is one of the
    first ``sinks`` tokens and j <= i + right (a sink stays visible once the window has moved past it)."""
    L = c["L"]
    i = torch.arange(L, device=DEV)[:, None]
    j = torch.arange(L, device=DEV)[None, :]
    vis = torch.ones(L, L, dtype=torch.bool, device=DEV)
    if c["left"] is not None:
        vis = vis & ((j >= i - c["left"]) | (j < c["sinks"]))
    if c["right"] is not None:
        vis = vis & (j <= i + c["right"])
    return vis


def _plain_attn(st):
    c = st["case"]
    G = c["H"] // c["Hkv"]
    scale = 1.0 / math.sqrt(c["d"])
    q = st["q"].float().permute(0, 2, 1, 3).contiguous()
    k = st["k"].float().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    v = st["v"].float().permute(0, 2, 1, 3).repeat_interleave(G, 1)
    hide = ~_visible(c)[None, None]
    if st["mask"] is not None:
        hide = hide | ~st["mask"][:, None, None, :]
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(hide, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(p, v)
    out = {"out": o.permute(0, 2, 1, 3).to(torch.bfloat16).contiguous()}
    if c["train"]:
        do = st["do"].float().permute(0, 2, 1, 3).contiguous()
        N, L, d = c["N"], c["L"], c["d"]
        heads = lambda t: t.view(N, c["Hkv"], G, L, d).sum(2).permute(0, 2, 1, 3).to(torch.bfloat16).contiguous()  # noqa: E731
        ds = torch.matmul(do, v.transpose(2, 3).contiguous())
        ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dv"] = heads(torch.matmul(p.transpose(2, 3).contiguous(), do))
        out["dq"] = torch.matmul(ds, k).permute(0, 2, 1, 3).to(torch.bfloat16).contiguous()
        out["dk"] = heads(torch.matmul(ds.transpose(2, 3).contiguous(), q))
    return out


def _plain_embed(st):
    c = st["case"]
    ids = st["ids"].long()
    out = {"out": (st["W"][ids] * c["scale"]).to(st["out"])}
    if c["train"]:
        g = st["do"].float() * (ids != 0).float()[:, None]
        out["dW"] = torch.zeros(c["V"], c["E"], device=DEV).index_add_(0, ids, g) * c["scale"]
    return out


def _blocks(u):
    T, D = u.shape
    pad = -D % BLOCK
    return torch.nn.functional.pad(u, (0, pad)).view(T, (D + pad) // BLOCK, BLOCK)


def _two_to(e):
    """2^e in 32 bits from its bit pattern (a power function may miss it by a rounding); -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _through_8_bits(u):
    """The values that the checkpoint of u (T, D) stands for: each block of 32 columns divided by the smallest power
    of two that brings its largest magnitude to at most 448, rounded to e4m3."""
    b = _blocks(u.float())
    mant, ex = torch.frexp(b.abs().amax(-1, keepdim=True))          # top = mant * 2^ex, mant in [0.5, 1)
    e = (ex - 9 + (mant > E4M3_TOP / 512.0).int()).clamp(-126, 126)  # 448 = 0.875 * 2^9
    q = (b * _two_to(-e)).to(torch.float8_e4m3fn).float()
    return (q * _two_to(e)).reshape(u.shape[0], -1)[:, :u.shape[1]]


def _plain_gelu8(st):
    u = st["x"].float() + st["b"]
    y = 0.5 * u * (1 + torch.tanh(GELU_K * (u + GELU_C * u * u * u)))
    h = _through_8_bits(u)
    t = torch.tanh(GELU_K * (h + GELU_C * h * h * h))
    slope = 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * GELU_K * (1 + 3 * GELU_C * h * h)
    du = st["dy"].float() * slope
    return {"y": y.to(torch.bfloat16), "dx": du.to(torch.bfloat16), "db": du.sum(0)}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op == "attn":
            return _plain_attn(state)
        if op == "embed":
            return _plain_embed(state)
        if op == "gelu8":
            return _plain_gelu8(state)
        return {"x": _through_8_bits(state["x"]).to(state["x"].dtype)}


# ------------------------------------------------------------------------------------------------ what a pass needs
def _pairs(c):
    """Visible (query, key) pairs of one sequence and head without padding."""
    L = c["L"]
    left = L if c["left"] is None else c["left"]
    right = L if c["right"] is None else c["right"]
    n = 0
    for i in range(L):
        lo, hi = max(0, i - left), min(L - 1, i + right)
        n += hi - lo + 1 + max(0, min(c["sinks"], lo, hi + 1))
    return n


def work(case):
    c = case
    if c["op"] == "attn":
        q, kv = c["N"] * c["L"] * c["H"] * c["d"], c["N"] * c["L"] * c["Hkv"] * c["d"]
        pairs = c["N"] * c["H"] * _pairs(c) * c["fill"]
        if c["train"]:  # out, dq, dk, dv written; q, k, v, do read; five products
            return {"bytes": 2 * (4 * q + 4 * kv), "flops": 14 * pairs * c["d"]}
        return {"bytes": 2 * (2 * q + 2 * kv), "flops": 4 * pairs * c["d"]}
    if c["op"] == "embed":
        T, V, E = c["T"], c["V"], c["E"]
        ob = 2 if c["out"] == "bfloat16" else 4
        rows = min(V, T)
        b = 4 * T + 4 * rows * E + ob * T * E
        if c["train"]:
            b += ob * T * E + 4 * V * E
        return {"bytes": b, "flops": (2 if c["train"] else 1) * T * E}
    n = c["T"] * c["D"]
    s = 2 if c["dtype"] == "bfloat16" else 4
    held = n + c["T"] * ((c["D"] + BLOCK - 1) // BLOCK)
    if c["op"] == "gelu8":  # x and dy read, y and dx written, the checkpoint written and read
        return {"bytes": 4 * s * n + 2 * held, "flops": 30 * n}
    return {"bytes": 2 * s * n + 2 * held, "flops": 4 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attn(c, st):
    if c["N"] * c["H"] * c["L"] ** 2 > 6e9:
        return None
    N, L, H, G, d = c["N"], c["L"], c["H"], c["H"] // c["Hkv"], c["d"]
    at = torch.arange(L, device=DEV)
    gap = at[None, :] - at[:, None]                    # key position minus query position
    allowed = torch.ones_like(gap, dtype=torch.bool)
    if c["right"] is not None:
        allowed &= gap <= c["right"]
    if c["left"] is not None:
        allowed &= (gap >= -c["left"]) | (at < c["sinks"])[None, :]
    # the padded keys of each sequence are left out of its products
    step = max(1, int(4e8 / (L * L)))
    res = {n: torch.zeros(N, L, h, d, dtype=torch.float64, device=DEV)
           for n, h in ([("out", H)] + ([("dq", H), ("dk", c["Hkv"]), ("dv", c["Hkv"])] if c["train"] else []))}
    for n in range(N):
        keys = L if st["mask"] is None else int(st["mask"][n].sum())
        ok = allowed[:, :keys]
        for h0 in range(0, H, step):
            hs = torch.arange(h0, min(H, h0 + step), device=DEV)
            q = st["q"].detach()[n][:, hs].double().transpose(0, 1).contiguous()
            k = st["k"].detach()[n, :keys][:, hs // G].double().transpose(0, 1).contiguous()
            v = st["v"].detach()[n, :keys][:, hs // G].double().transpose(0, 1).contiguous()
            w = torch.bmm(q, k.transpose(1, 2).contiguous()) / d ** 0.5
            w = torch.softmax(torch.where(ok, w, torch.full((), -1e300, dtype=torch.float64, device=DEV)), -1) * ok
            o = torch.bmm(w, v)
            res["out"][n][:, hs] = o.transpose(0, 1)
            if c["train"]:
                g = st["do"][n][:, hs].double().transpose(0, 1).contiguous()
                res["dv"][n, :keys].index_add_(1, hs // G, torch.bmm(w.transpose(1, 2).contiguous(), g).transpose(0, 1))
                e = torch.bmm(g, v.transpose(1, 2).contiguous())
                e = w * (e - (e * w).sum(-1, keepdim=True)) / d ** 0.5
                res["dq"][n][:, hs] = torch.bmm(e, k).transpose(0, 1)
                res["dk"][n, :keys].index_add_(1, hs // G, torch.bmm(e.transpose(1, 2).contiguous(), q).transpose(0, 1))
    return res


def _exact_embed(c, st):
    ids = st["ids"].long()
    out = {"out": torch.index_select(st["W"].detach().double(), 0, ids) * c["scale"]}
    if c["train"]:
        # sums of runs of the sorted tokens, as differences of one running sum
        at = torch.nonzero(ids != 0).flatten()
        order = torch.argsort(ids[at], stable=True)
        rows, n = torch.unique_consecutive(ids[at][order], return_counts=True)
        dW = torch.zeros(c["V"], c["E"], dtype=torch.float64, device=DEV)
        if at.numel():
            ends = torch.cumsum(n, 0)
            run = torch.cumsum(st["do"].double()[at[order]] * c["scale"], 0)[ends - 1]
            dW[rows] = torch.diff(run, dim=0, prepend=torch.zeros(1, c["E"], dtype=torch.float64, device=DEV))
        out["dW"] = dW
    return out


def _power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(v):
    """v (64 bits, magnitudes up to 448) to the nearest e4m3 value: steps of 2^(exponent - 3), no finer than 2^-9."""
    _, ex = torch.frexp(v)
    step = _power((ex - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_8_bits(u):
    out = torch.empty_like(u)
    for c0 in range(0, u.shape[1], BLOCK):
        part = u[:, c0:c0 + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        e = torch.log2(top.clamp(min=1e-300) / E4M3_TOP).round() - 1     # one of the two next to the right one
        e = e + (top > E4M3_TOP * _power(e)) + (top > 2 * E4M3_TOP * _power(e))
        unit = _power(e.clamp(min=-126))
        out[:, c0:c0 + BLOCK] = _round_e4m3(part / unit) * unit
    return out


def _exact_gelu8(c, st):
    u = st["x"].detach().double() + st["b"].detach().double()
    inner = lambda z: GELU_K * (z + GELU_C * z ** 3)  # noqa: E731
    y = u * torch.sigmoid(2 * inner(u))
    h = _exact_8_bits(u.float().double())  # by definition the checkpoint rounds the sum as 32 bits hold it
    s = torch.sigmoid(2 * inner(h))
    du = st["dy"].double() * (s + h * s * (1 - s) * 2 * GELU_K * (1 + 3 * GELU_C * h * h))
    return {"y": y, "dx": du, "db": du.sum(0)}


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attn":
            return _exact_attn(case, st)
        if case["op"] == "embed":
            return _exact_embed(case, st)
        if case["op"] == "gelu8":
            return _exact_gelu8(case, st)
        return {"x": _exact_8_bits(st["x"].double())}

"""The decode-step operators over block-quantised data, as measured cases: a key/value cache that is quantised as it
is written (and read back), attention of drafted tokens over that cache, and a mixture-of-experts layer whose experts
are block-quantised matrices.

`own = False` computes each operator with elementary torch operations in f32; `own = True` makes the calls that a user
of the library makes.  `exact` is the definition in f64.  Q8_0 and Q4_0 are blocks of 32 values with one f16 scale d:
    Q8_0  d = f16(max|v| / 127)                                q = clamp(round_half_away(v / d), -127, 127)
    Q4_0  d = f16(m / 7), m the element of largest magnitude   q = clamp(round_half_away(v / d), -8, 7)
both quotients rounded to f32, as the format prescribes; the value that a code stands for is d * q.
"""
import math

import torch

own = False

PAGE = 64  # tokens of a cache page in all cases


# ------------------------------------------------------------------------------------------------- cases ----
def listed():
    """kv: n rows of each of `seqs` sequences are written behind `context` tokens and read back.
    tree: n drafted tokens of each sequence attend to its context and along their tree ("chain": to the earlier ones).
    moe: a routed layer of `experts` gated experts for `tokens` tokens."""
    return [
        # one new token of one conversation: nothing but latency
        dict(name="kv one token", op="kv", seqs=1, n=1, context=1000, kv_heads=8, dim=128, ktype="q8_0", vtype="q8_0"),
        # prompt chunks of a few conversations, keys kept finer than values
        dict(name="kv prompt chunks", op="kv", seqs=5, n=333, context=77, kv_heads=4, dim=96, ktype="q8_0", vtype="q4_0"),
        # long prompts of a full server, written at once
        dict(name="kv long prompts", op="kv", seqs=16, n=1024, context=0, kv_heads=8, dim=128, ktype="q4_0", vtype="q4_0"),
        # the next token of one short conversation
        dict(name="tree single short", op="tree", seqs=1, n=1, tree="chain", context=500, heads=32, kv_heads=8, dim=128, ktype="q8_0", vtype="q8_0"),
        # the next token of many conversations of unequal length: the cache's bytes count
        dict(name="tree single batch", op="tree", seqs=16, n=1, tree="chain", context=16384, heads=32, kv_heads=8, dim=128, ktype="q8_0", vtype="q8_0"),
        # one long document, four-bit cache, one head of keys for each query head
        dict(name="tree single long", op="tree", seqs=1, n=1, tree="chain", context=60001, heads=16, kv_heads=16, dim=64, ktype="q4_0", vtype="q4_0"),
        # a small tree of drafts in a few conversations
        dict(name="tree drafts", op="tree", seqs=4, n=8, tree="random", context=4000, heads=32, kv_heads=8, dim=128, ktype="q8_0", vtype="q4_0"),
        # a wide tree of drafts over a long context: products count
        dict(name="tree wide drafts", op="tree", seqs=2, n=48, tree="random", context=12000, heads=32, kv_heads=8, dim=128, ktype="q8_0", vtype="q8_0"),
        # the next token through many small experts
        dict(name="moe single token", op="moe", tokens=1, experts=64, top_k=8, hidden=2048, inner=1024, normalise=False, gtype="q4_0", dtype="q4_0"),
        # drafts or a few users through small experts of odd width
        dict(name="moe few tokens", op="moe", tokens=7, experts=16, top_k=3, hidden=1120, inner=608, normalise=True, gtype="q8_0", dtype="q8_0"),
        # a few users through large experts, the second product kept finer
        dict(name="moe large experts", op="moe", tokens=8, experts=8, top_k=2, hidden=4096, inner=14336, normalise=True, gtype="q4_0", dtype="q8_0"),
        # a full server's decode step: nearly every expert has a few tokens
        dict(name="moe full step", op="moe", tokens=32, experts=32, top_k=4, hidden=2048, inner=1408, normalise=True, gtype="q4_0", dtype="q4_0"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(("kv", "tree", "tree", "moe", "moe"))
    q = lambda: rng.choice(("q8_0", "q4_0"))  # noqa: E731
    if op == "kv":
        seqs, heads, dim = _log(rng, 1, 16), rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((32, 64, 96, 128, 160, 256))
        n = _log(rng, 1, max(1, 16 * 1024 * 8 * 128 // (seqs * heads * dim)))
        return dict(op="kv", seqs=seqs, n=min(n, 8192), context=_log(rng, 1, 3000) - 1, kv_heads=heads, dim=dim, ktype=q(), vtype=q())
    if op == "tree":
        heads, group, dim = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 4, 5, 7, 8, 16)), rng.choice((64, 96, 128, 256))
        n, seqs = _log(rng, 1, 64), _log(rng, 1, 16)
        most = min(60000, 16 * 16384 * 8 * 128 // (seqs * heads * dim), 2 * 48 * 32 * 12000 * 128 // (seqs * n * heads * group * dim))
        return dict(op="tree", seqs=seqs, n=n, tree=rng.choice(("chain", "random", "random")), context=_log(rng, 1, max(1, most)) - 1,
                    heads=heads * group, kv_heads=heads, dim=dim, ktype=q(), vtype=q())
    experts = rng.choice((2, 5, 8, 16, 32, 64, 100))
    hidden = 32 * _log(rng, 8, 128)
    inner = 32 * _log(rng, 8, max(8, min(448, 8 * 4096 * 14336 // (32 * experts * hidden))))
    return dict(op="moe", tokens=_log(rng, 1, 32), experts=experts, top_k=rng.randint(1, min(8, experts)), hidden=hidden, inner=inner,
                normalise=rng.random() < 0.5, gtype=q(), dtype=q())


def _contexts(case):
    """Tokens that each sequence holds before the call: unequal, the first one has `context`."""
    return [case["context"] - (case["context"] * 2 * s) // (3 * case["seqs"]) for s in range(case["seqs"])]


def _bytes(kind, values):
    return values * (34 if kind == "q8_0" else 18) // 32


def work(case):
    if case["op"] == "kv":
        v = case["seqs"] * case["n"] * case["kv_heads"] * case["dim"]
        # f32 in, codes out; codes in, f32 out
        return {"bytes": 2 * (2 * 4 * v + _bytes(case["ktype"], v) + _bytes(case["vtype"], v)), "flops": 6 * v}
    if case["op"] == "tree":
        held = sum(c + case["n"] for c in _contexts(case))
        per = case["kv_heads"] * case["dim"]
        q = case["seqs"] * case["n"] * case["heads"] * case["dim"]
        pairs = sum(case["n"] * c + case["n"] * (case["n"] + 1) // 2 for c in _contexts(case))
        return {"bytes": _bytes(case["ktype"], held * per) + _bytes(case["vtype"], held * per) + 8 * q, "flops": 4 * pairs * case["heads"] * case["dim"]}
    t, e, k, h, f = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inner"))
    used = e * (1 - (1 - k / e) ** t)  # experts that are expected to get a token
    return {"bytes": int(used * (2 * _bytes(case["gtype"], f * h) + _bytes(case["dtype"], f * h))) + 4 * e * h + 8 * t * h,
            "flops": 6 * t * k * f * h + 2 * t * e * h}


# ---------------------------------------------------------------------------------------------- the format ----
def _quantise(kind, v):
    """Codes (int8) and scales (f16) of v, blocks of 32 along the last axis."""
    b = v.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    if kind == "q8_0":
        # by a tensor: by a plain number torch multiplies with the rounded reciprocal
        d, lo, hi = (amax / torch.full_like(amax, 127)).half(), -127, 127
    else:
        at = (b.abs() == amax).int().argmax(-1, keepdim=True)  # the first one on ties
        d, lo, hi = (b.gather(-1, at) / torch.full_like(amax, 7)).half(), -8, 7
    x = torch.where(d == 0, torch.zeros_like(b), b / d.float())
    t = x.trunc()
    q = t + ((x - t).abs() >= 0.5) * x.sign()
    return q.clamp(lo, hi).to(torch.int8).flatten(-2), d.squeeze(-1)


def _values(codes, scales):
    return (codes.unflatten(-1, (-1, 32)).float() * scales.float().unsqueeze(-1)).flatten(-2)


def _exact_values(kind, v):
    """What the codes of v stand for, in f64; the roundings that the format prescribes are made on the way."""
    b = v.double().reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    a = b.abs()
    amax = a.amax(-1, keepdim=True)
    if kind == "q8_0":
        s, most, least = amax / 127, 127, -127
    else:
        first = torch.where(a == amax, torch.arange(32, device=v.device).expand_as(a), torch.full_like(a, 32, dtype=torch.int64)).amin(-1, keepdim=True)
        s, most, least = torch.take_along_dim(b, first, -1) / 7, 7, -8
    d = s.to(torch.float32).to(torch.float16).double()
    x = (b / d).to(torch.float32).double()
    q = torch.where(x < 0, torch.ceil(x - 0.5), torch.floor(x + 0.5)).clamp(least, most)
    return torch.where(d == 0, torch.zeros_like(b), d * q).reshape(v.shape)


# -------------------------------------------------------------------------------------------------- inputs ----
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _kv_inputs(case, seed):
    """Keys and values of the context and of the n new tokens (keys with a few strong channels, as models have them), page table."""
    g = _generator(seed)
    seqs, n, heads, dim = (case[k] for k in ("seqs", "n", "kv_heads", "dim"))
    contexts = _contexts(case)
    longest = max(contexts) + n
    gain = 1 + 3 * (torch.rand(heads, dim, generator=g, device="cuda") > 0.95)
    k = _normal(g, seqs, longest, heads, dim) * gain
    v = _normal(g, seqs, longest, heads, dim) * 0.5
    pages = -(-longest // PAGE)
    table = torch.randperm(seqs * pages, generator=g, device="cuda").reshape(seqs, pages).to(torch.int32)
    start = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    begin = (torch.arange(seqs + 1, device="cuda") * n).to(torch.int32)
    return g, k, v, table, start, begin


def _tree(case, g):
    """may[s, i, j]: whether drafted token i of sequence s attends to drafted token j: itself and its ancestors."""
    n, seqs = case["n"], case["seqs"]
    if case["tree"] == "chain":
        return torch.ones(n, n, dtype=torch.bool, device="cuda").tril().expand(seqs, n, n).contiguous()
    draws = torch.rand(seqs, n, generator=g, device="cuda").tolist()
    may = torch.zeros(seqs, n, n, dtype=torch.bool)
    for s in range(seqs):
        for i in range(n):
            parent = int(draws[s][i] * (i + 1)) - 1  # -1: a root
            if parent >= 0:
                may[s, i] = may[s, parent]
            may[s, i, i] = True
    return may.cuda()


def _new_rows(x, start, n):
    at = start.long()[:, None] + torch.arange(n, device="cuda")
    return x[torch.arange(x.shape[0], device="cuda")[:, None], at].flatten(0, 1).contiguous()


def _moe_inputs(case, seed):
    g = _generator(seed)
    e, h, f, t = (case[k] for k in ("experts", "hidden", "inner", "tokens"))
    x = _normal(g, t, h)
    router = _normal(g, e, h) * (1.5 / math.sqrt(h))
    gate, up = (_normal(g, e * f, h) * (1 / math.sqrt(h)) for _ in range(2))
    down = _normal(g, e * h, f) * (1 / math.sqrt(f))
    return x, router, gate, up, down


def _type(vb, kind):
    return vb.Q8_0 if kind == "q8_0" else vb.Q4_0


def _device(vb, backend, t):
    import numpy as np
    dtype = {torch.float32: np.float32, torch.int32: np.int32}[t.dtype]
    return vb.GpuBuffer(backend, t.data_ptr(), t.numel(), dtype, owned=False)


def prepare(case, seed):
    s = {"case": case}
    if own:
        import vortx_b200 as vb
        s["backend"] = backend = vb.Backend(0, stream=torch.cuda.current_stream().cuda_stream)
        dev = lambda t: _device(vb, backend, t)  # noqa: E731
    if case["op"] == "moe":
        x, router, gate, up, down = _moe_inputs(case, seed)
        t, h, k = case["tokens"], case["hidden"], case["top_k"]
        s.update(x=x, router=router)
        if own:
            mats = [vb.QuantizedMatrix.from_device_f32(backend, _type(vb, kind), w.data_ptr(), w.shape[0], w.shape[1])
                    for kind, w in ((case["gtype"], gate), (case["gtype"], up), (case["dtype"], down))]
            backend.synchronize()
            s["layer"] = vb.MoeLayer(backend, dev(router), *mats, experts=case["experts"], top_k=k, normalise=case["normalise"], max_tokens=t)
            s["y"], s["ids"] = torch.empty(t, h, device="cuda"), torch.empty(t, k, dtype=torch.int32, device="cuda")
            s["views"] = [dev(s[n]) for n in ("y", "x", "ids")]
            return s
        for name, kind, w in (("gate", case["gtype"], gate), ("up", case["gtype"], up), ("down", case["dtype"], down)):
            parts = [_quantise(kind, p) for p in w.chunk(case["experts"])]
            s[name] = (torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]))
        return s
    g, k, v, table, start, begin = _kv_inputs(case, seed)
    n, seqs, heads, dim = (case[i] for i in ("n", "seqs", "kv_heads", "dim"))
    s.update(table=table, start=start, begin=begin, k=_new_rows(k, start, n), v=_new_rows(v, start, n))
    if case["op"] == "tree":
        s["q"] = _normal(g, seqs * n, case["heads"], dim)
        s["may"] = _tree(case, g)
    if own:
        s["cache"] = cache = vb.QuantizedCache(backend, _type(vb, case["ktype"]), _type(vb, case["vtype"]), heads, dim, table.numel(), PAGE)
        s["rows"] = vb.CacheRows(dev(table), dev(begin), dev(start), seqs * n)
        if case["op"] == "kv":
            s["out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
            s["views"] = [dev(x) for x in (s["k"], s["v"], *s["out"])]
            return s
        longest = k.shape[1]  # the context and the drafted tokens are in the cache when attention is called
        every = torch.arange(seqs + 1, device="cuda").mul(longest).to(torch.int32)
        zero = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        cache.append(None, dev(k), dev(v), vb.CacheRows(dev(table), dev(every), dev(zero), seqs * longest))
        backend.synchronize()
        s["attention"] = vb.CacheAttention(backend, cache, case["heads"], max_seqs=seqs)
        s["out"], s["mask"] = torch.empty_like(s["q"]), None
        if case["tree"] != "chain":
            words = -(-n // 32)
            bits = torch.zeros(seqs, n, words * 32, dtype=torch.int64, device="cuda")
            bits[..., :n] = s["may"]
            packed = (bits.unflatten(-1, (words, 32)) << torch.arange(32, device="cuda")).sum(-1)
            s["bits"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32).reshape(seqs * n, words).contiguous()
            s["mask"] = dev(s["bits"])
        s["views"] = [dev(s["out"]), dev(s["q"])]
        return s
    slots = table.numel() * PAGE
    s["cache"] = []
    for kind, x in ((case["ktype"], k), (case["vtype"], v)):
        codes = torch.zeros(slots, heads, dim, dtype=torch.int8, device="cuda")
        scales = torch.zeros(slots, heads, dim // 32, dtype=torch.float16, device="cuda")
        if case["op"] == "tree":
            at = _slots(table, torch.arange(x.shape[1], device="cuda").expand(seqs, -1))
            codes[at], scales[at] = _quantise(kind, x)
        s["cache"].append((codes, scales))
    return s


def _slots(table, positions):
    """Where the tokens at `positions` [seqs, any] lie in the cache."""
    return table.long().gather(1, positions // PAGE) * PAGE + positions % PAGE


# ------------------------------------------------------------------------------------------------- one pass ----
def run(state):
    return {"kv": _run_kv, "tree": _run_tree, "moe": _run_moe}[state["case"]["op"]](state)


def _run_kv(s):
    if own:
        k, v, ko, vo = s["views"]
        s["cache"].append(None, k, v, s["rows"])
        s["cache"].read(None, ko, vo, s["rows"])
        return s["out"]
    case = s["case"]
    at = _slots(s["table"], s["start"].long()[:, None] + torch.arange(case["n"], device="cuda")).flatten()
    out = []
    for kind, x, (codes, scales) in ((case["ktype"], s["k"], s["cache"][0]), (case["vtype"], s["v"], s["cache"][1])):
        codes[at], scales[at] = _quantise(kind, x)
        out.append(_values(codes[at], scales[at]))
    return tuple(out)


def _run_tree(s):
    if own:
        s["attention"].dispatch(s["backend"], None, s["views"][0], s["views"][1], s["rows"], mask=s["mask"])
        return s["out"]
    case = s["case"]
    seqs, n, heads, kv_heads, dim = (case[k] for k in ("seqs", "n", "heads", "kv_heads", "dim"))
    longest = max(_contexts(case)) + n
    positions = torch.arange(longest, device="cuda")
    at = _slots(s["table"], positions.expand(seqs, -1))
    k, v = (_values(codes[at], scales[at]) for codes, scales in s["cache"])
    q = s["q"].reshape(seqs, n, kv_heads, heads // kv_heads, dim)
    scores = torch.einsum("snhgd,slhd->shgnl", q, k) / math.sqrt(dim)
    behind = positions - s["start"][:, None]  # < 0: context, else the drafted token's number
    draft = s["may"].gather(2, behind.clamp(0, n - 1)[:, None].expand(-1, n, -1)) & (behind < n)[:, None]
    may = (behind < 0)[:, None] | draft
    scores = scores.masked_fill(~may[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    out = torch.einsum("shgnl,slhd->snhgd", p, v) / p.sum(-1).clamp_min(1e-30).permute(0, 3, 1, 2)[..., None]
    return out.reshape(seqs * n, heads, dim)


def _run_moe(s):
    if own:
        y, x, ids = s["views"]
        s["layer"].dispatch(s["backend"], None, y, x, s["case"]["tokens"], ids=ids)
        return s["y"], s["ids"]
    case, x = s["case"], s["x"]
    t, e, k, h, f = (case[n] for n in ("tokens", "experts", "top_k", "hidden", "inner"))
    logits = x @ s["router"].T
    best, ids = logits.sort(dim=-1, descending=True, stable=True)
    best, ids = best[:, :k], ids[:, :k]
    if case["normalise"]:
        weights = torch.softmax(best, -1)
    else:
        weights = torch.softmax(logits, -1).gather(1, ids)
    if t * k < e:  # fewer products than experts: only the chosen ones' weights
        gate, up, down = (_values(c[ids], d[ids]) for c, d in (s["gate"], s["up"], s["down"]))
        g, u = (torch.einsum("th,tkfh->tkf", x, w) for w in (gate, up))
        y = torch.einsum("tkf,tkhf,tk->th", g * torch.sigmoid(g) * u, down, weights)
    else:
        gate, up, down = (_values(c, d) for c, d in (s["gate"], s["up"], s["down"]))
        g, u = (torch.einsum("th,efh->etf", x, w) for w in (gate, up))
        all_weights = torch.zeros(t, e, device="cuda").scatter(1, ids, weights)
        y = (torch.bmm(g * torch.sigmoid(g) * u, down.transpose(1, 2)) * all_weights.T[..., None]).sum(0)
    return y, ids.to(torch.int32)


# ------------------------------------------------------------------------------------------------ in 64 bits ----
def exact(case, seed):
    if case["op"] == "moe":
        return _exact_moe(case, seed)
    g, k, v, table, start, begin = _kv_inputs(case, seed)
    n, seqs, dim = case["n"], case["seqs"], case["dim"]
    if case["op"] == "kv":
        return _exact_values(case["ktype"], _new_rows(k, start, n)), _exact_values(case["vtype"], _new_rows(v, start, n))
    q = _normal(g, seqs * n, case["heads"], dim).double().reshape(seqs, n, case["heads"], dim)
    may = _tree(case, g)
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    for s, held in enumerate(_contexts(case)):
        for h in range(case["kv_heads"]):
            key = _exact_values(case["ktype"], k[s, :held + n, h])
            value = _exact_values(case["vtype"], v[s, :held + n, h])
            for i in range(h * group, (h + 1) * group):
                score = q[s, :, i] @ key.T / math.sqrt(dim)
                score[:, held:][~may[s]] = -math.inf
                out[s, :, i] = torch.softmax(score, -1) @ value
    return out.reshape(seqs * n, case["heads"], dim)


def _exact_moe(case, seed):
    x, router, gate, up, down = _moe_inputs(case, seed)
    e, h, f, k = (case[n] for n in ("experts", "hidden", "inner", "top_k"))
    x = x.double()
    logits = x @ router.double().T
    order = sorted_ids = torch.argsort(logits, dim=-1, descending=True, stable=True)[:, :k]
    chosen = logits.gather(1, order)
    scale = chosen.logsumexp(-1, keepdim=True) if case["normalise"] else logits.logsumexp(-1, keepdim=True)
    weights = torch.exp(chosen - scale)
    y = torch.zeros_like(x)
    for i in range(e):
        tokens, places = (sorted_ids == i).nonzero(as_tuple=True)
        if len(tokens):
            a = x[tokens] @ _exact_values(case["gtype"], gate[i * f:(i + 1) * f]).T
            b = x[tokens] @ _exact_values(case["gtype"], up[i * f:(i + 1) * f]).T
            out = (a / (1 + torch.exp(-a)) * b) @ _exact_values(case["dtype"], down[i * h:(i + 1) * h]).T
            y.index_add_(0, tokens, out * weights[tokens, places, None])
    return y, None

"""The decode-step operators together, as a decoder calls them: projections, cache, attention, expert layer; and what
their own tests leave out (many sequences, arrays that make no sense, results in place of inputs)."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import DOT, attention, moe, quantised

pytestmark = pytest.mark.gpu


def _rng(seed):
    return np.random.Generator(np.random.Philox(seed))


def _read(backend, buf):
    out = np.empty(buf.len(), buf.dtype)
    backend.slow_read_buffer(buf, out)
    return out


class Decoder:
    """One layer for `seqs` sequences with up to `tokens` new tokens in a call."""
    hidden, heads, kv_heads, dim, experts, inner, top_k, page = 256, 8, 2, 64, 8, 128, 2, 32

    def __init__(self, b, seqs, tokens, pages=16, kt=vb.Q8_0, vt=vb.Q4_0, seed=0):
        rng = _rng(seed)
        self.b, self.seqs = b, seqs
        w = lambda r, c: (rng.standard_normal((r, c)) / np.sqrt(c)).astype(np.float32)  # noqa: E731
        q, kv = self.heads * self.dim, self.kv_heads * self.dim
        self.host = {n: w(r, self.hidden) for n, r in (("q", q), ("k", kv), ("v", kv))} | {"o": w(self.hidden, q)}
        self.w = {n: vb.QuantizedMatrix.from_f32(b, vb.Q8_0, m) for n, m in self.host.items()}
        self.router = w(self.experts, self.hidden)
        mats = [w(self.experts * self.inner, self.hidden), w(self.experts * self.inner, self.hidden), w(self.experts * self.hidden, self.inner)]
        self.gate, self.up = (quantised(vb.Q4_0, m).reshape(self.experts, self.inner, self.hidden) for m in mats[:2])
        self.down = quantised(vb.Q8_0, mats[2]).reshape(self.experts, self.hidden, self.inner)
        self.mats = [vb.QuantizedMatrix.from_f32(b, t, m) for t, m in zip((vb.Q4_0, vb.Q4_0, vb.Q8_0), mats)]
        self.cache = vb.QuantizedCache(b, kt, vt, self.kv_heads, self.dim, seqs * pages, self.page)
        self.table = rng.permutation(seqs * pages).reshape(seqs, pages).astype(np.int32)
        self.attention = vb.CacheAttention(b, self.cache, self.heads, seqs)
        self.layer = vb.MoeLayer(b, b.init_buffer(self.router.ravel()), *self.mats, experts=self.experts, top_k=self.top_k, max_tokens=tokens)
        f = lambda width: b.init_buffer(np.zeros(tokens * width, np.float32))  # noqa: E731
        self.x, self.q, self.k, self.v, self.a, self.p, self.y = f(self.hidden), f(q), f(q), f(q), f(q), f(self.hidden), f(self.hidden)
        self.table_dev = b.init_buffer(self.table.ravel())

    def rows(self, begin, start, n):
        return vb.CacheRows(self.table_dev, begin, start, n, seqs=self.seqs)

    def step(self, rows, mask=None):
        b, g, n = self.b, vb.Gemv(), rows.rows
        width = self.heads * self.dim                   # of q; k and v come with its stride
        g.dispatch_multi(b, None, [self.q, self.k, self.v], [self.w["q"], self.w["k"], self.w["v"]], self.x, batch=n)
        self.cache.append(None, self.k, self.v, rows, k_stride=width, v_stride=width)
        self.attention.dispatch(b, None, self.a, self.q, rows, mask=mask)
        g.dispatch(b, None, self.p, self.w["o"], self.a, batch=n)
        self.layer.dispatch(b, None, self.y, self.p, n)

    def free(self):
        self.attention.free()
        self.layer.free()
        self.cache.free()
        for m in [*self.w.values(), *self.mats]:
            m.free()


def test_a_decoder_layer_step_by_step(backend):
    """Prompts, then single tokens: every stage against its statement on what the stage before it left."""
    d = Decoder(backend, 3, 40, seed=1)
    i32 = lambda a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    past = [np.zeros((0, 2, d.kv_heads, d.dim), np.float32) for _ in range(3)]
    rng = _rng(2)
    for n in ([33, 1, 5], [1, 1, 1], [1, 0, 7], [1, 1, 1]):
        begin, start, total = np.concatenate([[0], np.cumsum(n)]), [len(p) for p in past], sum(n)
        x = rng.standard_normal((total, d.hidden)).astype(np.float32)
        backend.write_buffer(d.x, 0, x.ravel())
        d.step(d.rows(i32(begin), i32(start), total))
        q, k, v, a = (_read(backend, t).reshape(40, -1)[:total] for t in (d.q, d.k, d.v, d.a))
        p, y = (_read(backend, t).reshape(40, -1)[:total] for t in (d.p, d.y))
        for name, got in (("q", q), ("k", k), ("v", v)):
            m = quantised(vb.Q8_0, d.host[name])
            err = np.abs(got[:, :len(m)] - x.astype(np.float64) @ m.T)
            assert (err <= 2 * DOT * (np.abs(x) @ np.abs(m).T)).all()
        for s in range(3):
            new = np.stack([t[begin[s]:begin[s + 1], :d.kv_heads * d.dim].reshape(-1, d.kv_heads, d.dim) for t in (k, v)], 1)
            past[s] = np.concatenate([past[s], new])
            kq, vq = quantised(vb.Q8_0, past[s][:, 0]), quantised(vb.Q4_0, past[s][:, 1])
            may = np.concatenate([np.ones((n[s], start[s]), bool), np.tril(np.ones((n[s], n[s]), bool))], 1)
            for h in range(d.heads):
                qh = q[begin[s]:begin[s + 1], h * d.dim:(h + 1) * d.dim]
                want, tol = attention(qh, kq[:, h // 4], vq[:, h // 4], may, d.dim ** -0.5)
                assert (np.abs(a[begin[s]:begin[s + 1], h * d.dim:(h + 1) * d.dim] - want) <= tol).all()
        m = quantised(vb.Q8_0, d.host["o"])
        assert (np.abs(p - a.astype(np.float64) @ m.T) <= 2 * DOT * (np.abs(a) @ np.abs(m).T)).all()
        want, _, _, tol, _ = moe(p, d.router, d.gate, d.up, d.down, d.top_k, True)
        assert (np.abs(y - want) <= tol).all()
    d.free()


def test_a_recorded_step_is_the_eager_step(backend):
    """The step captured once and replayed over ten tokens gives what calls give, bit for bit."""
    import torch
    eager = Decoder(backend, 2, 2, seed=3)
    stream = torch.cuda.Stream()
    with vb.Backend(0, stream=stream.cuda_stream) as b:
        d = Decoder(b, 2, 2, seed=3)
        begin, start = b.init_buffer(np.array([0, 1, 2], np.int32)), b.init_buffer(np.zeros(2, np.int32))
        e_begin, e_start = backend.init_buffer(np.array([0, 1, 2], np.int32)), backend.init_buffer(np.zeros(2, np.int32))
        rows, e_rows = d.rows(begin, start, 2), eager.rows(e_begin, e_start, 2)
        d.step(rows)                                    # the projections' scratch is made by their first call
        b.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d.step(rows)
        rng = _rng(4)
        for i in range(10):
            x = rng.standard_normal(2 * d.hidden).astype(np.float32)
            for bk, buf, st in ((b, d.x, start), (backend, eager.x, e_start)):
                bk.write_buffer(buf, 0, x)
                bk.write_buffer(st, 0, np.array([i, 2 * i], np.int32))
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            eager.step(e_rows)
            assert np.array_equal(_read(b, d.y), _read(backend, eager.y))
        del graph
        d.free()
    eager.free()


def test_a_drafted_branch_is_the_sequence_it_stands_for(backend):
    """Rows of a tree of drafted tokens attend as if their branch had been decoded token by token."""
    rng = _rng(5)
    heads, kv, dim, context = 6, 2, 128, 70
    parents = [-1, 0, 0, 1, 2, 2, 4, 6, 3, 5]
    n = len(parents)
    draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    k, v, q = draw(context + n, kv, dim), draw(context + n, kv, dim), draw(n, heads, dim)
    dev = lambda a: backend.init_buffer(np.ascontiguousarray(a).ravel())  # noqa: E731
    i32 = lambda *a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, kv, dim, 8, 32)
    att = vb.CacheAttention(backend, cache, heads, 1)
    table = [i32(5, 0, 7), i32(1, 2, 3)]
    cache.append(None, dev(k[:context]), dev(v[:context]), vb.CacheRows(table[0], i32(0, context), i32(0), context))
    rows = vb.CacheRows(table[0], i32(0, n), i32(context), n)
    cache.append(None, dev(k[context:]), dev(v[context:]), rows)
    out = backend.uninit_buffer(n * heads * dim)
    att.dispatch(backend, None, out, dev(q), rows, mask=dev(vb.tree_mask(parents)))
    drafted = _read(backend, out).reshape(n, heads, dim)
    branch = [7]
    while parents[branch[0]] >= 0:
        branch.insert(0, parents[branch[0]])
    tokens = list(range(context)) + [context + i for i in branch]
    kq, vq = quantised(vb.Q8_0, k[tokens]), quantised(vb.Q8_0, v[tokens])
    cache.append(None, dev(k[:context]), dev(v[:context]), vb.CacheRows(table[1], i32(0, context), i32(0), context))
    one = backend.uninit_buffer(heads * dim)
    for depth, i in enumerate(branch):
        rows = vb.CacheRows(table[1], i32(0, 1), i32(context + depth), 1)
        cache.append(None, dev(k[context + i]), dev(v[context + i]), rows)
        att.dispatch(backend, None, one, dev(q[i]), rows)
        decoded = _read(backend, one).reshape(heads, dim)
        upto = context + depth + 1
        for h in range(heads):
            want, tol = attention(q[i:i + 1, h], kq[:upto, h // 3], vq[:upto, h // 3], np.ones((1, upto), bool), dim ** -0.5)
            assert (np.abs(decoded[h] - want[0]) <= tol[0]).all() and (np.abs(drafted[i, h] - want[0]) <= tol[0]).all()


@pytest.mark.parametrize("seqs", [32, 33, 70, 300])
def test_many_sequences(backend, seqs):
    """More sequences than a warp has lanes take another way to their shares; some have no rows."""
    rng = _rng(seqs)
    heads, kv, dim = 4, 2, 64
    context, n = rng.integers(0, 150, seqs), rng.integers(0, 4, seqs)
    context[seqs // 2], n[seqs // 2] = 900, 2
    n[0] = 0
    total = context + n
    per = int(-(-total.max() // 32))
    table = rng.permutation(seqs * per).astype(np.int32)
    dev = lambda a: backend.init_buffer(np.ascontiguousarray(a).ravel())  # noqa: E731
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    k, v = ([rng.standard_normal((t, kv, dim)).astype(np.float32) for t in total] for _ in range(2))
    every, begin = (np.concatenate([[0], np.cumsum(a)]) for a in (total, n))
    q = rng.standard_normal((begin[-1], heads, dim)).astype(np.float32)
    cache = vb.QuantizedCache(backend, vb.Q4_0, vb.Q8_0, kv, dim, seqs * per, 32)
    cache.append(None, dev(np.concatenate(k)), dev(np.concatenate(v)), vb.CacheRows(dev(table), i32(every), i32(np.zeros(seqs)), int(every[-1])))
    att = vb.CacheAttention(backend, cache, heads, seqs)
    out = backend.uninit_buffer(q.size)
    att.dispatch(backend, None, out, dev(q), vb.CacheRows(dev(table), i32(begin), i32(context), int(begin[-1])))
    got = _read(backend, out).reshape(q.shape)
    for s in range(seqs):
        kq, vq = quantised(vb.Q4_0, k[s]), quantised(vb.Q8_0, v[s])
        may = np.concatenate([np.ones((n[s], context[s]), bool), np.tril(np.ones((n[s], n[s]), bool))], 1)
        for h in range(heads):
            at = slice(begin[s], begin[s + 1])
            want, tol = attention(q[at, h], kq[:, h // 2], vq[:, h // 2], may, dim ** -0.5)
            assert (np.abs(got[at, h] - want) <= tol).all()


@pytest.mark.parametrize("begin,start", [([0, 5, 2, 9, 8], [0, 40, 3, 7]), ([-7, 3, 100, 1, 2 ** 31 - 1], [10, 2 ** 31 - 1, -1, 0]),
                                         ([8, 6, 4, 2, 0], [1, 2, 3, 4]), ([3, 3, 3, 3, 3], [2 ** 31 - 20] * 4),
                                         ([-2 ** 31, 2, 4, 6, 8], [-2 ** 31, 60, 63, 2 ** 30])])
def test_arrays_that_make_no_sense_stay_within_the_tensors(backend, begin, start):
    """Rows and tokens come out clamped: nothing outside the call's rows and the table's pages is written."""
    kv, dim, rows, pad = 2, 64, 8, 16
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, kv, dim, 9, 32)
    i32 = lambda a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    ones = backend.init_buffer(np.ones(9 * 32 * kv * dim, np.float32))
    every = vb.CacheRows(i32(range(9)), i32([0, 288]), i32([0]), 288)
    cache.append(None, ones, ones, every)
    r = vb.CacheRows(i32([0, 1, 2, 3, 4, 5, 6, 7]), i32(begin), i32(start), rows)
    x = backend.init_buffer(np.full(rows * kv * dim, 2.0, np.float32))
    cache.append(None, x, x, r)
    back = backend.uninit_buffer(288 * kv * dim)
    cache.read(None, back, None, every)
    assert (_read(backend, back)[256 * kv * dim:] == quantised(vb.Q8_0, np.ones((1, 32), np.float32))[0, 0]).all()  # page 8 is in no table
    for run in (lambda o: cache.read(None, o, o, r), lambda o: vb.CacheAttention(backend, cache, 2, 4).dispatch(backend, None, o, x, r),
                lambda o: vb.CacheAttention(backend, cache, 2, 4).dispatch(backend, None, o, x, r, mask=i32([-1] * rows))):
        out = backend.init_buffer(np.full((rows + 2 * pad) * kv * dim, 7.5, np.float32))
        run(out.ptr + 4 * pad * kv * dim)
        got = _read(backend, out).reshape(-1, kv * dim)
        assert (got[:pad] == 7.5).all() and (got[pad + rows:] == 7.5).all() and np.isfinite(got).all()


def test_results_in_place_of_inputs(backend):
    rng = _rng(9)
    d = Decoder(backend, 2, 9, seed=6)
    i32 = lambda a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    rows = d.rows(i32([0, 4, 9]), i32([300, 0]), 9)
    backend.write_buffer(d.x, 0, rng.standard_normal(9 * d.hidden).astype(np.float32))
    d.step(rows)
    want, y = _read(backend, d.a), _read(backend, d.y)
    d.attention.dispatch(backend, None, d.q, d.q, rows)
    assert np.array_equal(_read(backend, d.q), want)
    with pytest.raises(vb.VortxError):
        d.attention.dispatch(backend, None, d.q.ptr, d.q.ptr, rows, out_stride=d.heads * d.dim + 4)
    d.layer.dispatch(backend, None, d.p, d.p, 9)
    assert np.array_equal(_read(backend, d.p), y)
    d.free()


def test_a_workspace_each_for_graphs_at_the_same_time(backend):
    """Two recorded calls over one cache, with a workspace each, replayed on two streams at once."""
    import torch
    rng = _rng(10)
    heads, kv, dim, context = 8, 2, 128, 4000
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, kv, dim, 32, 128)
    k, v = (rng.standard_normal((context, kv, dim)).astype(np.float32) for _ in range(2))
    dev = lambda a: backend.init_buffer(np.ascontiguousarray(a).ravel())  # noqa: E731
    i32 = lambda *a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    table = i32(*range(32))
    cache.append(None, dev(k), dev(v), vb.CacheRows(table, i32(0, context), i32(0), context))
    rows = vb.CacheRows(table, i32(0, 1), i32(context - 1), 1)
    backend.synchronize()
    sides = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        b = vb.Backend(0, stream=stream.cuda_stream)
        q = b.init_buffer(rng.standard_normal(heads * dim).astype(np.float32))
        out, att, graph = b.uninit_buffer(heads * dim), vb.CacheAttention(b, cache, heads, 1), torch.cuda.CUDAGraph()
        att.dispatch(b, None, out, q, rows)
        want = _read(b, out)
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(20):
                att.dispatch(b, None, out, q, rows)
        sides.append((stream, b, q, out, att, graph, want))
    for _ in range(5):
        for stream, b, q, out, att, graph, want in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    for stream, b, q, out, att, graph, want in sides:
        stream.synchronize()
        assert np.array_equal(_read(b, out), want)
    while sides:
        stream, b, q, out, att, graph, want = sides.pop()
        del graph
        att.free()
        q.free()
        out.free()
        b.close()


FIRST_CALL = """
import sys, numpy as np, torch, vortx_b200 as vb
from test_gpu_decode_step import Decoder, _read
torch.zeros(1, device="cuda")
stream = torch.cuda.Stream()
with vb.Backend(0, stream=stream.cuda_stream) as b:
    d = Decoder(b, 2, 2, seed=3)
    rows = d.rows(b.init_buffer(np.array([0, 1, 2], np.int32)), b.init_buffer(np.array([0, 40], np.int32)), 2)
    rng = np.random.Generator(np.random.Philox(1))
    for t in (d.k, d.v, d.q, d.p):
        b.write_buffer(t, 0, rng.standard_normal(t.len()).astype(np.float32))
    b.synchronize()
    width = d.heads * d.dim
    def calls():
        d.cache.append(None, d.k, d.v, rows, k_stride=width, v_stride=width)
        d.attention.dispatch(b, None, d.a, d.q, rows)
        d.layer.dispatch(b, None, d.y, d.p, 2)
        d.cache.read(None, d.k, d.v, rows, k_stride=width, v_stride=width)
    k, v = _read(b, d.k), _read(b, d.v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    with torch.cuda.stream(stream):
        graph.replay()
    stream.synchronize()
    got = [_read(b, t) for t in (d.a, d.y, d.k)]
    b.write_buffer(d.k, 0, k)
    b.write_buffer(d.v, 0, v)
    calls()
    assert all(np.array_equal(g, _read(b, t)) for g, t in zip(got, (d.a, d.y, d.k))) and np.abs(got[0]).max() > 0 and np.abs(got[1]).max() > 0
    del graph
    d.free()
print("ok")
"""


def test_the_first_call_of_a_process_may_be_a_recorded_one():
    """Making the objects loads the code of every kernel that their calls launch."""
    import os
    import subprocess
    import sys
    from pathlib import Path
    here = Path(__file__).resolve().parent
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(here.parent), str(here), os.environ.get("PYTHONPATH", "")]))
    res = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300, env=env)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stdout + res.stderr

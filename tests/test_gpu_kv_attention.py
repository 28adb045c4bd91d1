"""Attention over the quantised cache against its f64 statement on the values that the codes stand for."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import attention, quantised
from vortx_b200 import _lib

pytestmark = pytest.mark.gpu


def _rng(seed):
    return np.random.Generator(np.random.Philox(seed))


def _read(backend, buf):
    out = np.empty(buf.len(), buf.dtype)
    backend.slow_read_buffer(buf, out)
    return out


class Scene:
    """Sequences of (context, new tokens) in a paged cache, with everything of them also on the host."""

    def __init__(self, backend, seqs, heads=8, kv_heads=2, dim=64, page=64, kt=vb.Q8_0, vt=vb.Q8_0, seed=0, pad=0, spread=1.0):
        rng = _rng(seed)
        self.backend, self.seqs, self.heads, self.kv_heads, self.dim, self.kt, self.vt = backend, seqs, heads, kv_heads, dim, kt, vt
        total = [c + n for c, n in seqs]
        per = max(1, max(-(-t // page) for t in total))
        pages = per * len(seqs) + 1
        self.table = rng.permutation(pages)[:per * len(seqs)].reshape(len(seqs), per).astype(np.int32)
        self.begin = np.concatenate([[0], np.cumsum([n for _, n in seqs])]).astype(np.int32)
        self.start = np.array([c for c, _ in seqs], np.int32)
        self.rows_n = int(self.begin[-1]) + pad
        self.k = [(rng.standard_normal((t, kv_heads, dim)) * spread).astype(np.float32) for t in total]
        self.v = [rng.standard_normal((t, kv_heads, dim)).astype(np.float32) for t in total]
        self.q = rng.standard_normal((self.rows_n, heads, dim)).astype(np.float32)
        self.cache = vb.QuantizedCache(backend, kt, vt, kv_heads, dim, pages, page)
        every = np.concatenate([[0], np.cumsum(total)]).astype(np.int32)
        if every[-1]:
            kv = [backend.init_buffer(np.concatenate([a.reshape(-1, kv_heads * dim) for a in x]).ravel()) for x in (self.k, self.v)]
            self.cache.append(None, *kv, vb.CacheRows(self._b(self.table), self._b(every), self._b(np.zeros(len(seqs), np.int32)), int(every[-1])))
        self.rows = vb.CacheRows(self._b(self.table), self._b(self.begin), self._b(self.start), self.rows_n, max_pages=per)

    def _b(self, a):
        return self.backend.init_buffer(np.ascontiguousarray(a).ravel())

    def run(self, mask=None, scale=None, **kw):
        att = vb.CacheAttention(self.backend, self.cache, self.heads, max(1, len(self.seqs)))
        out = self.backend.init_buffer(np.full(self.rows_n * self.heads * self.dim + 5, 7.5, np.float32))
        att.dispatch(self.backend, None, out, self._b(self.q), self.rows, mask=None if mask is None else self._b(mask), scale=scale, **kw)
        got = _read(self.backend, out)
        att.free()
        assert (got[self.rows_n * self.heads * self.dim:] == 7.5).all()
        return got[:self.rows_n * self.heads * self.dim].reshape(self.rows_n, self.heads, self.dim)

    def check(self, got, may=None, scale=None, k=None, v=None):
        """may[s]: [n, n] among the new tokens; None: those up to a row's own."""
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.heads // self.kv_heads
        worst = 0.0
        for s, (c, n) in enumerate(self.seqs):
            kq = quantised(self.kt, self.k[s]) if k is None else k[s]
            vq = quantised(self.vt, self.v[s]) if v is None else v[s]
            among = np.tril(np.ones((n, n), bool)) if may is None else may[s]
            ok = np.concatenate([np.ones((n, c), bool), among], 1)
            for h in range(self.heads):
                want, tol = attention(self.q[self.begin[s]:self.begin[s] + n, h], kq[:, h // group], vq[:, h // group], ok, scale)
                err = np.abs(got[self.begin[s]:self.begin[s] + n, h] - want)
                assert (err <= tol).all(), (s, h, float((err / tol).max()))
                worst = max(worst, float((err / tol).max(initial=0.0)))
        assert (got[self.begin[-1]:] == 7.5).all()     # rows behind the last sequence
        return worst


@pytest.mark.parametrize("kt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,n", [(4, 4, 1), (8, 1, 1), (6, 2, 5), (8, 2, 9), (5, 1, 13)])
def test_types_and_heads(backend, kt, vt, dim, heads, kv_heads, n):
    s = Scene(backend, [(100, n), (31, n), (0, n)], heads, kv_heads, dim, 64, kt, vt, seed=dim + n, pad=2)
    s.check(s.run())


@pytest.mark.parametrize("context", [0, 1, 30, 31, 32, 33, 63, 64, 65, 127, 128, 1000, 1999])
@pytest.mark.parametrize("n", [1, 2])
def test_lengths_of_one_sequence(backend, context, n):
    s = Scene(backend, [(context, n)], 4, 2, 64, 32, vb.Q8_0, vb.Q4_0, seed=context)
    s.check(s.run())


@pytest.mark.parametrize("kv_heads,page", [(1, 32), (3, 96), (8, 256)])
def test_ragged_batches(backend, kv_heads, page):
    """Sequences of very different lengths and row counts, some without rows."""
    seqs = [(1500, 1), (0, 1), (3, 0), (700, 17), (64, 3), (31, 1), (900, 0), (1, 40)]
    s = Scene(backend, seqs, kv_heads * 3, kv_heads, 64, page, vb.Q8_0, vb.Q8_0, seed=kv_heads, pad=3)
    s.check(s.run())


def _trees(rng, seqs):
    may, masks = [], []
    words = max(-(-n // 32) for _, n in seqs)
    for _, n in seqs:
        parents = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
        m = vb.tree_mask(parents)
        masks.append(np.pad(m, ((0, 0), (0, words - m.shape[1]))))
        bits = np.unpackbits(m.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        may.append(bits)
    return may, np.concatenate(masks).astype(np.uint32)


@pytest.mark.parametrize("dim,heads,kv_heads,kt,vt", [(128, 8, 2, vb.Q8_0, vb.Q4_0), (64, 4, 4, vb.Q4_0, vb.Q4_0), (256, 4, 1, vb.Q8_0, vb.Q8_0)])
def test_trees(backend, dim, heads, kv_heads, kt, vt):
    rng = _rng(dim)
    seqs = [(200, 48), (0, 7), (1000, 33), (31, 1)]
    s = Scene(backend, seqs, heads, kv_heads, dim, 64, kt, vt, seed=3)
    may, mask = _trees(rng, seqs)
    s.check(s.run(mask), may)


def test_masks_that_leave_nothing_and_masks_that_end_early(backend):
    seqs = [(0, 5), (40, 40)]
    s = Scene(backend, seqs, 4, 2, 64, seed=9)
    may = [np.zeros((5, 5), bool), np.eye(40, dtype=bool)]
    may[0][2, 4] = True                                # forward in the call: a mask is any set of bits
    mask = np.zeros((45, 1), np.uint32)
    mask[2, 0] = 1 << 4
    for i in range(40):
        mask[5 + i, 0] = 1 << i if i < 32 else 0xffffffff
        if i >= 32:
            may[1][i] = np.arange(40) < 32             # one word: tokens from 32 on are not attended to
    got = s.run(mask)
    assert (got[[0, 1, 3, 4]] == 0).all()
    s.check(got, may)
    mask[:5] |= np.uint32(0xffffffe0)                  # bits of tokens that the sequence does not have
    assert np.array_equal(s.run(mask), got)


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
def test_what_lies_in_masked_places_does_not_matter(backend, vt):
    """NaN and large numbers in the tokens behind the sequence's end and in tokens that the mask leaves out."""
    seqs = [(50, 6)]
    s = Scene(backend, seqs, 4, 2, 64, 64, vb.Q8_0, vt, seed=4)
    may = [np.tril(np.ones((6, 6), bool))]
    may[0][:, 1] = may[0][:, 3] = False
    mask = (may[0] << np.arange(6)).sum(1).astype(np.uint32).reshape(6, 1)
    clean = s.run(mask)
    s.check(clean, may)
    width = s.kv_heads * s.dim
    for poison in (np.nan, 6e4):
        x = s._b(np.full(8 * width, poison, np.float32))
        bad = lambda at, n: vb.CacheRows(s._b(s.table), s._b(np.array([0, n], np.int32)), s._b(np.array([at], np.int32)), n)  # noqa: E731
        s.cache.append(None, x, x, bad(51, 1))
        s.cache.append(None, x, x, bad(53, 1))
        s.cache.append(None, x, x, bad(56, 8))
        got = s.run(mask)
        if np.isnan(poison):
            assert np.array_equal(got, clean)
        s.check(got, may)


@pytest.mark.parametrize("kt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 2])
def test_small_trees_and_what_they_leave_out(backend, kt, vt, dim, group):
    """Up to four, or eight, rows of a head of keys on average (the products' columns are laid out differently), more in one
    sequence; NaN in a token that the mask leaves out."""
    rng = _rng(dim + group)
    seqs = [(37, 3), (0, 2), (64, 6), (1130, 1), (31, 3)]
    s = Scene(backend, seqs, 2 * group, 2, dim, 32, kt, vt, seed=dim, pad=1)
    may, mask = _trees(rng, seqs)
    mask = np.concatenate([mask, np.zeros((1, 1), np.uint32)])
    for i in range(6):                                 # token 2 of the third sequence is for nobody
        may[2][i, 2] = False
        mask[5 + i, 0] &= ~np.uint32(4)
    clean = s.run(mask)
    s.check(clean, may)
    x = s._b(np.full(2 * dim, np.nan, np.float32))
    s.cache.append(None, x, x, vb.CacheRows(s._b(s.table[2:3]), s._b(np.array([0, 1], np.int32)), s._b(np.array([66], np.int32)), 1))
    assert np.array_equal(s.run(mask), clean)


def test_nan_in_the_context_and_in_q_reaches_its_own_rows_only(backend):
    s = Scene(backend, [(40, 2), (70, 2)], 4, 2, 64, seed=6)
    clean = s.run()
    x = s._b(np.full(s.kv_heads * s.dim, np.nan, np.float32))
    one = vb.CacheRows(s._b(s.table[:1]), s._b(np.array([0, 1], np.int32)), s._b(np.array([10], np.int32)), 1)
    s.cache.append(None, x, x, one)
    got = s.run()
    assert np.isnan(got[:2]).all() and np.array_equal(got[2:], clean[2:])
    s.q[3, 1, 5] = np.inf
    got = s.run()
    assert np.isnan(got[3, 1]).all()
    others = np.ones(4, bool)
    others[1] = False
    assert np.array_equal(got[2], clean[2]) and np.array_equal(got[3][others], clean[3][others])


@pytest.mark.parametrize("gain", [1e-30, 1e-3, 30.0, 1e4])
def test_scores_of_any_size(backend, gain):
    """Softmaxes from uniform to one-hot; queries far below and above one."""
    s = Scene(backend, [(600, 3)], 4, 1, 128, seed=12)
    s.q *= np.float32(gain)
    s.check(s.run())
    s.check(s.run(scale=0.0), scale=0.0)
    s.check(s.run(scale=-0.25), scale=-0.25)


def test_values_whose_scales_grow_and_shrink(backend):
    """The power of two that the value scales are lifted by changes on the way."""
    s = Scene(backend, [(900, 2)], 2, 1, 64, seed=13)
    g = np.exp(np.linspace(-12, 8, 902)).astype(np.float32)
    for order in (g, g[::-1]):
        v = (s.v[0] * order[:, None, None]).astype(np.float32)
        r = vb.CacheRows(s._b(s.table), s._b(np.array([0, 902], np.int32)), s._b(np.array([0], np.int32)), 902)
        s.cache.append(None, s._b(s.k[0]), s._b(v), r)
        s.check(s.run(), v=[quantised(s.vt, v)])


def test_bad_pages_and_table_ends_are_left_out(backend):
    s = Scene(backend, [(100, 1)], 2, 1, 64, 32, seed=14)
    table = s.table.copy()
    table[0, 1] = -3
    table[0, 2] = 1 << 20
    s.rows = vb.CacheRows(s._b(table), s._b(s.begin), s._b(s.start), s.rows_n, max_pages=4)
    got = s.run()
    keep = np.r_[0:32, 96:101]
    want, tol = attention(s.q[0, :1], quantised(s.kt, s.k[0])[keep, 0], quantised(s.vt, s.v[0])[keep, 0], np.ones((1, 37), bool), 0.125)
    assert (np.abs(got[0, :1] - want) <= tol).all()
    # a table of three pages for a sequence that says it has 101 tokens: the first 96 count
    s.rows = vb.CacheRows(s._b(s.table[:, :3]), s._b(s.begin), s._b(s.start), s.rows_n, max_pages=3)
    got = s.run()
    want, tol = attention(s.q[0, :1], quantised(s.kt, s.k[0])[:96, 0], quantised(s.vt, s.v[0])[:96, 0], np.ones((1, 96), bool), 0.125)
    assert (np.abs(got[0, :1] - want) <= tol).all()
    # and one whose pages all are bad attends to nothing
    s.rows = vb.CacheRows(s._b(np.full((1, 4), -1, np.int32)), s._b(s.begin), s._b(s.start), s.rows_n)
    assert (s.run() == 0).all()


def test_strides_and_odd_addresses(backend):
    s = Scene(backend, [(77, 5)], 4, 2, 96, 32, vb.Q4_0, vb.Q8_0, seed=15)
    want = s.run()
    w = s.heads * s.dim
    q = np.full((5, w + 9), np.nan, np.float32)
    q[:, 3:3 + w] = s.q.reshape(5, w)
    qb, out = s._b(q), s._b(np.full((5, w + 3), 1.25, np.float32))
    att = vb.CacheAttention(backend, s.cache, s.heads, 1)
    att.dispatch(backend, None, out.ptr + 4, qb.ptr + 12, s.rows, q_stride=w + 9, out_stride=w + 3)
    got = _read(backend, out).reshape(5, w + 3)
    assert np.array_equal(got[:, 1:1 + w].reshape(want.shape), want)
    assert (got[:, 0] == 1.25).all() and (got[:, 1 + w:] == 1.25).all()


def test_long_context_is_split_and_repeats_bit_for_bit(backend):
    """A context long enough that every thread block has a share of one sequence."""
    s = Scene(backend, [(30000, 1)], 2, 1, 64, 64, vb.Q8_0, vb.Q8_0, seed=16)
    first = s.run()
    assert np.array_equal(first, s.run())
    kq, vq = quantised(s.kt, s.k[0]), quantised(s.vt, s.v[0])
    for h in range(2):
        want, tol = attention(s.q[:, h], kq[:, 0], vq[:, 0], np.ones((1, 30001), bool), 0.125)
        assert (np.abs(first[:, h] - want) <= tol).all()


def test_recorded_call_follows_its_arrays(backend):
    """Captured once; the replays see new lengths, queries and cache contents."""
    import torch
    stream = torch.cuda.Stream()
    with vb.Backend(0, stream=stream.cuda_stream) as b:
        s = Scene(b, [(90, 1), (10, 1)], 8, 2, 128, 64, seed=17)
        b.synchronize()
        att = vb.CacheAttention(b, s.cache, 8, 2)
        q, out = s._b(s.q), b.uninit_buffer(s.q.size)
        start = s._b(s.start)
        rows = vb.CacheRows(s._b(s.table), s._b(s.begin), start, 2, max_pages=s.table.shape[1])
        b.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            att.dispatch(b, None, out, q, rows)
        for new in ([90, 10], [33, 0], [64, 7]):
            b.write_buffer(start, 0, np.array(new, np.int32))
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            got = _read(b, out).reshape(2, 8, 128)
            for i, c in enumerate(new):
                for h in range(8):
                    want, tol = attention(s.q[i:i + 1, h], quantised(s.kt, s.k[i])[:c + 1, h // 4], quantised(s.vt, s.v[i])[:c + 1, h // 4],
                                          np.ones((1, c + 1), bool), 128 ** -0.5)
                    assert (np.abs(got[i:i + 1, h] - want) <= tol).all()
        del graph
        att.free()
        s.cache.free()


def test_refusals(backend):
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, 2, 64, 1, 32)

    def status(c, *a):
        with pytest.raises(vb.VortxError) as e:
            vb.CacheAttention(backend, c, *a)
        return e.value.status
    assert status(cache, 3, 1) == _lib.VX_ERR_SHAPE and status(cache, 0, 1) == _lib.VX_ERR_SHAPE
    assert status(cache, 4, 0) == _lib.VX_ERR_INVALID_ARGUMENT
    assert status(vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, 2, 32, 1, 32), 4, 1) == _lib.VX_ERR_UNSUPPORTED
    backend.set_option("debug.fail_alloc_after", 1)
    assert status(cache, 4, 1) == _lib.VX_ERR_OUT_OF_MEMORY
    att = vb.CacheAttention(backend, cache, 4, 1)
    i32 = lambda *a: backend.init_buffer(np.array(a, np.int32))  # noqa: E731
    rows = vb.CacheRows(i32(0), i32(0, 2), i32(0), 2)
    q = backend.init_buffer(np.zeros(2 * 256, np.float32))
    with pytest.raises(IndexError):
        att.dispatch(backend, None, q, backend.init_buffer(np.zeros(511, np.float32)), rows)
    with pytest.raises(IndexError):
        att.dispatch(backend, None, q, q, rows, mask=backend.init_buffer(np.zeros(3, np.uint32)), mask_words=2)
    with pytest.raises(vb.VortxError):                 # a mask of no words
        att.dispatch(backend, None, q, q, rows, mask=backend.init_buffer(np.zeros(1, np.uint32)))
    with pytest.raises(vb.VortxError):                 # more sequences than it was made for
        att.dispatch(backend, None, q, q, vb.CacheRows(i32(0, 0), i32(0, 1, 2), i32(0, 0), 2))
    with pytest.raises(vb.VortxError):
        att.dispatch(backend, None, q.ptr, q.ptr, rows, q_stride=255)
    with vb.Backend(0) as other, pytest.raises(vb.VortxError):
        att.dispatch(other, None, q, q, rows)
    before = backend.launch_count()
    att.dispatch(backend, None, q, q, vb.CacheRows(0, 0, 0, 0, seqs=0, max_pages=1))
    assert backend.launch_count() == before

"""Decode-step shapes that take ways through the kernels which the operators' own tests do not: expert layers whose rows are whole
chunks and many of them, units of whole chunks that four warps share, and batches of up to 32 sequences whose tiles are dealt out
evenly, so that a block ends one item and begins another."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import attention, quantised
from test_gpu_kv_attention import Scene, _trees
from test_gpu_moe import Layer, _rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("experts,hidden,inner,top_k,tokens", [(3, 96, 2304, 2, 5), (2, 64, 4096, 2, 4), (4, 160, 2560, 2, 24), (1, 32, 2304, 1, 7),
                                                               (2, 2656, 2304, 1, 3), (5, 4128, 768, 3, 9), (2, 32, 7168, 2, 17)])
def test_down_rows_of_many_whole_chunks(backend, dt, experts, hidden, inner, top_k, tokens):
    """9 to 56 chunks a row: several for every warp, shares that begin and end inside an expert, one to three passes over them."""
    l = Layer(backend, experts, hidden, inner, top_k, True, vb.Q8_0, dt, max_tokens=tokens, seed=experts + tokens)
    x = _rng(tokens).standard_normal((tokens, hidden)).astype(np.float32)
    first = l.run(x)
    l.check(x, first)
    assert all(np.array_equal(a, b) for a, b in zip(first, l.run(x)))


@pytest.mark.parametrize("gt,experts,hidden,inner,top_k,tokens", [
    (vb.Q8_0, 8, 768, 1376, 2, 6),      # 344 units of 12 chunks: 4 turns of eight warps, 3 of four
    (vb.Q8_0, 4, 192, 4000, 2, 9),      # 3 chunks: one warp has none
    (vb.Q4_0, 4, 640, 4000, 2, 9),
    (vb.Q8_0, 2, 1024, 2304, 2, 8),     # 144 units: eight warps
    (vb.Q4_0, 2, 1024, 2304, 2, 3)])
def test_units_of_whole_chunks(backend, gt, experts, hidden, inner, top_k, tokens):
    l = Layer(backend, experts, hidden, inner, top_k, False, gt, vb.Q4_0, max_tokens=tokens, seed=experts + hidden)
    x = _rng(tokens).standard_normal((tokens, hidden)).astype(np.float32)
    first = l.run(x)
    l.check(x, first)
    assert all(np.array_equal(a, b) for a, b in zip(first, l.run(x)))


@pytest.mark.parametrize("gt,dt", [(vb.Q8_0, vb.Q4_0), (vb.Q4_0, vb.Q8_0)])
@pytest.mark.parametrize("experts,hidden,inner,top_k,tokens", [(256, 64, 64, 16, 64), (256, 96, 32, 1, 64), (129, 128, 96, 7, 63), (2, 8224, 64, 2, 64)])
def test_the_most_experts_and_tokens(backend, gt, dt, experts, hidden, inner, top_k, tokens):
    l = Layer(backend, experts, hidden, inner, top_k, tokens % 2 == 0, gt, dt, max_tokens=tokens, seed=experts + top_k)
    l.check(_rng(tokens).standard_normal((tokens, hidden)).astype(np.float32))


def _repeat(s, *args):
    first = s.run(*args)
    assert np.array_equal(first, s.run(*args))
    return first


def _lengths(seed, seqs, lo, hi, n):
    return [(int(c), n) for c in _rng(seed).integers(lo, hi, seqs)]


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("seqs,heads,kv_heads,dim,lo,hi,n", [
    (32, 16, 16, 64, 260, 700, 1),      # 512 items, more than there are blocks
    (16, 10, 10, 64, 700, 3000, 1),     # 160 items of unequal length over 444 blocks
    (16, 20, 10, 96, 1000, 2400, 3),    # eight rows to a block
    (12, 128, 16, 128, 300, 1200, 2)])  # sixteen
def test_tiles_of_few_sequences_dealt_out_evenly(backend, vt, seqs, heads, kv_heads, dim, lo, hi, n):
    s = Scene(backend, _lengths(seqs + dim, seqs, lo, hi, n), heads, kv_heads, dim, 64, vb.Q8_0, vt, seed=seqs)
    s.check(_repeat(s))


def test_drafts_of_two_sequences_dealt_out_evenly(backend):
    """2 x 48 rows of 4 query heads to a head of keys over thousands of tokens: 192 items of 16 rows and a hundred tiles."""
    rng = _rng(5)
    seqs = [(4000, 48), (2900, 48)]
    s = Scene(backend, seqs, 32, 8, 64, 64, vb.Q8_0, vb.Q8_0, seed=21)
    may, mask = _trees(rng, seqs)
    got = _repeat(s, mask)
    group = 4
    for i, (c, n) in enumerate(seqs):                  # L > 2000: sqrt(L / 4) additions per warp, twice that of decode_ref's 2000
        kq, vq = quantised(s.kt, s.k[i]), quantised(s.vt, s.v[i])
        ok = np.concatenate([np.ones((n, c), bool), may[i]], 1)
        for h in range(32):
            at = slice(s.begin[i], s.begin[i + 1])
            want, tol = attention(s.q[at, h], kq[:, h // group], vq[:, h // group], ok, 0.125)
            assert (np.abs(got[at, h] - want) <= 2 * tol).all()


@pytest.mark.parametrize("seqs,heads,kv_heads,dim,kt,vt", [
    ([(0, 300)], 4, 2, 64, vb.Q8_0, vb.Q8_0), ([(513, 257)], 8, 2, 128, vb.Q8_0, vb.Q4_0), ([(31, 1), (700, 190), (0, 0), (5, 64)], 6, 2, 96, vb.Q4_0, vb.Q8_0),
    ([(1000, 1)] * 9 + [(200, 180)], 4, 4, 64, vb.Q4_0, vb.Q4_0), ([(40, 140)], 2, 1, 256, vb.Q8_0, vb.Q8_0)])
def test_pieces_of_prompts(backend, seqs, heads, kv_heads, dim, kt, vt):
    """Hundreds of rows of a sequence, each attending to the tokens up to itself, alone and next to sequences of one row or none."""
    s = Scene(backend, seqs, heads, kv_heads, dim, 64, kt, vt, seed=len(seqs) + dim, pad=3)
    s.check(_repeat(s))


def test_pages_behind_four_gigabytes(backend):
    """A cache of 5.9 GB whose sequences lie in its first and last pages: byte offsets of more than 32 bits."""
    rng = _rng(40)
    heads, kv, dim, page, pages, context = 8, 4, 256, 64, 42000, 200
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, kv, dim, pages, page)
    assert cache.device_bytes() > 5 << 30
    dev = lambda a: backend.init_buffer(np.ascontiguousarray(a).ravel())  # noqa: E731
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    table = i32([[pages - 1, 0, pages - 7, 31000], [1, pages - 2, 30900, 2]])
    k, v = (rng.standard_normal((2, context, kv, dim)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((2, heads, dim)).astype(np.float32)
    cache.append(None, dev(k), dev(v), vb.CacheRows(table, i32([0, context, 2 * context]), i32([0, 0]), 2 * context))
    back = backend.uninit_buffer(v.size)
    cache.read(None, None, back, vb.CacheRows(table, i32([0, context, 2 * context]), i32([0, 0]), 2 * context))
    got = np.empty(v.size, np.float32)
    backend.slow_read_buffer(back, got)
    assert np.array_equal(got.reshape(v.shape), quantised(vb.Q8_0, v).astype(np.float32))
    att = vb.CacheAttention(backend, cache, heads, 2)
    out = backend.uninit_buffer(q.size)
    att.dispatch(backend, None, out, dev(q), vb.CacheRows(table, i32([0, 1, 2]), i32([context - 1] * 2), 2))
    got = np.empty(q.size, np.float32)
    backend.slow_read_buffer(out, got)
    kq, vq = quantised(vb.Q8_0, k), quantised(vb.Q8_0, v)
    for s in range(2):
        for h in range(heads):
            want, tol = attention(q[s, h:h + 1], kq[s, :, h // 2], vq[s, :, h // 2], np.ones((1, context), bool), dim ** -0.5)
            assert (np.abs(got.reshape(q.shape)[s, h] - want[0]) <= tol[0]).all()
    att.free()
    cache.free()

"""Attention over the quantised cache where values are not numbers or differ by many powers of two: each number of the result is held
to the tolerance of its own sum, whatever other rows, tokens or blocks hold.

Tolerance.  decode_ref.attention's (2 d + 2^-18) sum p |v|, over the tokens of the number's row and its place j in the head, and
where tokens' weights in the block of 32 values differ widely, what the two f16 parts of a weight leave: with w_t = p_t |scale_t| of
that block, at most 2^-21 max(w) |code_tj| for each token.  For the largest w of the block is at least 2^-1 in the units in which it is
split (a row's largest weight in [2^12, 2^13), times scales of 2^-13 and more; or w itself in [2^14, 2^15)), and in them a
weight's parts miss at most 2^-25, times a scale below 4, and their product's two roundings 2^-25 each: 2^-22.4 in all, next
to the 2^-22 of w_t itself that 2^-18 covers."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import attention, quantised
from test_gpu_kv_attention import Scene, _rng

pytestmark = pytest.mark.gpu


def _with_values(s, v):
    """The scene's sequences with other values; returns what their codes stand for."""
    s.v = [a.astype(np.float32) for a in v]
    total = [len(a) for a in s.v]
    every = np.concatenate([[0], np.cumsum(total)]).astype(np.int32)
    kv = [s._b(np.concatenate([a.reshape(len(a), -1) for a in x])) for x in (s.k, s.v)]
    s.cache.append(None, *kv, vb.CacheRows(s._b(s.table), s._b(every), s._b(np.zeros(len(total), np.int32)), int(every[-1])))
    return [quantised(s.vt, a) for a in s.v]


def _check(s, got, v, may=None, scale=None):
    """v: what the values' codes stand for; may[s]: [n, n] among the new tokens, None: those up to a row's own."""
    scale = s.dim ** -0.5 if scale is None else scale
    for at, (c, n) in enumerate(s.seqs):
        k = quantised(s.kt, s.k[at])
        blocks = np.abs(s.v[at]).reshape(c + n, s.kv_heads, -1, 32).max(-1)
        d = (blocks / np.float32(127 if s.vt == vb.Q8_0 else 7)).astype(np.float16).astype(np.float64).repeat(32, -1)
        code = np.divide(np.abs(v[at]), d, out=np.zeros_like(v[at]), where=d > 0)
        ok = np.concatenate([np.ones((n, c), bool), np.tril(np.ones((n, n), bool)) if may is None else may[at]], 1)
        for h in range(s.heads):
            q, hk = s.q[s.begin[at]:s.begin[at] + n, h].astype(np.float64), h // (s.heads // s.kv_heads)
            want, tol = attention(q, k[:, hk], v[at][:, hk], ok, scale)
            score = np.where(ok, scale * q @ k[:, hk].T, -np.inf)
            p = np.exp(score - score.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            for i in range(n):
                tol[i] += 2.0 ** -21 * (p[i][:, None] * d[:, hk]).max(0) * code[ok[i], hk].sum(0)
            err = np.abs(got[s.begin[at]:s.begin[at] + n, h] - want)
            assert (err <= tol).all(), (at, h, float((err / tol).max()))


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim,heads,kv_heads,n", [(64, 2, 2, 1), (96, 4, 2, 2), (128, 8, 2, 3), (256, 2, 2, 1)])
@pytest.mark.parametrize("at", [3, 70])
def test_nan_in_a_value_whose_weight_is_nothing(backend, vt, dim, heads, kv_heads, n, at):
    """0 times NaN is NaN in a sum: a row that attends to the token gets it, whether the token's tile is one of context alone (token 3)
    or the one in which the call's own tokens begin (token 70), and nobody else does."""
    s = Scene(backend, [(80, n), (80, n)], heads, kv_heads, dim, 32, vb.Q8_0, vt, seed=dim + at)
    for sq in range(2):
        s.q[:, :, 0] = 100.0
        s.k[sq][:, :, 0] = 0.0
        s.k[sq][at, :, 0] = -100.0                     # a score of -1250 and less
    s.v[0][at, :, 40] = np.nan
    want = _with_values(s, s.v)
    got = s.run()
    assert np.isnan(got[:n, :, 32:64]).all() and np.isfinite(got[:n, :, :32]).all() and np.isfinite(got[n:]).all()
    want[0][at] = 0.0
    got[:n, :, 32:64] = 0.0
    want[0][:, :, 32:64] = 0.0
    s.v[0][at] = 0.0
    _check(s, got, want)


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_rows_that_attend_to_large_and_to_small_values(backend, vt, dim, group):
    """Four drafted tokens in one tile, two of large values and two whose values are 2^-22 of that; each attends to its own
    kind.  With 1, 2 and 4 query heads to a head of keys: 4, 8 and 16 rows to a thread block."""
    s = Scene(backend, [(0, 4), (0, 4)], 2 * group, 2, dim, 32, vb.Q8_0, vt, seed=dim + group)
    v = [a * np.float32(2.0) ** np.array([16, -6, 16, -6], np.float32)[:, None, None] for a in s.v]
    may = np.array([[1, 0, 0, 0], [0, 1, 0, 0], [1, 0, 1, 0], [0, 1, 0, 1]], bool)
    mask = np.tile((may << np.arange(4)).sum(1).astype(np.uint32), 2).reshape(8, 1)
    want = _with_values(s, v)
    _check(s, s.run(mask), want, [may, may])


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim,heads,kv_heads,n", [(64, 2, 2, 1), (96, 4, 2, 3), (128, 8, 2, 3), (256, 4, 2, 1)])
@pytest.mark.parametrize("down", [10, 14, 15, 16, 18, 22])
@pytest.mark.parametrize("pattern", ["every token", "in turns"])
def test_blocks_of_a_token_that_differ(backend, vt, dim, heads, kv_heads, n, down, pattern):
    """A block of 32 values is 2^-down of the others': the second one of every token, or the first and second of tokens in turn."""
    s = Scene(backend, [(100, n), (3, n)], heads, kv_heads, dim, 32, vb.Q8_0, vt, seed=dim + down)
    v = [a * np.float32(2.0 ** 14) for a in s.v]
    for a in v:
        small = np.float32(2.0 ** -down)
        a[:, :, 32:64] *= small
        if pattern == "in turns":
            a[::2, :, 32:64] /= small
            a[::2, :, :32] *= small
    want = _with_values(s, v)
    _check(s, s.run(), want)


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (96, 4, 2), (128, 8, 2), (256, 2, 2)])
def test_blocks_that_only_tokens_of_little_weight_have(backend, vt, dim, heads, kv_heads):
    """The heaviest tokens' second block is zeros; what stands there comes from tokens of 2^-24 of their weight.  The last block is
    zeros in every token."""
    s = Scene(backend, [(90, 1)], heads, kv_heads, dim, 32, vb.Q8_0, vt, seed=dim)
    light = np.arange(91) % 3 == 1
    s.q[:] = 0.0
    s.q[:, :, 0] = 1.0
    s.k[0][:, :, 0] = np.where(light, -16.6, 0.0)[:, None]       # 16.6 = 24 ln 2
    s.k[0][:, :, 1:] *= np.float32(0.01)
    v = s.v[0].copy()
    v[~light, :, 32:64] = 0.0
    if dim > 64:
        v[:, :, -32:] = 0.0
    want = _with_values(s, [v])
    got = s.run(scale=1.0)
    _check(s, got, want, scale=1.0)
    assert np.abs(got[:, :, 32:64]).max() > 0 and (dim == 64 or (got[:, :, -32:] == 0).all())


@pytest.mark.parametrize("kt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim,heads,kv_heads,n", [(64, 2, 2, 1), (96, 4, 2, 2), (128, 8, 2, 3), (256, 4, 2, 4)])
@pytest.mark.parametrize("up", [16, 18, 20, 24])
def test_query_rows_of_a_wide_range(backend, kt, dim, heads, kv_heads, n, up):
    """An element of q is 2^up times the others, where the keys are zero.  The two f16 parts of the others miss at most 2^-39 of the
    largest (and 2^-23 of themselves): a score moves by that times scale sum |k|, and the result by twice as much of sum p |v|."""
    s = Scene(backend, [(60, n), (9, n)], heads, kv_heads, dim, 32, kt, vb.Q8_0, seed=dim + up)
    s.q[:, :, 5] = np.float32(2.0 ** up)
    for k in s.k:
        k[:, :, 5] = 0.0
    _with_values(s, s.v)
    got, group, scale = s.run(), heads // kv_heads, dim ** -0.5
    for at, (c, m) in enumerate(s.seqs):
        k, v = quantised(s.kt, s.k[at]), quantised(s.vt, s.v[at])
        ok = np.concatenate([np.ones((m, c), bool), np.tril(np.ones((m, m), bool))], 1)
        for h in range(heads):
            q, kh, vh = s.q[s.begin[at]:s.begin[at] + m, h].astype(np.float64), k[:, h // group], v[:, h // group]
            want, tol = attention(q, kh, vh, ok, scale)
            score = np.where(ok, scale * q @ kh.T, -np.inf)
            p = np.exp(score - score.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            tol += 2 * scale * 2.0 ** (up - 39) * np.abs(kh).sum(1).max() * (p @ np.abs(vh))
            assert (np.abs(got[s.begin[at]:s.begin[at] + m, h] - want) <= tol).all()


@pytest.mark.parametrize("vt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (96, 4, 2), (128, 16, 2), (256, 2, 2)])
def test_tiles_that_only_have_tokens_of_little_weight(backend, vt, dim, heads, kv_heads):
    """Small values of the last two of eight tiles, of 2^-44 of the earlier tokens' weight, are all that stands in the second block."""
    s = Scene(backend, [(254, 1)], heads, kv_heads, dim, 64, vb.Q8_0, vt, seed=dim + heads)
    light = np.arange(255) >= 192
    s.q[:] = 0.0
    s.q[:, :, 0] = 1.0
    s.k[0][:, :, 0] = np.where(light, -30.5, 0.0)[:, None]       # 44 ln 2
    s.k[0][:, :, 1:] *= np.float32(0.01)
    v = s.v[0] * np.float32(2.0 ** (-8 if vt == vb.Q8_0 else -12))
    v[~light, :, 32:64] = 0.0
    want = _with_values(s, [v])
    _check(s, s.run(scale=1.0), want, scale=1.0)

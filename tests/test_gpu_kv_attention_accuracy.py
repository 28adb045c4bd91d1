"""Attention over the quantised cache where values are not numbers or differ by many powers of two: each number of the result is held
to the tolerance of its own sum, (2 d + 2^-18) sum p |v| over the tokens of its row and its place in the head
(decode_ref.attention), whatever other rows, tokens or blocks hold."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import quantised
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
    s.check(got, v=want, k=[quantised(s.kt, k) for k in s.k])


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
    s.check(s.run(mask), [may, may], v=want)

"""The quantised cache: what is written and read back is bit for bit what the host quantiser makes of the same rows, at
every alignment of rows, tiles and pages; rows without a place and rows of no sequence; strides and odd addresses."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import quantised

pytestmark = pytest.mark.gpu

TYPES = [(vb.Q8_0, vb.Q8_0), (vb.Q8_0, vb.Q4_0), (vb.Q4_0, vb.Q8_0), (vb.Q4_0, vb.Q4_0)]


def _rows(backend, table, begin, start, rows):
    return vb.CacheRows(*(backend.init_buffer(np.asarray(a, np.int32).ravel()) for a in (table, begin, start)), rows)


def _rng(seed):
    return np.random.Generator(np.random.Philox(seed))


def _read(backend, buf):
    out = np.empty(buf.len(), buf.dtype)
    backend.slow_read_buffer(buf, out)
    return out


@pytest.mark.parametrize("kt,vt", TYPES)
@pytest.mark.parametrize("heads,dim,page,seqs", [
    (1, 32, 32, [(0, 1)]), (2, 64, 32, [(31, 1), (0, 33)]), (3, 96, 64, [(5, 100), (63, 1), (64, 64), (17, 0), (1, 62)]),
    (8, 128, 64, [(0, 64), (40, 41)]), (1, 256, 128, [(100, 200)]), (2, 512, 32, [(3, 70)]), (4, 160, 96, [(95, 2), (0, 96)]),
])
def test_round_trip_is_the_host_quantiser_bit_for_bit(backend, kt, vt, heads, dim, page, seqs):
    rng = _rng(dim + heads)
    n = [c for _, c in seqs]
    begin = np.concatenate([[0], np.cumsum(n)])
    rows = int(begin[-1])
    per = max(-(-(s + c) // page) for s, c in seqs)
    pages = per * len(seqs) + 3
    table = rng.permutation(pages)[:per * len(seqs)].reshape(len(seqs), per)
    cache = vb.QuantizedCache(backend, kt, vt, heads, dim, pages, page)
    k = (rng.standard_normal((rows, heads * dim)) * np.exp(rng.uniform(-8, 8, (rows, 1)))).astype(np.float32)
    v = rng.standard_normal((rows, heads * dim)).astype(np.float32)
    k[0, :32] = 0.0                                    # a block of zeros
    v[0, :32] = [3.0, -3.0] * 16                       # ties of the largest magnitude: the first one's sign counts
    r = _rows(backend, table, begin, [s for s, _ in seqs], rows)
    cache.append(None, backend.init_buffer(k.ravel()), backend.init_buffer(v.ravel()), r)
    ko, vo = (backend.init_buffer(np.full(rows * heads * dim + 7, np.nan, np.float32)) for _ in range(2))
    cache.read(None, ko, vo, r)
    for got, a, t in ((_read(backend, ko), k, kt), (_read(backend, vo), v, vt)):
        want = quantised(t, a).astype(np.float32)
        assert np.array_equal(got[:rows * heads * dim].reshape(want.shape), want)
        assert np.isnan(got[rows * heads * dim:]).all()
    # one of the two alone
    only = backend.init_buffer(np.zeros(rows * heads * dim, np.float32))
    cache.read(None, None, only, r)
    assert np.array_equal(_read(backend, only).reshape(v.shape), quantised(vt, v).astype(np.float32))
    cache.free()


@pytest.mark.parametrize("kt,vt", TYPES)
def test_writing_token_by_token_equals_writing_at_once(backend, kt, vt):
    heads, dim, page, n = 2, 64, 32, 75
    rng = _rng(3)
    k, v = (rng.standard_normal((n, heads * dim)).astype(np.float32) for _ in range(2))
    table = [[2, 0, 1]]
    out = []
    for piece in (n, 1, 13):
        cache = vb.QuantizedCache(backend, kt, vt, heads, dim, 3, page)
        for at in range(0, n, piece):
            m = min(piece, n - at)
            cache.append(None, backend.init_buffer(k[at:at + m].ravel()), backend.init_buffer(v[at:at + m].ravel()),
                         _rows(backend, table, [0, m], [at], m))
        bufs = [backend.uninit_buffer(n * heads * dim) for _ in range(2)]
        cache.read(None, *bufs, _rows(backend, table, [0, n], [0], n))
        out.append([_read(backend, b) for b in bufs])
        cache.free()
    for other in out[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(out[0], other))
    assert np.array_equal(out[0][0].reshape(k.shape), quantised(kt, k).astype(np.float32))


def test_strides_and_odd_addresses(backend):
    heads, dim, rows = 3, 64, 20
    w = heads * dim
    rng = _rng(5)
    wide = rng.standard_normal((rows, w + 37)).astype(np.float32)
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q4_0, heads, dim, 1, 32)
    buf = backend.init_buffer(wide.ravel())
    r = _rows(backend, [[0]], [0, rows], [4], rows)
    # rows inside wider ones, at an address that no vector load takes: k from column 1, v from column 5
    cache.append(None, buf.ptr + 4, buf.ptr + 20, r, k_stride=w + 37, v_stride=w + 37)
    out = backend.init_buffer(np.full((rows, 2 * w + 3), -1.0, np.float32).ravel())
    cache.read(None, out.ptr + 4, out.ptr + (w + 2) * 4, r, k_stride=2 * w + 3, v_stride=2 * w + 3)
    got = _read(backend, out).reshape(rows, -1)
    assert np.array_equal(got[:, 1:1 + w], quantised(vb.Q8_0, wide[:, 1:1 + w]).astype(np.float32))
    assert np.array_equal(got[:, w + 2:2 * w + 2], quantised(vb.Q4_0, wide[:, 5:5 + w]).astype(np.float32))
    assert (got[:, 0] == -1).all() and (got[:, w + 1] == -1).all() and (got[:, 2 * w + 2:] == -1).all()


def test_rows_and_tokens_without_a_place(backend):
    """Rows of no sequence stay as they were; tokens of a bad page, or behind the table's end, are zeros; nothing else of the
    cache changes."""
    heads, dim, page = 1, 32, 32
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, heads, dim, 4, page)
    full = np.ones((128, dim), np.float32)
    every = _rows(backend, [[0, 1, 2, 3]], [0, 128], [0], 128)
    one = backend.init_buffer(full.ravel())
    cache.append(None, one, one, every)
    rng = _rng(8)
    rows = 80
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    xb = backend.init_buffer(x.ravel())
    # sequence 0: rows 2..40 at tokens 20..58, pages -1 and 3; 1: no rows; 2: rows 41..60 at 50.., page 7 (too large) behind page 1 and then
    # past the table; 3: a negative start; rows 0, 1 and 70.. of no sequence
    table = [[-1, 3], [0, 0], [1, 7], [2, 2]]
    r = _rows(backend, table, [2, 41, 41, 61, 70], [20, 0, 50, -5], rows)
    cache.append(None, xb, xb, r)
    got = backend.init_buffer(np.full(rows * dim, 9.0, np.float32))
    cache.read(None, got, None, r)
    got = _read(backend, got).reshape(rows, dim)
    want = np.full((rows, dim), 9.0, np.float32)
    deq = quantised(vb.Q8_0, x).astype(np.float32)
    want[2:41] = 0.0
    want[2 + 12:41] = deq[2 + 12:41]                   # tokens 32..58 in page 3
    want[41:61] = 0.0                                  # tokens 50.. : page 7, then past the end
    assert np.array_equal(got, want)
    back = backend.uninit_buffer(128 * dim)
    cache.read(None, back, None, every)
    back = _read(backend, back).reshape(128, dim)
    keep = quantised(vb.Q8_0, full).astype(np.float32)
    keep[96:96 + 27] = deq[14:41]
    assert np.array_equal(back, keep)


@pytest.mark.parametrize("qt", [vb.Q8_0, vb.Q4_0])
def test_what_is_not_finite_reads_back_as_nan(backend, qt):
    dim = 128
    x = np.ones((5, dim), np.float32)
    x[0, 3], x[1, 40], x[2, 127] = np.nan, np.inf, -np.inf
    x[3, 70] = 3e38                                    # its scale passes f16
    x[4, 0] = 1e-20                                    # a tiny one does not
    cache = vb.QuantizedCache(backend, qt, qt, 1, dim, 1, 32)
    r = _rows(backend, [[0]], [0, 5], [0], 5)
    b = backend.init_buffer(x.ravel())
    cache.append(None, b, b, r)
    for which in (0, 1):
        out = backend.uninit_buffer(5 * dim)
        cache.read(None, out if which == 0 else None, out if which == 1 else None, r)
        got = _read(backend, out).reshape(5, 4, 32)
        bad = np.zeros((5, 4), bool)
        bad[0, 0] = bad[1, 1] = bad[2, 3] = bad[3, 2] = True
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("qt", [vb.Q8_0, vb.Q4_0])
def test_ties_borders_signs_and_small_scales(backend, qt):
    """Values of equal magnitude and different signs, values half way between two codes, scales next to a border of f16, f16's
    small numbers and zeros of both signs: still the host quantiser's codes."""
    rng = _rng(30)
    heads, dim, n = 2, 128, 96
    step, top = (127.0, 127) if qt == vb.Q8_0 else (7.0, 7)
    x = np.zeros((n, heads * dim // 32, 32), np.float32)
    for t in range(n):
        for b in range(x.shape[1]):
            kind = (t * x.shape[1] + b) % 8
            v = rng.integers(-top, top + 1, 32).astype(np.float32)
            if kind == 1:                              # half way: the scale is 1 / 8, exact
                v = (rng.integers(-top, top, 32) + 0.5).astype(np.float32) / 8
                v[5] = -top / 8 if t % 2 else top / 8
            elif kind == 2:                            # next to half way
                v = np.nextafter((rng.integers(-top, top, 32) + 0.5).astype(np.float32), rng.choice([-np.inf, np.inf], 32).astype(np.float32)) / 16
                v[3] = top / 16
            elif kind == 3:                            # the scale half way between two f16 numbers, or next to it
                s = np.float32((1024 + int(rng.integers(0, 1024)) + 0.5) / 1024)
                v = rng.standard_normal(32).astype(np.float32)
                v[7] = np.nextafter(np.float32(s * step), np.float32(rng.choice([0.0, s * step, np.inf])))
            elif kind == 4:
                v = (rng.standard_normal(32) * 10.0 ** rng.uniform(-9, -3)).astype(np.float32)
            elif kind == 5:
                v = np.where(rng.random(32) < 0.5, np.float32(-0.0), np.float32(0.0)).astype(np.float32)
            elif kind == 6:
                v = (rng.standard_normal(32) * 1e-30).astype(np.float32)
            elif kind == 7:                            # one magnitude, both signs
                v = np.where(rng.random(32) < 0.5, -1.0, 1.0).astype(np.float32) * np.float32(rng.uniform(0.1, 10))
            x[t, b] = v
    flat = x.reshape(n, heads * dim)
    cache = vb.QuantizedCache(backend, qt, qt, heads, dim, 3, 32)
    xb = backend.init_buffer(flat.ravel())
    rows = _rows(backend, [[2, 0, 1]], [0, n], [0], n)
    cache.append(None, xb, xb, rows)
    k, v = backend.uninit_buffer(flat.size), backend.uninit_buffer(flat.size)
    cache.read(None, k, v, rows)
    want = vb.dequantize_host(qt, vb.quantize(qt, flat), n, heads * dim).astype(np.float32).reshape(-1, 32)
    for got in (_read(backend, k).reshape(-1, 32), _read(backend, v).reshape(-1, 32)):
        bad = [i for i in range(len(want)) if not np.array_equal(got[i], want[i])]
        assert not bad, (len(bad), bad[0] % 8, got[bad[0]], want[bad[0]])


def test_many_sequences_and_empty_calls(backend):
    """More sequences than one step of the search sees, most of them without rows."""
    rng = _rng(11)
    seqs, heads, dim, page = 1500, 1, 32, 32
    n = rng.integers(0, 4, seqs) * (rng.random(seqs) < 0.3)
    begin = np.concatenate([[0], np.cumsum(n)])
    rows = int(begin[-1])
    start = rng.integers(0, 29, seqs)
    cache = vb.QuantizedCache(backend, vb.Q4_0, vb.Q8_0, heads, dim, seqs, page)
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    r = _rows(backend, rng.permutation(seqs).reshape(-1, 1), begin, start, rows)
    b, out = backend.init_buffer(x.ravel()), backend.uninit_buffer(rows * dim)
    cache.append(None, b, b, r)
    cache.read(None, out, None, r)
    assert np.array_equal(_read(backend, out).reshape(x.shape), quantised(vb.Q4_0, x).astype(np.float32))
    before = backend.launch_count()
    cache.append(None, b, b, vb.CacheRows(0, 0, 0, 0, seqs=0, max_pages=1))
    cache.read(None, None, None, r)
    assert backend.launch_count() == before


def test_two_contexts_on_two_streams_share_a_cache(backend):
    with vb.Backend(0) as other:
        cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, 1, 64, 2, 32)
        x = _rng(2).standard_normal((40, 64)).astype(np.float32)
        b = other.init_buffer(x.ravel())
        arrays = [other.init_buffer(np.asarray(a, np.int32)) for a in ([1, 0], [0, 40], [0])]
        other.synchronize()
        cache.append(None, b, b, vb.CacheRows(*arrays, 40), backend=other)
        other.synchronize()
        out = backend.uninit_buffer(40 * 64)
        cache.read(None, None, out, vb.CacheRows(*arrays, 40))
        assert np.array_equal(_read(backend, out).reshape(x.shape), quantised(vb.Q8_0, x).astype(np.float32))
        b.free()
        for a in arrays:
            a.free()


def test_refusals(backend):
    def status(*a, **kw):
        with pytest.raises(vb.VortxError) as e:
            vb.QuantizedCache(backend, *a, **kw)
        return e.value.status
    from vortx_b200 import _lib
    bad = _lib.VX_ERR_INVALID_ARGUMENT
    assert status(5, vb.Q8_0, 1, 64, 1) == bad and status(vb.Q8_0, 9, 1, 64, 1) == bad
    assert status(vb.Q8_0, vb.Q8_0, 0, 64, 1) == bad and status(vb.Q8_0, vb.Q8_0, 1, 48, 1) == bad
    assert status(vb.Q8_0, vb.Q8_0, 1, 0, 1) == bad and status(vb.Q8_0, vb.Q8_0, 1, 64, 0) == bad
    assert status(vb.Q8_0, vb.Q8_0, 1, 64, 1, 33) == bad and status(vb.Q8_0, vb.Q8_0, 1, 64, 1, 0) == bad
    assert status(vb.Q8_0, vb.Q8_0, 1, 544, 1) == _lib.VX_ERR_UNSUPPORTED
    assert status(vb.Q8_0, vb.Q8_0, 64, 512, 2 ** 30, 2 ** 20) == _lib.VX_ERR_OUT_OF_MEMORY
    backend.set_option("debug.fail_alloc_after", 1)
    assert status(vb.Q8_0, vb.Q8_0, 1, 64, 1) == _lib.VX_ERR_OUT_OF_MEMORY
    cache = vb.QuantizedCache(backend, vb.Q8_0, vb.Q8_0, 2, 64, 1, 32)
    assert cache.device_bytes() == 2 * 2 * (32 * 64 + 32 * 2 * 2)
    r = _rows(backend, [[0]], [0, 4], [0], 4)
    buf = backend.init_buffer(np.zeros(4 * 128, np.float32))
    short = backend.init_buffer(np.zeros(4 * 128 - 1, np.float32))
    with pytest.raises(IndexError):
        cache.append(None, short, buf, r)
    with pytest.raises(IndexError):
        cache.read(None, buf, short, r)
    with pytest.raises(TypeError):
        cache.append(None, backend.init_buffer(np.zeros(4 * 128, np.int32)), buf, r)
    with pytest.raises(vb.VortxError):
        cache.append(None, None, buf, r)
    with pytest.raises(vb.VortxError):
        cache.append(None, buf.ptr, buf.ptr, r, k_stride=127)
    with pytest.raises(IndexError):
        vb.CacheRows(backend.init_buffer(np.zeros(1, np.int32)), backend.init_buffer(np.zeros(1, np.int32)), backend.init_buffer(np.zeros(1, np.int32)), 4)

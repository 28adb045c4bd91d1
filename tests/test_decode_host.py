"""The decode-step operators without a GPU: the mask of a tree, what the Python layer refuses, null arguments."""
import ctypes as C

import numpy as np
import pytest

import vortx_b200 as vb
from vortx_b200 import _lib
from vortx_b200.backend import GpuBuffer

BAD = _lib.VX_ERR_INVALID_ARGUMENT


class _NoBackend:
    _ctx = None


def _buf(n, dtype=np.float32):
    return GpuBuffer(_NoBackend(), 0x1000, n, dtype, owned=False)


def _i32(n):
    return _buf(n, np.int32)


@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 64, 65, 100])
def test_tree_mask(n):
    rng = np.random.Generator(np.random.Philox(n))
    parents = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
    m = vb.tree_mask(parents)
    assert m.dtype == np.uint32 and m.shape == (n, -(-n // 32))
    for i in range(n):
        want, j = set(), i
        while j >= 0:
            want.add(j)
            j = parents[j]
        assert want == {j for j in range(32 * m.shape[1]) if m[i, j // 32] >> (j % 32) & 1}


def test_tree_mask_of_a_chain_is_the_lower_triangle():
    m = vb.tree_mask([i - 1 for i in range(40)])
    assert [int(r[0]) | int(r[1]) << 32 for r in m] == [(2 << i) - 1 for i in range(40)]


@pytest.mark.parametrize("parents", [[0], [-2], [-1, 1], [-1, 0, 5]])
def test_tree_mask_refuses(parents):
    with pytest.raises(ValueError):
        vb.tree_mask(parents)


def test_rows_struct():
    assert C.sizeof(_lib.VxKvRows) == 48
    assert [f for f, _ in _lib.VxKvRows._fields_] == ["table", "max_pages", "begin", "start", "seqs", "rows"]
    r = vb.CacheRows(_i32(12), _i32(4), _i32(3), 7)
    assert (r.seqs, r.max_pages, r.rows) == (3, 4, 7)
    assert (r._c.table, r._c.begin, r._c.start, r._c.seqs, r._c.max_pages, r._c.rows) == (0x1000, 0x1000, 0x1000, 3, 4, 7)


@pytest.mark.parametrize("error,args,kw", [
    (TypeError, (_buf(1), _i32(2), _i32(1), 1), {}),                     # a table of floats
    (TypeError, (_i32(1), _buf(2, np.int64), _i32(1), 1), {}),
    (TypeError, ([0], _i32(2), _i32(1), 1), {}),                         # host memory
    (IndexError, (_i32(1), _i32(1), _i32(1), 1), {}),                    # begin has seqs + 1 entries
    (IndexError, (_i32(3), _i32(3), _i32(2), 1), {"max_pages": 2}),
    (IndexError, (_i32(4), _i32(4), _i32(2), 1), {"seqs": 3}),
    (ValueError, (0x1000, 0x1000, 0x1000, 1), {"max_pages": 1}),
    (ValueError, (0x1000, 0x1000, 0x1000, 1), {"seqs": 1}),
    (ValueError, (_i32(1), _i32(2), _i32(1), -1), {}),
    (ValueError, (_i32(7), _i32(4), _i32(3), 1), {}),                    # not the same number of pages each
    (ValueError, (0x1000, 0x1000, 0x1000, 1), {"seqs": -1, "max_pages": 1}),
])
def test_rows_refuse(error, args, kw):
    with pytest.raises(error):
        vb.CacheRows(*args, **kw)


def _cache():
    c = vb.QuantizedCache.__new__(vb.QuantizedCache)
    c.backend, c._h, c.heads, c.head_dim, c.width = _NoBackend(), None, 2, 64, 128
    return c


def test_freed_and_short_are_refused():
    cache, rows = _cache(), vb.CacheRows(_i32(1), _i32(2), _i32(1), 3)
    for call in (cache.append, cache.read):
        with pytest.raises(IndexError):
            call(None, _buf(3 * 128 - 1), _buf(3 * 128), rows)
        with pytest.raises(IndexError):
            call(None, _buf(3 * 128), _buf(3 * 128), rows, v_stride=129)
        with pytest.raises(ValueError):
            call(None, _buf(3 * 128), _buf(3 * 128), rows, k_stride=-1)
        with pytest.raises(TypeError):
            call(None, _buf(3 * 128, np.float16), _buf(3 * 128), rows)
        with pytest.raises(vb.VortxError) as e:               # no cache behind it
            call(None, _buf(3 * 128), _buf(3 * 128), rows)
        assert e.value.status == BAD
    with pytest.raises(ValueError):
        vb.CacheAttention(_NoBackend(), cache, 4, 1)
    with pytest.raises(ValueError):
        vb.CacheAttention(_NoBackend(), cache, -4, 1)
    with pytest.raises(ValueError):
        vb.QuantizedCache(_NoBackend(), vb.Q8_0, vb.Q8_0, 1, 64, -1)
    att = vb.CacheAttention.__new__(vb.CacheAttention)
    att.cache, att.width, att.backend, att._h = cache, 256, _NoBackend(), None
    with pytest.raises(ValueError):
        att.dispatch(_NoBackend(), None, _buf(3 * 256), _buf(3 * 256), rows)
    with pytest.raises(ValueError):
        att.dispatch(_NoBackend(), None, _buf(3 * 256), _buf(3 * 256), rows, mask=0x1000)
    with pytest.raises(ValueError, match="words"):
        att.dispatch(_NoBackend(), None, _buf(3 * 256), _buf(3 * 256), rows, mask=_buf(4, np.uint32))
    layer = vb.MoeLayer.__new__(vb.MoeLayer)
    w = vb.QuantizedMatrix.__new__(vb.QuantizedMatrix)
    w._h, w.backend = None, _NoBackend()
    layer._gate = layer._up = layer._down = w
    layer._router_buffer, layer._h, layer.backend = None, None, _NoBackend()
    with pytest.raises(ValueError, match="freed"):
        layer.dispatch(_NoBackend(), None, _buf(1), _buf(1), 1)
    with pytest.raises(ValueError):
        layer.dispatch(_NoBackend(), None, _buf(1), _buf(1), -1)


def test_null_arguments():
    lib = _lib.load()
    h, n = C.c_void_p(), C.c_size_t()
    rows = _lib.VxKvRows(0x1000, 1, 0x1000, 0x1000, 1, 1)
    calls = [
        lambda: lib.vx_kv_cache_create(None, 0, 0, 1, 64, 1, 32, C.byref(h)),
        lambda: lib.vx_kv_cache_free(None, None),
        lambda: lib.vx_kv_cache_info(None, None, None, None, None, None, None, C.byref(n)),
        lambda: lib.vx_kv_append(None, None, C.byref(rows), 0x1000, 64, 0x1000, 64),
        lambda: lib.vx_kv_read(None, None, C.byref(rows), 0x1000, 64, 0x1000, 64),
        lambda: lib.vx_kv_attention_create(None, None, 1, 1, C.byref(h)),
        lambda: lib.vx_kv_attention_free(None, None),
        lambda: lib.vx_kv_attention_run(None, None, C.byref(rows), 0x1000, 64, 0x1000, 64, 1.0, None, 0),
        lambda: lib.vx_moe_create(None, 0x1000, 1, None, None, None, 1, 1, 1, C.byref(h)),
        lambda: lib.vx_moe_free(None, None),
        lambda: lib.vx_moe_run(None, None, 0x1000, 64, 0x1000, 64, 1, None, None),
    ]
    for call in calls:
        assert call() == BAD and b"null" in lib.vx_last_error()
    assert h.value is None

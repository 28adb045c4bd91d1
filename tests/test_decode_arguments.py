"""What the decode-step operators' Python layer refuses of buffers that have been freed and of views with gaps (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import vortx_b200 as vb
from vortx_b200 import _lib
from vortx_b200.backend import GpuBuffer
from vortx_b200.shapes import TensorLayout
from vortx_b200.tensor import TensorRef


class _NoBackend:
    _ctx = None


def _buf(n, dtype=np.float32):
    return GpuBuffer(_NoBackend(), 0x1000, n, dtype, owned=False)


def _i32(n):
    return _buf(n, np.int32)


def _objects():
    """A cache, an attention and a layer without a library object behind them: a call that passes the checks is refused there."""
    cache = vb.QuantizedCache.__new__(vb.QuantizedCache)
    cache.backend, cache._h, cache.heads, cache.head_dim, cache.width = _NoBackend(), C.c_void_p(0), 2, 64, 128
    att = vb.CacheAttention.__new__(vb.CacheAttention)
    held = vb.QuantizedCache.__new__(vb.QuantizedCache)
    held.backend, held._h, held.heads, held.head_dim, held.width = _NoBackend(), C.c_void_p(1), 2, 64, 128
    att.cache, att.width, att.backend, att._h = held, 256, _NoBackend(), None
    w = vb.QuantizedMatrix.__new__(vb.QuantizedMatrix)
    w._h, w.backend = C.c_void_p(1), _NoBackend()
    layer = vb.MoeLayer.__new__(vb.MoeLayer)
    layer._gate = layer._up = layer._down = w
    layer._router_buffer, layer._h, layer.backend = None, None, _NoBackend()
    layer.hidden, layer.top_k, layer.inner, layer.experts, layer.max_tokens = 64, 2, 32, 4, 8
    return cache, att, layer


def _calls(rows, k=None, q=None, mask=None, x=None, ids=None, weights=None):
    cache, att, layer = _objects()
    b, k, q, x = _NoBackend(), k or _buf(384), q or _buf(768), x or _buf(192)
    return {
        "append k": lambda: cache.append(None, k, _buf(384), rows), "append v": lambda: cache.append(None, _buf(384), k, rows),
        "read k": lambda: cache.read(None, k, _buf(384), rows), "read v": lambda: cache.read(None, _buf(384), k, rows),
        "attention q": lambda: att.dispatch(b, None, _buf(768), q, rows, mask=mask), "attention out": lambda: att.dispatch(b, None, q, _buf(768), rows, mask=mask),
        "layer x": lambda: layer.dispatch(b, None, _buf(192), x, 3, ids=ids, weights=weights),
        "layer y": lambda: layer.dispatch(b, None, x, _buf(192), 3, ids=ids, weights=weights),
    }


def _freed(n, dtype=np.float32):
    b = _buf(n, dtype)
    b.free()
    return b


def _behind(b):
    """A view that begins behind the buffer's start, so that its address is not zero when the buffer's is."""
    return TensorRef(TensorLayout.contiguous([b.len()]), b).narrow(0, 4, b.len() - 4)


def test_calls_that_pass_reach_the_library():
    rows = vb.CacheRows(_i32(1), _i32(2), _i32(1), 3)
    for name, call in _calls(rows, mask=_buf(3, np.uint32), ids=_i32(6), weights=_buf(6)).items():
        with pytest.raises(vb.VortxError) as e:
            call()
        assert e.value.status == _lib.VX_ERR_INVALID_ARGUMENT, name


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("view", [False, True])
def test_rows_whose_arrays_have_been_freed(which, view):
    """The pointers were taken when the rows were made; a call would read memory that is somebody else's by now."""
    arrays = [_i32(1), _i32(2), _i32(1)]
    given = list(arrays)
    if view:
        arrays[which] = _i32(6)
        given[which] = _behind(arrays[which])
    rows = vb.CacheRows(*given, 3, seqs=1, max_pages=1)
    arrays[which].free()
    for name, call in _calls(rows).items():
        if not name.startswith("layer"):
            with pytest.raises(ValueError, match="freed"):
                call()


@pytest.mark.parametrize("view", [False, True])
def test_tensors_that_have_been_freed(view):
    """A freed mask would be no mask, a freed k of read one that is not wanted, a freed view an address near zero."""
    rows = vb.CacheRows(_i32(1), _i32(2), _i32(1), 3)
    of = (lambda n, dtype=np.float32: _behind(_freed(n + 4, dtype))) if view else _freed
    for name, call in _calls(rows, k=of(384), q=of(768), x=of(192)).items():
        with pytest.raises(ValueError, match="freed"):
            call()
    for kw in ({"mask": of(3, np.uint32)}, {"ids": of(6, np.int32)}, {"weights": of(6)}):
        for name, call in _calls(rows, **kw).items():
            if name.startswith("attention" if "mask" in kw else "layer"):
                with pytest.raises(ValueError, match="freed"):
                    call()


def test_empty_tensors_need_no_address():
    """A buffer of no elements may have the address zero."""
    none = GpuBuffer(_NoBackend(), 0, 0, np.int32, owned=False)
    rows = vb.CacheRows(none, none, none, 0)
    empty = GpuBuffer(_NoBackend(), 0, 0, np.float32, owned=False)
    cache, _, _ = _objects()
    with pytest.raises(vb.VortxError):
        cache.append(None, empty, empty, rows)


def _view(shape, stride, dtype=np.float32, offset=0, size=1 << 16):
    return TensorRef(TensorLayout.contiguous([size]).view(offset, shape, stride), _buf(size, dtype))


@pytest.mark.parametrize("what,shape,stride,dtype", [("table", [3, 4], [9, 1], np.int32), ("begin", [4], [2], np.int32), ("start", [3, 1], [5, 1], np.int32)])
def test_rows_of_arrays_with_gaps_are_refused(what, shape, stride, dtype):
    """Four columns of a page table of nine: the kernels take the pages of all sequences one after the other."""
    arrays = {"table": _i32(12), "begin": _i32(4), "start": _i32(3)}
    arrays[what] = _view(shape, stride, dtype)
    with pytest.raises(ValueError, match="dense|stride 1"):
        vb.CacheRows(**arrays, rows=3, seqs=3, max_pages=4)
    arrays[what] = _view(shape, [int(np.prod(shape[i + 1:])) for i in range(len(shape))], dtype)
    vb.CacheRows(**arrays, rows=3, seqs=3, max_pages=4)


def test_views_with_gaps_need_the_stride_argument():
    """Rows of a wider matrix (q, k and v of one projection) without saying how far apart they are; heads that are not next to each
    other; a mask, ids or weights with gaps, which have no stride argument."""
    rows = vb.CacheRows(_i32(1), _i32(2), _i32(1), 3)
    gaps = dict(k=_view([3, 128], [384, 1]), q=_view([3, 256], [512, 1]), x=_view([3, 64], [96, 1]))
    for name, call in _calls(rows, **gaps).items():
        with pytest.raises(ValueError, match="dense"):
            call()
    for kw in ({"mask": _view([3, 1], [2, 1], np.uint32)}, {"ids": _view([3, 2], [4, 1], np.int32)}, {"weights": _view([3, 2], [4, 1])}):
        for name, call in _calls(rows, **kw).items():
            if name.startswith("attention" if "mask" in kw else "layer"):
                with pytest.raises(ValueError, match="dense"):
                    call()
    cache, att, layer = _objects()
    b = _NoBackend()
    # with the stride they reach the library, which has no object here
    for call in (lambda: cache.append(None, gaps["k"], gaps["k"], rows, k_stride=384, v_stride=384), lambda: cache.read(None, gaps["k"], None, rows, k_stride=384),
                 lambda: att.dispatch(b, None, _buf(768), gaps["q"], rows, q_stride=512), lambda: att.dispatch(b, None, gaps["q"], _buf(768), rows, out_stride=512),
                 lambda: layer.dispatch(b, None, _buf(192), gaps["x"], 3, x_stride=96), lambda: layer.dispatch(b, None, gaps["x"], _buf(192), 3, y_stride=96)):
        with pytest.raises(vb.VortxError):
            call()
    apart = _view([3, 2, 64], [64, 192, 1])             # [heads, rows, 64] seen as [rows, heads, 64]
    with pytest.raises(ValueError, match="dense"):
        cache.append(None, apart, _buf(384), rows, k_stride=64)
    # dense views and single rows of a wider matrix need no stride
    one = vb.CacheRows(_i32(1), _i32(2), _i32(1), 1)
    for call in (lambda: cache.append(None, _view([3, 2, 64], [128, 64, 1]), _view([3, 128], [128, 1], offset=512), rows),
                 lambda: cache.append(None, _view([1, 128], [384, 1]), _view([128], [1], offset=256), one)):
        with pytest.raises(vb.VortxError):
            call()


def test_a_router_with_gaps_is_refused():
    w = vb.QuantizedMatrix.__new__(vb.QuantizedMatrix)
    w._h, w.backend, w.rows, w.cols = None, _NoBackend(), 128, 64
    for router, error in ((_view([4, 64], [80, 1]), ValueError), (_view([4, 64], [64, 1]), vb.VortxError)):
        with pytest.raises(error):
            vb.MoeLayer(_NoBackend(), router, w, w, w, 4, 2)

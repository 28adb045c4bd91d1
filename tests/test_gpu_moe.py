"""The mixture-of-experts layer against its f64 statement on the weights' dequantised values."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import moe, quantised
from vortx_b200 import _lib

pytestmark = pytest.mark.gpu


def _rng(seed):
    return np.random.Generator(np.random.Philox(seed))


def _read(backend, buf):
    out = np.empty(buf.len(), buf.dtype)
    backend.slow_read_buffer(buf, out)
    return out


class Layer:
    def __init__(self, backend, experts, hidden, inner, top_k, normalise=True, gt=vb.Q4_0, dt=vb.Q4_0, max_tokens=32, seed=0, router=None):
        rng = _rng(seed)
        self.backend, self.hidden, self.inner, self.top_k, self.normalise, self.experts = backend, hidden, inner, top_k, normalise, experts
        w = lambda r, c: (rng.standard_normal((r, c)) / np.sqrt(c)).astype(np.float32)  # noqa: E731
        self.router = (1.5 * w(experts, hidden)).astype(np.float32) if router is None else router
        gate, up, down = w(experts * inner, hidden), w(experts * inner, hidden), w(experts * hidden, inner)
        self.gate, self.up = (quantised(gt, m).reshape(experts, inner, hidden) for m in (gate, up))
        self.down = quantised(dt, down).reshape(experts, hidden, inner)
        self.mats = [vb.QuantizedMatrix.from_f32(backend, t, m) for t, m in ((gt, gate), (gt, up), (dt, down))]
        self.router_buf = backend.init_buffer(self.router.ravel())
        self.layer = vb.MoeLayer(backend, self.router_buf, *self.mats, experts=experts, top_k=top_k, normalise=normalise, max_tokens=max_tokens)

    def run(self, x):
        t = len(x)
        b = self.backend
        y = b.init_buffer(np.full(t * self.hidden + 3, 7.5, np.float32))
        ids, w = b.init_buffer(np.full(t * self.top_k + 1, -9, np.int32)), b.init_buffer(np.full(t * self.top_k + 1, 7.5, np.float32))
        before = b.launch_count()
        self.layer.dispatch(b, None, y, b.init_buffer(x.ravel()), t, ids=ids, weights=w)
        assert b.launch_count() - before == 3
        y, ids, w = _read(b, y), _read(b, ids), _read(b, w)
        assert (y[t * self.hidden:] == 7.5).all() and ids[-1] == -9 and w[-1] == 7.5
        return y[:-3].reshape(t, -1), ids[:-1].reshape(t, -1), w[:-1].reshape(t, -1)

    def check(self, x, got=None):
        y, ids, w = self.run(x) if got is None else got
        want, wi, ww, tol, dw = moe(x, self.router, self.gate, self.up, self.down, self.top_k, self.normalise)
        assert np.array_equal(ids, wi)
        assert (np.abs(w - ww) <= (dw[:, None] + 2.0 ** -20) * ww).all()
        assert (np.abs(y - want) <= tol).all(), float((np.abs(y - want) / tol).max())


@pytest.mark.parametrize("gt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("dt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("experts,hidden,inner,top_k,tokens", [
    (1, 32, 32, 1, 1), (2, 64, 96, 2, 3), (5, 160, 224, 3, 9), (8, 256, 128, 2, 17), (16, 1120, 608, 3, 7), (33, 96, 32, 8, 32), (256, 64, 32, 16, 5),
    (3, 1056, 32, 1, 64), (2, 32, 1376, 2, 33),
])
def test_types_and_shapes(backend, gt, dt, experts, hidden, inner, top_k, tokens):
    l = Layer(backend, experts, hidden, inner, top_k, tokens % 2 == 0, gt, dt, max_tokens=tokens, seed=experts + tokens)
    l.check(_rng(tokens).standard_normal((tokens, hidden)).astype(np.float32))


@pytest.mark.parametrize("tokens", range(1, 20))
def test_every_group_size_of_one_expert(backend, tokens):
    """One expert takes all tokens: groups of 1 to 16 and the next pass."""
    l = Layer(backend, 2, 128, 64, 2, max_tokens=24, seed=1)
    l.check(_rng(tokens).standard_normal((tokens, 128)).astype(np.float32))


@pytest.mark.parametrize("gt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("experts,hidden,inner,top_k,tokens", [(8, 1536, 1376, 2, 6), (2, 512, 4800, 2, 11), (4, 160, 4000, 2, 5), (3, 96, 3424, 3, 8)])
def test_units_that_four_warps_share(backend, gt, experts, hidden, inner, top_k, tokens):
    """More units than thread blocks and columns that do not fill eight warps: two units of a block at a time."""
    l = Layer(backend, experts, hidden, inner, top_k, True, gt, vb.Q8_0, max_tokens=tokens, seed=experts)
    x = _rng(tokens).standard_normal((tokens, hidden)).astype(np.float32)
    first = l.run(x)
    l.check(x, first)
    assert all(np.array_equal(a, b) for a, b in zip(first, l.run(x)))


@pytest.mark.parametrize("hidden,tokens", [(2624, 3), (4128, 5), (9504, 2), (32, 4)])
def test_output_tiles_share_out_the_columns(backend, hidden, tokens):
    """Three, two, one and four blocks add up an output tile's columns."""
    l = Layer(backend, 2, hidden, 192, 2, False, vb.Q8_0, vb.Q4_0, max_tokens=tokens, seed=hidden)
    l.check(_rng(tokens).standard_normal((tokens, hidden)).astype(np.float32))


def test_calls_follow_each_other_and_repeat_bit_for_bit(backend):
    """Different token counts through one layer; the same call again gives the same bits."""
    l = Layer(backend, 16, 512, 256, 4, max_tokens=32, seed=2)
    rng = _rng(7)
    xs = [rng.standard_normal((t, 512)).astype(np.float32) for t in (32, 1, 7, 32, 2)]
    first = [l.run(x) for x in xs]
    for x, f in zip(xs, first):
        l.check(x, f)
    for x, f in list(zip(xs, first))[::-1]:
        assert all(np.array_equal(a, b) for a, b in zip(l.run(x), f))


def test_ties_go_to_the_lowest_expert(backend):
    router = np.zeros((9, 64), np.float32)
    router[4], router[7] = 1.0, 1.0
    l = Layer(backend, 9, 64, 32, 4, max_tokens=4, router=router)
    x = np.ones((2, 64), np.float32)
    x[1] *= -1
    _, ids, w = l.run(x)
    assert ids.tolist() == [[4, 7, 0, 1], [0, 1, 2, 3]]
    assert (np.abs(w[1] - 0.25) <= 2.0 ** -22).all()
    x[:] = 0.0                                         # every logit is 0 or -0
    x[1] = -0.0
    assert l.run(x)[1].tolist() == [[0, 1, 2, 3]] * 2


def test_what_is_not_finite_stays_with_its_token(backend):
    l = Layer(backend, 6, 96, 64, 2, max_tokens=8, seed=5)
    x = _rng(3).standard_normal((5, 96)).astype(np.float32)
    clean = l.run(x)
    x[1, 7], x[3, 90] = np.nan, np.inf
    y, ids, w = l.run(x)
    for t in (0, 2, 4):
        assert np.array_equal(y[t], clean[0][t]) and np.array_equal(ids[t], clean[1][t])
    assert not np.isfinite(y[[1, 3]]).any()
    for t in (1, 3):                                   # still two different experts
        assert len(set(ids[t])) == 2 and ids[t].min() >= 0 and ids[t].max() < 6
    assert ids[1].tolist() == [0, 1]


@pytest.mark.parametrize("gain", [1e-30, 1e-4, 1e3])
def test_inputs_of_any_size(backend, gain):
    router = (_rng(1).standard_normal((4, 128)) * (0.1 / gain)).astype(np.float32)
    l = Layer(backend, 4, 128, 64, 2, max_tokens=4, seed=6, router=router)
    x = (_rng(4).standard_normal((3, 128)) * gain).astype(np.float32)
    x[0, 64:96] *= 1e-5                                # blocks of their own size
    x[2] = 0.0
    l.check(x)


def test_strides_odd_addresses_and_optional_outputs(backend):
    l = Layer(backend, 5, 96, 64, 2, max_tokens=8, seed=7)
    x = _rng(9).standard_normal((4, 96)).astype(np.float32)
    want = l.run(x)[0]
    wide = np.full((4, 103), np.nan, np.float32)
    wide[:, 5:101] = x
    xb, y = backend.init_buffer(wide.ravel()), backend.init_buffer(np.full(4 * 99, 1.5, np.float32))
    l.layer.dispatch(backend, None, y.ptr + 4, xb.ptr + 20, 4, x_stride=103, y_stride=99)
    got = _read(backend, y).reshape(4, 99)
    # the router's sums are taken in another order at this alignment: within the weights' rounding of the same result
    assert (np.abs(got[:, 1:97] - want) <= 2.0 ** -18 * np.abs(want).max()).all()
    assert (got[:, 0] == 1.5).all() and (got[:, 97:] == 1.5).all()


def test_recorded_layer(backend):
    import torch
    stream = torch.cuda.Stream()
    with vb.Backend(0, stream=stream.cuda_stream) as b:
        l = Layer(b, 8, 256, 128, 2, max_tokens=4, seed=8)
        rng = _rng(10)
        x, y = b.uninit_buffer(3 * 256), b.uninit_buffer(3 * 256)
        b.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            l.layer.dispatch(b, None, y, x, 3)
        for _ in range(3):
            v = rng.standard_normal((3, 256)).astype(np.float32)
            b.write_buffer(x, 0, v.ravel())
            with torch.cuda.stream(stream):
                graph.replay()
            stream.synchronize()
            got = _read(b, y).reshape(3, 256)
            want, _, _, tol, _ = moe(v, l.router, l.gate, l.up, l.down, 2, True)
            assert (np.abs(got - want) <= tol).all()
        del graph
        l.layer.free()
        for m in l.mats:
            m.free()


def test_refusals(backend):
    m = lambda r, c, t=vb.Q4_0: vb.QuantizedMatrix.from_f32(backend, t, np.ones((r, c), np.float32))  # noqa: E731
    router = backend.init_buffer(np.zeros(4 * 64, np.float32))
    gate, up, down = m(4 * 32, 64), m(4 * 32, 64), m(4 * 64, 32)

    def status(*a, **kw):
        with pytest.raises(vb.VortxError) as e:
            vb.MoeLayer(backend, *a, **kw)
        return e.value.status
    assert status(router, gate, m(4 * 32, 64, vb.Q8_0), down, 4, 2) == _lib.VX_ERR_UNSUPPORTED
    assert status(router, gate, m(4 * 32, 32), down, 4, 2) == _lib.VX_ERR_SHAPE
    assert status(router, gate, up, m(4 * 32, 32), 4, 2) == _lib.VX_ERR_SHAPE
    assert status(router, gate, up, down, 3, 2) == _lib.VX_ERR_SHAPE
    assert status(router, gate, up, down, 4, 5) == _lib.VX_ERR_UNSUPPORTED
    assert status(router, gate, up, down, 4, 0) == _lib.VX_ERR_UNSUPPORTED
    assert status(router, gate, up, down, 4, 2, max_tokens=65) == _lib.VX_ERR_UNSUPPORTED
    assert status(router.ptr, gate, up, down, 257, 2) == _lib.VX_ERR_UNSUPPORTED
    with pytest.raises(IndexError):
        vb.MoeLayer(backend, backend.init_buffer(np.zeros(255, np.float32)), gate, up, down, 4, 2)
    backend.set_option("debug.fail_alloc_after", 1)
    assert status(router, gate, up, down, 4, 2) == _lib.VX_ERR_OUT_OF_MEMORY
    layer = vb.MoeLayer(backend, router, gate, up, down, 4, 2, max_tokens=2)
    x = backend.init_buffer(np.zeros(3 * 64, np.float32))
    y = backend.init_buffer(np.zeros(3 * 64, np.float32))
    with pytest.raises(vb.VortxError):
        layer.dispatch(backend, None, y, x, 3)
    with pytest.raises(IndexError):
        layer.dispatch(backend, None, backend.init_buffer(np.zeros(64, np.float32)), x, 2)
    with pytest.raises(IndexError):
        layer.dispatch(backend, None, y, x, 2, ids=backend.init_buffer(np.zeros(3, np.int32)))
    with pytest.raises(TypeError):
        layer.dispatch(backend, None, y, x, 2, ids=backend.init_buffer(np.zeros(4, np.float32)))
    with pytest.raises(vb.VortxError):
        layer.dispatch(backend, None, y.ptr, x.ptr, 2, x_stride=63)
    with vb.Backend(0) as other, pytest.raises(vb.VortxError):
        layer.dispatch(other, None, y, x, 1)
    before = backend.launch_count()
    layer.dispatch(backend, None, y, x, 0)
    assert backend.launch_count() == before

"""The expert layer next to inputs that stand out of their block: what a product is off by is measured against the sum of
|weight| |input| of its own row, not against the largest input or output of the call.

Tolerance.  That of decode_ref.moe, 2 * 2^-20 of sum |w||x| for a product, covers them: x is split into two f16 parts with the
largest of a block (or of a few together) in [2^14, 2^15), so every x keeps 22 bits down to 2^-16 of that and misses at most 2^-39
of it below; with a gain of up to 2^10, as here, an ordinary x keeps them.  Codes are exact, products are exact, and sums of
products rise no higher than sum |w||x| of the row."""
import numpy as np
import pytest

import vortx_b200 as vb
from decode_ref import moe, quantised

pytestmark = pytest.mark.gpu


def _rng(seed):
    return np.random.Generator(np.random.Philox(seed))


def _read(backend, buf):
    out = np.empty(buf.len(), buf.dtype)
    backend.slow_read_buffer(buf, out)
    return out


def _error(backend, x, router, gate, up, down, gt, dt, top_k):
    """Largest error of the layer's output next to its tolerance; gate, up [E, F, H], down [E, H, F] in f32."""
    mats = [vb.QuantizedMatrix.from_f32(backend, t, m.reshape(-1, m.shape[-1])) for t, m in ((gt, gate), (gt, up), (dt, down))]
    layer = vb.MoeLayer(backend, backend.init_buffer(router.ravel()), *mats, experts=len(gate), top_k=top_k, max_tokens=len(x))
    y = backend.uninit_buffer(x.size)
    layer.dispatch(backend, None, y, backend.init_buffer(x.ravel()), len(x))
    got = _read(backend, y).reshape(x.shape)
    want, _, _, tol, _ = moe(x, router, quantised(gt, gate), quantised(gt, up), quantised(dt, down), top_k, True)
    layer.free()
    for m in mats:
        m.free()
    return float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("gt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("gain", [30.0, 1000.0])
@pytest.mark.parametrize("hidden,tokens", [(512, 1), (512, 4), (512, 8), (160, 3)])
def test_inputs_that_stand_out_of_their_block(backend, gt, gain, hidden, tokens):
    """One input of every block is `gain` times the others, where the weights' codes are -1, 0 or 1.  The down product takes the
    result apart again: its row j has the inner value j alone."""
    rng = _rng(hidden + tokens)
    inner = hidden
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    w = [(rng.standard_normal((2, inner, hidden)) / np.sqrt(hidden)).astype(np.float32) for _ in range(2)]
    at = np.arange(hidden // 32) * 32 + rng.integers(0, 32, hidden // 32)
    x[:, at] *= np.float32(gain)
    for m in w:                                        # below one and a half of a code's step
        step = np.abs(m).reshape(2, inner, -1, 32).max(-1) / (127 if gt == vb.Q8_0 else 7)
        m[:, :, at] = (rng.integers(-1, 2, m[:, :, at].shape) * step).astype(np.float32)
    down = np.zeros((2, hidden, inner), np.float32)
    down[:, np.arange(hidden), np.arange(inner)] = 1.0
    router = (rng.standard_normal((2, hidden)) * 1e-3 / gain).astype(np.float32)
    assert _error(backend, x, router, *w, down, gt, vb.Q8_0, 2) <= 1.0


@pytest.mark.parametrize("dt", [vb.Q8_0, vb.Q4_0])
@pytest.mark.parametrize("gain", [30.0, 1000.0])
@pytest.mark.parametrize("inner,tokens", [(512, 1), (512, 4), (512, 7), (96, 2)])
def test_inner_values_that_stand_out_of_their_block(backend, dt, gain, inner, tokens):
    """The same for the down product: a row of `up` that is `gain` times the others makes the inner value, and no code of `down`
    takes it (its own rounding in the first product would be allowed for otherwise)."""
    rng = _rng(inner + tokens)
    hidden = 64
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    w = [(rng.standard_normal((2, inner, hidden)) / np.sqrt(hidden)).astype(np.float32) for _ in range(2)]
    at = np.arange(inner // 32) * 32 + rng.integers(0, 32, inner // 32)
    w[1][:, at] *= np.float32(gain)
    down = (rng.standard_normal((2, hidden, inner)) / np.sqrt(inner)).astype(np.float32)
    down[:, :, at] = 0.0
    router = (rng.standard_normal((2, hidden)) * 1e-2).astype(np.float32)
    assert _error(backend, x, router, *w, down, vb.Q8_0, dt, 2) <= 1.0

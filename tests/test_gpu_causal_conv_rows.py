"""The causal convolution and its gradients where a thread goes through 16 or 32 rows of a chunk, as in training on long sequences, against plain forms in 64 bits in some of the channels."""
import numpy as np
import pytest

import sequence_reference as ref

pytestmark = pytest.mark.gpu

LENGTH, CHANNELS = 1100, 4102  # rows that no chunk divides, channels that no piece of 4 or 8 does


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


@pytest.fixture(scope='module')
def inputs():
    rng = np.random.default_rng(0)
    wide = {k: rng.standard_normal((1, LENGTH, CHANNELS), dtype=np.float32) for k in ('x', 'gy')}
    return {dtype: {k: v.astype(dtype) for k, v in wide.items()} for dtype in ('float16', 'float32')}


def chunk_rows(length, lines, units):
    rows = 32
    while rows > 8 and lines * -(-length // rows) < units * 1024:
        rows //= 2
    return rows


def device_units():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('taps', [1, 2, 4, 5, 6, 8])
@pytest.mark.parametrize('batch,rows', [(16, 32), (5, 16)])
def test_causal_conv_of_long_chunks(chx, inputs, batch, rows, taps, dtype):
    """The sequences are the same numbers, read with a stride of 0, and end in other places."""
    units = device_units()
    assert chunk_rows(LENGTH, batch * -(-CHANNELS // 4), units) == rows  # the gradients; the forward call has as many rows in float32, and as few as half of them in float16
    assert chunk_rows(LENGTH, batch * -(-CHANNELS // (8 if dtype == 'float16' else 4)), units) >= rows // 2
    rng = np.random.default_rng(taps)
    one = inputs[dtype]
    n = lambda *s: rng.standard_normal(s).astype(dtype)  # noqa: E731
    w, b, state, gnew = n(CHANNELS, taps), n(CHANNELS), n(batch, taps - 1, CHANNELS), n(batch, taps - 1, CHANNELS)
    lengths = rng.integers(0, LENGTH + 1, batch).astype(np.int32)
    lengths[:4] = [LENGTH, 0, 3, 32 * 20 + 5]
    some = np.array([0, 1, 3, 4, 7, 8, 2051, 4092, 4095, 4096, 4097, 4098, 4099, 4100, 4101])  # of the first, an inner and the last pieces, which overlap
    shape = (batch, LENGTH, CHANNELS)
    x, gy = (chx.array(one[k]).broadcast_to(shape) for k in ('x', 'gy'))
    for activation, ends in (('silu', lengths), (None, None)):
        args = [x, chx.array(w), chx.array(b)]
        more = dict(state=chx.array(state), lengths=None if ends is None else chx.array(ends), activation=activation)
        y, new = chx.causal_conv(*args, **more)
        gx, gw, gb, gstate = chx.causal_conv_grad(*args, gy, gnew_state=chx.array(gnew), **more)
        few = dict(x=np.broadcast_to(one['x'][..., some], shape[:2] + some.shape), w=w[some], b=b[some])
        want, size, want_new = ref.causal_conv(**few, state=state[..., some], lengths=ends, activation=activation)
        ref.assert_within(y.get()[..., some], want, size, 1, 'y')
        assert np.array_equal(new.get()[..., some], want_new.astype(dtype))
        wants, sizes = ref.causal_conv_grad(**few, gy=np.broadcast_to(one['gy'][..., some], shape[:2] + some.shape), state=state[..., some], lengths=ends, activation=activation,
                                            gnew=gnew[..., some])
        for name, got, want, size in (('gx', gx.get()[..., some], wants[0], sizes[0]), ('gw', gw.get()[some], wants[1], sizes[1]), ('gb', gb.get()[some], wants[2], sizes[2]),
                                      ('gstate', gstate.get()[..., some], wants[3], sizes[3])):
            ref.assert_within(got, want, size, 1, '%s %s %s' % (name, taps, activation))
            if got.size:
                got, rounding = got.astype(np.float64), 2.0 ** -11 if dtype == 'float16' else 0
                assert np.linalg.norm(got - want) <= (1e-5 + rounding) * np.linalg.norm(want), name  # 168 roundings of 2^-24, and float16's own

"""Layer norm of arrays whose rows repeat, as the gradient of a sum or a mean over time does."""
import numpy as np
import pytest

import block_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


# the shape of what is there, and the one that it is broadcast to
BROADCAST = [((3, 1, 5), (3, 4, 5)), ((1, 4, 5), (3, 4, 5)), ((1, 1, 5), (3, 4, 5)), ((5, 1, 650), (5, 35, 650)), ((1, 35, 650), (5, 35, 650)), ((2, 1, 3, 70), (2, 4, 3, 70)), ((2, 3, 1, 70), (2, 3, 4, 70)),
             ((2, 1, 1, 70), (2, 3, 4, 70)), ((3, 4, 1), (3, 4, 6)), ((6, 1, 1), (6, 7, 9)), ((3, 1, 20001), (3, 2, 20001)), ((40, 1, 4096), (40, 100, 4096))]


@pytest.mark.parametrize('dtype', ['float16', 'float32', 'float64'])
@pytest.mark.parametrize('there,shape', BROADCAST)
def test_layer_norm_of_broadcast_arrays(chx, there, shape, dtype):
    """x, gy and both as views that repeat give what their copies give, bit for bit, and those are right."""
    rng = np.random.default_rng(1)
    params = 'float64' if dtype == 'float64' else 'float32'
    gamma, beta = (chx.array(rng.standard_normal(shape[-1]).astype(params)) for _ in range(2))
    x, gy = (rng.standard_normal(shape).astype(dtype) for _ in range(2))
    few_x, few_gy = (rng.standard_normal(there).astype(dtype) for _ in range(2))
    views = [chx.array(a).broadcast_to(shape) for a in (few_x, few_gy)]
    copies = [np.ascontiguousarray(np.broadcast_to(a, shape)) for a in (few_x, few_gy)]
    for broadcast_x, broadcast_gy in ((True, False), (False, True), (True, True)):
        a, b = (views[0] if broadcast_x else chx.array(x)), (views[1] if broadcast_gy else chx.array(gy))
        c, d = copies[0] if broadcast_x else x, copies[1] if broadcast_gy else gy
        y, state = chx.layer_norm(a, gamma, beta)
        want, want_state = chx.layer_norm(chx.array(c), gamma, beta)
        assert y.shape == shape
        for got, w in zip((y, state.mean, state.inv_std), (want, want_state.mean, want_state.inv_std)):
            assert np.array_equal(got.get(), w.get())
        for got, w in zip(chx.layer_norm_grad(a, gamma, b, state), chx.layer_norm_grad(chx.array(c), gamma, chx.array(d), want_state)):
            assert np.array_equal(got.get(), w.get())
        exact, off = ref.layer_norm(c, gamma.get(), beta.get(), 2e-5, 2.0 ** -53 if dtype == 'float64' else 2.0 ** -24)
        if dtype == 'float64':  # whose plain form needs more bits than the kernel: a mean of six equal numbers, rounded, leaves 2^-53 of them, which 1 / sqrt(eps) makes 224 times as much
            wide = c.astype(np.longdouble)
            d = wide - wide.mean(-1, keepdims=True)
            exact['y'] = (d / np.sqrt((d * d).mean(-1, keepdims=True) + np.longdouble(2e-5)) * gamma.get() + beta.get()).astype(np.float64)
        ref.assert_off(y.get(), exact['y'], off['y'], '%s to %s %s' % (there, shape, dtype))

"""States that are infinite, or zeros that grow, where the selective scan cuts the time axis into chunks: a chunk's decay may leave float32's range though no row's does."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


def run(chx, c):
    return [v.get() for v in chx.selective_scan(**{k: chx.array(v) for k, v in c.items()})]


def plain(length, channels, states, seed=0):
    rng = np.random.default_rng(seed)
    f = lambda *s: (np.abs(rng.standard_normal(s)) + 0.1).astype(np.float32)  # noqa: E731
    return {'u': f(1, length, channels), 'delta': np.full((1, length, channels), 2, np.float32), 'a': np.full((channels, states), -1, np.float32), 'b': f(1, length, states),
            'c': f(1, length, states), 'd': f(channels), 'state': f(1, channels, states)}


@pytest.mark.parametrize('states', [1, 5, 16, 64])
@pytest.mark.parametrize('length', [40, 300, 1500])
def test_an_infinite_state_stays_infinite(chx, length, states):
    """Decays of exp(-2) a row, exp(-96) and less a chunk: an infinite state is as infinite as before, of whatever sequence came before or of an infinite input."""
    c = plain(length, 7, states)
    c['state'][0, 3] = np.inf
    c['u'][0, 5, 4] = np.inf
    y, new = run(chx, c)
    assert np.isposinf(y[0, :, 3]).all() and np.isposinf(y[0, 5:, 4]).all() and np.isposinf(new[0, 3:5]).all()
    others = [0, 1, 2, 5, 6]
    assert np.isfinite(y[..., others]).all() and np.isfinite(y[0, :5, 4]).all() and np.isfinite(new[0, others]).all()


@pytest.mark.parametrize('states', [1, 5, 16, 64])
@pytest.mark.parametrize('length', [40, 300, 1500])
def test_a_state_that_grows_out_of_zeros(chx, length, states):
    """Growth of exp(2) a row, exp(96) and more a chunk, of nothing until ten rows before the end."""
    c = plain(length, 7, states)
    c['a'][:] = 1
    c['state'][:] = 0
    c['u'][:, :length - 10] = 0
    y, new = run(chx, c)
    h, wants = np.zeros((7, states)), []
    for t in range(length):
        h = h * np.exp(2.0) + 2.0 * c['u'][0, t].astype(np.float64)[:, None] * c['b'][0, t]
        wants.append((h * c['c'][0, t]).sum(1) + c['d'].astype(np.float64) * c['u'][0, t])
    # ten rows and a sum over states and d u of positive numbers: a row rounds its product, its sum and dt u b, and its exponential, of an argument of 2, is off by 2 + 3 * 2 half steps
    limit = (10 * 12 + states + 1) * 2.0 ** -24
    np.testing.assert_allclose(y[0], np.array(wants), rtol=limit, atol=0)
    np.testing.assert_allclose(new[0], h, rtol=limit, atol=0)


def test_a_small_state_that_grows(chx):
    """A state of 1e-30 that a chunk makes exp(96) times as large: neither it nor what comes of it is out of range."""
    c = plain(300, 7, 16)
    c['a'][:] = 1
    c['delta'][:, :48] = c['delta'][:, 96:] = 0
    c['state'][:] = 1e-30
    c['u'][:] = 0
    _, new = run(chx, c)
    exact = np.exp(96.0) * np.float64(np.float32(1e-30))
    # 48 rows of products and exponentials; or sums of steps, exact here, and an exponential of 96: 2 + 3 * 96 half steps
    np.testing.assert_allclose(new, np.full(new.shape, exact), rtol=(48 * 12 + 290) * 2.0 ** -24, atol=0)

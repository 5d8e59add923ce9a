"""Infinite inputs and states of the selective scan: sequences at once give what they give token by token, and what the definition gives."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


def case(batch, length, channels, states, dtype, seed=0):
    """Products of one sign, so that an infinite state gives an infinite sum over the states."""
    rng = np.random.default_rng(seed)
    n = lambda *s: (np.abs(rng.standard_normal(s)) + 0.1).astype(dtype)  # noqa: E731
    f = lambda *s: (np.abs(rng.standard_normal(s)) + 0.1).astype(np.float32)  # noqa: E731
    return {'u': n(batch, length, channels), 'delta': n(batch, length, channels), 'a': -f(channels, states), 'b': n(batch, length, states), 'c': n(batch, length, states),
            'd': f(channels), 'z': n(batch, length, channels), 'state': f(batch, channels, states)}


def on_device(chx, c):
    return {k: chx.array(v) for k, v in c.items()}


def by_tokens(chx, c):
    """Outputs row by row, with the state that each row leaves."""
    state, ys = chx.array(c['state']), []
    dev = on_device(chx, c)
    for t in range(c['u'].shape[1]):
        y, state = chx.selective_scan(**dict(dev, state=state, **{k: dev[k][:, t:t + 1] for k in ('u', 'delta', 'b', 'c', 'z')}))
        ys.append(y.get())
    return np.concatenate(ys, 1), state.get()


def assert_same_kinds(got, want, what):
    for kind in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(kind(got), kind(want)), '%s: %s' % (what, kind.__name__)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [40, 300])
@pytest.mark.parametrize('states', [1, 3, 5, 12, 16, 24, 33, 64])
def test_infinite_inputs(chx, states, length, dtype):
    """Channels whose u, or whose step, is infinite in one row: that row and those behind it are infinite, the others are as they were."""
    c = case(2, length, 21, states, dtype)
    row = length // 2 + 3
    c['a'] /= 4  # no decay of a row, or of a chunk, becomes 0 (the steps of 48 rows add up to 45)
    c['u'][0, row, 2] = c['delta'][0, row, 7] = c['u'][1, row, 20] = np.inf
    finite = dict(c, **{k: np.where(np.isinf(c[k]), 1, c[k]).astype(dtype) for k in ('u', 'delta')})
    finite = chx.selective_scan(**on_device(chx, finite))[0].get()
    y, new = (v.get() for v in chx.selective_scan(**on_device(chx, c)))
    want = np.zeros(y.shape, bool)
    for b, channel in ((0, 2), (0, 7), (1, 20)):
        want[b, row:, channel] = True
    assert np.array_equal(np.isposinf(y), want) and not np.isnan(y).any()
    assert np.array_equal(y[~want], finite[~want])
    assert np.array_equal(np.isposinf(new), np.broadcast_to(want[:, -1, :, None], new.shape)) and not np.isnan(new).any()
    token_y, token_new = by_tokens(chx, c)
    assert_same_kinds(y, token_y, 'tokens')
    assert_same_kinds(new, token_new, 'state of tokens')


@pytest.mark.parametrize('length', [1, 40, 300])
@pytest.mark.parametrize('states', [1, 5, 16])
def test_infinite_inputs_without_a_skip(chx, states, length):
    """Without `d` an infinite u counts by its states alone."""
    c = case(1, length, 21, states, 'float32', seed=3)
    c['a'] /= 4
    del c['d']
    row = length // 2
    c['u'][0, row, 2] = np.inf
    y, new = (v.get() for v in chx.selective_scan(**on_device(chx, c)))
    want = np.zeros(y.shape, bool)
    want[0, row:, 2] = True
    assert np.array_equal(np.isposinf(y), want) and not np.isnan(y).any()
    token_y, token_new = by_tokens(chx, c)
    assert_same_kinds(y, token_y, 'tokens')
    assert_same_kinds(new, token_new, 'state of tokens')


@pytest.mark.parametrize('states', [1, 5, 16, 24])
def test_infinite_inputs_leave_the_gradients_before_them(chx, states):
    length, row = 300, 150
    c = case(1, length, 21, states, 'float32', seed=4)
    c['a'] /= 4
    gy = np.random.default_rng(5).standard_normal(c['u'].shape).astype(np.float32)
    want = chx.selective_scan_grad(gy=chx.array(gy), **on_device(chx, c))
    c['u'][0, row, 7] = np.inf
    got = chx.selective_scan_grad(gy=chx.array(gy), **on_device(chx, c))
    others = np.arange(21) != 7
    for k in ('u', 'delta', 'z'):
        a, b = getattr(got, k).get(), getattr(want, k).get()
        assert np.array_equal(a[:, :row], b[:, :row]) and np.array_equal(a[..., others], b[..., others]) and np.isfinite(b).all(), k
    for k in ('b', 'c'):
        a, b = getattr(got, k).get(), getattr(want, k).get()
        assert np.array_equal(a[:, :row], b[:, :row]), k
    assert np.array_equal(got.u.get(), want.u.get())  # of which the states are no part
    assert np.array_equal(got.state.get(), want.state.get())
    for k in ('a', 'd', 'delta_bias'):
        a, b = getattr(got, k), getattr(want, k)
        assert (a is None) == (b is None) and (a is None or np.array_equal(a.get()[others], b.get()[others])), k


@pytest.mark.parametrize('states', [1, 5, 16, 24])
def test_infinite_steps_leave_the_gradients_before_them(chx, states):
    """Behind a step without end nothing is left of the state, so that it takes no part in the gradients of the rows before: those are the gradients without it."""
    length, row = 90, 50
    c = case(1, length, 21, states, 'float32', seed=1)
    gy = np.random.default_rng(2).standard_normal(c['u'].shape).astype(np.float32)
    far = dict(c, delta=c['delta'].copy())
    far['delta'][0, row, 7] = 1e30  # forgets everything too: exp(-1e30 |a|) is 0
    c['delta'][0, row, 7] = np.inf
    got, want = (chx.selective_scan_grad(gy=chx.array(gy), **on_device(chx, v)) for v in (c, far))
    for k in ('u', 'delta', 'z'):
        a, b = getattr(got, k).get(), getattr(want, k).get()
        assert np.isfinite(a[:, :row]).all() and np.array_equal(a[:, :row], b[:, :row]), k
        others = np.arange(21) != 7
        assert np.isfinite(a[..., others]).all() and np.array_equal(a[..., others], b[..., others]), k
    for k in ('b', 'c'):
        a, b = getattr(got, k).get(), getattr(want, k).get()
        assert np.isfinite(a[:, :row]).all() and np.array_equal(a[:, :row], b[:, :row]), k
    assert np.isfinite(got.state.get()).all() and np.array_equal(got.state.get(), want.state.get())

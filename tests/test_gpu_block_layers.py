"""Layer norm, linear attention and AdamW on the device against plain forms (block_reference.py)."""
import numpy as np
import pytest

import block_reference as ref
import sequence_reference as seq

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


def up(chx, a):
    return None if a is None else chx.array(a)


def apart(chx, a, extra=3):
    """`a` on the device as a part of wider rows, whose other elements are NaN."""
    wide = np.full(a.shape[:-1] + (a.shape[-1] + extra,), np.nan, a.dtype)
    wide[..., 1:1 + a.shape[-1]] = a
    return chx.array(wide)[..., 1:1 + a.shape[-1]]


# ---------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------
NORMS = [(1, 1), (3, 2), (5, 7), (4, 8), (129, 9), (20, 64), (33, 127), (7, 128), (5, 250), (1000, 33), (6, 512), (257, 650), (3, 1023), (9, 2048), (70, 3333), (2, 4096), (3, 8200), (2, 16384),
         (5, 20001), (2, 32769), (3, 70001)]


def norm_case(rows, cols, dtype, params, seed=0):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal(cols)) + 0.5 * rng.standard_normal(cols)).astype(dtype)
    return x, (1 + 0.1 * rng.standard_normal(cols)).astype(params), (0.1 * rng.standard_normal(cols)).astype(params), rng.standard_normal((rows, cols)).astype(dtype)


@pytest.mark.parametrize('dtype,params', [('float16', 'float16'), ('float16', 'float32'), ('float32', 'float32'), ('float64', 'float64')])
@pytest.mark.parametrize('rows,cols', NORMS)
def test_layer_norm(chx, rows, cols, dtype, params):
    u = 2.0 ** -53 if dtype == 'float64' else seq.U32
    for i, (with_gamma, with_beta, wide) in enumerate(((True, True, False), (True, True, True), (False, True, False), (True, False, True), (False, False, False))):
        x, gamma, beta, gy = norm_case(rows, cols, dtype, params, seed=i)
        gamma, beta = gamma if with_gamma else None, beta if with_beta else None
        place = (lambda a: apart(chx, a)) if wide else (lambda a: up(chx, a))
        what = '%d x %d %s %s %d' % (rows, cols, dtype, params, i)
        y, state = chx.layer_norm(place(x), up(chx, gamma), up(chx, beta))
        want, off = ref.layer_norm(x, gamma, beta, 2e-5, u)
        assert state.mean.dtype == state.inv_std.dtype == (np.float64 if dtype == 'float64' else np.float32) and y.dtype == x.dtype
        for name, got in (('y', y), ('mean', state.mean), ('inv_std', state.inv_std)):
            ref.assert_off(got.get(), want[name], off[name], what + ' ' + name)
        grads = chx.layer_norm_grad(place(x), up(chx, gamma), place(gy), state)
        want, off = ref.layer_norm_grad(x, gamma, gy, 2e-5, u)
        assert (grads[1] is None) == (gamma is None) and (grads[2] is None) == (beta is None)
        for name, got in zip(('gx', 'ggamma', 'gbeta'), grads):
            if got is not None:
                ref.assert_off(got.get(), want[name].reshape(got.shape), off[name].reshape(got.shape), what + ' ' + name)
                assert got.dtype == (x.dtype if name == 'gx' else np.dtype(params))


@pytest.mark.parametrize('rows,cols,dtype', [(132000, 3, 'float16'), (132001, 40, 'float32'), (33003, 300, 'float16'), (33001, 250, 'float32'), (17001, 600, 'float16'), (4101, 2500, 'float16'),
                                             (4097, 1700, 'float32'), (2050, 5000, 'float16')])
def test_layer_norm_of_many_rows(chx, rows, cols, dtype):
    """So many that a thread takes several at once, the last ones not all there."""
    x, gamma, beta, gy = norm_case(rows, cols, dtype, 'float32')
    y, state = chx.layer_norm(up(chx, x), up(chx, gamma), up(chx, beta))
    want, off = ref.layer_norm(x, gamma, beta, 2e-5)
    for name, got in (('y', y), ('mean', state.mean), ('inv_std', state.inv_std)):
        ref.assert_off(got.get(), want[name], off[name], name)
    grads = chx.layer_norm_grad(up(chx, x), up(chx, gamma), up(chx, gy), state)
    want, off = ref.layer_norm_grad(x, gamma, gy, 2e-5)
    for name, got in zip(('gx', 'ggamma', 'gbeta'), grads):
        ref.assert_off(got.get(), want[name].reshape(got.shape), off[name].reshape(got.shape), name)


def test_layer_norm_of_many_axes_and_of_none(chx):
    x, gamma, beta, gy = norm_case(24, 40, 'float32', 'float32')
    want, state = chx.layer_norm(up(chx, x), up(chx, gamma), up(chx, beta))
    got, state4 = chx.layer_norm(up(chx, x.reshape(2, 3, 4, 40)), up(chx, gamma), up(chx, beta))
    assert got.shape == (2, 3, 4, 40) and state4.mean.shape == (2, 3, 4) and np.array_equal(got.get().reshape(24, 40), want.get())
    turned = chx.array(np.ascontiguousarray(x.reshape(4, 6, 40).transpose(1, 0, 2))).transpose(1, 0, 2)  # rows in no even order: copied
    assert np.array_equal(chx.layer_norm(turned, up(chx, gamma), up(chx, beta))[0].get().reshape(24, 40), want.get())
    columns = chx.array(np.ascontiguousarray(x.T)).T
    assert np.array_equal(chx.layer_norm(columns, up(chx, gamma), up(chx, beta))[0].get(), want.get())
    one, state1 = chx.layer_norm(up(chx, x[3]), up(chx, gamma), up(chx, beta))
    assert state1.mean.shape == () and np.array_equal(one.get(), want.get()[3])
    gx = chx.layer_norm_grad(up(chx, x.reshape(2, 3, 4, 40)), up(chx, gamma), up(chx, gy.reshape(2, 3, 4, 40)), state4)[0]
    assert np.array_equal(gx.get().reshape(24, 40), chx.layer_norm_grad(up(chx, x), up(chx, gamma), up(chx, gy), state)[0].get())
    none, state0 = chx.layer_norm(chx.zeros((0, 7)), chx.ones((7,)), chx.zeros((7,)))
    assert none.shape == (0, 7)
    gx, ggamma, gbeta = chx.layer_norm_grad(chx.zeros((0, 7)), chx.ones((7,)), chx.zeros((0, 7)), state0)
    assert gx.shape == (0, 7) and not ggamma.get().any() and not gbeta.get().any()
    with pytest.raises(chx.DimensionError):
        chx.layer_norm(chx.zeros((3, 0)))


def test_layer_norm_of_rows_far_from_zero_and_of_constant_ones(chx):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((40, 333)) + 1000 * rng.standard_normal((40, 1))).astype(np.float32)
    x[7] = 5.25
    x[8] = 3e4 + 1e-3 * np.arange(333)
    (y, state), (want, off) = chx.layer_norm(up(chx, x)), ref.layer_norm(x, None, None, 2e-5)
    ref.assert_off(y.get(), want['y'], off['y'], 'y')
    ref.assert_off(state.inv_std.get(), want['inv_std'], off['inv_std'], 'inv_std')
    assert not y.get()[7].any()
    x[9, 5], x[10, 300], x[11, 0] = np.nan, np.inf, -np.inf
    with_nan = chx.layer_norm(up(chx, x))[0].get()
    assert np.isnan(with_nan[9:12]).all() and np.array_equal(np.delete(with_nan, [9, 10, 11], 0), np.delete(y.get(), [9, 10, 11], 0))


@pytest.mark.parametrize('cols', [64, 900, 4096, 40000])
def test_layer_norm_means_of_float16_are_those_of_its_values(chx, cols):
    """Differences from a mean with more bits than the values would all be rounded alike, and the mean of 4096 values off by up to 6e-8.

    Exact ones of variance 1 leave what their sum loses: an addition rounds by at most 2^-25 of its result where that is a power of two, by 2^-24 of it at most, with a deviation of half of that.
    m <= 40 terms one after another in a thread have results of order sqrt(m) at most, and the levels of the tree behind, ten at most, cols / (m 2^l) results of order sqrt(m 2^l):
    together a deviation of 2^-25 sqrt(cols (m + 10)), so that six of them are below 2^-19.5 sqrt(cols), and cols times less in the mean.  The division and the last addition round the mean."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((50, cols)).astype(np.float16)
    _, state = chx.layer_norm(up(chx, x))
    want = x.astype(np.float64).mean(1)
    assert (np.abs(state.mean.get() - want) <= 2.0 ** -19.5 / cols ** 0.5 + 2.0 ** -23 * np.abs(want)).all()


@pytest.mark.parametrize('rows,cols,dtype', [(20003, 64, 'float16'), (9001, 600, 'float16'), (4099, 2500, 'float16'), (300, 5, 'float32'), (3, 20001, 'float32')])
def test_layer_norm_keeps_to_the_row(chx, rows, cols, dtype):
    """A row with an infinity or NaN is NaN; those that are taken with it are as without it."""
    x, gamma, beta, gy = norm_case(rows, cols, dtype, dtype)
    args = [up(chx, a) for a in (gamma, beta)]
    y, state = chx.layer_norm(up(chx, x), *args)
    gx = chx.layer_norm_grad(up(chx, x), args[0], up(chx, gy), state)[0].get()
    bad = x.copy()
    touched = [0, rows // 2, rows - 1] if rows > 3 else [1]
    for n, row in enumerate(touched):
        bad[row, n * 7 % cols] = (np.inf, np.nan, -np.inf)[n]
    y2, state2 = chx.layer_norm(up(chx, bad), *args)
    gx2 = chx.layer_norm_grad(up(chx, bad), args[0], up(chx, gy), state2)[0].get()
    others = np.setdiff1d(np.arange(rows), touched)
    for got, want in ((y2.get(), y.get()), (state2.mean.get(), state.mean.get()), (state2.inv_std.get(), state.inv_std.get()), (gx2, gx)):
        assert np.array_equal(got[others], want[others])
    assert np.isnan(y2.get()[touched]).all() and np.isnan(gx2[touched]).all()


@pytest.mark.parametrize('rows,cols,dtype', [(40, 5, 'float16'), (9, 70, 'float32'), (20001, 100, 'float16'), (4099, 2500, 'float16'), (7, 4100, 'float32'), (3, 40000, 'float16')])
def test_layer_norm_in_place(chx, rows, cols, dtype):
    """y may be x, for which the routine has no argument: the entry itself."""
    x, gamma, beta, _ = norm_case(rows, cols, dtype, 'float32')
    want, state = chx.layer_norm(up(chx, x), up(chx, gamma), up(chx, beta))
    a, g, b, mean, inv = up(chx, x), up(chx, gamma), up(chx, beta), chx.zeros((rows,)), chx.zeros((rows,))
    chx._lib.call('hipcx_layer_norm', a.desc(), g.desc(), b.desc(), 2e-5, a.desc(), mean.desc(), inv.desc(), None)
    chx.synchronize()
    for got, w in ((a, want), (mean, state.mean), (inv, state.inv_std)):
        assert np.array_equal(got.get(), w.get())


def test_layer_norm_gradients_against_differences(chx):
    """In float64: central differences of sum(y * gy), whose error is h^2 / 6 of the third derivative (of order 1 here) and 2^-53 of the sum (of order 20) over h."""
    x, gamma, beta, gy = norm_case(3, 11, 'float64', 'float64')
    grads = [g.get() for g in chx.layer_norm_grad(up(chx, x), up(chx, gamma), up(chx, gy), chx.layer_norm(up(chx, x), up(chx, gamma), up(chx, beta))[1])]
    h = 1e-5
    for a, grad in zip((x, gamma, beta), grads):
        flat = a.reshape(-1)
        for i in range(flat.size):
            was, sums = flat[i], []
            for s in (h, -h):
                flat[i] = was + s
                sums.append((chx.layer_norm(up(chx, x), up(chx, gamma), up(chx, beta))[0].get() * gy).sum())
            flat[i] = was
            assert abs((sums[0] - sums[1]) / (2 * h) - grad.reshape(-1)[i]) < 1e-7


# ---------------------------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------------------------
# batch, length, heads, share, keys, values
ATTENDS = [(1, 1, 1, 1, 1, 1), (2, 1, 3, 1, 50, 50), (1, 8, 2, 1, 64, 64), (2, 9, 2, 2, 5, 3), (1, 63, 1, 1, 16, 80), (3, 64, 2, 1, 33, 65), (2, 65, 4, 4, 64, 128), (1, 200, 2, 1, 128, 128),
           (2, 130, 2, 2, 100, 31), (1, 70, 1, 1, 256, 200), (1, 66, 1, 1, 130, 256), (1, 600, 3, 1, 50, 50), (1, 1100, 1, 1, 32, 64)]


def attend_case(sizes, dtype, seed=0, ragged=False, decay='rows', strong=False):
    batch, length, heads, share, keys, values = sizes
    rng = np.random.default_rng(seed)
    n = lambda *s: rng.standard_normal(s).astype(dtype)  # noqa: E731
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    c = {'q': n(batch, length, heads // share, keys), 'k': n(batch, length, heads // share, keys), 'v': n(batch, length, heads, values), 'gy': n(batch, length, heads, values),
         'state': f(batch, heads, keys, values), 'gnew': f(batch, heads, keys, values), 'lengths': None, 'log_decay': None}
    if decay == 'rows':
        c['log_decay'] = -np.exp(1.5 * f(batch, length, heads) - (0 if strong else 3))
    elif decay == 'heads':
        c['log_decay'] = np.log1p(-np.exp2(-3 - np.arange(heads, dtype=np.float32) % 8))
    if ragged:
        c['lengths'] = rng.integers(-1, length + 3, batch).astype(np.int32 if seed % 2 else np.int64)
        c['lengths'][batch // 2] = 0
        behind = ~seq.inside(seq.ends_of(c['lengths'], batch, length), length)[..., 0]
        for k in ('q', 'k', 'v', 'gy') + (('log_decay',) if decay == 'rows' else ()):
            c[k][behind] = np.nan
    return c


def check_attend(chx, c, place, scale, state, gnew, what):
    s, g = c['state'] if state else None, c['gnew'] if gnew else None
    args, more = [place(c[k]) for k in ('q', 'k', 'v')], dict(log_decay=up(chx, c['log_decay']), scale=scale, state=up(chx, s), lengths=up(chx, c['lengths']))
    y, new = chx.linear_attention(*args, **more)
    (want, want_new), (off, off_new) = ref.linear_attention(c['q'], c['k'], c['v'], c['log_decay'], scale, s, c['lengths'])
    ref.assert_off(y.get(), want, off, what + ' y')
    ref.assert_off(new.get(), want_new, off_new, what + ' state')
    grads = chx.linear_attention_grad(*args, place(c['gy']), gnew_state=up(chx, g), **more)
    wants, offs, n = ref.linear_attention_grad(c['q'], c['k'], c['v'], c['gy'], c['log_decay'], scale, s, c['lengths'], g)
    assert (grads.log_decay is None) == (c['log_decay'] is None) and (grads.state is None) == (s is None)
    for name, got in grads._asdict().items():
        if got is not None:
            ref.assert_off(got.get(), wants[name], offs[name], '%s g%s' % (what, name))
            # together: terms pass through some hundreds of roundings of either sign, which add up like their squares.  A log decay's gradient is a difference of sums that is exactly zero where
            # there is nothing that decays, so that its error is one of those sums', whose absolute values' 2-norm is offs / (n U)
            norm = np.linalg.norm(wants[name] if name != 'log_decay' else offs[name] / (n * seq.U32))
            assert np.linalg.norm(got.get() - wants[name]) <= (1e-5 + np.finfo(got.dtype).eps / 2) * norm, '%s g%s' % (what, name)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', ATTENDS)
def test_linear_attention(chx, sizes, dtype):
    for i, (decay, ragged, state, gnew, wide, scale) in enumerate((('rows', False, True, True, False, None), ('heads', True, True, False, True, 0.3), (None, False, False, True, False, 1.0),
                                                                   ('rows', True, False, False, True, None))):
        c = attend_case(sizes, dtype, seed=i, ragged=ragged, decay=decay, strong=i == 3)
        check_attend(chx, c, (lambda a: apart(chx, a)) if wide else (lambda a: up(chx, a)), scale, state, gnew, '%s %s %d' % (sizes, dtype, i))


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_linear_attention_of_views(chx, dtype):
    """Parts of one projection, sequences and heads in other orders, decays with strides and broadcast ones."""
    c = attend_case((2, 90, 4, 2, 24, 40), dtype)
    b, l = 2, 90
    wide = chx.array(np.concatenate([c['q'].reshape(b, l, -1), c['k'].reshape(b, l, -1), c['v'].reshape(b, l, -1)], 2))
    q, k, v = wide[:, :, :48].reshape(b, l, 2, 24), wide[:, :, 48:96].reshape(b, l, 2, 24), wide[:, :, 96:].reshape(b, l, 4, 40)
    decay, state = up(chx, c['log_decay']), up(chx, c['state'])
    y, new = chx.linear_attention(up(chx, c['q']), up(chx, c['k']), up(chx, c['v']), decay, state=state)
    for got, want in zip(chx.linear_attention(q, k, v, decay, state=state), (y, new)):
        assert np.array_equal(got.get(), want.get())
    turned = [chx.array(np.ascontiguousarray(c[n].transpose(2, 1, 0, 3))).transpose(2, 1, 0, 3) for n in ('q', 'k', 'v')]
    of_rows = chx.array(np.ascontiguousarray(c['log_decay'].transpose(2, 0, 1))).transpose(1, 2, 0)
    for got, want in zip(chx.linear_attention(*turned, of_rows, state=state), (y, new)):
        assert np.array_equal(got.get(), want.get())
    grads = chx.linear_attention_grad(up(chx, c['q']), up(chx, c['k']), up(chx, c['v']), up(chx, c['gy']), decay, state=state)
    for got, want in zip(chx.linear_attention_grad(*turned, up(chx, c['gy']), of_rows, state=state), grads):
        assert np.array_equal(got.get(), want.get())


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('keys,values', [(50, 50), (128, 64), (7, 100)])
def test_linear_attention_in_pieces_and_tokens(chx, keys, values, dtype):
    """Pieces of a sequence, the state moved forward in place, are the sequence at once."""
    c = attend_case((3, 150, 2, 1, keys, values), dtype)
    (want, want_new), (off, off_new) = ref.linear_attention(c['q'], c['k'], c['v'], c['log_decay'], None, c['state'])
    state, at = up(chx, c['state']), 0
    for n in (1, 1, 64, 3, 8, 70, 1, 2):
        piece = slice(at, at + n)
        y, same = chx.linear_attention(*(up(chx, c[k][:, piece]) for k in ('q', 'k', 'v')), up(chx, c['log_decay'][:, piece]), state=state, out_state=state)
        assert same is state
        ref.assert_off(y.get(), want[:, piece], off[:, piece], 'rows %d to %d' % (at, at + n))
        at += n
    ref.assert_off(state.get(), want_new, off_new, 'state')


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [5, 100, 700])
def test_linear_attention_keeps_what_comes_before_an_infinity(chx, length, dtype):
    """Infinities and NaN of a row reach no earlier one, and no other column, head or sequence."""
    c = attend_case((2, length, 2, 1, 40, 70), dtype)
    args = lambda c: ([up(chx, c[k]) for k in ('q', 'k', 'v')], dict(log_decay=up(chx, c['log_decay']), state=up(chx, c['state'])))  # noqa: E731
    a, more = args(c)
    plain, plain_new = (x.get() for x in chx.linear_attention(*a, **more))
    (_, _), (off, off_new) = ref.linear_attention(c['q'], c['k'], c['v'], c['log_decay'], None, c['state'])
    t = length * 3 // 5
    for name, value in (('v', np.inf), ('v', np.nan), ('k', np.nan), ('q', np.inf)):
        bad = dict(c, **{name: c[name].copy()})
        bad[name][1, t, 0, 17] = value
        a, more = args(bad)
        y, new = (x.get() for x in chx.linear_attention(*a, **more))
        touched = np.zeros(y.shape, bool)
        touched_new = np.zeros(new.shape, bool)
        if name == 'q':
            touched[1, t, 0] = True
        elif name == 'k':
            touched[1, t:, 0] = True
            touched_new[1, 0, 17] = True
        else:
            touched[1, t:, 0, 17] = True
            touched_new[1, 0, :, 17] = True
        for got, want, at, far in ((y, plain, touched, off), (new, plain_new, touched_new, off_new)):
            assert not np.isfinite(got[at]).any(), name
            # elsewhere as without it; a tile that has one goes row by row, in another order
            limit = 2 * far + (np.finfo(dtype).eps * ab_of(want) if got is y else 0)
            assert (np.abs(got - want) <= limit + 1e-7)[~at].all(), name


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [5, 100, 900])
def test_linear_attention_of_a_state_that_is_not_finite(chx, length, dtype):
    """An infinity or NaN in a state stays in its column of values, its head and its sequence, whatever power of two the others are counted in."""
    c = attend_case((2, length, 2, 1, 40, 70), dtype)
    args, decay = [up(chx, c[k]) for k in ('q', 'k', 'v')], up(chx, c['log_decay'])
    plain, plain_new = (x.get() for x in chx.linear_attention(*args, decay, state=up(chx, c['state'])))
    for value in (np.inf, np.nan):
        state = c['state'].copy()
        state[1, 0, 7, 17] = value
        y, new = (x.get() for x in chx.linear_attention(*args, decay, state=up(chx, state)))
        touched, touched_new = np.zeros(y.shape, bool), np.zeros(new.shape, bool)
        touched[1, :, 0, 17] = touched_new[1, 0, :, 17] = True
        assert not np.isfinite(new[1, 0, 7, 17]) and not np.isfinite(y[1, 0, 0, 17])
        assert np.array_equal(y[~touched], plain[~touched]) and np.array_equal(new[~touched_new], plain_new[~touched_new])


def ab_of(x):
    return np.abs(x.astype(np.float64))


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [6, 150, 700])
def test_linear_attention_starts_anew_where_nothing_is_kept(chx, length, dtype):
    """A log decay of -infinity, or of the type's lowest value, ends what was gathered: documents behind one another are as if alone."""
    c = attend_case((1, length, 2, 1, 30, 40), dtype)
    cuts = sorted({0, 2, length // 3, length // 3 + 1, length - 1, length})
    for lowest in (-np.inf, np.finfo(np.float32).min):
        decay = c['log_decay'].copy()
        decay[:, cuts[:-1]] = lowest
        y, new = chx.linear_attention(*(up(chx, c[k]) for k in ('q', 'k', 'v')), up(chx, decay), state=up(chx, c['state']))
        for first, last in zip(cuts, cuts[1:]):
            alone = np.zeros_like(c['log_decay'])
            alone[:, first:last] = c['log_decay'][:, first:last]
            piece = slice(first, last)
            (want, want_new), (off, off_new) = ref.linear_attention(c['q'][:, piece], c['k'][:, piece], c['v'][:, piece], np.where(np.arange(last - first)[:, None] == 0, 0, decay[0, piece])[None])
            ref.assert_off(y.get()[:, piece], want, off, 'rows %d to %d' % (first, last))
        ref.assert_off(new.get(), want_new, off_new, 'state')
        grads = chx.linear_attention_grad(*(up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')), up(chx, decay), state=up(chx, c['state']), gnew_state=up(chx, c['gnew']))
        assert all(np.isfinite(g.get()).all() for g in grads) and not grads.state.get().any()
        wants, offs, _ = ref.linear_attention_grad(c['q'], c['k'], c['v'], c['gy'], decay, None, c['state'], None, c['gnew'])
        for name, got in grads._asdict().items():
            ref.assert_off(got.get(), wants[name], offs[name], name)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('keys,values', [(24, 40), (6, 90), (130, 33)])
def test_linear_attention_of_the_largest_and_smallest_numbers(chx, keys, values, dtype):
    """A state that all but vanishes and comes back, one that starts near the type's end, growing and fading by sixteens of powers of two, a scale that takes products far away."""
    c = attend_case((4, 260, 1, 1, keys, values), dtype)
    c['log_decay'][:] = -0.01
    c['state'][0] *= 1e-30
    c['log_decay'][0, :130] = -0.5                   # 2^-94 of it is left ...
    c['v'][0, :200] = 0
    c['v'][0, 200:] *= 8000                          # ... when rows of 2^13 come
    c['state'][1] *= 1e30
    c['log_decay'][1, :] = -0.7
    c['v'][2] *= np.exp2(np.arange(260) // 64 * 6.0 - 12).astype(dtype)[:, None, None]
    c['log_decay'][2, :] = 0.02                      # (grows)
    c['k'][3] *= np.exp2(-(np.arange(260) // 64) * 3.0).astype(dtype)[:, None, None]
    c['log_decay'][3, 128] = -80
    for scale in (None, 2.0 ** -20, 2.0 ** 12):
        with np.errstate(over='ignore'):
            check_attend_outputs(chx, c, scale)


def check_attend_outputs(chx, c, scale):
    more = dict(log_decay=up(chx, c['log_decay']), scale=scale, state=up(chx, c['state']))
    y, new = chx.linear_attention(*(up(chx, c[k]) for k in ('q', 'k', 'v')), **more)
    (want, want_new), (off, off_new) = ref.linear_attention(c['q'], c['k'], c['v'], c['log_decay'], scale, c['state'])
    grads = chx.linear_attention_grad(*(up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')), gnew_state=up(chx, c['gnew']), **more)
    wants, offs, _ = ref.linear_attention_grad(c['q'], c['k'], c['v'], c['gy'], c['log_decay'], scale, c['state'], None, c['gnew'])
    for b in range(y.shape[0]):  # (each has its own numbers, and limits that follow from them)
        ref.assert_off(y.get()[b], want[b], off[b], 'y of %d' % b)
        ref.assert_off(new.get()[b], want_new[b], off_new[b], 'state of %d' % b)
        for name, got in grads._asdict().items():
            ref.assert_off(got.get()[b], wants[name][b], offs[name][b], 'g%s of %d' % (name, b))


def test_linear_attention_of_nothing(chx):
    state = np.random.default_rng(0).standard_normal((2, 3, 4, 5)).astype(np.float32)
    z = lambda *s: chx.zeros(s, 'float32')  # noqa: E731
    y, new = chx.linear_attention(z(2, 0, 3, 4), z(2, 0, 3, 4), z(2, 0, 3, 5), state=up(chx, state))
    assert y.shape == (2, 0, 3, 5) and np.array_equal(new.get(), state)
    g = chx.linear_attention_grad(z(2, 0, 3, 4), z(2, 0, 3, 4), z(2, 0, 3, 5), z(2, 0, 3, 5), z(3), state=up(chx, state), gnew_state=up(chx, state))
    assert np.array_equal(g.state.get(), state) and not g.log_decay.get().any() and g.q.shape == (2, 0, 3, 4)
    y, new = chx.linear_attention(z(0, 7, 3, 4), z(0, 7, 3, 4), z(0, 7, 3, 5))
    assert y.shape == (0, 7, 3, 5) and new.shape == (0, 3, 4, 5)
    g = chx.linear_attention_grad(z(0, 7, 3, 4), z(0, 7, 3, 4), z(0, 7, 3, 5), z(0, 7, 3, 5), z(3))
    assert not g.log_decay.get().any()
    with pytest.raises(chx.DimensionError):
        chx.linear_attention(z(2, 4, 3), z(2, 4, 3), z(2, 4, 3))


def test_linear_attention_gradients_against_differences(chx):
    """float32 through the kernels: central differences of sum(y * gy) + sum(new * gnew) in 64 bits of the plain form agree with its gradients, and the kernels' with those."""
    c = attend_case((1, 6, 2, 2, 3, 4), 'float32')
    grads = chx.linear_attention_grad(*(up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')), up(chx, c['log_decay']), state=up(chx, c['state']), gnew_state=up(chx, c['gnew']))
    wide = {k: c[k].astype(np.float64) for k in ('q', 'k', 'v', 'log_decay', 'state')}
    h = 1e-5

    def loss():
        (y, new), _ = ref.linear_attention(**wide)
        return (y * c['gy']).sum() + (new * c['gnew']).sum()

    _, offs, _ = ref.linear_attention_grad(c['q'], c['k'], c['v'], c['gy'], c['log_decay'], None, c['state'], None, c['gnew'])
    for name, a in wide.items():
        flat, got = a.reshape(-1), getattr(grads, name).get().reshape(-1)
        for i in range(flat.size):
            was, sums = flat[i], []
            for s in (h, -h):
                flat[i] = was + s
                sums.append(loss())
            flat[i] = was
            # h^2 / 6 of a third derivative of order 100 and 2^-52 of sums of order 100 over h
            assert abs((sums[0] - sums[1]) / (2 * h) - got[i]) <= offs[name].reshape(-1)[i] + 1e-7 + 1e-7 * abs(got[i]), name


# ---------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------
def adamw_arrays(sizes, dtype, grad_dtype, bits, master, seed=0):
    rng = np.random.default_rng(seed)
    f = np.float32
    arrays = []
    for n in sizes:
        size = np.repeat(np.exp(rng.standard_normal(n // 64 + 1)), 64)[:n].astype(f) * f(1e-3)
        p, g, m, v = (rng.standard_normal(n).astype(f) for _ in range(4))
        w, m, v = p * f(0.05), m * size * f(0.3), size * size * np.exp(f(0.3) * v)
        scales = [None, None]
        if bits == 8:
            zero = np.zeros(n, f)
            code, m_scale, _ = ref.stored(np.abs(m), 16, zero)
            m, (v, v_scale) = np.where(m < 0, code + 128, code).astype(np.uint8), ref.stored(np.sqrt(v), 32, zero)[:2]
            v, scales = v.astype(np.uint8), [m_scale, v_scale]
        arrays.append([w.astype(dtype), (g * size).astype(grad_dtype), m, v] + scales + [w.copy() if master and dtype == 'float16' else None])
    return arrays


def check_adamw(chx, arrays, t, device_t=False, **hyper):
    hyper = dict(dict(alpha=0.001, beta1=0.9, beta2=0.999, eps=1e-8, eta=1.0, weight_decay_rate=0.01, seed=77), **hyper)
    dev = [[up(chx, a) for a in x] for x in arrays]
    step = up(chx, np.array([t], np.int64)) if device_t else t
    chx.adamw_update([x[0] for x in dev], [x[1] for x in dev], [chx.AdamWState(*x[2:]) for x in dev], step, **hyper)
    for i, (x, d) in enumerate(zip(arrays, dev)):
        flat = [None if a is None else a.reshape(-1) for a in x]
        want = ref.adamw(*flat[:7], i, t, **hyper)
        for name, got, w in zip(('p', 'm', 'v', 'm_scale', 'v_scale', 'master'), [d[0]] + d[2:], want):
            assert (got is None) == (w is None)
            if got is not None:
                g = got.get().reshape(-1)
                same = (g == w) | (np.isnan(g.astype(np.float64)) & np.isnan(w.astype(np.float64)))
                if name in 'mv' and want[3] is not None:  # codes of blocks that are not a number mean nothing
                    same |= np.isnan(ref.of_blocks(want[3 if name == 'm' else 4], g.size))
                assert g.dtype == w.dtype and same.all(), '%s of array %d: %d of %d differ, first %r, expected %r' % (name, i, (~same).sum(), g.size, g[~same][0], w[~same][0])
    return dev


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,grad_dtype,master', [('float32', 'float32', False), ('float16', 'float16', False), ('float16', 'float32', False), ('float16', 'float16', True),
                                                     ('float16', 'float32', True)])
def test_adamw(chx, dtype, grad_dtype, master, bits):
    """Every bit of it, for arrays of all sizes."""
    sizes = [1, 7, 8, 255, 256, 257, 2047, 2048, 2049, 5000, 100003] + list(range(300, 360))
    check_adamw(chx, adamw_arrays(sizes, dtype, grad_dtype, bits, master), 13)
    check_adamw(chx, adamw_arrays([3000, 129], dtype, grad_dtype, bits, master, 1), 1, alpha=0.1, beta1=0.0, beta2=0.5, eps=1e-3, eta=0.5, weight_decay_rate=0.0, seed=-5)
    check_adamw(chx, adamw_arrays([3000, 129], dtype, grad_dtype, bits, master, 2), (3 << 32) + 17, device_t=True)
    check_adamw(chx, adamw_arrays([3000, 129], dtype, grad_dtype, bits, master, 3), 1000, device_t=True, seed=1 << 40)


def test_adamw_of_mixed_arrays_step_by_step(chx):
    """States of both kinds in one list, a float16 array between float32 ones, arrays without elements, gradients that are views; two steps with states from adamw_state."""
    arrays = adamw_arrays([600, 0], 'float32', 'float32', 8, False) + adamw_arrays([600, 70], 'float16', 'float32', 32, True) + adamw_arrays([33], 'float32', 'float32', 32, False)
    check_adamw(chx, arrays, 5)
    rng = np.random.default_rng(1)
    w, half = rng.standard_normal((20, 30)).astype(np.float32), rng.standard_normal(500).astype(np.float16)
    params = [up(chx, w), up(chx, half)]
    states = [chx.adamw_state(params[0], bits=8), chx.adamw_state(params[1], master=True)]
    flat = [[w.reshape(-1), np.zeros(600, np.uint8), np.zeros(600, np.uint8), np.zeros(3, np.float32), np.zeros(3, np.float32), None],
            [half, np.zeros(500, np.float32), np.zeros(500, np.float32), None, None, half.astype(np.float32)]]
    for t in (1, 2):
        g = [rng.standard_normal((30, 20)).astype(np.float32), rng.standard_normal((500, 3)).astype(np.float16)]
        chx.adamw_update(params, [up(chx, g[0]).T, up(chx, g[1])[:, 1]], states, t, weight_decay_rate=0.1, seed=4)
        for i, grad in enumerate((g[0].T.reshape(-1), g[1][:, 1])):
            p, m, v, ms, vs, master = flat[i]
            flat[i] = list(ref.adamw(p, grad, m, v, ms, vs, master, i, t, 0.001, 0.9, 0.999, 1e-8, 1.0, 0.1, 4))
    for i in range(2):
        for got, want in zip([params[i], states[i].m, states[i].v, states[i].m_scale, states[i].v_scale, states[i].master], flat[i]):
            assert (got is None) == (want is None) and (got is None or np.array_equal(got.get().reshape(-1), want))


def test_adamw_of_special_values(chx):
    """Zeros, subnormal and huge gradients, infinities and NaN: states of 32 bits as the formulas say, a block of 8 bits that cannot be told is NaN and its neighbours are not touched."""
    for bits in (32, 8):
        for seed in range(2):
            (p, g, m, v, ms, vs, master), = adamw_arrays([2048], 'float32', 'float32', bits, False, seed)
            g[:256] = 0
            g[256:512] *= np.float32(1e-36)
            g[512:768:7] = 0
            g[768:1024] *= np.float32(1e17)
            g[1024 + 5] = np.inf
            g[1280 + 100] = np.nan
            g[1536 + 3] = np.float32(1e32)  # its square is infinite
            if bits == 8:
                ms[0] = vs[0] = 0
            check_adamw(chx, [[p, g, m, v, ms, vs, master]], 3)
            check_adamw(chx, [[p, g, m, v, ms, vs, master]], 3, eps=0.0)


def test_adamw_states_of_8_bits_follow_those_of_32(chx):
    """Rounded at random in proportion, a state of 8 bits is right on average: over many elements with one gradient, m and v after 50 steps are those of 32 bits.

    m: a step leaves at most an eighth of a value as spread, of m's mean over the steps since (1 / (1 - beta) of them count): the mean of 2^16 elements is within
    6 / 2^8 * 1/8 of it even if every step's rounding were kept whole.

    v: sqrt(v) is what is right on average, so that v is larger by the variance of each rounding.  With a constant gradient v grows like the step s and its root r, next to a code, by r / (2 s), which
    is 8 / s of a step of r / 16, or 4 / s of one of r / 8: a variance of at most r^2 / 256 where that is over half a step, and of at most the movement times the step's square,
    r^2 / (16 s), elsewhere.  What a step s adds stays, and is var / v(T) = (s / T) min(1 / 256, 1 / (16 s)) of v at the end: together (136 / 256 + 34 / 16) / 50 = 5.3 % at T = 50; and the mean of
    2^16 elements whose relative spread is below sqrt(0.053) is within 6 / 2^8 of that spread."""
    n = 1 << 16
    g = np.full(n, 0.01, np.float32)
    p = [chx.zeros((n,)), chx.zeros((n,))]
    states = [chx.adamw_state(p[0], bits=8), chx.adamw_state(p[1])]
    grad = up(chx, g)
    for t in range(1, 51):
        chx.adamw_update(p, [grad, grad], states, t, seed=9)
    m = ref.part_of(states[0].m.get().astype(np.int64) & 127, 16) * ref.of_blocks(states[0].m_scale.get(), n)
    root = ref.part_of(states[0].v.get().astype(np.int64), 32) * ref.of_blocks(states[0].v_scale.get(), n)
    assert abs(m.mean() / states[1].m.get()[0] - 1) < 6 / 256 / 8
    more, noise = (root.astype(np.float64) ** 2).mean() / states[1].v.get()[0] - 1, 6 / 256 * 0.053 ** 0.5
    assert -noise < more < 0.053 + noise


def test_adamw_refuses_what_would_be_written_twice(chx):
    p, q = chx.zeros((600,)), chx.zeros((600,))
    s, r = chx.adamw_state(p), chx.adamw_state(q)
    g = chx.ones((600,))
    for params, grads, states in (([p, p], [g, g], [s, r]), ([p, q], [g, g], [s, s]), ([p], [p], [s]), ([p[:400], p[300:]], [g[:400], g[300:]], [chx.adamw_state(p[:400]), chx.adamw_state(p[300:])]),
                                  ([p], [s.m], [s])):
        with pytest.raises(chx.ChainerxError):
            chx.adamw_update(params, grads, states, 1)
    assert not p.get().any()
    chx.adamw_update([p[:300], p[300:]], [g[:300], g[:300]], [chx.adamw_state(p[:300]), chx.adamw_state(p[300:])], 1)  # halves of one array, a gradient for both
    assert (p.get() == p.get()[0]).all() and p.get()[0] != 0
    with pytest.raises(chx.DimensionError):
        chx.adamw_update([p], [g, g], [s], 1)
    with pytest.raises(chx.ChainerxError):
        chx.adamw_update([p], [g], [s], 0)


# ---------------------------------------------------------------------------------------------
# long sequences in segments, addresses far apart
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', [(1, 2100, 2, 2, 256, 70), (2, 1500, 4, 4, 100, 130), (3, 900, 2, 1, 50, 50), (1, 1281, 1, 1, 5, 6)])
def test_linear_attention_of_long_sequences(chx, sizes, dtype):
    """Time in segments: with states and without, heads that share keys, sequences that end in the first segment, the last, and before any; the state moved forward in place."""
    for i, (decay, ragged, state, gnew) in enumerate((('heads', False, True, True), ('rows', True, True, False), (None, True, False, True))):
        c = attend_case(sizes, dtype, seed=i, ragged=ragged, decay=decay)
        if decay is None:  # (all that there is stays: values that keep the sums in float16's range)
            c['v'] = c['v'] * np.asarray(0.1, dtype)
        check_attend(chx, c, lambda a: up(chx, a), None, state, gnew, '%s %s %d' % (sizes, dtype, i))
    state = up(chx, c['state'])
    y, new = chx.linear_attention(*(up(chx, c[k]) for k in ('q', 'k', 'v')), state=up(chx, c['state']), lengths=up(chx, c['lengths']))
    y2, same = chx.linear_attention(*(up(chx, c[k]) for k in ('q', 'k', 'v')), state=state, lengths=up(chx, c['lengths']), out_state=state)
    assert same is state and np.array_equal(y.get(), y2.get()) and np.array_equal(state.get(), new.get())


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [4, 90])
def test_linear_attention_of_sequences_far_apart(chx, length, dtype):
    """Sequences and rows whose distance in memory takes more than 31 bits, results among them; at 2^24 elements from row to row the call is refused."""
    c = attend_case((2, length, 2, 1, 16, 24), dtype)
    dev = {k: up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')}
    more = dict(log_decay=up(chx, c['log_decay']), state=up(chx, c['state']))
    want, want_new = chx.linear_attention(dev['q'], dev['k'], dev['v'], **more)
    grads = chx.linear_attention_grad(dev['q'], dev['k'], dev['v'], dev['gy'], **more)
    item = np.dtype(dtype).itemsize
    batch, row = 1 << 33, ((1 << 24) - 3) * item
    buffer = chx._array.alloc_bytes(batch + length * row + (1 << 16))
    far = {}
    for i, k in enumerate(('q', 'k', 'v', 'gy')):
        far[k] = chx.ndarray(buffer, 8192 * i, c[k].shape, (batch, row, c[k].shape[3] * item + 256, item), np.dtype(dtype))
        chx.routines._copy_into(far[k], dev[k])
    y, new = chx.linear_attention(far['q'], far['k'], far['v'], **more)
    assert np.array_equal(y.get(), want.get()) and np.array_equal(new.get(), want_new.get())
    for got, w in zip(chx.linear_attention_grad(far['q'], far['k'], far['v'], far['gy'], **more), grads):
        assert np.array_equal(got.get(), w.get())
    beyond = chx.ndarray(buffer, 0, c['q'].shape, (batch, item << 24, 512, item), np.dtype(dtype))
    with pytest.raises(chx.ChainerxNotImplementedError):
        chx.linear_attention(beyond, far['k'], far['v'])


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length', [3, 100])
def test_linear_attention_of_strides_that_repeat_and_run_backwards(chx, length, dtype):
    """Inputs broadcast over the batch and read backwards in time, and a single row of any stride."""
    c = attend_case((3, length, 2, 1, 18, 20), dtype)
    dev = {k: up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')}
    for k in ('q', 'k', 'v'):
        c[k] = np.ascontiguousarray(np.broadcast_to(c[k][:1, ::-1], c[k].shape))
        dev[k] = dev[k][:1, ::-1].broadcast_to(c[k].shape)
    dense = [up(chx, c[k]) for k in ('q', 'k', 'v')]
    views = [dev[k] for k in ('q', 'k', 'v')]
    for got, want in zip(chx.linear_attention(*views), chx.linear_attention(*dense)):
        assert np.array_equal(got.get(), want.get())
    for got, want in zip(chx.linear_attention_grad(*views, dev['gy'])[:3], chx.linear_attention_grad(*dense, dev['gy'])[:3]):
        assert np.array_equal(got.get(), want.get())
    q, k, v = (a[:, :1] for a in dense)
    want = chx.linear_attention(up(chx, q.get()), up(chx, k.get()), up(chx, v.get()))
    for far in (1 << 40, -(1 << 40), 0):
        odd = [chx.ndarray(a._buf, a._offset, a.shape, (a.strides[0], far) + a.strides[2:], a.dtype) for a in (q, k, v)]
        for got, w in zip(chx.linear_attention(*odd), want):
            assert np.array_equal(got.get(), w.get())


@pytest.mark.parametrize('seed', range(16))
def test_layers_of_drawn_sizes(chx, seed):
    """Any widths, lengths, heads and shares, padded and not, in both types; rows of any number and width."""
    rng = np.random.default_rng(1000 + seed)
    share = int(rng.choice([1, 1, 2, 3]))
    sizes = (int(rng.integers(1, 4)), int(np.exp(rng.uniform(0, np.log(420)))), share * int(rng.integers(1, 3)), share, int(rng.integers(1, 257)), int(rng.integers(1, 257)))
    dtype, ragged, decay = ('float16', 'float32')[seed % 2], bool(rng.integers(2)), (None, 'rows', 'heads')[int(rng.integers(3))]
    c = attend_case(sizes, dtype, seed=seed, ragged=ragged, decay=decay)
    if decay is None:
        c['v'] = c['v'] * np.asarray(0.1, dtype)
    check_attend(chx, c, (lambda a: apart(chx, a)) if rng.integers(2) else (lambda a: up(chx, a)), None, bool(rng.integers(2)), bool(rng.integers(2)), '%s %s' % (sizes, dtype))
    rows, cols = int(np.exp(rng.uniform(0, np.log(3000)))), int(np.exp(rng.uniform(0, np.log(9000))))
    x, gamma, beta, gy = norm_case(rows, cols, dtype, 'float32', seed=seed)
    y, state = chx.layer_norm(apart(chx, x, 5), up(chx, gamma), up(chx, beta))
    want, off = ref.layer_norm(x, gamma, beta, 2e-5)
    for name, got in (('y', y), ('mean', state.mean), ('inv_std', state.inv_std)):
        ref.assert_off(got.get(), want[name], off[name], '%d x %d %s' % (rows, cols, name))
    want, off = ref.layer_norm_grad(x, gamma, gy, 2e-5)
    for name, got in zip(('gx', 'ggamma', 'gbeta'), chx.layer_norm_grad(up(chx, x), up(chx, gamma), apart(chx, gy, 2), state)):
        ref.assert_off(got.get(), want[name].reshape(got.shape), off[name].reshape(got.shape), '%d x %d %s' % (rows, cols, name))


# ---------------------------------------------------------------------------------------------
# the layers together, graphs, streams, threads
# ---------------------------------------------------------------------------------------------
NAMES = ('gamma', 'beta', 'in_w', 'out_w')


def block_case(rng, units, heads, width, dtype='float32'):
    n = lambda *s: (rng.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731
    return {'gamma': 1 + 0.1 * n(units) * units ** 0.5, 'beta': n(units), 'in_w': n(3 * heads * width, units), 'out_w': n(units, heads * width)}


def block(chx, p, x, decay, state=None, lengths=None):
    """layer norm -> linear -> linear attention -> linear, added to what went in; (the result, the state, what the gradients need)."""
    batch, length, units = x.shape
    heads, width = decay.shape[-1], p['out_w'].shape[1] // decay.shape[-1]
    n, stats = chx.layer_norm(x, p['gamma'], p['beta'])
    rows = n.reshape(batch * length, units)
    wide = chx.linear(rows, p['in_w']).reshape(batch, length, 3, heads, width)
    qkv = [wide[:, :, i] for i in range(3)]
    y, new = chx.linear_attention(*qkv, decay, state=state, lengths=lengths)
    out = chx.add(chx.linear(y.reshape(batch * length, heads * width), p['out_w']).reshape(x.shape), x)
    return out, new, (stats, rows, qkv, y)


def block_grad(chx, p, x, decay, kept, gout, state=None, lengths=None, gnew=None):
    """The gradients of the parameters, by name, and those of x and the state."""
    batch, length, units = x.shape
    stats, rows, qkv, y = kept
    g = gout.reshape(batch * length, units)
    flat = y.reshape(batch * length, -1)
    grads = {'out_w': chx.dot(g.T, flat)}
    a = chx.linear_attention_grad(*qkv, chx.dot(g, p['out_w']).reshape(y.shape), decay, state=state, lengths=lengths, gnew_state=gnew)
    gwide = chx.concatenate([v.reshape(batch * length, -1) for v in (a.q, a.k, a.v)], 1)
    grads['in_w'] = chx.dot(gwide.T, rows)
    gx, grads['gamma'], grads['beta'] = chx.layer_norm_grad(x, p['gamma'], chx.dot(gwide, p['in_w']).reshape(x.shape), stats)
    return grads, chx.add(gx, gout), a.state


def plain_block(p, x, decay, state, lengths):
    heads, width = decay.shape[-1], p['out_w'].shape[1] // decay.shape[-1]
    n = ref.layer_norm(x, p['gamma'], p['beta'], 2e-5)[0]['y']
    wide = (n @ p['in_w'].T).reshape(x.shape[:2] + (3, heads, width))
    (y, new), _ = ref.linear_attention(wide[:, :, 0], wide[:, :, 1], wide[:, :, 2], decay, None, state, lengths)
    return y.reshape(x.shape[:2] + (-1,)) @ p['out_w'].T + x, new


def test_a_block_is_trained_as_its_formulas_say(chx):
    """Its gradients against differences of the plain forms in 64 bits along random directions, and the step that AdamW takes with them bit by bit."""
    rng = np.random.default_rng(5)
    host, x = block_case(rng, 20, 2, 9), rng.standard_normal((3, 70, 20)).astype(np.float32)
    decay, state, lengths = -np.exp(rng.standard_normal((3, 70, 2)) - 2).astype(np.float32), rng.standard_normal((3, 2, 9, 9)).astype(np.float32), np.array([70, 0, 41])
    gout, gnew = rng.standard_normal(x.shape).astype(np.float32), rng.standard_normal(state.shape).astype(np.float32)
    p, dx, dd, ds, dl = {k: up(chx, v) for k, v in host.items()}, up(chx, x), up(chx, decay), up(chx, state), up(chx, lengths)
    _, _, kept = block(chx, p, dx, dd, ds, dl)
    grads, gx, gstate = block_grad(chx, p, dx, dd, kept, up(chx, gout), ds, dl, up(chx, gnew))

    def loss(**over):
        v = {k: over.get(k, a).astype(np.float64) for k, a in dict(host, x=x, state=state).items()}
        out, new = plain_block(v, v['x'], decay.astype(np.float64), v['state'], lengths)
        return (out * gout).sum() + (new * gnew).sum()

    for name, base, got in [(k, host[k], grads[k]) for k in NAMES] + [('x', x, gx), ('state', state, gstate)]:
        along, base, step, got = rng.standard_normal(base.shape), base.astype(np.float64), 1e-4, got.get().astype(np.float64)
        change = (loss(**{name: base + step * along}) - loss(**{name: base - step * along})) / (2 * step)
        # differences are exact to step^2; a float32 gradient's elements to some 1e-6 of their size
        assert abs((got * along).sum() - change) <= 1e-4 * (np.abs(got * along).sum() + 1), name
    states = [chx.adamw_state(p[k], bits=8 if k.endswith('w') else 32) for k in NAMES]
    want = []
    for i, k in enumerate(NAMES):
        s = states[i]
        want.append(ref.adamw(host[k].reshape(-1), grads[k].get().reshape(-1), *[None if a is None else a.get().reshape(-1) for a in (s.m, s.v, s.m_scale, s.v_scale)], None, i, 1, 0.01, 0.9, 0.999,
                              1e-8, 1.0, 0.1, 3))
    chx.adamw_update([p[k] for k in NAMES], [grads[k] for k in NAMES], states, 1, alpha=0.01, weight_decay_rate=0.1, seed=3)
    for k, s, w in zip(NAMES, states, want):
        for got, expected in zip((p[k], s.m, s.v, s.m_scale, s.v_scale), w):
            assert (got is None) == (expected is None) and (got is None or np.array_equal(got.get().reshape(-1), expected)), k


@pytest.mark.parametrize('length', [30, 400])
def test_a_block_answers_a_prompt_and_then_token_by_token(chx, length):
    """As a server runs it, a state for each layer, moved forward in place: what the whole sequences give."""
    rng = np.random.default_rng(6)
    layers = [{k: up(chx, v) for k, v in block_case(rng, 24, 3, 8).items()} for _ in range(2)]
    x = rng.standard_normal((3, length, 24)).astype(np.float32)
    decay = up(chx, np.log1p(-np.exp2(-3.0 - np.arange(3))).astype(np.float32))

    def run(x, states):
        h = up(chx, x)
        for i, p in enumerate(layers):
            h, new, _ = block(chx, p, h, decay, states[i])
            states[i] = new
        return h.get()

    want, states = run(x, [None, None]), [None, None]
    cuts = [0, length - 12, length - 11, length - 10, length - 4, length]
    got = [run(x[:, a:b], states) for a, b in zip(cuts, cuts[1:])]
    # sums of some tens of terms in other orders, through two layers that divide by a deviation of order 1: far from any mistake in a row or a state
    np.testing.assert_allclose(np.concatenate(got, 1), want, rtol=0, atol=1e-4)


def test_a_step_replays_in_a_graph(chx):
    """The block's forward pass, gradients and AdamW's step in a captured graph, replayed between eager steps from the same weights: each replay is the next step."""
    from chainer_amd import graph
    rng = np.random.default_rng(9)
    host, x = block_case(rng, 24, 2, 16), up(chx, rng.standard_normal((2, 700, 24)).astype(np.float32))
    decay, lengths, gout = up(chx, -np.exp(rng.standard_normal((2, 700, 2)) - 2).astype(np.float32)), up(chx, np.array([700, 333])), up(chx, rng.standard_normal((2, 700, 24)).astype(np.float32))
    make = lambda: ({k: up(chx, v) for k, v in host.items()}, up(chx, np.array([1], np.int64)))  # noqa: E731
    (p, t), (q, u) = make(), make()
    s, r = ([chx.adamw_state(w[k], bits=b) for k, b in zip(NAMES, (32, 32, 8, 8))] for w in (p, q))

    def step(p, s, t):
        out, new, kept = block(chx, p, x, decay, None, lengths)
        grads, gx, _ = block_grad(chx, p, x, decay, kept, gout, None, lengths)
        chx.adamw_update([p[k] for k in NAMES], [grads[k] for k in NAMES], s, t, alpha=0.01, weight_decay_rate=0.1, seed=3)
        return out, new, gx

    everything = lambda p, s, t: [p[k] for k in NAMES] + [a for state in s for a in state if a is not None] + [t]  # noqa: E731
    captured = graph.capture(lambda: step(p, s, t))
    for _ in range(4):
        for a, b in zip(everything(q, r, u), everything(p, s, t)):  # (the passes before the capture were steps, too)
            chx.routines._copy_into(a, b)
        want = [a.get() for a in step(q, r, u)]
        captured.replay()
        chx.synchronize()
        for a, w in zip(captured.result, want):
            assert np.array_equal(a.get(), w)
        for a, b in zip(everything(p, s, t), everything(q, r, u)):
            assert np.array_equal(a.get(), b.get())
        chx.add(t, chx.array(np.array([1], np.int64)), out=t)  # the next step
    captured.release()


def test_layers_on_two_streams_and_threads_at_once(chx):
    """Calls at the same time have workspaces of their own, on whatever stream is current where they are made."""
    import threading

    import torch
    c = attend_case((2, 1500, 2, 1, 50, 50), 'float16', ragged=True)
    args = [up(chx, c[k]) for k in ('q', 'k', 'v')]
    more = dict(log_decay=up(chx, c['log_decay']), lengths=up(chx, c['lengths']))
    x, gamma, beta, gy = (up(chx, a) for a in norm_case(900, 650, 'float32', 'float32'))

    def everything():
        y, stats = chx.layer_norm(x, gamma, beta)
        p = chx.array(np.linspace(-1, 1, 5000, dtype=np.float32))
        s = chx.adamw_state(p, bits=8)
        chx.adamw_update([p], [chx.ones((5000,))], [s], 1)
        return [y] + list(chx.layer_norm_grad(x, gamma, gy, stats)) + list(chx.linear_attention(*args, **more)) + list(chx.linear_attention_grad(*args, up(chx, c['gy']), **more))[:4] + [p, s.v]

    want = [a.get() for a in everything()]
    chx.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], {}

    def work(i):
        with torch.cuda.stream(streams[i]):
            results[i] = [everything() for _ in range(3)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for s in streams:
        s.synchronize()
    for i in range(3):
        for r in results[i]:
            for a, w in zip(r, want):
                assert np.array_equal(a.get(), w)

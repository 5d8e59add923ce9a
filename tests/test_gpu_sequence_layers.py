"""Dropout, the causal convolution and the selective scan on the device against plain forms in 64 bits (sequence_reference.py)."""
import numpy as np
import pytest

import sequence_reference as ref

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
# dropout
# ---------------------------------------------------------------------------------------------
KEY = np.array([0x0123456789ABCDEF, (5 << 32) + 7], np.int64)


@pytest.mark.parametrize('dtype', ['float16', 'float32', 'float64'])
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (9,), (3, 5), (129, 650), (2, 3, 4, 5), (4099,)])
def test_dropout(chx, shape, dtype):
    rng = np.random.default_rng(1)
    x, r = rng.standard_normal(shape).astype(dtype), rng.standard_normal(shape).astype(dtype)
    for ratio, residual in ((0.5, None), (0.1, r), (0.0, r), (0.0, None), (0.999, None), (1 - 2.0 ** -30, r)):
        got = chx.dropout(up(chx, x), ratio, up(chx, KEY), site=9, residual=up(chx, residual)).get()
        want = ref.dropout(x, ratio, KEY, 9, residual)
        assert got.dtype == x.dtype
        dropped = ~ref.kept(x.size, ratio, KEY, 9).reshape(shape)
        assert np.array_equal(got[dropped], np.zeros(1, dtype).repeat(dropped.sum()) if residual is None else r[dropped])
        # two roundings of 32 (64) bits -- the scale and the product, or the scale and the sum -- and the one to the type
        size = np.abs(x.astype(np.float64)) * 65536 / (65536 - ref.threshold(ratio)) + (0 if residual is None else np.abs(r.astype(np.float64)))
        if dtype == 'float64':
            assert (np.abs(got - want) <= 4 * 2.0 ** -53 * size).all()
        else:
            ref.assert_within(got, want, size, 2, '%s %s' % (shape, ratio))


def test_dropout_masks(chx):
    """Another seed, step or layer is another mask, a gradient's is the forward one's; the share of what is kept is the ratio's."""
    n = 1 << 16
    ones = chx.ones((n,), 'float32')
    masks = {}
    for name, key, site in (('a', KEY, 0), ('site', KEY, 1), ('seed', KEY + [1, 0], 0), ('step', KEY + [0, 1], 0), ('wrap', np.array([-1, -1], np.int64), (1 << 32) - 1)):
        masks[name] = chx.dropout(ones, 0.25, up(chx, key), site).get() != 0
        assert np.array_equal(masks[name], ref.kept(n, 0.25, key, site)), name
        assert np.array_equal(masks[name], chx.dropout(ones.astype('float16'), 0.25, up(chx, key), site).get() != 0)
        # 2^16 draws of probability 3/4: six standard deviations
        assert abs(masks[name].mean() - 0.75) < 6 * np.sqrt(0.75 * 0.25 / n)
    for a in masks:
        for b in masks:
            # masks that have nothing to do with each other agree in 3/4^2 + 1/4^2 of the places
            assert a == b or abs((masks[a] == masks[b]).mean() - 0.625) < 6 * np.sqrt(0.625 * 0.375 / n)


def test_dropout_takes_views_and_keeps_what_is_dropped_out(chx):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((33, 20)).astype(np.float32)
    want = chx.dropout(chx.array(x), 0.3, up(chx, KEY)).get()
    assert np.array_equal(chx.dropout(chx.array(np.ascontiguousarray(x.T)).T, 0.3, up(chx, KEY)).get(), want)
    assert np.array_equal(chx.dropout(apart(chx, x), 0.3, up(chx, KEY)).get(), want)
    flat = chx.array(np.concatenate([np.zeros(1, np.float32), x.reshape(-1)]))[1:].reshape(33, 20)  # an odd address
    assert np.array_equal(chx.dropout(flat, 0.3, up(chx, KEY)).get(), want)
    # NaN and infinities that are dropped leave nothing behind
    dropped = ~ref.kept(x.size, 0.3, KEY, 0).reshape(x.shape)
    x[dropped] = np.where(np.arange(dropped.sum()) % 2 == 0, np.nan, np.inf)
    assert np.array_equal(chx.dropout(chx.array(x), 0.3, up(chx, KEY)).get(), want)
    empty = chx.dropout(chx.zeros((0, 4), 'float16'), 0.3, up(chx, KEY))
    assert empty.shape == (0, 4)


def test_dropout_in_place_and_beyond_2_31_elements(chx):
    from chainer_amd import _lib
    n = (1 << 31) + 13
    x = chx.ones((n,), 'float16')
    _lib.call('hipcx_dropout', x.desc(), 0.5, up(chx, KEY).desc(), 2, x.desc(), x.desc(), chx.routines.current_stream())  # x + dropout(x)
    first = n // 8 * 8 - 4096
    assert np.array_equal(x[first:].get(), np.where(ref.kept(n - first, 0.5, KEY, 2, first), 3, 1).astype(np.float16))
    assert np.array_equal(x[:4096].get(), np.where(ref.kept(4096, 0.5, KEY, 2), 3, 1).astype(np.float16))


# ---------------------------------------------------------------------------------------------
# the causal convolution
# ---------------------------------------------------------------------------------------------
CONVS = [(1, 1, 1, 1), (2, 3, 5, 2), (3, 40, 8, 3), (2, 37, 33, 4), (1, 300, 650, 4), (4, 9, 12, 8), (5, 70, 24, 7), (2, 16, 7, 5), (130, 1, 36, 4), (1, 1000, 3, 6)]


def conv_case(batch, length, channels, taps, dtype, seed=0, ragged=False):
    rng = np.random.default_rng(seed)
    n = lambda *s: rng.standard_normal(s).astype(dtype)  # noqa: E731
    c = {'x': n(batch, length, channels), 'w': n(channels, taps), 'b': n(channels), 'state': n(batch, taps - 1, channels), 'gy': n(batch, length, channels),
         'gnew': n(batch, taps - 1, channels), 'lengths': None}
    if ragged:
        c['lengths'] = rng.integers(-1, length + 3, batch).astype(np.int32 if seed % 2 else np.int64)
        c['lengths'][batch // 2] = 0
        ends = ref.ends_of(c['lengths'], batch, length)
        for k in ('x', 'gy'):
            c[k][~ref.inside(ends, length)[..., 0]] = np.nan
    return c


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', CONVS)
def test_causal_conv(chx, sizes, dtype):
    for i, (activation, ragged, bias, state) in enumerate((('silu', False, True, True), (None, True, False, True), ('silu', True, True, False))):
        c = conv_case(*sizes, dtype, seed=i, ragged=ragged)
        b, s = c['b'] if bias else None, c['state'] if state else None
        y, new = chx.causal_conv(apart(chx, c['x']), up(chx, c['w']), up(chx, b), state=up(chx, s), lengths=up(chx, c['lengths']), activation=activation)
        want, size, want_new = ref.causal_conv(c['x'], c['w'], b, s, c['lengths'], activation)
        what = '%s %s %s' % (sizes, dtype, activation)
        ref.assert_within(y.get(), want, size, 1, what)
        assert np.array_equal(new.get(), want_new.astype(dtype)), what
        grads = chx.causal_conv_grad(apart(chx, c['x']), up(chx, c['w']), up(chx, b), apart(chx, c['gy']), state=up(chx, s), lengths=up(chx, c['lengths']),
                                     activation=activation, gnew_state=up(chx, c['gnew']) if i else None)
        wants, sizes_of = ref.causal_conv_grad(c['x'], c['w'], b, c['gy'], s, c['lengths'], activation, c['gnew'] if i else None)
        for name, got, w, n in zip(('gx', 'gw', 'gb', 'gstate'), grads, wants, sizes_of):
            if got is not None:
                ref.assert_within(got.get(), w, n, 1, '%s %s' % (what, name))
        assert (grads[2] is None) == (b is None) and (grads[3] is None) == (s is None)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('channels,taps', [(19, 4), (1301, 8), (8, 7), (3, 8), (67, 2)])
def test_causal_conv_pieces_and_tokens(chx, channels, taps, dtype):
    """A sequence in pieces and token by token, the state moved forward in place, is the sequence at once, bit for bit."""
    c = conv_case(3, 50, channels, taps, dtype)
    w, b = up(chx, c['w']), up(chx, c['b'])
    whole, last = chx.causal_conv(up(chx, c['x']), w, b, state=up(chx, c['state']), activation='silu')
    state, ys, t = chx.array(c['state']), [], 0
    for n in (1, 1, 2, 0, 17, 1, 3, 25):
        y, new = chx.causal_conv(up(chx, c['x'])[:, t:t + n], w, b, state=state, activation='silu', out_state=state)
        assert new is state
        ys.append(y.get())
        t += n
    assert t == 50
    assert np.array_equal(np.concatenate(ys, 1), whole.get()) and np.array_equal(state.get(), last.get())
    assert np.array_equal(last.get(), c['x'][:, 51 - taps:])


def test_causal_conv_empty(chx):
    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        c = conv_case(*shape, 3, 'float32')
        y, new = chx.causal_conv(up(chx, c['x']), up(chx, c['w']), up(chx, c['b']), state=up(chx, c['state']))
        assert y.shape == shape and np.array_equal(new.get(), ref.causal_conv(c['x'], c['w'], c['b'], c['state'])[2].astype(np.float32))
        gx, gw, gb, gstate = chx.causal_conv_grad(up(chx, c['x']), up(chx, c['w']), up(chx, c['b']), up(chx, c['gy']), state=up(chx, c['state']), gnew_state=up(chx, c['gnew']))
        assert gx.shape == shape and not gw.get().any() and not gb.get().any()
        if shape[1] == 0:
            assert np.array_equal(gstate.get(), c['gnew'])


def test_causal_conv_beyond_2_31_elements(chx):
    """Rows whose place in memory takes more than 32 bits, with the window of the last ones."""
    length, channels = (1 << 20) + 5, 2056
    x = chx.zeros((1, length, channels), 'float16')
    c = conv_case(1, 40, channels, 4, 'float16')
    chx.routines._copy_into(x[:, length - 40:], chx.array(c['x']))
    w, b = chx.array(c['w']), chx.array(c['b'])
    y, new = chx.causal_conv(x, w, b, activation='silu')
    short, short_new = chx.causal_conv(chx.array(c['x']), w, b, state=chx.zeros((1, 3, channels), 'float16'), activation='silu')
    assert np.array_equal(y[:, length - 40:].get(), short.get()) and np.array_equal(new.get(), short_new.get())


# ---------------------------------------------------------------------------------------------
# the selective scan
# ---------------------------------------------------------------------------------------------
# batch, length, channels, states, groups (None: b and c without that axis)
SCANS = [(1, 1, 1, 1, None), (2, 5, 3, 4, None), (3, 17, 65, 16, None), (2, 33, 70, 5, 2), (1, 64, 128, 16, 1), (2, 40, 48, 64, None), (2, 19, 60, 24, 3), (1, 130, 16, 32, None),
         (20, 35, 50, 16, None), (1, 700, 20, 16, None), (2, 333, 6, 7, 2), (65, 1, 33, 16, None), (2, 1, 70, 10, 2), (1, 16, 64, 16, None), (1, 300, 5, 64, None)]


def scan_case(batch, length, channels, states, groups, dtype, seed=0, ragged=False):
    rng = np.random.default_rng(seed)
    n = lambda *s: rng.standard_normal(s).astype(dtype)  # noqa: E731
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    shared = (batch, length, states) if groups is None else (batch, length, groups, states)
    c = {'u': n(batch, length, channels), 'delta': n(batch, length, channels), 'a': -np.exp(f(channels, states)), 'b': n(*shared), 'c': n(*shared), 'd': f(channels),
         'z': n(batch, length, channels), 'delta_bias': f(channels) - 2, 'state': f(batch, channels, states)}
    more = {'gy': n(batch, length, channels), 'gnew': f(batch, channels, states)}
    lengths = None
    if ragged:
        lengths = rng.integers(-1, length + 3, batch).astype(np.int32 if seed % 2 else np.int64)
        lengths[batch // 2] = 0
        outside = ~ref.inside(ref.ends_of(lengths, batch, length), length)[..., 0]
        for v in [c[k] for k in ('u', 'delta', 'b', 'c', 'z')] + [more['gy']]:
            v[outside] = np.nan
    return c, more, lengths


VARIANTS = [('all', (), True, False), ('ragged', ('state',), True, True), ('bare', ('d', 'z', 'delta_bias', 'state'), False, False), ('no gate', ('z',), True, True)]


def scan_on_device(chx, c, lengths, softplus):
    args = {k: None if v is None else apart(chx, v) if k in ('u', 'delta', 'b', 'c', 'z') else up(chx, v) for k, v in c.items()}
    return dict(args, lengths=up(chx, lengths), delta_softplus=softplus)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', SCANS)
def test_selective_scan(chx, sizes, dtype):
    for i, (name, without, softplus, ragged) in enumerate(VARIANTS):
        c, _, lengths = scan_case(*sizes, dtype, seed=i, ragged=ragged)
        c = {k: None if k in without else v for k, v in c.items()}
        if not softplus:
            c['delta'] = np.abs(c['delta']) / 4
        y, new = chx.selective_scan(**scan_on_device(chx, c, lengths, softplus))
        (want, want_new), (size, new_size), n = ref.selective_scan(delta_softplus=softplus, lengths=lengths, **c)
        what = '%s %s %s' % (sizes, dtype, name)
        ref.assert_within(y.get(), want, size, n, what)
        ref.assert_within(new.get(), want_new, new_size, n, what + ' state')


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', SCANS)
def test_selective_scan_grad(chx, sizes, dtype):
    for i, (name, without, softplus, ragged) in enumerate(VARIANTS):
        c, more, lengths = scan_case(*sizes, dtype, seed=i, ragged=ragged)
        c = {k: None if k in without else v for k, v in c.items()}
        if not softplus:
            c['delta'] = np.abs(c['delta']) / 4
        gnew = more['gnew'] if i % 2 == 0 else None
        args = scan_on_device(chx, c, lengths, softplus)
        grads = chx.selective_scan_grad(gy=apart(chx, more['gy']), gnew_state=up(chx, gnew), **args)
        again = chx.selective_scan_grad(gy=apart(chx, more['gy']), gnew_state=up(chx, gnew), **args)
        wants, sizes_of, n = ref.selective_scan_grad(gy=more['gy'], gnew=gnew, delta_softplus=softplus, lengths=lengths, **c)
        for k, got in grads._asdict().items():
            assert (got is None) == (c[k] is None), k
            if got is None:
                continue
            assert got.shape == c[k].shape and got.dtype == c[k].dtype
            ref.assert_within(got.get(), wants[k].reshape(got.shape), sizes_of[k].reshape(got.shape), n, '%s %s %s: %s' % (sizes, dtype, name, k))
            assert np.array_equal(got.get(), getattr(again, k).get()), k


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', [(300, 18, 5, 16, None), (260, 9, 6, 3, 2), (131, 21, 190, 24, 1), (258, 17, 3, 64, None)])
def test_selective_scan_grad_many_short(chx, sizes, dtype):
    """More workgroups than compute units, whole sequences each: the tiles' states come from a launch of their own."""
    test_selective_scan_grad(chx, sizes, dtype)


@pytest.mark.parametrize('batch,length,ragged', [(2, 1, False), (3, 21, False), (3, 150, True), (1, 300, False), (300, 5, False)])
def test_selective_scan_forgetting_states(chx, batch, length, ragged):
    """A state whose decay is exp(-inf), what a = -exp(a_log) overflows to, holds its last row alone: rows and chunks behind the last one change nothing."""
    c, more, lengths = scan_case(batch, length, 9, 16, None, 'float32', seed=1, ragged=ragged)
    c['a'][3], c['a'][:, 5], c['a'][7, 2] = -np.inf, -np.inf, -3e38
    finite = dict(c, a=np.maximum(c['a'], np.float32(-1e30)))  # the same decays, 0, and no product of 0 and inf; every step is above 1e-4
    results = []
    for v in (c, finite):
        dev = scan_on_device(chx, v, lengths, True)
        y, new = chx.selective_scan(**dev)
        grads = chx.selective_scan_grad(gy=apart(chx, more['gy']), gnew_state=up(chx, more['gnew']), **dev)
        results.append(dict(grads._asdict(), y=y, new=new))
    for k, got in results[0].items():
        assert np.isfinite(got.get()).all(), k
        assert np.array_equal(got.get(), results[1][k].get()), k
    ends = ref.ends_of(lengths, batch, length)
    for b in range(batch):
        if ends[b] == 0:
            assert np.array_equal(new.get()[b], c['state'][b])
            continue
        t = ends[b] - 1
        raw = c['delta'][b, t].astype(np.float64) + c['delta_bias']
        want = np.log1p(np.exp(raw)) * c['u'][b, t] * c['b'][b, t, 5]
        # the softplus 9 and its argument's |raw|, as in the plain form's bound; two products, and a sum with 0
        assert (np.abs(new.get()[b, :, 5] - want) <= (12 + np.abs(raw)) * ref.U32 * np.abs(want)).all()


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('channels,states', [(19, 16), (33, 6), (4, 64)])
def test_selective_scan_pieces_and_tokens(chx, channels, states, dtype):
    """A sequence in pieces and token by token, the state moved forward in place, is the sequence at once."""
    c, _, _ = scan_case(3, 50, channels, states, None, dtype)
    dev = scan_on_device(chx, c, None, True)
    state, ys, t = chx.array(c['state']), [], 0
    for n in (1, 1, 2, 0, 17, 1, 3, 25):
        part = dict(dev, state=state, out_state=state, **{k: dev[k][:, t:t + n] for k in ('u', 'delta', 'b', 'c', 'z')})
        y, new = chx.selective_scan(**part)
        assert new is state
        ys.append(y.get())
        t += n
    (want, want_new), (size, new_size), n = ref.selective_scan(delta_softplus=True, **c)
    ref.assert_within(np.concatenate(ys, 1), want, size, n, 'pieces')
    ref.assert_within(state.get(), want_new, new_size, n, 'state')


def test_selective_scan_empty(chx):
    for shape in ((0, 5, 4), (2, 0, 4), (2, 5, 0)):
        c, more, _ = scan_case(*shape, 3, None, 'float32')
        dev = {k: up(chx, v) for k, v in c.items()}
        y, new = chx.selective_scan(delta_softplus=True, **dev)
        assert y.shape == shape and new.shape == c['state'].shape
        g = chx.selective_scan_grad(gy=up(chx, more['gy']), gnew_state=up(chx, more['gnew']), delta_softplus=True, **dev)
        assert g.u.shape == shape and g.b.shape == c['b'].shape and not g.a.get().any() and not g.d.get().any() and not g.delta_bias.get().any()
        assert not g.b.get().any() and not g.c.get().any()
        if shape[1] == 0:
            assert np.array_equal(new.get(), c['state']) and np.array_equal(g.state.get(), more['gnew'])


def test_selective_scan_of_steps_that_forget_and_that_do_not_move(chx):
    """Steps so long that nothing is left of the state, so short that nothing is added, and gates at infinity."""
    c, more, _ = scan_case(2, 21, 5, 4, None, 'float32')
    c['delta'][:, 5] = 1e4
    c['delta'][:, 9] = -200
    c['z'][:, 3], c['z'][:, 4] = np.inf, -1e30
    dev = scan_on_device(chx, c, None, True)
    y, new = chx.selective_scan(**dev)
    c['z'][:, 3], c['z'][:, 4] = 1, -100  # what the plain form can say of the other rows
    (want, want_new), (size, new_size), n = ref.selective_scan(delta_softplus=True, **c)
    rows = [i for i in range(21) if i not in (3, 4)]
    # dt of 1e4 counts its roundings |dt a| times in the exponent of e^(-1e4 |a|) = 0: they move nothing, what follows is as exact as ever
    ref.assert_within(y.get()[:, rows], want[:, rows], size[:, rows], 21 * 60 + 60, 'y')
    ref.assert_within(new.get(), want_new, new_size, 21 * 60 + 60, 'state')
    assert not np.isnan(y.get()[:, 3]).any() and not y.get()[:, 4].any()


def test_selective_scan_of_sequences_far_apart(chx):
    """Sequences and rows whose distance in memory takes more than 31 bits."""
    c, more, _ = scan_case(2, 40, 70, 16, None, 'float16')
    dev = scan_on_device(chx, c, None, True)
    gy = up(chx, more['gy'])
    want, want_new = chx.selective_scan(**dev)
    grads = chx.selective_scan_grad(gy=gy, **dev)
    batch, row = 1 << 32, (1 << 26) - 2  # bytes
    buffer = chx._array.alloc_bytes(batch + 40 * row + 4096)
    for i, k in enumerate(('u', 'delta', 'z')):
        far = chx.ndarray(buffer, 512 * i, (2, 40, 70), (batch, row, 2), np.dtype('float16'))
        chx.routines._copy_into(far, dev[k])
        dev[k] = far
    got, new = chx.selective_scan(**dev)
    assert np.array_equal(got.get(), want.get()) and np.array_equal(new.get(), want_new.get())
    for a, b in zip(chx.selective_scan_grad(gy=gy, **dev), grads):
        assert (a is None) == (b is None) and (a is None or np.array_equal(a.get(), b.get()))


def test_selective_scan_of_a_single_row_of_any_stride(chx):
    """A unit axis' stride says nothing."""
    c, more, _ = scan_case(2, 1, 70, 16, None, 'float16')
    dev, gy = scan_on_device(chx, c, None, True), up(chx, more['gy'])
    want, want_new = chx.selective_scan(**dev)
    grads = chx.selective_scan_grad(gy=gy, **dev)
    for far in (1 << 40, -(1 << 40), 0):
        odd = dict(dev, **{k: chx.ndarray(dev[k]._buf, dev[k]._offset, dev[k].shape, (dev[k].strides[0], far, 2), dev[k].dtype) for k in ('u', 'delta', 'z', 'b', 'c')})
        got, new = chx.selective_scan(**odd)
        assert np.array_equal(got.get(), want.get()) and np.array_equal(new.get(), want_new.get())
        for a, b in zip(chx.selective_scan_grad(gy=gy, **odd), grads):
            assert (a is None) == (b is None) and (a is None or np.array_equal(a.get(), b.get()))


@pytest.mark.parametrize('seed', range(10))
def test_layers_of_drawn_sizes(chx, seed):
    rng = np.random.default_rng(1000 + seed)
    groups = int(rng.choice([1, 1, 2, 3]))
    batch, length, per = int(rng.integers(1, 9)), int(np.exp(rng.uniform(0, 5.5))), int(np.exp(rng.uniform(0, 4.5)))
    dtype, states, ragged = str(rng.choice(['float16', 'float32'])), int(rng.integers(1, 65)), bool(rng.random() < 0.5)
    sizes = (batch, length, per * groups, states, groups)
    c, more, lengths = scan_case(*sizes, dtype, seed=seed, ragged=ragged)
    dev = scan_on_device(chx, c, lengths, True)
    y, new = chx.selective_scan(**dev)
    (want, want_new), (size, new_size), n = ref.selective_scan(delta_softplus=True, lengths=lengths, **c)
    ref.assert_within(y.get(), want, size, n, '%s %s' % (sizes, dtype))
    ref.assert_within(new.get(), want_new, new_size, n, '%s %s state' % (sizes, dtype))
    grads = chx.selective_scan_grad(gy=apart(chx, more['gy']), gnew_state=up(chx, more['gnew']), **dev)
    wants, sizes_of, n = ref.selective_scan_grad(gy=more['gy'], gnew=more['gnew'], delta_softplus=True, lengths=lengths, **c)
    for k, got in grads._asdict().items():
        ref.assert_within(got.get(), wants[k].reshape(got.shape), sizes_of[k].reshape(got.shape), n, '%s %s: %s' % (sizes, dtype, k))
    taps = int(rng.integers(1, 9))
    c = conv_case(batch, length, per * groups, taps, dtype, seed=seed, ragged=ragged)
    x, w, b, state, ends = apart(chx, c['x']), up(chx, c['w']), up(chx, c['b']), up(chx, c['state']), up(chx, c['lengths'])
    y, new = chx.causal_conv(x, w, b, state=state, lengths=ends, activation='silu')
    want, size, want_new = ref.causal_conv(c['x'], c['w'], c['b'], c['state'], c['lengths'], 'silu')
    ref.assert_within(y.get(), want, size, 1, 'conv %s %s' % (sizes, taps))
    assert np.array_equal(new.get(), want_new.astype(dtype))
    grads = chx.causal_conv_grad(x, w, b, apart(chx, c['gy']), state=state, lengths=ends, activation='silu', gnew_state=up(chx, c['gnew']))
    for got, want, size in zip(grads, *ref.causal_conv_grad(c['x'], c['w'], c['b'], c['gy'], c['state'], c['lengths'], 'silu', c['gnew'])):
        ref.assert_within(got.get(), want, size, 1, 'conv %s %s gradients' % (sizes, taps))


# ---------------------------------------------------------------------------------------------
# streams, graphs, the layers together
# ---------------------------------------------------------------------------------------------
def block_params(chx, rng, units, inner, states, taps):
    n = lambda *s: (rng.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32)  # noqa: E731
    host = {'in_w': n(2 * inner, units), 'conv_w': n(inner, taps), 'conv_b': n(inner), 'step_w': n(inner, inner), 'step_b': n(inner) - 2, 'bc_w': n(2 * states, inner),
            'a': -np.exp(rng.standard_normal((inner, states))).astype(np.float32), 'd': n(inner), 'out_w': n(units, inner)}
    return {k: chx.array(v) for k, v in host.items()}


def block(chx, p, x, conv_state, scan_state, key, ratio=0.25):
    """linear -> causal convolution -> linears -> selective scan -> linear -> dropout, added to what went in."""
    batch, length, units = x.shape
    states = p['a'].shape[1]
    wide = chx.linear(x.reshape(batch * length, units), p['in_w']).reshape(batch, length, -1)
    inner = wide.shape[2] // 2
    h, conv_state = chx.causal_conv(wide[:, :, :inner], p['conv_w'], p['conv_b'], state=conv_state, activation='silu')
    rows = h.reshape(batch * length, inner)
    delta = chx.linear(rows, p['step_w']).reshape(h.shape)
    bc = chx.linear(rows, p['bc_w']).reshape(batch, length, 2 * states)
    y, scan_state = chx.selective_scan(h, delta, p['a'], bc[:, :, :states], bc[:, :, states:], p['d'], wide[:, :, inner:], p['step_b'], True, state=scan_state)
    out = chx.linear(y.reshape(batch * length, inner), p['out_w']).reshape(batch, length, units)
    return chx.dropout(out, ratio, key, site=1, residual=x), conv_state, scan_state


def test_block_prompt_then_tokens(chx):
    """A prompt and then token by token, as a server runs the layers, gives what the whole sequence gives (without dropout, whose mask goes by position)."""
    rng = np.random.default_rng(7)
    p, key = block_params(chx, rng, 24, 40, 16, 4), up(chx, KEY)
    x = chx.array(rng.standard_normal((3, 30, 24)).astype(np.float32))
    whole, _, _ = block(chx, p, x, None, None, key, 0.0)
    y, conv_state, scan_state = block(chx, p, x[:, :20], None, None, key, 0.0)
    ys = [y.get()]
    for t in range(20, 30):
        y, conv_state, scan_state = block(chx, p, x[:, t:t + 1], conv_state, scan_state, key, 0.0)
        ys.append(y.get())
    # products of 40 and 24 terms in other orders, and the scan's own roundings: far from any mistake in a row or a state
    np.testing.assert_allclose(np.concatenate(ys, 1), whole.get(), rtol=0, atol=1e-4)


def test_block_gradients_agree_with_differences(chx):
    """The layers' gradients chained by hand, in float32, against differences of the forward pass of the plain forms in 64 bits."""
    rng = np.random.default_rng(8)
    batch, length, channels, states, taps, ratio = 2, 23, 9, 5, 4, 0.5
    c, more, _ = scan_case(batch, length, channels, states, None, 'float32')
    cc = conv_case(batch, length, channels, taps, 'float32')
    gy, key = more['gy'], up(chx, KEY)
    x, w = up(chx, cc['x']), up(chx, cc['w'])
    dev = {k: up(chx, v) for k, v in c.items()}

    h, _ = chx.causal_conv(x, w, up(chx, cc['b']), activation='silu')
    dev['u'] = h
    y, _ = chx.selective_scan(delta_softplus=True, **dev)
    chx.dropout(y, ratio, key, site=4)
    g = chx.dropout(up(chx, gy), ratio, key, site=4)
    sg = chx.selective_scan_grad(gy=g, delta_softplus=True, **dev)
    gx, gw, gb, _ = chx.causal_conv_grad(x, w, up(chx, cc['b']), sg.u, activation='silu')

    def loss(**over):
        v = {**{k: cc[k].astype(np.float64) for k in ('x', 'w', 'b')}, **over}
        u = ref.causal_conv(v['x'], v['w'], v['b'], activation='silu')[0]
        scan = {k: over.get('scan_' + k, a.astype(np.float64)) for k, a in c.items()}
        scan['u'] = u
        out = ref.selective_scan(delta_softplus=True, **scan)[0][0]
        return (ref.dropout(out, ratio, KEY, 4) * gy).sum()

    for name, base, got in (('x', cc['x'], gx), ('w', cc['w'], gw), ('b', cc['b'], gb), ('scan_delta', c['delta'], sg.delta), ('scan_a', c['a'], sg.a), ('scan_b', c['b'], sg.b),
                            ('scan_c', c['c'], sg.c), ('scan_d', c['d'], sg.d), ('scan_z', c['z'], sg.z), ('scan_delta_bias', c['delta_bias'], sg.delta_bias), ('scan_state', c['state'], sg.state)):
        along = rng.standard_normal(base.shape)
        base, step = base.astype(np.float64), 1e-4
        change = (loss(**{name: base + step * along}) - loss(**{name: base - step * along})) / (2 * step)
        got = got.get().astype(np.float64)
        # differences are exact to step^2; a float32 gradient's elements to some 1e-6 of their size
        assert abs((got * along).sum() - change) <= 1e-4 * (np.abs(got * along).sum() + 1), name


def test_layers_replay_in_a_graph(chx):
    """The block and its gradients in a captured graph, replayed between eager calls of the same layers; a changed step draws another mask."""
    from chainer_amd import graph
    rng = np.random.default_rng(9)
    p, key = block_params(chx, rng, 24, 40, 16, 4), chx.array(KEY)
    x = chx.array(rng.standard_normal((3, 70, 24)).astype(np.float32))
    c, more, lengths = scan_case(2, 40, 24, 16, None, 'float16', seed=1, ragged=True)
    dev, gy = scan_on_device(chx, c, lengths, True), apart(chx, more['gy'])
    cc = conv_case(2, 40, 24, 4, 'float16')
    conv = [up(chx, cc[k]) for k in ('x', 'w', 'b', 'gy')]

    def step():
        return (block(chx, p, x, None, None, key) + tuple(g for g in chx.selective_scan_grad(gy=gy, **dev) if g is not None) +
                tuple(g for g in chx.causal_conv_grad(*conv, activation='silu') if g is not None))

    captured = graph.capture(step)
    first = None
    for i in range(4):
        captured.replay()
        chx.synchronize()
        got = [a.get() for a in captured.result]
        for a, b in zip(got, step()):
            assert np.array_equal(a, b.get())
        assert first is None or not np.array_equal(first, got[0])
        first = got[0]
        chx.add(key, chx.array(np.array([0, 1], np.int64)), out=key)  # the next step
    captured.release()


def test_layers_on_two_streams_at_once(chx):
    """Calls on another stream than the current one's usual, at the same time as others, have workspaces of their own."""
    import torch
    c, more, lengths = scan_case(4, 300, 40, 16, None, 'float32', seed=1, ragged=True)
    dev, gy = scan_on_device(chx, c, lengths, True), apart(chx, more['gy'])
    cc = conv_case(4, 300, 40, 4, 'float32')
    conv = [up(chx, cc[k]) for k in ('x', 'w', 'b', 'gy')]

    def everything():
        return [chx.selective_scan(**dev)[0]] + list(chx.selective_scan_grad(gy=gy, **dev)) + list(chx.causal_conv_grad(*conv))[:3]

    want = [a.get() for a in everything() if a is not None]
    chx.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append([a for a in everything() if a is not None])
    for s in streams:
        s.synchronize()
    for r in results:
        for a, w in zip(r, want):
            assert np.array_equal(a.get(), w)


def test_strides_that_repeat_and_run_backwards(chx):
    """Inputs broadcast over the batch and read backwards in time."""
    c, more, _ = scan_case(3, 20, 6, 4, None, 'float32')
    dev = {k: up(chx, v) for k, v in c.items()}
    for k in ('u', 'b', 'z'):
        c[k] = np.ascontiguousarray(np.broadcast_to(c[k][:1, ::-1], c[k].shape))
        dev[k] = dev[k][:1, ::-1].broadcast_to(c[k].shape)
    y, new = chx.selective_scan(delta_softplus=True, **dev)
    (want, want_new), (size, new_size), n = ref.selective_scan(delta_softplus=True, **c)
    ref.assert_within(y.get(), want, size, n, 'y')
    ref.assert_within(new.get(), want_new, new_size, n, 'state')
    cc = conv_case(3, 20, 6, 4, 'float32')
    x = chx.array(cc['x'])[:1, ::-1].broadcast_to(cc['x'].shape)
    cc['x'] = np.ascontiguousarray(np.broadcast_to(cc['x'][:1, ::-1], cc['x'].shape))
    want, size, _ = ref.causal_conv(cc['x'], cc['w'])
    ref.assert_within(chx.causal_conv(x, chx.array(cc['w']))[0].get(), want, size, 1, 'conv')


def test_language_model_with_dropout(chx):
    """The language model's forward pass with dropout before its layers, step by step against the oracle and masks in Python's integers."""
    from chainer_amd import configs as cfg
    from oracle import native as oracle

    class WithDropout(object):
        dropout = staticmethod(lambda x, ratio, key, site: ref.dropout(x, ratio, key, site).astype(x.dtype))

        def __getattr__(self, name):
            return getattr(oracle, name)

    p, ids = cfg.lstm_lm_params(vocab=50, units=20), cfg.lstm_lm_input(batch=3, seq=4, vocab=50)
    want, want_h, want_c = cfg.lstm_lm_forward(WithDropout(), p, ids, np.zeros, step=False, dropout=(0.5, KEY))
    plain, _, _ = cfg.lstm_lm_forward(oracle, p, ids, np.zeros, step=False)
    dev, key = cfg.tree_map(chx.array, p), up(chx, KEY)
    for step in (None, False):
        got, h, c = cfg.lstm_lm_forward(chx, dev, chx.array(ids), chx.zeros, step=step, dropout=(0.5, key))
        for a, b in zip([got] + h + c, [want] + want_h + want_c):
            # sums of 20 products of |weights| <= 0.05 through four steps: some dozens of roundings of values of at most 5
            np.testing.assert_allclose(a.get(), b, rtol=0, atol=64 * 2.0 ** -24 * 5)
        assert np.abs(got.get() - plain).max() > 1e-4
        none, _, _ = cfg.lstm_lm_forward(chx, dev, chx.array(ids), chx.zeros, step=step, dropout=(0.0, key))
        same, _, _ = cfg.lstm_lm_forward(chx, dev, chx.array(ids), chx.zeros, step=step)
        assert np.array_equal(none.get(), same.get())

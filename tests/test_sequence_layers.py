"""CPU tests of dropout, the causal convolution and the selective scan: what their entry points refuse, and the plain forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import sequence_reference as ref

F16, F32, F64, I32, I64 = 7, 8, 9, 4, 5
SIZE = {F16: 2, F32: 4, F64: 8, I32: 4, I64: 8}


def described(shape, dtype=F32, strides=None):
    """A descriptor of memory that is never read."""
    from chainer_amd import _lib
    if strides is None:
        strides, n = [], SIZE[dtype]
        for s in reversed(shape):
            strides.insert(0, n)
            n *= max(1, s)
    return _lib.CArray(0x10000, dtype, len(shape), (ctypes.c_int64 * 10)(*shape), (ctypes.c_int64 * 10)(*strides))


def refused(name, error, *args):
    """The entry point ends in `error` before it launches anything (this machine may have no device)."""
    from chainer_amd import _lib
    with pytest.raises(error) as e:
        _lib.call(name, *[ctypes.byref(a) if isinstance(a, _lib.CArray) else a for a in args], None)
    assert type(e.value) is error and str(e.value)


def errors():
    import chainer_amd as chx
    return chx.ChainerxError, chx.DimensionError, chx.DtypeError, chx.ChainerxNotImplementedError


def test_dropout_refusals():
    plain, dimension, dtype, missing = errors()
    x, key, out = described((4, 5)), described((2,), I64), described((4, 5))

    def call(error, x=x, ratio=0.5, key=key, site=0, residual=None, out=out):
        refused('hipcx_dropout', error, x, ratio, key, site, residual, out)

    for ratio in (-0.1, 1.0, 1.5, float('nan'), float('inf')):
        call(plain, ratio=ratio)
    for site in (-1, 1 << 32):
        call(plain, site=site)
    call(plain, x=None)
    call(plain, key=None)
    call(plain, out=None)
    call(dtype, x=described((4, 5), I32), out=described((4, 5), I32))
    call(dtype, out=described((4, 5), F16))
    call(dtype, residual=described((4, 5), F16))
    call(dtype, key=described((2,), I32))
    call(dimension, key=described((3,), I64))
    call(dimension, key=described((2,), I64, [16]))
    call(dimension, key=described((2, 1), I64))
    call(dimension, out=described((5, 4)))
    call(dimension, residual=described((5,)))
    call(dimension, x=described((4, 5), F32, [4, 16]))
    call(dimension, out=described((4, 5), F32, [40, 4]))
    call(missing, x=described((1 << 18, (1 << 17) + 1)), out=described((1 << 18, (1 << 17) + 1)))


def conv_arguments(batch=2, length=6, channels=5, taps=4, dtype=F32, **over):
    rows, window = described((batch, length, channels), dtype), described((batch, taps - 1, channels), dtype)
    args = {'x': rows, 'w': described((channels, taps), dtype), 'b': described((channels,), dtype), 'state': window, 'lengths': described((batch,), I32),
            'activation': 1, 'y': rows, 'new_state': window}
    assert set(over) <= set(args)
    args.update(over)
    return list(args.values())


CONV_REFUSALS = [('plain', dict(x=None)), ('plain', dict(w=None)), ('plain', dict(y=None)), ('plain', dict(new_state=None)), ('plain', dict(activation=2)), ('plain', dict(activation=-1)),
                 ('dtype', dict(x=described((2, 6, 5), F64))), ('dtype', dict(w=described((5, 4), F16))), ('dtype', dict(b=described((5,), F16))),
                 ('dtype', dict(state=described((2, 3, 5), F16))), ('dtype', dict(y=described((2, 6, 5), F16))), ('dtype', dict(lengths=described((2,), F32))),
                 ('dimension', dict(x=described((12, 5)))), ('dimension', dict(w=described((4, 5)))), ('dimension', dict(w=described((5, 4), F32, [4, 20]))),
                 ('dimension', dict(b=described((4,)))), ('dimension', dict(b=described((5,), F32, [8]))), ('dimension', dict(state=described((2, 4, 5)))),
                 ('dimension', dict(new_state=described((1, 3, 5)))), ('dimension', dict(y=described((2, 7, 5)))), ('dimension', dict(lengths=described((3,), I32))),
                 ('dimension', dict(x=described((2, 6, 5), F32, [240, 40, 8]))), ('dimension', dict(x=described((2, 6, 5), F32, [122, 20, 4]))),
                 ('dimension', dict(y=described((2, 6, 5), F32, [4, 8, 48])))]


@pytest.mark.parametrize('i', range(len(CONV_REFUSALS)))
def test_causal_conv_refusals(i):
    kind, over = CONV_REFUSALS[i]
    refused('hipcx_causal_conv', dict(zip(('plain', 'dimension', 'dtype', 'missing'), errors()))[kind], *conv_arguments(**over))


def test_causal_conv_takes_one_to_eight_taps():
    missing = errors()[3]
    refused('hipcx_causal_conv', missing, *conv_arguments(taps=9))
    refused('hipcx_causal_conv', missing, *conv_arguments(w=described((5, 0))))


def test_causal_conv_grad_refusals():
    plain, dimension, dtype, _ = errors()
    rows, w, b, window = described((2, 6, 5)), described((5, 4)), described((5,)), described((2, 3, 5))

    def call(error, x=rows, w=w, b=b, state=window, lengths=None, activation=1, gy=rows, gnew=window, gx=rows, gw=w, gb=b, gstate=window, workspace=0x20000,
             size=1 << 20):
        refused('hipcx_causal_conv_grad', error, x, w, b, state, lengths, activation, gy, gnew, gx, gw, gb, gstate, workspace, size)

    for name in ('x', 'w', 'gy', 'gx', 'gw'):
        call(plain, **{name: None})
    call(plain, size=16)
    call(plain, workspace=None)
    call(plain, activation=7)
    call(dtype, gy=described((2, 6, 5), F16))
    call(dtype, gw=described((5, 4), F16))
    call(dimension, gy=described((2, 5, 5)))
    call(dimension, gw=described((4, 5)))
    call(dimension, gw=described((5, 4), F32, [4, 20]))
    call(dimension, gstate=described((2, 4, 5)))
    call(dimension, gnew=described((2, 3, 4)))
    call(dimension, gb=described((6,)))


SCAN = ('u', 'delta', 'a', 'b', 'c', 'd', 'z', 'bias', 'softplus', 'state', 'lengths')


def scan_arguments(batch=2, length=6, channels=6, states=4, groups=None, dtype=F32, grad=False, **over):
    rows, shared = described((batch, length, channels), dtype), described((batch, length, states) if groups is None else (batch, length, groups, states), dtype)
    a, d, state = described((channels, states)), described((channels,)), described((batch, channels, states))
    args = {'u': rows, 'delta': rows, 'a': a, 'b': shared, 'c': shared, 'd': d, 'z': rows, 'bias': d, 'softplus': 1, 'state': state,
            'lengths': described((batch,), I64)}
    if grad:
        args.update(gy=rows, gnew=state, gu=rows, gdelta=rows, ga=a, gb=shared, gc=shared, gd=d, gz=rows, gbias=d, gstate=state, workspace=0x20000, size=1 << 24)
    else:
        args.update(y=rows, new_state=state, workspace=0x20000, size=1 << 24)
    assert set(over) <= set(args)
    args.update(over)
    return list(args.values())


SCAN_REFUSALS = [('plain', dict(u=None)), ('plain', dict(delta=None)), ('plain', dict(a=None)), ('plain', dict(b=None)), ('plain', dict(c=None)),
                 ('dtype', dict(u=described((2, 6, 6), F64))), ('dtype', dict(delta=described((2, 6, 6), F16))), ('dtype', dict(b=described((2, 6, 4), F16))),
                 ('dtype', dict(z=described((2, 6, 6), F16))), ('dtype', dict(a=described((6, 4), F16))), ('dtype', dict(d=described((6,), F16))),
                 ('dtype', dict(bias=described((6,), F64))), ('dtype', dict(state=described((2, 6, 4), F16))), ('dtype', dict(lengths=described((2,), F32))),
                 ('dimension', dict(u=described((12, 6)))), ('dimension', dict(a=described((4, 6)))), ('dimension', dict(b=described((2, 6)))),
                 ('dimension', dict(c=described((2, 6, 5)))), ('dimension', dict(c=described((2, 6, 1, 4)))), ('dimension', dict(d=described((5,)))),
                 ('dimension', dict(z=described((2, 5, 6)))), ('dimension', dict(state=described((2, 4, 6)))), ('dimension', dict(lengths=described((2, 1), I64))),
                 ('dimension', dict(delta=described((2, 6, 6), F32, [4, 8, 48]))), ('dimension', dict(a=described((6, 4), F32, [4, 24]))),
                 ('dimension', dict(state=described((2, 6, 4), F32, [4, 32, 8]))), ('dimension', dict(b=described((2, 6, 4), F32, [400, 50, 4])))]


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('i', range(len(SCAN_REFUSALS)))
def test_selective_scan_refusals(i, grad):
    kind, over = SCAN_REFUSALS[i]
    error = dict(zip(('plain', 'dimension', 'dtype', 'missing'), errors()))[kind]
    refused('hipcx_selective_scan_grad' if grad else 'hipcx_selective_scan', error, *scan_arguments(grad=grad, **over))


def test_selective_scan_limits():
    plain, dimension, dtype, missing = errors()
    for grad in (False, True):
        name = 'hipcx_selective_scan_grad' if grad else 'hipcx_selective_scan'
        refused(name, missing, *scan_arguments(grad=grad, states=65))
        refused(name, missing, *scan_arguments(grad=grad, a=described((6, 0))))
        refused(name, dimension, *scan_arguments(grad=grad, groups=4))  # of 6 channels
        refused(name, dimension, *scan_arguments(grad=grad, groups=0))
        for far in (1 << 28, -(1 << 28)):  # bytes from a row to the next
            for k in ('u', 'delta', 'z'):
                refused(name, missing, *scan_arguments(grad=grad, **{k: described((2, 6, 6), F32, [24, far, 4])}))
        refused(name, missing, *scan_arguments(grad=grad, c=described((2, 6, 4), F32, [24, 1 << 28, 4])))
    refused('hipcx_selective_scan', plain, *scan_arguments(y=None))
    refused('hipcx_selective_scan', plain, *scan_arguments(new_state=None))
    refused('hipcx_selective_scan', dtype, *scan_arguments(new_state=described((2, 6, 4), F16)))
    refused('hipcx_selective_scan', dimension, *scan_arguments(new_state=described((2, 6, 4), F32, [4, 32, 8])))
    refused('hipcx_selective_scan', dimension, *scan_arguments(y=described((2, 7, 6))))
    for name in ('gy', 'gu', 'gdelta', 'ga', 'gb', 'gc', 'gz', 'z'):
        refused('hipcx_selective_scan_grad', plain, *scan_arguments(grad=True, **{name: None}))
    refused('hipcx_selective_scan_grad', plain, *scan_arguments(grad=True, size=64))
    refused('hipcx_selective_scan_grad', plain, *scan_arguments(grad=True, workspace=None))
    refused('hipcx_selective_scan', missing, *scan_arguments(y=described((2, 6, 6), F32, [24, 1 << 28, 4])))
    refused('hipcx_selective_scan_grad', missing, *scan_arguments(grad=True, gu=described((2, 6, 6), F32, [24, 1 << 28, 4])))
    refused('hipcx_selective_scan_grad', dimension, *scan_arguments(grad=True, gb=described((2, 6, 4), F32, [200, 32, 4])))
    refused('hipcx_selective_scan_grad', dtype, *scan_arguments(grad=True, ga=described((6, 4), F16)))
    refused('hipcx_selective_scan_grad', dimension, *scan_arguments(grad=True, gstate=described((2, 4, 6))))


# ---------------------------------------------------------------------------------------------
# the plain forms themselves
# ---------------------------------------------------------------------------------------------
def test_philox_known_answers():
    """The known-answer vectors that the generator's authors publish with it (Random123, kat_vectors: philox4x32, 10 rounds)."""
    ones = 0xFFFFFFFF
    assert ref.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.philox((ones, ones, ones, ones), (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert ref.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def _differences(f, x, gy, step=1e-5):
    """The gradient of sum(f(x) * gy) by central differences."""
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        g[i] = sum(((p - m) * w).sum() for p, m, w in zip(f(up), f(down), gy)) / (2 * step)
    return g


@pytest.mark.parametrize('activation', [None, 'silu'])
def test_causal_conv_gradients_agree_with_differences(activation):
    rng = np.random.default_rng(3)
    x, w, b, state = rng.standard_normal((3, 4, 2)), rng.standard_normal((2, 3)), rng.standard_normal(2), rng.standard_normal((3, 2, 2))
    lengths = [4, 0, 1]
    gy, gnew = rng.standard_normal(x.shape), rng.standard_normal(state.shape)
    got = ref.causal_conv_grad(x, w, b, gy, state, lengths, activation, gnew)[0]
    values = dict(x=x, w=w, b=b, state=state)
    for name, g in zip(('x', 'w', 'b', 'state'), got):
        f = lambda v: ref.causal_conv(**dict(values, **{name: v}), lengths=lengths, activation=activation)[::2]  # noqa: E731
        np.testing.assert_allclose(g, _differences(f, values[name], (gy, gnew)), rtol=1e-6, atol=1e-8, err_msg=name)


@pytest.mark.parametrize('softplus,gate,groups', [(True, True, 1), (False, False, 2), (True, False, None)])
def test_selective_scan_gradients_agree_with_differences(softplus, gate, groups):
    rng = np.random.default_rng(4)
    n = lambda *s: rng.standard_normal(s)  # noqa: E731
    shared = (3, 4, 2) if groups is None else (3, 4, groups, 2)
    values = dict(u=n(3, 4, 2), delta=n(3, 4, 2) * 0.3, a=-np.exp(n(2, 2)), b=n(*shared), c=n(*shared), d=n(2), z=n(3, 4, 2) if gate else None, delta_bias=n(2) * 0.1,
                  state=n(3, 2, 2))
    more = dict(delta_softplus=softplus, lengths=[4, 0, 2])
    gy, gnew = n(3, 4, 2), n(3, 2, 2)
    got = ref.selective_scan_grad(gy=gy, gnew=gnew, **values, **more)[0]
    for name, v in values.items():
        if v is None:
            continue
        f = lambda v: ref.selective_scan(**dict(values, **{name: v}), **more)[0]  # noqa: E731
        np.testing.assert_allclose(got[name].reshape(v.shape), _differences(f, v, (gy, gnew)), rtol=1e-6, atol=1e-8, err_msg=name)

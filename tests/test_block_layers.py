"""CPU tests of layer norm, linear attention and AdamW: what their entry points refuse, the workspaces they ask for, and the plain forms that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_sequence_layers import F16, F32, F64, I32, I64, SIZE, described, errors, refused

U8 = 6
SIZE[U8] = 1
KINDS = ('plain', 'dimension', 'dtype', 'missing')


# ---------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------
def norm_arguments(grad, dtype=F32, **over):
    rows, cols, stats = described((3, 4, 5), dtype), described((5,), dtype), described((3, 4), F64 if dtype == F64 else F32)
    args = {'x': rows, 'gamma': cols, 'beta': cols, 'eps': 1e-5, 'y': rows, 'mean': stats, 'inv_std': stats}
    if grad:
        args = {'x': rows, 'gamma': cols, 'gy': rows, 'mean': stats, 'inv_std': stats, 'gx': rows, 'ggamma': cols, 'gbeta': cols, 'workspace': 0x20000, 'size': 1 << 24}
    assert set(over) <= set(args)
    args.update(over)
    return list(args.values())


NORM_REFUSALS = [('plain', dict(eps=-1e-5)), ('plain', dict(eps=float('nan'))), ('plain', dict(eps=float('inf'))), ('plain', dict(x=None)), ('plain', dict(y=None)), ('plain', dict(mean=None)),
                 ('plain', dict(inv_std=None)), ('dtype', dict(x=described((3, 4, 5), I32), y=described((3, 4, 5), I32))), ('dtype', dict(y=described((3, 4, 5), F16))),
                 ('dtype', dict(gamma=described((5,), F16))), ('dtype', dict(beta=described((5,), F64))), ('dtype', dict(mean=described((3, 4), F16))),
                 ('dimension', dict(y=described((4, 3, 5)))), ('dimension', dict(y=described((3, 4, 5), F32, [80, 16, 4]))), ('dimension', dict(gamma=described((4,)))),
                 ('dimension', dict(gamma=described((1, 5)))), ('dimension', dict(beta=described((5,), F32, [8]))), ('dimension', dict(mean=described((4, 3)))),
                 ('dimension', dict(inv_std=described((3, 4), F32, [4, 12]))), ('dimension', dict(x=described((3, 4, 5), F32, [160, 40, 8]))),
                 ('dimension', dict(x=described((3, 4, 5), F32, [100, 20, 4]))), ('dimension', dict(x=described((3, 4, 5), F32, [88, 22, 4]))),
                 ('dimension', dict(x=described((), F32))), ('dimension', dict(x=described((3, 0)), y=described((3, 0)), mean=described((3,)), inv_std=described((3,)), gamma=None, beta=None))]
NORM_GRAD_REFUSALS = [('plain', dict(workspace=None)), ('plain', dict(size=39)), ('plain', dict(workspace=0x20004)), ('plain', dict(gy=None)), ('plain', dict(gx=None)), ('plain', dict(x=None)),
                      ('dtype', dict(gy=described((3, 4, 5), F16))), ('dtype', dict(ggamma=described((5,), F16))), ('dtype', dict(gx=described((3, 4, 5), F64))),
                      ('dimension', dict(gy=described((3, 5, 4)))), ('dimension', dict(gx=described((3, 4, 5), F32, [20, 60, 4]))), ('dimension', dict(gbeta=described((6,)))),
                      ('dimension', dict(mean=described((12,)))), ('dimension', dict(gy=described((3, 4, 5), F32, [100, 20, 4])))]


@pytest.mark.parametrize('i', range(len(NORM_REFUSALS)))
def test_layer_norm_refusals(i):
    kind, over = NORM_REFUSALS[i]
    refused('hipcx_layer_norm', dict(zip(KINDS, errors()))[kind], *norm_arguments(False, **over))


@pytest.mark.parametrize('i', range(len(NORM_GRAD_REFUSALS)))
def test_layer_norm_grad_refusals(i):
    kind, over = NORM_GRAD_REFUSALS[i]
    refused('hipcx_layer_norm_grad', dict(zip(KINDS, errors()))[kind], *norm_arguments(True, **over))


def test_layer_norm_parameters_share_a_type():
    for over in (dict(gamma=described((5,), F16), beta=described((5,), F32)), dict(gamma=described((5,), F32), beta=described((5,), F16))):
        refused('hipcx_layer_norm', errors()[2], *norm_arguments(False, F16, **over))
    refused('hipcx_layer_norm_grad', errors()[2], *norm_arguments(True, F16, ggamma=described((5,), F32)))


def test_layer_norm_workspaces():
    from chainer_amd import _lib
    size = lambda *a: _lib.load().hipcx_layer_norm_grad_workspace_size(ctypes.byref(described(*a)))  # noqa: E731
    for shape in ((1, 1), (4480, 650), (16384, 4096), (2, 3, 100000), (1 << 20, 3)):
        for dtype, item in ((F16, 4), (F32, 4), (F64, 8)):
            n = size(shape, dtype)
            assert n > 0 and n % (2 * shape[-1] * item) == 0 and n <= 2048 * shape[-1] * 2 * item
    for bad in (((), F32), ((3, 0), F32), ((0, 3), F32), ((3, 4), I32), ((3, 1 << 41), F32)):
        assert size(*bad) == 0


def differences(f, a, step=1e-5):
    out = np.zeros(a.shape)
    for at in np.ndindex(*a.shape):
        was, sums = a[at], []
        for s in (step, -step):
            a[at] = was + s
            sums.append(f())
        a[at] = was
        out[at] = (sums[0] - sums[1]) / (2 * step)
    return out


def test_layer_norm_gradients_agree_with_differences():
    rng = np.random.default_rng(1)
    x, gamma, beta, gy = rng.standard_normal((4, 7)), rng.standard_normal(7), rng.standard_normal(7), rng.standard_normal((4, 7))
    grads, _ = ref.layer_norm_grad(x, gamma, gy, 1e-3)
    loss = lambda: (ref.layer_norm(x, gamma, beta, 1e-3)[0]['y'] * gy).sum()  # noqa: E731
    for name, a in (('gx', x), ('ggamma', gamma), ('gbeta', beta)):
        assert np.abs(differences(loss, a) - grads[name]).max() < 1e-7


# ---------------------------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------------------------
def attend_arguments(grad, dtype=F32, batch=2, length=70, key_heads=2, heads=4, keys=6, values=10, **over):
    of_keys, of_values = described((batch, length, key_heads, keys), dtype), described((batch, length, heads, values), dtype)
    decay, state = described((batch, length, heads)), described((batch, heads, keys, values))
    args = {'q': of_keys, 'k': of_keys, 'v': of_values, 'log_decay': decay, 'scale': 0.5, 'state': state, 'lengths': described((batch,), I32)}
    if grad:
        args.update(gy=of_values, gnew=state, gq=of_keys, gk=of_keys, gv=of_values, glog_decay=decay, gstate=state, workspace=0x20000, size=1 << 30)
    else:
        args.update(y=of_values, new_state=state, workspace=0x20000, size=1 << 30)
    assert set(over) <= set(args)
    args.update(over)
    return list(args.values())


Q, V, S = (2, 70, 2, 6), (2, 70, 4, 10), (2, 4, 6, 10)
ATTEND_REFUSALS = [('plain', dict(q=None)), ('plain', dict(k=None)), ('plain', dict(v=None)), ('plain', dict(scale=float('nan'))), ('plain', dict(scale=1e39)),
                   ('dtype', dict(q=described(Q, F64))), ('dtype', dict(k=described(Q, F16))), ('dtype', dict(v=described(V, F16))), ('dtype', dict(log_decay=described((2, 70, 4), F16))),
                   ('dtype', dict(state=described(S, F16))), ('dtype', dict(lengths=described((2,), F32))),
                   ('dimension', dict(q=described((140, 2, 6)))), ('dimension', dict(k=described((2, 70, 2, 5)))), ('dimension', dict(v=described((2, 69, 4, 10)))),
                   ('dimension', dict(v=described((3, 70, 4, 10)))), ('dimension', dict(v=described((2, 70, 3, 10)))), ('dimension', dict(v=described((2, 70, 0, 10)))),
                   ('dimension', dict(log_decay=described((2,)))), ('dimension', dict(log_decay=described((2, 70)))), ('dimension', dict(log_decay=described((2, 70, 4), F32, [1120, 16, 6]))),
                   ('dimension', dict(state=described((2, 2, 6, 10)))), ('dimension', dict(state=described(S, F32, [960, 240, 4, 24]))), ('dimension', dict(lengths=described((3,), I64))),
                   ('dimension', dict(q=described(Q, F32, [3360, 48, 4, 8]))), ('dimension', dict(v=described(V, F32, [11200, 160, 40, 8]))),
                   ('dimension', dict(k=described(Q, F32, [3362, 48, 24, 4]))), ('missing', dict(q=described(Q, F32, [4 << 24, 4 << 24, 24, 4]))),
                   ('missing', dict(v=described(V, F32, [-(4 << 24), -(4 << 24), 40, 4])))]


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('i', range(len(ATTEND_REFUSALS)))
def test_linear_attention_refusals(i, grad):
    kind, over = ATTEND_REFUSALS[i]
    refused('hipcx_linear_attention_grad' if grad else 'hipcx_linear_attention', dict(zip(KINDS, errors()))[kind], *attend_arguments(grad, **over))


def test_linear_attention_refuses_results_that_do_not_fit():
    plain, dimension, dtype, missing = errors()
    for over, error in ((dict(y=None), plain), (dict(new_state=None), plain), (dict(y=described(V, F16)), dtype), (dict(y=described(Q)), dimension), (dict(new_state=described((2, 4, 10, 6))), dimension),
                        (dict(new_state=described(S, F32, [960, 240, 4, 24])), dimension), (dict(y=described(V, F32, [11200, 160, 4, 16])), dimension)):
        refused('hipcx_linear_attention', error, *attend_arguments(False, **over))
    for over, error in ((dict(gy=None), plain), (dict(gq=None), plain), (dict(gk=None), plain), (dict(gv=None), plain), (dict(log_decay=None), plain), (dict(workspace=None), plain),
                        (dict(size=15), plain), (dict(workspace=0x20004), plain), (dict(gq=described(Q, F16)), dtype), (dict(glog_decay=described((2, 70, 4), F16)), dtype),
                        (dict(gv=described(Q)), dimension), (dict(glog_decay=described((4,))), dimension), (dict(glog_decay=described((2, 70, 4), F32, [1120, 4, 280])), dimension),
                        (dict(gstate=described((2, 4, 10, 6))), dimension), (dict(gnew=described(S, F32, [960, 240, 4, 24])), dimension),
                        (dict(gk=described(Q, F32, [4 << 24, 4 << 24, 24, 4])), missing)):
        refused('hipcx_linear_attention_grad', error, *attend_arguments(True, **over))


def test_linear_attention_limits():
    missing = errors()[3]
    for grad in (False, True):
        name = 'hipcx_linear_attention_grad' if grad else 'hipcx_linear_attention'
        refused(name, missing, *attend_arguments(grad, keys=257))
        refused(name, missing, *attend_arguments(grad, values=257))
        refused(name, missing, *attend_arguments(grad, keys=0))
        refused(name, missing, *attend_arguments(grad, length=1 << 30))
        refused(name, missing, *attend_arguments(grad, key_heads=1, heads=1 << 20))
        refused(name, missing, *attend_arguments(grad, batch=1 << 24))


def test_linear_attention_workspaces():
    from chainer_amd import _lib
    lib = _lib.load()

    def sizes(q, v, decay=True, padded=False, dtype=F32):
        q, v = described(q, dtype), described(v, dtype)
        g, n = ctypes.byref(described((v.shape[0], v.shape[1], v.shape[2]))) if decay else None, ctypes.byref(described((v.shape[0],), I32)) if padded else None
        return (lib.hipcx_linear_attention_workspace_size(ctypes.byref(q), ctypes.byref(v), n), lib.hipcx_linear_attention_grad_workspace_size(ctypes.byref(q), ctypes.byref(v), g, n))

    assert sizes((128, 1, 16, 128), (128, 1, 16, 128))[0] == 0  # next tokens take none
    forward, grad = sizes((1, 16384, 16, 128), (1, 16384, 16, 128))
    assert forward % (16 * 4 * (128 * 128 + 1)) == 0 and forward > 0  # (segments are counted for each by itself)
    assert sizes((1, 16384, 16, 128), (1, 16384, 16, 128), False)[1] < grad < sizes((1, 16384, 4, 128), (1, 16384, 16, 128))[1]
    assert sizes((1, 16384, 16, 128), (1, 16384, 16, 128), padded=True)[0] % (16 * 4 * (128 * 128 + 1)) == 0
    assert sizes((1, 16384, 16, 128), (1, 16384, 16, 128), dtype=F64) == (0, 0)
    for q, v in (((2, 70, 2, 257), (2, 70, 4, 10)), ((2, 70, 2, 6), (2, 70, 3, 10)), ((2, 70, 2, 6), (2, 71, 4, 10)), ((70, 2, 6), (2, 70, 4, 10)), ((2, 1 << 30, 2, 6), (2, 1 << 30, 4, 10))):
        assert sizes(q, v) == (0, 0)


@pytest.mark.parametrize('share,heads_decay', [(1, False), (2, True)])
def test_linear_attention_gradients_agree_with_differences(share, heads_decay):
    rng = np.random.default_rng(2)
    b, l, h, n, m = 2, 5, 2, 3, 2
    a = {'q': rng.standard_normal((b, l, h // share, n)), 'k': rng.standard_normal((b, l, h // share, n)), 'v': rng.standard_normal((b, l, h, m)),
         'log_decay': -np.exp(rng.standard_normal((h,) if heads_decay else (b, l, h))), 'state': rng.standard_normal((b, h, n, m))}
    gy, gnew, lengths = rng.standard_normal((b, l, h, m)), rng.standard_normal((b, h, n, m)), np.array([3, 5])

    def loss():
        (y, new), _ = ref.linear_attention(a['q'], a['k'], a['v'], a['log_decay'], 0.7, a['state'], lengths)
        return (y * gy).sum() + (new * gnew).sum()

    grads, _, _ = ref.linear_attention_grad(a['q'], a['k'], a['v'], gy, a['log_decay'], 0.7, a['state'], lengths, gnew)
    for name, x in a.items():
        assert np.abs(differences(loss, x) - grads[name]).max() < 1e-7, name


# ---------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------
def adamw(error, arrays, t=1, t_array=None, alpha=0.1, beta1=0.9, beta2=0.999, eps=1e-8, eta=1.0, decay=0.0):
    """``arrays``: of (parameter, gradient, m, v, m_scale, v_scale, master)."""
    from chainer_amd import _lib
    lists = []
    for column in zip(*arrays):
        pointers = (ctypes.POINTER(_lib.CArray) * len(column))()
        for i, a in enumerate(column):
            if a is not None:
                pointers[i] = ctypes.pointer(a)
        lists.append(pointers)
    with pytest.raises(error) as e:
        _lib.call('hipcx_adamw_many', *lists, len(arrays), t, None if t_array is None else ctypes.byref(t_array), alpha, beta1, beta2, eps, eta, decay, 0, None)
    assert type(e.value) is error and str(e.value)


def at(place, shape, dtype=F32, strides=None):
    a = described(shape, dtype, strides)
    a.data = 0x100000 * (1 + place)
    return a


def one(bits=32, dtype=F32, place=0, **over):
    n, state, scale = (1000,), F32 if bits == 32 else U8, None if bits == 32 else (4,)
    names = ('p', 'g', 'm', 'v', 'm_scale', 'v_scale', 'master')
    args = dict(zip(names, [at(place, n, dtype), at(place + 1, n, dtype), at(place + 2, n, state), at(place + 3, n, state), scale and at(place + 4, scale), scale and at(place + 5, scale), None]))
    assert set(over) <= set(args)
    args.update(over)
    return [args[name] for name in names]


def test_adamw_refusals():
    plain, dimension, dtype, missing = errors()
    nan, inf = float('nan'), float('inf')
    for over in (dict(t=0), dict(t=-3), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(beta2=nan), dict(eps=-1e-8), dict(eps=inf), dict(alpha=nan), dict(eta=inf), dict(decay=nan)):
        adamw(plain, [one()], **over)
    adamw(dtype, [one()], t_array=at(9, (1,), I32))
    adamw(dimension, [one()], t_array=at(9, (2,), I64))
    for name in 'pgmv':
        adamw(plain, [one(**{name: None})])
    for over in (dict(p=at(0, (1000,), F64), g=at(1, (1000,), F64)), dict(g=at(1, (1000,), F16)), dict(m=at(2, (1000,), F16)), dict(v=at(3, (1000,), U8)), dict(master=at(6, (1000,)))):
        adamw(dtype, [one(**over)])
    adamw(dtype, [one(dtype=F16, master=at(6, (1000,), F16))])
    for over in (dict(g=at(1, (10, 100))), dict(m=at(2, (999,))), dict(v=at(3, (1001,))), dict(p=at(0, (1000,), F32, [8])), dict(m=at(2, (1000,), F32, [-4]))):
        adamw(dimension, [one(**over)])
    adamw(dimension, [one(dtype=F16, master=at(6, (999,)))])
    for over, error in ((dict(m_scale=None), plain), (dict(v_scale=None), plain), (dict(m_scale=at(4, (3,))), dimension), (dict(v_scale=at(5, (4, 1))), dimension), (dict(v_scale=at(5, (4,), F16)), dtype),
                        (dict(v=at(3, (1000,))), dtype)):
        adamw(error, [one(8, **over)])
    adamw(plain, [one(m_scale=at(4, (4,)))])
    big = (1 << 33) + 1
    adamw(missing, [one(p=at(0, (big,)), g=at(1, (big,)), m=at(2, (big,)), v=at(3, (big,)))])
    adamw(dimension, [one(), one(place=10, g=at(11, (5,)))])  # a later one of several


def test_adamw_refuses_what_shares_memory():
    plain = errors()[0]
    inside = lambda place, offset, *a: setattr_data(at(place, *a), offset)  # noqa: E731

    def setattr_data(a, offset):
        a.data += offset
        return a

    adamw(plain, [one(), one()])
    adamw(plain, [one(g=at(0, (1000,)))])
    adamw(plain, [one(m=at(3, (1000,)))])
    adamw(plain, [one(), one(place=10, p=inside(0, 3996, (1000,)))])
    adamw(plain, [one(), one(place=10, g=inside(2, 400, (1000,)))])
    adamw(plain, [one(), one(8, place=10, m_scale=inside(3, 8, (4,)))])
    adamw(plain, [one(8, v_scale=at(4, (4,)))])

"""The selective scan and its gradients within bounds that every element has for itself (sequence_bounds.py), and sequences that end inside a chunk, where the batch is one sequence too."""
import numpy as np
import pytest

import sequence_bounds as bounds
import sequence_reference as ref
from test_gpu_sequence_layers import SCANS, apart, conv_case, scan_case, scan_on_device, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


def ends_inside(batch, length, seed):
    """A sequence by itself ends in the middle, inside a tile; of several the first is whole and one is empty."""
    if batch == 1:
        n = max(1, length * 5 // 8)
        return np.array([n + 5 if n % 16 == 0 and n + 5 < length else n], np.int32)
    n = np.random.default_rng(seed).integers(1, length + 1, batch)
    n[batch // 2], n[0] = 0, length
    return n


VARIANTS = [('all', (), True, False), ('ragged', ('state',), True, True), ('bare', ('d', 'z', 'delta_bias', 'state'), False, False), ('no gate', ('z',), True, False),
            ('no gate, ragged', ('z', 'd'), True, True)]
MORE = [(2, 333, 130, 16, None), (1, 610, 66, 12, 2), (300, 18, 5, 16, None), (260, 9, 6, 3, 2), (131, 21, 190, 24, 1), (258, 17, 3, 64, None)]


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('sizes', SCANS + MORE)
def test_selective_scan(chx, sizes, dtype):
    batch, length = sizes[:2]
    for i, (name, without, softplus, ragged) in enumerate(VARIANTS):
        c, more, _ = scan_case(*sizes, dtype, seed=10 + i)
        c = {k: None if k in without else v for k, v in c.items()}
        if not softplus:
            c['delta'] = np.abs(c['delta']) / 4
        gy, gnew, lengths = more['gy'], more['gnew'] if i % 2 == 0 else None, None
        if ragged:
            lengths = ends_inside(batch, length, i)
            outside = ~ref.inside(ref.ends_of(lengths, batch, length), length)[..., 0]
            for v in [c[k] for k in ('u', 'delta', 'b', 'c', 'z') if c[k] is not None] + [gy]:
                v[outside] = np.nan
        what = '%s %s %s: ' % (sizes, dtype, name)
        dev = scan_on_device(chx, c, lengths, softplus)
        y, new = chx.selective_scan(**dev)
        wants = bounds.selective_scan(c, softplus, lengths)
        for k, got in (('y', y), ('state', new)):
            assert wants[k][0].any()
            bounds.assert_close(got.get(), *wants[k], what + k)
        grads = chx.selective_scan_grad(gy=apart(chx, gy), gnew_state=up(chx, gnew), **dev)
        wants = bounds.selective_scan_grad(c, gy, gnew, softplus, lengths)
        for k, got in grads._asdict().items():
            assert (got is None) == (c[k] is None), k
            if got is not None:
                assert wants[k][0].any() or k in ('a', 'state')  # (of one row that starts from zeros, or forgets them)
                bounds.assert_close(got.get(), *wants[k], what + 'g' + k)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('activation', [None, 'silu'])
@pytest.mark.parametrize('sizes', [(1, 300, 650, 4), (1, 1000, 3, 6), (1, 40, 8, 3), (1, 77, 24, 8), (1, 90, 13, 1)])
def test_causal_conv_of_one_sequence_that_ends_inside(chx, sizes, activation, dtype):
    batch, length, channels, taps = sizes
    c = conv_case(*sizes, dtype, seed=3)
    lengths = ends_inside(batch, length, 0)
    for k in ('x', 'gy'):
        c[k][0, lengths[0]:] = np.nan
    args = [apart(chx, c['x']), up(chx, c['w']), up(chx, c['b'])]
    more = dict(state=up(chx, c['state']), lengths=up(chx, lengths), activation=activation)
    y, new = chx.causal_conv(*args, **more)
    want, size, want_new = ref.causal_conv(c['x'], c['w'], c['b'], c['state'], lengths, activation)
    assert want.any()
    ref.assert_within(y.get(), want, size, 1, 'y')
    assert np.array_equal(new.get(), want_new.astype(dtype))
    grads = chx.causal_conv_grad(*args, apart(chx, c['gy']), gnew_state=up(chx, c['gnew']), **more)
    for name, got, want, size in zip(('gx', 'gw', 'gb', 'gstate'), grads, *ref.causal_conv_grad(c['x'], c['w'], c['b'], c['gy'], c['state'], lengths, activation, c['gnew'])):
        assert want.any() or taps == 1
        ref.assert_within(got.get(), want, size, 1, name)


@pytest.mark.parametrize('groups', [None, 2])
@pytest.mark.parametrize('states', range(1, 65))
def test_selective_scan_of_every_number_of_states(chx, states, groups):
    """Lanes that have not enough states for themselves: whole and padded, moved forward in place, in chunks."""
    for i, length in enumerate((21, 100)):
        c, _, _ = scan_case(3, length, 6, states, groups, 'float32', seed=states + i)
        lengths = ends_inside(3, length, states)
        outside = ~ref.inside(ref.ends_of(lengths, 3, length), length)[..., 0]
        for k in ('u', 'delta', 'b', 'c', 'z'):
            c[k][outside] = np.nan
        state = chx.array(c['state'])
        y, new = chx.selective_scan(**dict(scan_on_device(chx, c, lengths, True), state=state, out_state=state))
        wants = bounds.selective_scan(c, True, lengths)
        assert new is state
        bounds.assert_close(y.get(), *wants['y'], 'y')
        bounds.assert_close(new.get(), *wants['state'], 'state')

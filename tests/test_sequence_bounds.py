"""The bounds of sequence_bounds.py: 32-bit arithmetic is within them, and results with a mistake are not."""
import numpy as np
import pytest

import sequence_bounds as bounds
import sequence_reference as ref

F = np.float32


def case(batch, length, channels, states, seed=0, gate=True):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(F)  # noqa: E731
    c = {'u': f(batch, length, channels), 'delta': f(batch, length, channels), 'a': -np.exp(f(channels, states)), 'b': f(batch, length, states), 'c': f(batch, length, states),
         'd': f(channels), 'z': f(batch, length, channels) if gate else None, 'delta_bias': f(channels) - 2, 'state': f(batch, channels, states)}
    return c, f(batch, length, channels), f(batch, channels, states)


SIZES = [(1, 700, 20, 16), (1, 300, 5, 64), (20, 35, 50, 16), (2, 130, 16, 5)]


def in_32_bits(c, gy, gnew):
    """Outputs and gradients row by row in float32."""
    raw = c['delta'] + c['delta_bias']
    e = np.exp(-np.abs(raw))
    s = e / (2 + e)
    dt = np.maximum(raw, 0) + 2 * np.arctanh(s)
    logistic = lambda x: 1 / (1 + np.exp(-x))  # noqa: E731
    gate = c['z'] * logistic(c['z']) if c['z'] is not None else np.ones_like(raw)
    length = raw.shape[1]
    decay, x = np.exp(dt[..., None] * c['a']), dt * c['u']
    hs, h = [c['state']], c['state']
    for t in range(length):
        h = decay[:, t] * h + x[:, t, :, None] * c['b'][:, t, None]
        hs.append(h)
    y0 = np.stack([(hs[t + 1] * c['c'][:, t, None]).sum(2) for t in range(length)], 1) + c['d'] * c['u']
    out = {'y': y0 * gate, 'state': h}
    g0 = gy * gate
    g = {k: np.zeros_like(v) for k, v in c.items() if v is not None}
    if c['z'] is not None:
        l = logistic(c['z'])
        g['z'] = gy * l * (1 + c['z'] * (1 - l)) * y0
    q, gdt = gnew, np.zeros_like(gy)
    for t in reversed(range(length)):
        q = q + g0[:, t, :, None] * c['c'][:, t, None]
        g['c'][:, t] = (g0[:, t, :, None] * hs[t + 1]).sum(1)
        g['b'][:, t] = (q * x[:, t, :, None]).sum(1)
        qb = (q * c['b'][:, t, None]).sum(2)
        q = q * decay[:, t]
        p = q * hs[t]
        g['a'] += (dt[:, t, :, None] * p).sum(0)
        g['u'][:, t] = c['d'] * g0[:, t] + dt[:, t] * qb
        gdt[:, t] = (p * c['a']).sum(2) + c['u'][:, t] * qb
    g['delta'] = gdt * logistic(raw)
    g['d'], g['delta_bias'], g['state'] = (g0 * c['u']).sum((0, 1)), g['delta'].sum((0, 1)), q
    assert all(v.dtype == F for v in list(g.values()) + list(out.values()))
    return out, g


@pytest.mark.parametrize('gate', [True, False])
@pytest.mark.parametrize('sizes', SIZES)
def test_32_bits_are_within(sizes, gate):
    c, gy, gnew = case(*sizes, gate=gate)
    out, g = in_32_bits(c, gy, gnew)
    for wants, gots in ((bounds.selective_scan(c, True), out), (bounds.selective_scan_grad(c, gy, gnew, True), g)):
        for k, (want, error) in wants.items():
            bounds.assert_close(gots[k], want, error, k)
            bounds.assert_close(want.astype(np.float16), want, error, k) if np.abs(want).max() < 6e4 else None


def test_values_are_the_plain_forms():
    c, gy, gnew = case(3, 20, 6, 5)
    lengths = np.array([20, 0, 13])
    (y, new), _, _ = ref.selective_scan(delta_softplus=True, lengths=lengths, **c)
    got = bounds.selective_scan(c, True, lengths)
    np.testing.assert_allclose(got['y'][0], y, rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(got['state'][0], new, rtol=1e-12, atol=1e-13)
    wants = ref.selective_scan_grad(gy=gy, gnew=gnew, delta_softplus=True, lengths=lengths, **c)[0]
    got = bounds.selective_scan_grad(c, gy, gnew, True, lengths)
    assert set(got) == {k for k, v in wants.items() if v is not None}
    for k, (value, _) in got.items():
        np.testing.assert_allclose(value, wants[k], rtol=1e-12, atol=1e-12, err_msg=k)


def rejected(got, want, what):
    with pytest.raises(AssertionError):
        bounds.assert_close(got.astype(F), *want, what)


def within_elements(got, want):
    """As many elements as pass one by one, of all."""
    value, error = want
    return (np.abs(got - value) <= error + 2.0 ** -126).mean()


@pytest.mark.parametrize('sizes', SIZES[:3])
def test_mistakes_are_not(sizes):
    c, gy, gnew = case(*sizes)
    batch, length = sizes[:2]
    outs, grads = bounds.selective_scan(c, True), bounds.selective_scan_grad(c, gy, gnew, True)
    for k, want in list(outs.items()) + list(grads.items()):
        rejected(np.zeros_like(want[0]), want, k)
        if k not in ('delta', 'z', 'u', 'y'):  # (gradients of some rows are next to nothing)
            assert within_elements(0, want) < 0.02, k
        assert within_elements(0, want) < 0.1, k
        rejected(want[0] * (1 + 1e-4), want, k)

    # a state that is 1 % off where a chunk of 32 rows begins
    state, ys = c['state'].astype(np.float64), []
    for t in range(0, length, 32):
        piece = {k: (v[:, t:t + 32] if k in ('u', 'delta', 'b', 'c', 'z') else v) for k, v in c.items()}
        piece['state'] = state * (1.01 if t else 1)
        (y, state), _, _ = ref.selective_scan(delta_softplus=True, **piece)
        ys.append(y)
    rejected(np.concatenate(ys, 1), outs['y'], 'a carry')
    assert within_elements(np.concatenate(ys, 1)[:, 32:36], [v[:, 32:36] for v in outs['y']]) < 0.5

    # the gradients without a softplus' slope, and a chunk's part of a sum over rows that is missing
    raw = c['delta'].astype(np.float64) + c['delta_bias']
    rejected(grads['delta'][0] / ref.logistic(raw), grads['delta'], 'no slope')
    rejected(grads['delta'][0][:, 32:].sum((0, 1)), grads['delta_bias'], 'rows missing')
    rejected((grads['delta'][0] / ref.logistic(raw)).sum((0, 1)), grads['delta_bias'], 'no slope')
    short = {k: (v[:, 32:] if k in ('u', 'delta', 'b', 'c', 'z') else v) for k, v in c.items()}
    short['state'] = ref.selective_scan(delta_softplus=True, **{k: (v[:, :32] if k in ('u', 'delta', 'b', 'c', 'z') else v) for k, v in c.items()})[0][1]
    if length > 32:
        rejected(bounds.selective_scan_grad(short, gy[:, 32:], gnew, True)['a'][0], grads['a'], 'rows missing')

    # steps in half precision
    rough = dict(c, delta=raw.astype(np.float16).astype(np.float64), delta_bias=None)
    (y, new), _, _ = ref.selective_scan(delta_softplus=True, **rough)
    rejected(y, outs['y'], 'half')
    rejected(new, outs['state'], 'half')

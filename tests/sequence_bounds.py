"""How far the selective scan and its gradients, in 32 bits, may be from their plain forms in 64 (sequence_reference.py), for every element by itself.

A row's errors go through the recurrence with the row's own decays: what is forgotten takes its error along.  `A` and `Q` are the recurrences of the absolute values, which bound a state, or its
gradient, wherever a chunk of the time axis begins; `E` and `F` are how far they may be off.  Errors are counted in units of U, half a step of float32; products of two errors are left out (they are
below 1e-4 of what is counted, whose counts are rounded up by more).

  exp2 and the reciprocal of the transcendental unit are within a step (2); the softplus of x takes (its argument rounded: |x|; the exponential's: the factor log2 e 0.22 |x|, the product |x|;
  the exponential 2; 2 + e 1, the reciprocal 2, the product 1; the series 2, the sum 1) less than 10 + 4 |x|; the logistic 8 + 2.5 |x|, 3.5 |x| where its argument is a rounded sum
"""
import numpy as np

import sequence_reference as ref
from sequence_reference import U32 as U

NORM = 1e-5  # of the 2-norm: 168 U.  A term passes through some dozens of roundings, of either sign, which add up like their squares; those of a sum over rows do so too


def _terms(c, softplus, lengths):
    c = dict(c)
    t = ref._scan_terms(c['u'], c['delta'], c['a'], c['b'], c['c'], c.get('d'), c.get('z'), c.get('delta_bias'), softplus, c.get('state'), lengths)
    raw = np.abs(t['raw'])
    t['of_dt'] = 10 + 4 * raw if softplus else np.ones_like(raw)
    t['x'] = t['dt'] * t['u']
    t['of_decay'] = np.where(t['keep'][..., None], np.abs(t['dt'][..., None] * t['a']) * (t['of_dt'][..., None] + 4) + 3, 0)
    if c.get('z') is not None:
        t['z'] = np.where(t['keep'], np.nan_to_num(c['z'].astype(np.float64)), 0)
    return t


def _states(t):
    """States, the recurrence of their absolute values, and their errors, from before the first row on."""
    h, size, error = [t['h0']], [np.abs(t['h0'])], [np.zeros_like(t['h0'])]
    for i in range(t['u'].shape[1]):
        decay, b = t['decay'][:, i], t['b'][:, i]
        xb = t['x'][:, i, :, None] * b
        h.append(h[-1] * decay + xb)
        size.append(size[-1] * decay + np.abs(xb))
        error.append(decay * (error[-1] + t['of_decay'][:, i] * U * size[-2]) + np.abs(xb) * (t['of_dt'][:, i, :, None] + 2) * U + np.where(t['keep'][:, i, :, None], U * size[-1], 0))
    return [np.stack(v, 1) for v in (h, size, error)]


def _outputs(t, h, size, error):
    """y before the gate, and its error."""
    n = t['a'].shape[1]
    y0 = (h[:, 1:] * t['c']).sum(3) + t['d'] * t['u']
    y0_size = (size[:, 1:] * np.abs(t['c'])).sum(3) + np.abs(t['d'] * t['u'])
    return y0, (error[:, 1:] * np.abs(t['c'])).sum(3) + (n // 4 + 8) * U * y0_size


def selective_scan(c, softplus, lengths=None):
    """{'y': (value, error), 'state': (value, error)}"""
    t = _terms(c, softplus, lengths)
    h, size, error = _states(t)
    y, y_error = _outputs(t, h, size, error)
    if t['gate'] is not None:
        y, y_error = y * t['gate'], np.abs(t['gate']) * y_error + (2.5 * np.abs(t['z']) + 9) * U * np.abs(y * t['gate'])
    keep = t['keep']
    return {'y': (np.where(keep, y, 0), np.where(keep, y_error, 0)), 'state': (h[:, -1], error[:, -1])}


def selective_scan_grad(c, gy, gnew, softplus, lengths=None):
    """{name: (value, error)}; b and c [batch, time, groups, states]"""
    t = _terms(c, softplus, lengths)
    keep = t['keep']
    h, size, error = _states(t)
    y0, y0_error = _outputs(t, h, size, error)
    batch, length, channels = t['u'].shape
    n, ab, out = t['a'].shape[1], np.abs, {}
    gy = np.where(keep, gy.astype(np.float64), 0)
    q = np.zeros_like(t['h0']) if gnew is None else gnew.astype(np.float64)
    if t['gate'] is None:
        g0, g0_error = gy, np.zeros_like(gy)
    else:
        z, l = t['z'], ref.logistic(t['z'])
        g0 = gy * t['gate']
        g0_error = (2.5 * ab(z) + 9) * U * ab(g0)
        slope_error = l * (1 + ab(z)) * (2.5 * ab(z) + 10) * U  # of l (1 + z (1 - l)): 1 - l is off by what l is
        out['z'] = (gy * y0 * t['gate_slope'], ab(gy) * (slope_error * ab(y0) + ab(t['gate_slope']) * (y0_error + 2 * U * ab(y0))))
    # sums over rows, one after another and then chunk by chunk, and over the channels of a wave, of a workgroup and of all
    of_rows, of_channels = length + batch + 8, 12 + channels // 64
    qs, qf = ab(q), np.zeros_like(q)
    rows = {k: np.zeros_like(gy) for k in ('u', 'u_error', 'dt', 'dt_error')}
    shared = {k: np.zeros(t['b'].shape) for k in ('b', 'b_error', 'c', 'c_error')}
    ga, ga_error = np.zeros(t['a'].shape), np.zeros(t['a'].shape)
    for i in reversed(range(length)):
        g, gf, dt, x = (v[:, i, :, None] for v in (g0, g0_error, t['dt'], t['x']))
        u, of_dt, b, c_ = t['u'][:, i], t['of_dt'][:, i], t['b'][:, i], t['c'][:, i]
        q = q + g * c_
        qs = qs + ab(g * c_)
        qf = qf + gf * ab(c_) + U * qs * keep[:, i, :, None]
        shared['c'][:, i] = g * h[:, i + 1]
        shared['c_error'][:, i] = ab(g) * error[:, i + 1] + gf * size[:, i + 1] + (1 + of_channels) * U * ab(g) * size[:, i + 1]
        shared['b'][:, i] = q * x
        shared['b_error'][:, i] = qf * ab(x) + (of_dt[..., None] + 2 + of_channels) * U * qs * ab(x)
        qb, qb_size = (q * b).sum(2), (qs * ab(b)).sum(2)
        qb_error = (qf * ab(b)).sum(2) + (n // 4 + 6) * U * qb_size
        decay = t['decay'][:, i]
        q, qf, qs = q * decay, decay * (qf + t['of_decay'][:, i] * U * qs), qs * decay
        p, p_size = q * h[:, i], qs * size[:, i]
        p_error = qf * size[:, i] + qs * error[:, i] + U * p_size
        ga += (dt * p).sum(0)
        ga_error += (ab(dt) * (p_error + (of_dt[..., None] + 1 + of_rows) * U * p_size)).sum(0)
        rows['u'][:, i] = t['d'] * g[..., 0] + dt[..., 0] * qb
        rows['u_error'][:, i] = ab(t['d']) * gf[..., 0] + ab(dt[..., 0]) * (qb_error + (of_dt + 2) * U * qb_size) + 2 * U * ab(t['d'] * g[..., 0])
        rows['dt'][:, i] = (p * t['a']).sum(2) + u * qb
        rows['dt_error'][:, i] = (p_error * ab(t['a'])).sum(2) + (n // 4 + 10) * U * (p_size * ab(t['a'])).sum(2) + ab(u) * (qb_error + 2 * U * qb_size)
    slope = ref.logistic(t['raw']) if softplus else np.ones_like(t['raw'])
    of_slope = 3.5 * ab(t['raw']) + 9 if softplus else 0
    gdelta = np.where(keep, rows['dt'] * slope, 0)
    gdelta_error = np.where(keep, rows['dt_error'] * slope + of_slope * U * ab(gdelta), 0)
    fold = lambda v: v.reshape(batch, length, t['groups'], channels // t['groups'], -1).sum(3)  # noqa: E731
    out.update(u=(rows['u'], rows['u_error']), delta=(gdelta, gdelta_error), a=(ga, ga_error), b=(fold(shared['b']), fold(shared['b_error'])), c=(fold(shared['c']), fold(shared['c_error'])),
               state=(q, qf), d=((g0 * t['u']).sum((0, 1)), ((g0_error + (1 + of_rows) * U * ab(g0)) * ab(t['u'])).sum((0, 1))),
               delta_bias=(gdelta.sum((0, 1)), (gdelta_error + of_rows * U * ab(gdelta)).sum((0, 1))))
    return out


def assert_close(got, want, error, what):
    """Every element within its error, and all together within NORM of their 2-norm; both and a rounding to got's type."""
    got, dtype = np.asarray(got).astype(np.float64), np.asarray(got).dtype
    want, error = want.reshape(got.shape), error.reshape(got.shape)
    half, tiny = (0, 2.0 ** -126) if dtype == np.float32 else (ref.half_step(dtype), 2.0 ** -25 + 2.0 ** -126)
    limit = error + half * (np.abs(want) + error) + tiny
    bad = ~(np.abs(got - want) <= limit)
    assert not bad.any(), '%s: %d of %d off; first %r, expected %r within %.3g' % (what, bad.sum(), bad.size, got[bad][0], want[bad][0], limit[bad][0])
    off, norm = np.linalg.norm(got - want), np.linalg.norm(want)
    assert off <= (NORM + half) * norm + tiny * np.sqrt(got.size), '%s: off by %.3g of its 2-norm' % (what, off / norm)

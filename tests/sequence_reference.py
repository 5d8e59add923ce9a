"""Plain forms in 64 bits of dropout, the causal convolution and the selective scan, their gradients, and how far 32-bit arithmetic may be from them.

Every linear operation is computed twice: on the values and on their absolute values ("size").  A sum of products in any order, each of whose terms has gone through
`n` roundings of relative size 2^-24, is at most n * 2^-24 * size from the exact one; `n` is counted beside each function.
"""
import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return np.finfo(dtype).eps / 2


def assert_within(got, ref, size, roundings, what):
    """|got - ref| <= roundings * 2^-24 * size, and a rounding to got's type (subnormal results: half of their step)."""
    got, dtype = np.asarray(got).astype(np.float64), np.asarray(got).dtype
    assert got.shape == ref.shape, '%s: shape %r, expected %r' % (what, got.shape, ref.shape)
    limit = roundings * U32 * size
    if dtype == np.float16:
        limit = limit + half_step(dtype) * (np.abs(ref) + limit) + 2.0 ** -25
    limit = limit + np.finfo(np.float32).tiny
    good = np.abs(got - ref) <= limit
    if dtype == np.float16:  # from 65520 on (65504 and half a step) a value rounds to infinity
        good |= (got == np.copysign(np.inf, ref)) & (np.abs(ref) + limit >= 65520)
    bad = ~good
    assert not bad.any(), '%s: %d of %d off; first %r, expected %r within %.3g' % (
        what, bad.sum(), bad.size, got[bad][0], ref[bad][0], limit[bad][0])


def logistic(x):
    return 0.5 * (1 + np.tanh(0.5 * x))


def ends_of(lengths, batch, length):
    return np.full(batch, length) if lengths is None else np.clip(np.asarray(lengths, np.int64), 0, length)


def inside(ends, length):
    return (np.arange(length)[None] < ends[:, None])[..., None]


# ---------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------
def threshold(ratio):
    return min(65535, int(np.floor(ratio * 65536 + 0.5)))


def philox(counter, key):
    """Philox4x32-10 of one counter (four words) and key (two), in Python's integers."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k[0], q & low, (p >> 32) ^ c[3] ^ k[1], p & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def kept(n, ratio, key, site, first=0):
    """Elements first .. first + n - 1 that are kept; first is a multiple of 8."""
    seed, step = (int(v) & 0xFFFFFFFFFFFFFFFF for v in key)
    words = [philox((i, site, step & 0xFFFFFFFF, step >> 32), (seed & 0xFFFFFFFF, seed >> 32)) for i in range(first // 8, first // 8 + (n + 7) // 8)]
    bits = np.array(words, np.uint64)
    return np.stack([bits & np.uint64(0xFFFF), bits >> np.uint64(16)], 2).reshape(-1)[:n] >= threshold(ratio)


def dropout(x, ratio, key, site=0, residual=None):
    y = np.where(kept(x.size, ratio, key, site).reshape(x.shape), x.astype(np.float64) * 65536 / (65536 - threshold(ratio)), 0)
    return y if residual is None else y + residual.astype(np.float64)


# ---------------------------------------------------------------------------------------------
# the causal convolution
# ---------------------------------------------------------------------------------------------
def _conv_inputs(x, w, state, lengths):
    b, length, d = x.shape
    ends = ends_of(lengths, b, length)
    clean = np.where(inside(ends, length), x.astype(np.float64), 0)
    before = np.zeros((b, w.shape[1] - 1, d)) if state is None else state.astype(np.float64)
    return ends, np.concatenate([before, clean], 1)


def _conv_sums(rows, w, b, length):
    s = np.zeros((rows.shape[0], length, rows.shape[2])) + b
    for k in range(w.shape[1]):
        s += rows[:, k:k + length] * w[:, k]
    return s


def causal_conv(x, w, b=None, state=None, lengths=None, activation=None):
    """(y, its size, new state).  A sum of taps + 1 terms takes taps roundings a term, of which the logistic of it makes at most (1 + |s|) times as many and adds
    2 |s| + 6 of its own: its argument has two, its exponential and reciprocal are within a step, its sum and the product are rounded."""
    ends, rows = _conv_inputs(x, w, state, lengths)
    w64, b64 = w.astype(np.float64), 0.0 if b is None else b.astype(np.float64)
    s = _conv_sums(rows, w64, b64, x.shape[1])
    size = _conv_sums(np.abs(rows), np.abs(w64), np.abs(b64), x.shape[1])
    taps = w.shape[1]
    if activation is not None:
        size = size * logistic(s) * (taps * (1 + np.abs(s)) + 2 * np.abs(s) + 6)
        s = s * logistic(s)
    else:
        size = size * taps
    keep = inside(ends, x.shape[1])
    new = np.stack([rows[i, n:n + taps - 1] for i, n in enumerate(ends)]) if len(ends) else rows[:, :taps - 1]
    return np.where(keep, s, 0), np.where(keep, size, 0), new


def causal_conv_grad(x, w, b, gy, state=None, lengths=None, activation=None, gnew=None):
    """(gx, gw, gb, gstate), and their sizes with the roundings counted in; gb and gstate of zeros for what is not given."""
    ends, rows = _conv_inputs(x, w, state, lengths)
    batch, length, d = x.shape
    taps = w.shape[1]
    w64, b64 = w.astype(np.float64), 0.0 if b is None else b.astype(np.float64)
    gp = np.where(inside(ends, length), gy.astype(np.float64), 0)
    gp_size = np.abs(gp)
    if activation is not None:
        s = _conv_sums(rows, w64, b64, length)
        size = _conv_sums(np.abs(rows), np.abs(w64), np.abs(b64), length)
        l = logistic(s)
        # the slope l (1 + s (1 - l)): its own derivative is below 1/2; the sum's taps roundings of `size`, and 2 |s| + 12 of the slope's terms
        gp_size = gp_size * (0.5 * taps * size + (2 * np.abs(s) + 12) * l * (1 + np.abs(s) * (1 - l)))
        gp = gp * l * (1 + s * (1 - l))
    else:
        gp_size = gp_size * 1

    def around(g, weights, last):
        out = np.zeros((batch, length + taps - 1, d))
        for k in range(taps):
            out[:, k:k + length] += g * weights[:, k]
        if last is not None:
            for i, n in enumerate(ends):
                out[i, n:n + taps - 1] += last[i]
        return out

    grows = around(gp, w64, None if gnew is None else gnew.astype(np.float64))
    size = around(gp_size + (taps + 1) * np.abs(gp), np.abs(w64), None if gnew is None else (taps + 1) * np.abs(gnew.astype(np.float64)))
    # sums over rows: at most 64 in a thread, 256 threads' of a workgroup, four chains over the parts
    n = 64 + 256 + batch * (length // 8 + 1) // 4 + 4
    gw, gw_size = np.zeros((d, taps)), np.zeros((d, taps))
    for k in range(taps):
        gw[:, k] = (gp * rows[:, k:k + length]).sum((0, 1))
        gw_size[:, k] = ((gp_size + n * np.abs(gp)) * np.abs(rows[:, k:k + length])).sum((0, 1))
    return ((grows[:, taps - 1:], gw, gp.sum((0, 1)), grows[:, :taps - 1]),
            (size[:, taps - 1:], gw_size, (gp_size + n * np.abs(gp)).sum((0, 1)), size[:, :taps - 1]))


# ---------------------------------------------------------------------------------------------
# the selective scan
# ---------------------------------------------------------------------------------------------
def _scan_terms(u, delta, a, b, c, d, z, bias, softplus, state, lengths):
    batch, length, channels = u.shape
    ends = ends_of(lengths, batch, length)
    keep = inside(ends, length)
    f = lambda v: np.where(keep if v.ndim == 3 else keep[..., None], v.astype(np.float64), 0)  # noqa: E731
    if b.ndim == 3:
        b, c = b[:, :, None], c[:, :, None]
    per_channel = lambda v: np.repeat(f(v), channels // v.shape[2], 2)  # noqa: E731
    raw = f(delta) + (0.0 if bias is None else bias.astype(np.float64))
    dt = np.where(keep, np.logaddexp(0, raw) if softplus else raw, 0)
    t = {'u': f(u), 'dt': dt, 'raw': raw, 'a': a.astype(np.float64), 'b': per_channel(b), 'c': per_channel(c), 'd': np.zeros(channels) if d is None else d.astype(np.float64),
         'h0': np.zeros((batch, channels, a.shape[1])) if state is None else state.astype(np.float64), 'keep': keep, 'groups': b.shape[2], 'softplus': softplus}
    t['decay'] = np.exp(dt[..., None] * t['a'])
    t['gate'] = t['gate_slope'] = None
    if z is not None:
        l = logistic(f(z))
        t['gate'], t['gate_slope'] = f(z) * l, l * (1 + f(z) * (1 - l))
    # Roundings that a step adds to a term: the product with the decay and the sum, and the decay's own -- dt has 9 of the softplus and |raw| of its argument, dt a
    # two more, all of which count |dt a| times, and the exponential is within a step (2).
    m, r = np.abs(dt[..., None] * t['a']).max(initial=0), np.abs(raw).max(initial=0)
    t['a_step'] = 4 + m * (11 + r)
    t['of_dt'] = 9 + r
    return t


def _sizes(t):
    s = dict(t)
    for k in ('u', 'dt', 'a', 'b', 'c', 'd', 'h0', 'gate', 'gate_slope'):
        if s[k] is not None:
            s[k] = np.abs(s[k])
    return s


def _states(t):
    h = np.zeros((t['u'].shape[1] + 1,) + t['h0'].shape)
    h[0] = t['h0']
    for i in range(t['u'].shape[1]):
        h[i + 1] = h[i] * t['decay'][:, i] + (t['dt'][:, i] * t['u'][:, i])[..., None] * t['b'][:, i]
    return np.moveaxis(h, 0, 1)


def _scan_outputs(t, h):
    y0 = (h[:, 1:] * t['c']).sum(3) + t['d'] * t['u']
    return y0, np.where(t['keep'], y0 if t['gate'] is None else y0 * t['gate'], 0), h[:, -1]


def selective_scan(u, delta, a, b, c, d=None, z=None, delta_bias=None, delta_softplus=False, state=None, lengths=None):
    """((y, new state), (their sizes), roundings)."""
    t = _scan_terms(u, delta, a, b, c, d, z, delta_bias, delta_softplus, state, lengths)
    h = _states(t)
    s = _sizes(t)
    _, y, new = _scan_outputs(t, h)
    _, y_size, new_size = _scan_outputs(s, _states(s))
    # the steps, dt u b and its place in the sum, the sum over states and d u, the gate (its argument 2 |z|, the logistic 6, two products)
    n = u.shape[1] * t['a_step'] + t['of_dt'] + a.shape[1] + 16 + (0 if z is None else 2 * np.abs(np.nan_to_num(z.astype(np.float64))).max(initial=0))
    return (y, new), (y_size, new_size), n


def _scan_gradients(t, h, y0, gy, gnew):
    """Of the values in `t`; given their sizes, the sizes."""
    batch, length, channels = t['u'].shape
    g0 = gy if t['gate'] is None else gy * t['gate']
    out = {'z': None if t['gate'] is None else gy * y0 * t['gate_slope'], 'd': (g0 * t['u']).sum((0, 1))}
    q = gnew.copy()
    gu, gdt, gb, gc = np.zeros_like(gy), np.zeros_like(gy), np.zeros_like(t['b']), np.zeros_like(t['c'])
    ga = np.zeros(t['a'].shape)
    for i in reversed(range(length)):
        q = q + g0[:, i, :, None] * t['c'][:, i]
        gc[:, i] = g0[:, i, :, None] * h[:, i + 1]
        gb[:, i] = q * (t['dt'][:, i] * t['u'][:, i])[..., None]
        qb = (q * t['b'][:, i]).sum(2)
        q = q * t['decay'][:, i]
        x = q * h[:, i]
        ga += (t['dt'][:, i, :, None] * x).sum(0)
        gu[:, i] = t['d'] * g0[:, i] + t['dt'][:, i] * qb
        gdt[:, i] = (x * t['a']).sum(2) + t['u'][:, i] * qb
    gdelta = np.where(t['keep'], gdt * (logistic(t['raw']) if t['softplus'] else 1), 0)
    groups = t['groups']
    fold = lambda v: v.reshape(batch, length, groups, channels // groups, -1).sum(3)  # noqa: E731
    out.update(u=gu, delta=gdelta, a=ga, b=fold(gb), c=fold(gc), delta_bias=gdelta.sum((0, 1)), state=q)
    return out


def selective_scan_grad(u, delta, a, b, c, gy, d=None, z=None, delta_bias=None, delta_softplus=False, state=None, lengths=None, gnew=None):
    """(gradients by name, their sizes, roundings); of b and c [batch, time, groups, states]."""
    t = _scan_terms(u, delta, a, b, c, d, z, delta_bias, delta_softplus, state, lengths)
    s = _sizes(t)
    gy = np.where(t['keep'], gy.astype(np.float64), 0)
    gnew = np.zeros_like(t['h0']) if gnew is None else gnew.astype(np.float64)
    h, h_size = _states(t), _states(s)
    grads = _scan_gradients(t, h, _scan_outputs(t, h)[0], gy, gnew)
    sizes = _scan_gradients(s, h_size, _scan_outputs(s, h_size)[0], np.abs(gy), np.abs(gnew))
    batch, length, channels = u.shape
    zmax = 0 if z is None else np.abs(np.nan_to_num(z.astype(np.float64))).max(initial=0)
    # the steps there and back, the terms as above, the sums over states, over rows (a thread's, then over sequences and chunks) and over channels
    n = 2 * length * t['a_step'] + 2 * t['of_dt'] + a.shape[1] + 32 + 4 * zmax + length + batch + 64 + channels // 64
    return grads, sizes, n

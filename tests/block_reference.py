"""Plain forms in 64 bits of layer norm and linear attention and their gradients, with how far 32-bit arithmetic may be from them, and AdamW operation by operation in 32 bits.

As in sequence_reference.py every sum is computed on the values and on their absolute values ("size"); a sum of products whose terms go through `n` roundings of 2^-24 is at most
n * 2^-24 * size from the exact one.  The matrix pipe may round an addition by a whole step, so its additions count twice.
"""
import numpy as np

from sequence_reference import U32, ends_of, inside

ab = np.abs


# ---------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------
def layer_norm(x, gamma, beta, eps, u=U32):
    """({'y', 'mean', 'inv_std'}, how far each may be off before its rounding to a type).

    The sums of a row go through at most 64 additions a term, and one for every 1024 columns beyond: `k`.  The first mean's error is taken out by the second sum, whose terms are rounded differences;
    the variance is off by k + 4 roundings, its root by half of them."""
    x = x.astype(np.float64)
    k = 64 + x.shape[-1] // 1024
    mean = x.mean(-1, keepdims=True)
    d = x - mean
    inv = 1 / np.sqrt((d * d).mean(-1, keepdims=True) + eps)
    xh = d * inv
    g = 1.0 if gamma is None else gamma.astype(np.float64)
    b = 0.0 if beta is None else beta.astype(np.float64)
    y = xh * g + b
    of_xh = u * ((k / 2 + 8) * ab(xh) + (k + 2) * ab(xh).mean(-1, keepdims=True))
    off = {'y': of_xh * ab(g) + u * (2 * ab(xh * g) + 2 * ab(y)), 'mean': u * (2 * ab(mean) + (k + 2) * ab(d).mean(-1, keepdims=True))[..., 0], 'inv_std': u * (k / 2 + 6) * inv[..., 0]}
    return {'y': y, 'mean': mean[..., 0], 'inv_std': inv[..., 0]}, off


def layer_norm_grad(x, gamma, gy, eps, u=U32):
    """({'gx', 'ggamma', 'gbeta'}, how far off): with a state whose mean and inverse deviation are rounded."""
    cols = x.shape[-1]
    value, off = layer_norm(x, None, None, eps, u)
    x, gy = x.reshape(-1, cols).astype(np.float64), gy.reshape(-1, cols).astype(np.float64)
    k = 64 + cols // 1024
    inv, mean = value['inv_std'].reshape(-1, 1), value['mean'].reshape(-1, 1)
    xh = value['y'].reshape(-1, cols)
    of_xh = off['y'].reshape(-1, cols) + (off['mean'].reshape(-1, 1) * inv + off['inv_std'].reshape(-1, 1) / inv * ab(xh))
    gw = 1.0 if gamma is None else gamma.astype(np.float64)
    g = gy * gw
    m = lambda v: v.mean(1, keepdims=True)  # noqa: E731
    a, b = m(g), m(g * xh)
    of_a = u * (k + 3) * m(ab(g))
    of_b = u * (k + 3) * m(ab(g * xh)) + m(ab(g) * of_xh)
    inner = g - a - xh * b
    of_inner = u * (2 * ab(g) + 2 * ab(a) + 3 * ab(xh * b) + 2 * ab(inner)) + of_a + ab(xh) * of_b + of_xh * ab(b)
    gx = inv * inner
    of_gx = inv * of_inner + (off['inv_std'].reshape(-1, 1) + u * inv) * ab(inner)
    n = 40 + x.shape[0] // 128  # a workgroup's rows one after another, its threads', then in 64 bits
    out = {'gx': gx, 'ggamma': (gy * xh).sum(0), 'gbeta': gy.sum(0)}
    return out, {'gx': of_gx, 'ggamma': (ab(gy) * of_xh + n * u * ab(gy * xh)).sum(0), 'gbeta': n * u * ab(gy).sum(0)}


def assert_off(got, want, off, what):
    """|got - want| <= off, and a rounding to got's type (subnormal results: half of their step)."""
    got, dtype = np.asarray(got).astype(np.float64), np.asarray(got).dtype
    assert got.shape == want.shape, '%s: shape %r, expected %r' % (what, got.shape, want.shape)
    half = 0.0 if dtype == np.float64 else np.finfo(dtype).eps / 2
    tiny = {'float16': 2.0 ** -25, 'float32': 2.0 ** -126, 'float64': 2.0 ** -1000}[dtype.name]
    limit = off + half * (ab(want) + off) + tiny
    bad = ~(ab(got - want) <= limit)
    if dtype == np.float16:  # from 65520 on (65504 and half a step) a value rounds to infinity
        bad &= ~((got == np.copysign(np.inf, want)) & (ab(want) + limit >= 65520))
    assert not bad.any(), '%s: %d of %d off; first %r, expected %r within %.3g' % (what, bad.sum(), bad.size, got[bad][0], want[bad][0], limit[bad][0])


# ---------------------------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------------------------
def _per_head(x, heads):
    return np.repeat(x, heads // x.shape[2], 2)


def _attend_inputs(q, k, v, log_decay, lengths):
    b, l, h = v.shape[:3]
    ends = ends_of(lengths, b, l)
    keep = inside(ends, l)[..., None]
    f = lambda x: np.where(keep, x.astype(np.float64), 0)  # noqa: E731
    g = np.zeros((b, l, h))
    if log_decay is not None:
        g = np.where(keep[..., 0], np.broadcast_to(log_decay.astype(np.float64), (b, l, h)), 0)
    return f(_per_head(q, h)), f(_per_head(k, h)), f(v), g, keep


def _states(k, v, g, state):
    s = [state]
    for t in range(k.shape[1]):
        s.append(s[-1] * np.exp(g[:, t])[..., None, None] + k[:, t][..., :, None] * v[:, t][..., None, :])
    return s


def _roundings(q, v, g):
    """Of a term: the product of q and k and the one with v on the matrix pipe (a reduction's additions, twice), a state's tile by tile, the tiles' decays, and what exponents lose: their sums
    are as good as a float's, and a decay by 2^-150 leaves nothing.  float16's products with two parts leave out 2^-22 of each of three factors."""
    l = v.shape[1]
    total = min(150.0, float(ab(g).sum(1).max(initial=0)) * 1.45)
    return 2 * (q.shape[3] + v.shape[3] + 128) + 8 * (l // 64 + 2) + 24 + 2 * total


def linear_attention(q, k, v, log_decay=None, scale=None, state=None, lengths=None):
    """((y, new state), (how far each may be off))"""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    q, k, v, g, keep = _attend_inputs(q, k, v, log_decay, lengths)
    state = np.zeros((v.shape[0], v.shape[2], k.shape[3], v.shape[3])) if state is None else state.astype(np.float64)

    def outputs(q, k, v, state, scale):
        s = _states(k, v, g, state)
        return np.stack([(q[:, t][..., :, None] * s[t + 1]).sum(2) * scale for t in range(q.shape[1])], 1) if q.shape[1] else np.zeros(v.shape), s[-1]

    n = _roundings(q, v, g)
    y, new = outputs(q, k, v, state, scale)
    y_size, new_size = outputs(ab(q), ab(k), ab(v), ab(state), ab(scale))
    return (np.where(keep, y, 0), new), (n * U32 * np.where(keep, y_size, 0), n * U32 * new_size)


def linear_attention_grad(q, k, v, gy, log_decay=None, scale=None, state=None, lengths=None, gnew=None):
    """({'q', 'k', 'v', 'log_decay', 'state'}, how far each may be off, in how many roundings)"""
    scale = q.shape[3] ** -0.5 if scale is None else scale
    key_heads = q.shape[2]
    b, l, h = v.shape[:3]
    q, k, v, g, keep = _attend_inputs(q, k, v, log_decay, lengths)
    gy = np.where(keep, gy.astype(np.float64), 0)
    zeros = np.zeros((b, h, k.shape[3], v.shape[3]))
    state = zeros if state is None else state.astype(np.float64)
    gnew = zeros if gnew is None else gnew.astype(np.float64)

    def gradients(q, k, v, gy, state, gnew, scale, sign):
        s = _states(k, v, g, state)
        gq, gk, gv, gg = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape), np.zeros(g.shape)
        r = gnew
        for t in reversed(range(l)):
            r = r + scale * q[:, t][..., :, None] * gy[:, t][..., None, :]
            gq[:, t] = scale * (s[t + 1] * gy[:, t][..., None, :]).sum(3)
            gk[:, t] = (r * v[:, t][..., None, :]).sum(3)
            gv[:, t] = (r * k[:, t][..., :, None]).sum(2)
            r = r * np.exp(g[:, t])[..., None, None]
            gg[:, t] = (s[t] * r).sum((2, 3))
        if sign < 0:  # what the kernel adds up instead: of q gq and k gk from a row on
            of_rows = ((q * gq).sum(3) + (k * gk).sum(3))[:, ::-1].cumsum(1)[:, ::-1] if l else gg
            gg = of_rows + (s[-1] * gnew).sum((2, 3))[:, None]
        return gq, gk, gv, gg, r

    n = 2 * _roundings(q, v, g) + 64
    fold = lambda x: x.reshape(b, l, key_heads, h // key_heads, -1).sum(3)  # noqa: E731

    def named(values):
        gq, gk, gv, gg, gs = values
        gq, gk, gv, gg = (np.where(m, x, 0) for m, x in ((keep, gq), (keep, gk), (keep, gv), (keep[..., 0], gg)))
        return {'q': fold(gq), 'k': fold(gk), 'v': gv, 'log_decay': gg.sum((0, 1)) if log_decay is not None and log_decay.ndim == 1 else gg, 'state': gs}

    value = named(gradients(q, k, v, gy, state, gnew, scale, 1))
    size = named(gradients(ab(q), ab(k), ab(v), ab(gy), ab(state), ab(gnew), ab(scale), -1))
    return value, {name: n * U32 * x for name, x in size.items()}, n


# ---------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------
def part_of(code, exponents):
    """What a code stands for, as a part of its block's scale."""
    e, f = np.maximum(code >> 3, 1), np.where(code >> 3 == 0, code, 8 + code % 8)
    return np.ldexp(f.astype(np.float64), e - exponents - 2).astype(np.float32)


def of_blocks(scale, n):
    return np.repeat(scale, 256)[:n]


def stored(x, exponents, up):
    """(codes, scales) of 32-bit values that are not negative."""
    n = x.size
    padded = np.zeros(-(-n // 256) * 256, np.float32)
    padded[:n] = x
    top = padded.reshape(-1, 256).max(1)
    f, e = np.frexp(top)
    e = np.clip(np.where(top > 0, e - (f == 0.5), -100), -100, 100)
    scale = np.where(top <= 2.0 ** 100, np.ldexp(np.float32(1), e), np.nan).astype(np.float32)
    with np.errstate(invalid='ignore'):
        y = (x / of_blocks(scale, n)).astype(np.float32)
        fine = np.isfinite(y)
        y = np.where(fine, y, 0).astype(np.float32)
    power = np.maximum(np.where(y > 0, np.frexp(y)[1] - 1 + exponents - 1, 1), 1)
    steps = np.floor(np.ldexp(y, exponents + 2 - power).astype(np.float32) + up).astype(np.int64)
    return np.minimum(8 * power + steps - 8, 8 * exponents - 1), scale, fine


def philox_words(n, site, t, seed):
    """n words of 32 bits, four to a counter."""
    c = np.arange((n + 3) // 4, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    c = [c, np.full_like(c, site), np.full_like(c, t & 0xFFFFFFFF), np.full_like(c, t >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n].astype(np.int64)


def adamw(p, g, m, v, m_scale, v_scale, master, site, t, alpha, beta1, beta2, eps, eta, weight_decay_rate, seed):
    """The new (p, m, v, m_scale, v_scale, master) of flat arrays, each operation rounded to 32 bits."""
    f = np.float32
    n = p.size
    step = f(eta * alpha * np.sqrt(1 - np.float64(beta2) ** t) / (1 - np.float64(beta1) ** t))
    weights, grad = (p if master is None else master).astype(f), g.astype(f)
    eight = m.dtype == np.uint8
    with np.errstate(all='ignore'):
        if eight:
            old_m = part_of(m.astype(np.int64) & 127, 16) * of_blocks(m_scale, n)
            old_m = np.where(m >= 128, -old_m, old_m)
            r = part_of(v.astype(np.int64), 32) * of_blocks(v_scale, n)
            old_v = r * r
        else:
            old_m, old_v = m, v
        new_m = old_m + f(1 - beta1) * (grad - old_m)
        new_v = old_v + f(1 - beta2) * (grad * grad - old_v)
        root = np.sqrt(new_v)
        new = weights - (step * (new_m / (root + f(eps))) + f(eta * weight_decay_rate) * weights)
        new_p = new.astype(p.dtype)
    assert new.dtype == f and new_m.dtype == f and new_v.dtype == f
    if not eight:
        return new_p, new_m, new_v, None, None, None if master is None else new
    words = philox_words(n, site, t, seed)
    up = lambda w: ((w.astype(f) + f(0.5)) * f(2.0 ** -16)).astype(f)  # noqa: E731
    m_code, m_scale, _ = stored(ab(new_m), 16, up(words & 0xFFFF))
    m_code = np.where(np.signbit(new_m), m_code + 128, m_code)
    v_code, v_scale, _ = stored(root, 32, up(words >> 16))
    v_code = np.where(root > 0, np.maximum(v_code, 1), v_code)
    return new_p, m_code.astype(np.uint8), v_code.astype(np.uint8), m_scale, v_scale, None if master is None else new

"""Performance cases of the selective recurrent layer's operators and of dropout: chainer_amd's kernels (`own`) and their plain forms in torch.

  conv     chainer_amd.causal_conv: a short causal convolution of every channel along time, with SiLU; `train` adds causal_conv_grad
  scan     chainer_amd.selective_scan: a diagonal state space whose steps depend on the input; `train` adds selective_scan_grad
  dropout  chainer_amd.dropout: from a counter-based generator, optionally added to a residual; `train` adds the gradient

`length` 1 is a server's next token.  Sizes are those of the package's language model (batches of 20 and 128, 35 steps, 650 units) and of wider
layers of the same kind.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one request's next token: the window of the convolution moves by one row
        {'name': 'conv_token_b1', 'kind': 'conv', 'batch': 1, 'length': 1, 'channels': 1300, 'taps': 4, 'dtype': 'float16', 'ragged': False, 'train': False},
        # prompts of several lengths, padded to the longest
        {'name': 'conv_prompts_f16', 'kind': 'conv', 'batch': 16, 'length': 2048, 'channels': 4096, 'taps': 4, 'dtype': 'float16', 'ragged': True,
         'train': False},
        # training on the language model's windows
        {'name': 'conv_train_lm_f32', 'kind': 'conv', 'batch': 20, 'length': 35, 'channels': 650, 'taps': 3, 'dtype': 'float32', 'ragged': False,
         'train': True},
        # training on long sequences
        {'name': 'conv_train_f16', 'kind': 'conv', 'batch': 8, 'length': 2048, 'channels': 2048, 'taps': 4, 'dtype': 'float16', 'ragged': False,
         'train': True},
        # a few requests' next tokens: latency
        {'name': 'scan_token_b3', 'kind': 'scan', 'batch': 3, 'length': 1, 'channels': 1300, 'states': 16, 'groups': 1, 'gate': True, 'dtype': 'float32',
         'ragged': False, 'train': False},
        # a full batch of next tokens: the states' bandwidth
        {'name': 'scan_token_b128_f16', 'kind': 'scan', 'batch': 128, 'length': 1, 'channels': 4096, 'states': 16, 'groups': 1, 'gate': True,
         'dtype': 'float16', 'ragged': False, 'train': False},
        # one long prompt: parallel along time
        {'name': 'scan_prompt_16384_f16', 'kind': 'scan', 'batch': 1, 'length': 16384, 'channels': 2048, 'states': 16, 'groups': 1, 'gate': True,
         'dtype': 'float16', 'ragged': False, 'train': False},
        # a padded batch, one sequence of it empty; no gate, sizes that no tile divides
        {'name': 'scan_prompts_777_f32', 'kind': 'scan', 'batch': 20, 'length': 777, 'channels': 650, 'states': 16, 'groups': 1, 'gate': False,
         'dtype': 'float32', 'ragged': True, 'train': False},
        # training on the language model's windows
        {'name': 'scan_train_lm_f32', 'kind': 'scan', 'batch': 20, 'length': 35, 'channels': 650, 'states': 16, 'groups': 1, 'gate': True,
         'dtype': 'float32', 'ragged': False, 'train': True},
        # training on long sequences
        {'name': 'scan_train_2048_f16', 'kind': 'scan', 'batch': 4, 'length': 2048, 'channels': 2048, 'states': 16, 'groups': 1, 'gate': True,
         'dtype': 'float16', 'ragged': False, 'train': True},
        # between the layers of the language model, one time step, there and back
        {'name': 'dropout_lm_f32', 'kind': 'dropout', 'rows': 128, 'cols': 650, 'ratio': 0.5, 'residual': False, 'dtype': 'float32', 'train': True},
        # at the end of a block, added to what went round it
        {'name': 'dropout_add_f16', 'kind': 'dropout', 'rows': 65536, 'cols': 2048, 'ratio': 0.1, 'residual': True, 'dtype': 'float16', 'train': False},
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(['conv', 'scan', 'scan', 'dropout'])
    case = {'kind': kind, 'dtype': rng.choice(['float16', 'float32']), 'train': rng.random() < 0.5}
    if kind == 'dropout':
        total = _log_int(rng, 1, 1 << 26)
        rows = _log_int(rng, 1, total)
        case.update(rows=rows, cols=total // rows, ratio=rng.choice([0.0, 0.1, 0.25, 0.5, 0.9, round(rng.uniform(0.01, 0.99), 3)]), residual=rng.random() < 0.5)
        return case
    length = rng.choice([1, _log_int(rng, 2, 16384), _log_int(rng, 2, 16384)])
    channels = _log_int(rng, 16, 4096)
    if kind == 'conv':
        batch = max(1, min(_log_int(rng, 1, 256), (1 << 25) // (length * channels)))
        case.update(batch=batch, length=length, channels=channels, taps=rng.choice([2, 3, 4, 4, 4, 5, 8]), ragged=rng.random() < 0.4)
        return case
    states, groups = rng.choice([16, 16, 16, 1, 5, 8, 12, 24, 32, 64]), rng.choice([1, 1, 1, 2, 3])
    channels = max(groups, channels // groups * groups)
    limit = 1 << (27 if case['train'] else 29)
    length = max(1, min(length, limit // (channels * states)))
    batch = max(1, min(_log_int(rng, 1, 256), limit // (length * channels * states)))
    case.update(batch=batch, length=length, channels=channels, states=states, groups=groups, gate=rng.random() < 0.7, ragged=rng.random() < 0.4)
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _lengths(case, gen):
    """Rows of each sequence of a padded batch: the first is as long as the batch, one in the middle is empty."""
    n = torch.randint(0, case['length'] + 1, (case['batch'],), generator=gen, device='cuda', dtype=torch.int32)
    n[case['batch'] // 2] = 0
    n[0] = case['length']
    return n


def _inside(lengths, length):
    return torch.arange(length, device='cuda')[None, :, None] < lengths[:, None, None]


def prepare(case, seed):
    gen = torch.Generator('cuda')
    gen.manual_seed(seed)
    dtype = getattr(torch, case['dtype'])

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(shape, generator=gen, device='cuda') * scale).to(to)

    if case['kind'] == 'dropout':
        shape = (case['rows'], case['cols'])
        state = {'x': normal(*shape), 'residual': normal(*shape) if case['residual'] else None, 'gy': normal(*shape) if case['train'] else None,
                 'key': torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 63), 1000 + seed], device='cuda')}
        return {'case': case, **state}

    b, l, d, train = case['batch'], case['length'], case['channels'], case['train']
    lengths = _lengths(case, gen) if case['ragged'] else None

    def rows(width, scale=1.0, pitch=None):
        """[b, l, width], a part of wider rows where `pitch` says so; what lies behind a sequence's end is not to be looked at."""
        x = normal(b, l, pitch or width, scale=scale)
        if lengths is not None:
            x.masked_fill_(~_inside(lengths, l), math.nan)
        return x[..., (pitch or width) - width:]

    if case['kind'] == 'conv':
        k = case['taps']
        return {'case': case, 'x': rows(d, pitch=2 * d), 'w': normal(d, k, scale=1 / math.sqrt(k)), 'b': normal(d, scale=0.1), 'state': normal(b, k - 1, d),
                'lengths': lengths, 'gy': rows(d) if train else None, 'gnew': normal(b, k - 1, d) if train else None}
    n, g = case['states'], case['groups']
    # a decays like 1 .. n, the steps are between 0.001 and 0.1 where delta is zero
    a = -torch.arange(1, n + 1, device='cuda', dtype=torch.float32) * torch.exp(normal(d, 1, scale=0.1, to=torch.float32))
    steps = torch.exp(torch.rand(d, generator=gen, device='cuda') * math.log(100.0) + math.log(0.001))
    shared = rows(2 * g * n).unflatten(2, (2, g, n))
    return {'case': case, 'u': rows(d), 'delta': rows(d, 0.5), 'a': a, 'b': shared[:, :, 0], 'c': shared[:, :, 1], 'd': normal(d, to=torch.float32),
            'z': rows(d, pitch=2 * d) if case['gate'] else None, 'bias': torch.log(torch.expm1(steps)), 'state': normal(b, d, n, to=torch.float32),
            'lengths': lengths, 'gy': rows(d) if train else None, 'gnew': normal(b, d, n, to=torch.float32) if train else None}


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
def _read(x, lengths):
    """In 32 bits, with zeros behind the sequences' ends."""
    if x is None:
        return None
    x = x.float()
    return x if lengths is None else torch.where(_inside(lengths, x.shape[1]) if x.ndim == 3 else _inside(lengths, x.shape[1])[..., None], x, 0.0)


def _zero_behind(y, lengths):
    return y if lengths is None else torch.where(_inside(lengths, y.shape[1]), y, 0.0)


def _windows(xs, taps, length):
    """[b, length, d, taps] of [b, taps - 1 + length, d]."""
    return xs.unfold(1, taps, 1)[:, :length]


def _conv_plain(s):
    k, length, lengths = s['w'].shape[1], s['x'].shape[1], s['lengths']
    dtype = s['x'].dtype
    w = s['w'].float()
    xs = torch.cat([s['state'].float(), _read(s['x'], lengths)], 1)
    p = (_windows(xs, k, length) * w).sum(3) + s['b'].float()
    sig = torch.sigmoid(p)
    y = _zero_behind(p * sig, lengths)
    ends = torch.full((xs.shape[0],), length, device='cuda') if lengths is None else lengths.long()
    last = (ends[:, None] + torch.arange(k - 1, device='cuda'))[:, :, None].expand(-1, -1, xs.shape[2])
    out = {'y': y.to(dtype), 'state': torch.gather(xs, 1, last).to(dtype)}
    if s['gy'] is not None:
        gp = _read(s['gy'], lengths) * sig * (1 + p * (1 - sig))
        around = torch.nn.functional.pad(gp, (0, 0, k - 1, k - 1))
        gxs = (_windows(around, k, length + k - 1) * w.flip(1)).sum(3)
        gxs = gxs.scatter_add(1, last, s['gnew'].float())
        out.update(gx=gxs[:, k - 1:].to(dtype), gw=(_windows(xs, k, length) * gp[..., None]).sum((0, 1), dtype=torch.float64).to(dtype),
                   gb=gp.sum((0, 1), dtype=torch.float64).to(dtype), gstate=gxs[:, :k - 1].to(dtype))
    return out


def _recurrence(decay, x):
    """h[t] = decay[t] h[t-1] + x[t] along axis 1, in log2 of the length many steps; decay[0] does not count.  Takes both arrays over."""
    step = 1
    while step < x.shape[1]:
        x = torch.cat([x[:, :step], x[:, step:] + decay[:, step:] * x[:, :-step]], 1)
        if 2 * step < x.shape[1]:
            decay = torch.cat([decay[:, :step], decay[:, step:] * decay[:, :-step]], 1)
        step *= 2
    return x


def _per_channel(x, d):
    """[b, l, g, n] -> [b, l, d, n]"""
    return x.repeat_interleave(d // x.shape[2], 2)


def _scan_plain(s):
    lengths, dtype, d = s['lengths'], s['u'].dtype, s['u'].shape[2]
    g, a = s['b'].shape[2], s['a']
    u, z = _read(s['u'], lengths), _read(s['z'], lengths)
    raw = s['delta'].float() + s['bias']
    dt = torch.nn.functional.softplus(raw)
    if lengths is not None:
        dt = torch.where(_inside(lengths, u.shape[1]), dt, 0.0)
    b, c = _per_channel(_read(s['b'], lengths), d), _per_channel(_read(s['c'], lengths), d)
    decay = torch.exp(dt[..., None] * a)
    x = (dt * u)[..., None] * b
    x[:, 0] += decay[:, 0] * s['state']
    h = _recurrence(decay, x)
    y0 = (h * c).sum(3) + s['d'] * u
    sig = None if z is None else torch.sigmoid(z)
    y = y0 if z is None else y0 * z * sig
    out = {'y': _zero_behind(y, lengths).to(dtype), 'state': h[:, -1].clone()}
    if s['gy'] is None:
        return out
    gy = _read(s['gy'], lengths)
    g0 = gy
    if z is not None:
        g0 = gy * z * sig
        out['gz'] = (gy * y0 * sig * (1 + z * (1 - sig))).to(dtype)
    q = g0[..., None] * c
    q[:, -1] += s['gnew']
    after = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], 1)
    q = _recurrence(after.flip(1), q.flip(1)).flip(1)
    before = torch.cat([s['state'][:, None], h[:, :-1]], 1)
    e = q * decay * before
    qb = (q * b).sum(3)
    gdelta = _zero_behind(((e * a).sum(3) + u * qb) * torch.sigmoid(raw), lengths)
    out.update(gu=(s['d'] * g0 + dt * qb).to(dtype), gdelta=gdelta.to(dtype), ga=(e * dt[..., None]).sum((0, 1), dtype=torch.float64).float(),
               gb=(q * (dt * u)[..., None]).unflatten(2, (g, d // g)).sum(3).to(dtype), gc=(h * g0[..., None]).unflatten(2, (g, d // g)).sum(3).to(dtype),
               gd=(g0 * u).sum((0, 1), dtype=torch.float64).float(), gbias=gdelta.sum((0, 1), dtype=torch.float64).float(), gstate=q[:, 0] * decay[:, 0])
    return out


_LOW = 0xFFFFFFFF


def _threshold(ratio):
    return min(65535, int(math.floor(ratio * 65536 + 0.5)))


def _kept_plain(n, ratio, key, site):
    """Which of n elements Philox4x32-10 keeps: eight numbers of 16 bits from each counter."""
    c0 = torch.arange((n + 7) // 8, device='cuda')
    k0, k1 = key[0] & _LOW, (key[0] >> 32) & _LOW
    c1, c2, c3 = torch.full_like(c0, site), (key[1] & _LOW).expand_as(c0), ((key[1] >> 32) & _LOW).expand_as(c0)
    for _ in range(10):  # the generator's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n] >= _threshold(ratio)


def _dropout_plain(s):
    x, ratio = s['x'], s['case']['ratio']
    kept = _kept_plain(x.numel(), ratio, s['key'], _SITE).reshape(x.shape)
    scale = 65536 / (65536 - _threshold(ratio))
    y = torch.where(kept, x.float() * scale, 0.0)
    out = {'y': (y if s['residual'] is None else s['residual'].float() + y).to(x.dtype)}
    if s['gy'] is not None:
        out['gx'] = torch.where(kept, s['gy'].float() * scale, 0.0).to(x.dtype)
    return out


# ---------------------------------------------------------------------------------------------
# the calls
# ---------------------------------------------------------------------------------------------
_SITE = 3  # a layer's number among those that drop out


class _Exported(object):
    """Device memory of an array, described for torch."""

    def __init__(self, a):
        self.array = a  # keeps the memory
        self.__cuda_array_interface__ = {'shape': a.shape, 'typestr': a.dtype.str, 'data': (a.data_ptr, False), 'version': 2}


def _named(**arrays):
    return {k: torch.as_tensor(_Exported(a), device='cuda') for k, a in arrays.items() if a is not None}


_NUMPY = {torch.float16: np.dtype('float16'), torch.float32: np.dtype('float32'), torch.int32: np.dtype('int32'), torch.int64: np.dtype('int64')}


def _own(s):
    import chainer_amd as chx

    def of(name):
        t = s[name]
        if t is None:
            return None
        dt = _NUMPY[t.dtype]
        return chx.ndarray(t, 0, tuple(t.shape), tuple(n * dt.itemsize for n in t.stride()), dt)

    case = s['case']
    if case['kind'] == 'dropout':
        key = of('key')
        y = chx.dropout(of('x'), case['ratio'], key, site=_SITE, residual=of('residual'))
        return _named(y=y, gx=None if s['gy'] is None else chx.dropout(of('gy'), case['ratio'], key, site=_SITE))
    if case['kind'] == 'conv':
        x, w, b, state, lengths = of('x'), of('w'), of('b'), of('state'), of('lengths')
        y, new = chx.causal_conv(x, w, b, state=state, lengths=lengths, activation='silu')
        if s['gy'] is None:
            return _named(y=y, state=new)
        gx, gw, gb, gstate = chx.causal_conv_grad(x, w, b, of('gy'), state=state, lengths=lengths, activation='silu', gnew_state=of('gnew'))
        return _named(y=y, state=new, gx=gx, gw=gw, gb=gb, gstate=gstate)
    args = [of(name) for name in ('u', 'delta', 'a', 'b', 'c')]
    more = dict(d=of('d'), z=of('z'), delta_bias=of('bias'), delta_softplus=True, state=of('state'), lengths=of('lengths'))
    y, new = chx.selective_scan(*args, **more)
    if s['gy'] is None:
        return _named(y=y, state=new)
    g = chx.selective_scan_grad(*args, of('gy'), gnew_state=of('gnew'), **more)
    return _named(y=y, state=new, gu=g.u, gdelta=g.delta, ga=g.a, gb=g.b, gc=g.c, gd=g.d, gz=g.z, gbias=g.delta_bias, gstate=g.state)


def run(state):
    if own:
        return _own(state)
    return {'conv': _conv_plain, 'scan': _scan_plain, 'dropout': _dropout_plain}[state['case']['kind']](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------------------------
def work(case):
    it, train = np.dtype(case['dtype']).itemsize, case['train']
    if case['kind'] == 'dropout':
        n = case['rows'] * case['cols']
        return {'bytes': it * n * (2 + case['residual'] + 2 * train), 'flops': n * (1 + case['residual'] + train)}
    b, l, d = case['batch'], case['length'], case['channels']
    if case['kind'] == 'conv':
        k = case['taps']
        states, weights = b * (k - 1) * d, (k + 1) * d
        flops = b * l * d * (2 * k + 4)
        return {'bytes': it * ((4 if train else 2) * b * l * d + (4 if train else 2) * states + (2 if train else 1) * weights), 'flops': (3 if train else 1) * flops}
    n, g = case['states'], case['groups']
    rows, shared = b * l * d * (3 + case['gate']), 2 * b * l * g * n
    more_rows = b * l * d * (3 + case['gate'])  # gy; gu, gdelta, gz
    nbytes = it * (rows + shared) + 4 * (2 * b * d * n + d * (n + 2))
    if train:
        nbytes += it * (more_rows + shared) + 4 * (2 * b * d * n + d * (n + 2))
    # per state: exp, 2 products, 2 multiply-adds; back: 9 more of which 4 are multiply-adds
    return {'bytes': nbytes, 'flops': b * l * d * (n * (7 + (13 if train else 0)) + 10)}


def _exact_mask(n, ratio, key, site):
    u = np.uint64
    c = [np.arange((n + 7) // 8, dtype=u), u(site), u(int(key[1]) & _LOW), u(int(key[1]) >> 32 & _LOW)]
    k = [int(key[0]) & _LOW, int(key[0]) >> 32 & _LOW]
    low, half = u(_LOW), u(32)
    for r in range(10):
        m, o = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(o >> half) ^ c[1] ^ u(k[0] + r * 0x9E3779B9 & _LOW), o & low, (m >> half) ^ c[3] ^ u(k[1] + r * 0xBB67AE85 & _LOW), m & low]
    bits = np.stack([w.astype('<u4') for w in c], 1).view('<u2')
    return bits.reshape(-1)[:n] >= _threshold(ratio)


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case['kind'] == 'dropout':
        kept = torch.from_numpy(_exact_mask(s['x'].numel(), case['ratio'], s['key'].tolist(), _SITE)).to('cuda').reshape(s['x'].shape)
        share = 1 - _threshold(case['ratio']) / 65536
        out = {'y': kept * wide['x'] / share + (0 if s['residual'] is None else wide['residual'])}
        if s['gy'] is not None:
            out['gx'] = kept * wide['gy'] / share
        return out
    lengths = s['lengths']
    ends = torch.full((case['batch'],), case['length'], device='cuda') if lengths is None else lengths
    for k in ('x', 'u', 'delta', 'b', 'c', 'z', 'gy'):  # what lies behind the ends counts nowhere
        if k in wide and wide[k] is not None and wide[k].ndim >= 3:
            wide[k] = torch.nan_to_num(wide[k])
    names = {'conv': ('x', 'w', 'b', 'state'), 'scan': ('u', 'delta', 'a', 'b', 'c', 'd', 'z', 'bias', 'state')}[case['kind']]
    leaves = {k: wide[k].requires_grad_(case['train']) for k in names if wide[k] is not None}
    with torch.set_grad_enabled(case['train']):
        y, new = _exact_conv(leaves, ends) if case['kind'] == 'conv' else _exact_scan(leaves, ends)
    out = {'y': y.detach(), 'state': new.detach()}
    if case['train']:
        grads = torch.autograd.grad([y, new], list(leaves.values()), [wide['gy'], wide['gnew']])
        out.update({'g' + k: v for k, v in zip(leaves, grads)})
    return out


def _exact_conv(s, ends):
    k, d = s['w'].shape[1], s['w'].shape[0]
    length = s['x'].shape[1]
    xs = torch.cat([s['state'], s['x']], 1)
    p = torch.zeros_like(s['x']) + s['b']
    for i in range(k):
        p = p + xs[:, i:i + length] * s['w'][:, i]
    y = torch.nn.functional.silu(p) * (torch.arange(length, device='cuda')[None, :, None] < ends[:, None, None])
    new = torch.stack([xs[i, int(n):int(n) + k - 1] for i, n in enumerate(ends.tolist())])
    return y, new


def _exact_scan(s, ends):
    h, ys = s['state'], []
    d, g = s['u'].shape[2], s['b'].shape[2]
    for t in range(s['u'].shape[1]):
        dt = torch.nn.functional.softplus(s['delta'][:, t] + s['bias']) * (t < ends)[:, None]
        b, c = (s[k][:, t].repeat_interleave(d // g, 1) for k in ('b', 'c'))
        h = h * torch.exp(dt[..., None] * s['a']) + (dt * s['u'][:, t])[..., None] * b
        y = (h * c).sum(2) + s['d'] * s['u'][:, t]
        ys.append((y * torch.nn.functional.silu(s['z'][:, t]) if 'z' in s else y) * (t < ends)[:, None])
    return torch.stack(ys, 1), h

"""Performance cases of layer norm, linear attention and AdamW: chainer_amd's kernels (`own`) and their plain forms in torch.

  norm    chainer_amd.layer_norm: rows normalised to mean 0 and variance 1, scaled and shifted; `train` adds layer_norm_grad
  attend  chainer_amd.linear_attention: a matrix for each head that decays and gathers keys and values; `train` adds linear_attention_grad
  adamw   chainer_amd.adamw_update: a step of AdamW over a list of arrays in place, its states in 32 bits or in 8

`length` 1 is a server's next token.  Sizes are those of the package's networks (the language model's batches of 20 and 128, 35 steps, 650 units as 13 heads of
50, its 10000 words; the 784-1000-1000-10 perceptron; ResNet-50's filters) and of wider layers of the same kind.
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # between the layers of the language model, one time step: latency
        {'name': 'norm_lm_step_f32', 'kind': 'norm', 'rows': 128, 'cols': 650, 'dtype': 'float32', 'params': 'float32', 'train': False},
        # training on the language model's windows
        {'name': 'norm_train_lm_f32', 'kind': 'norm', 'rows': 4480, 'cols': 650, 'dtype': 'float32', 'params': 'float32', 'train': True},
        # training a wide block in float16, its weights in float32
        {'name': 'norm_train_4096_f16', 'kind': 'norm', 'rows': 16384, 'cols': 4096, 'dtype': 'float16', 'params': 'float32', 'train': True},
        # one request's next token: the states move by one row
        {'name': 'attend_token_b1', 'kind': 'attend', 'batch': 1, 'length': 1, 'heads': 13, 'shared': 1, 'keys': 50, 'values': 50, 'dtype': 'float32',
         'decay': 'rows', 'ragged': False, 'train': False},
        # a full batch of next tokens: the states' bandwidth
        {'name': 'attend_token_b128_f16', 'kind': 'attend', 'batch': 128, 'length': 1, 'heads': 16, 'shared': 1, 'keys': 128, 'values': 128, 'dtype': 'float16',
         'decay': 'rows', 'ragged': False, 'train': False},
        # one long prompt: parallel along time; a fixed decay for each head
        {'name': 'attend_prompt_16384_f16', 'kind': 'attend', 'batch': 1, 'length': 16384, 'heads': 16, 'shared': 1, 'keys': 128, 'values': 128,
         'dtype': 'float16', 'decay': 'heads', 'ragged': False, 'train': False},
        # a padded batch, one sequence of it empty; sizes that no tile divides
        {'name': 'attend_prompts_777_f32', 'kind': 'attend', 'batch': 20, 'length': 777, 'heads': 13, 'shared': 1, 'keys': 50, 'values': 50, 'dtype': 'float32',
         'decay': 'rows', 'ragged': True, 'train': False},
        # training on the language model's windows
        {'name': 'attend_train_lm_f32', 'kind': 'attend', 'batch': 20, 'length': 35, 'heads': 13, 'shared': 1, 'keys': 50, 'values': 50, 'dtype': 'float32',
         'decay': 'rows', 'ragged': False, 'train': True},
        # training on long sequences
        {'name': 'attend_train_2048_f16', 'kind': 'attend', 'batch': 4, 'length': 2048, 'heads': 16, 'shared': 1, 'keys': 128, 'values': 128, 'dtype': 'float16',
         'decay': 'rows', 'ragged': False, 'train': True},
        # a small network's step: latency
        {'name': 'adamw_mlp_f32', 'kind': 'adamw', 'arrays': 'mlp', 'total': 0, 'count': 0, 'bits': 32, 'dtype': 'float32', 'master': False},
        # many arrays of all sizes, float16 weights with a copy in 32 bits
        {'name': 'adamw_resnet50_f16', 'kind': 'adamw', 'arrays': 'resnet50', 'total': 0, 'count': 0, 'bits': 32, 'dtype': 'float16', 'master': True},
        # the language model's weights with states in 8 bits
        {'name': 'adamw_lm_8bits_f16', 'kind': 'adamw', 'arrays': 'lm', 'total': 0, 'count': 0, 'bits': 8, 'dtype': 'float16', 'master': False},
    ]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(['norm', 'attend', 'attend', 'adamw'])
    case = {'kind': kind, 'dtype': rng.choice(['float16', 'float32'])}
    if kind == 'norm':
        cols = _log_int(rng, 8, 16384)
        return dict(case, rows=_log_int(rng, 1, min(65536, (1 << 26) // cols)), cols=cols, params=rng.choice([case['dtype'], 'float32']), train=rng.random() < 0.6)
    if kind == 'adamw':
        total = _log_int(rng, 1000, 20000000)
        return dict(case, arrays='drawn', total=total, count=_log_int(rng, 1, min(300, total)), bits=rng.choice([32, 8]), master=rng.random() < 0.5)
    train = rng.random() < 0.5
    keys, values = rng.choice([(128, 128), (64, 64), (32, 32), (50, 50), (128, 64), (64, 128), (16, 80), (100, 100), (rng.randint(8, 128), rng.randint(8, 128))])
    shared = rng.choice([1, 1, 1, 2, 4])
    heads = shared * rng.randint(1, 16 // shared)
    length = rng.choice([1, _log_int(rng, 2, 16384), _log_int(rng, 2, 16384)])
    limit = 1 << (17 if train else 18)  # rows of all heads
    length = max(1, min(length, limit // heads, 4096 if train else 16384))
    batch = max(1, min(_log_int(rng, 1, 128), limit // (heads * length), (1 << 28) // (heads * keys * values)))
    return dict(case, batch=batch, length=length, heads=heads, shared=shared, keys=keys, values=values, decay=rng.choice(['rows', 'rows', 'heads', 'none']),
                ragged=rng.random() < 0.4, train=train)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _resnet50_arrays():
    """Elements of ResNet-50's filters, norms and last layer."""
    sizes, width = [3 * 64 * 49, 64, 64], 64
    for stage, blocks in enumerate((3, 4, 6, 3)):
        mid = 64 << stage
        for b in range(blocks):
            sizes += [width * mid, mid, mid, mid * mid * 9, mid, mid, mid * 4 * mid, 4 * mid, 4 * mid]
            if b == 0:
                sizes += [width * 4 * mid, 4 * mid, 4 * mid]
            width = 4 * mid
    return sizes + [width * 1000, 1000]


def _arrays(case):
    if case['arrays'] == 'mlp':
        return [784 * 1000, 1000, 1000 * 1000, 1000, 1000 * 10, 10]
    if case['arrays'] == 'resnet50':
        return _resnet50_arrays()
    if case['arrays'] == 'lm':
        return [10000 * 650] + 2 * [4 * 650 * 650, 4 * 650, 4 * 650 * 650, 4 * 650] + [10000 * 650, 10000]
    # a list of all sizes that sum up to about the total
    rng = random.Random(case['total'] * 1009 + case['count'])
    shares = [math.exp(rng.gauss(0, 2)) for _ in range(case['count'])]
    return [max(1, int(case['total'] * s / sum(shares))) for s in shares]


def _lengths(case, gen):
    """Rows of each sequence of a padded batch: the first is as long as the batch, one in the middle is empty."""
    n = torch.randint(0, case['length'] + 1, (case['batch'],), generator=gen, device='cuda', dtype=torch.int32)
    n[case['batch'] // 2] = 0
    n[0] = case['length']
    return n


def _inside(lengths, length):
    """[batch, length, 1, 1]"""
    return (torch.arange(length, device='cuda')[None, :] < lengths[:, None])[..., None, None]


_BLOCK = 256  # elements that share the scales of their 8-bit states


def _values_of(exponents):
    """What the codes of 8 bits stand for, as parts of a block's scale: `exponents` powers of two of eight steps each, the lowest with the same steps down to 0."""
    c = np.arange(8 * exponents)
    e, f = np.maximum(c >> 3, 1), np.where(c >> 3 == 0, c, 8 + c % 8)
    return np.ldexp(f.astype(np.float64), e - exponents + 1 - 3)


_M_VALUES = np.concatenate([_values_of(16), -_values_of(16)]).astype(np.float32)
_R_VALUES = _values_of(32).astype(np.float32)


def prepare(case, seed):
    gen = torch.Generator('cuda')
    gen.manual_seed(seed)
    dtype = getattr(torch, case['dtype'])

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(shape, generator=gen, device='cuda') * scale).to(to)

    if case['kind'] == 'norm':
        rows, cols, params = case['rows'], case['cols'], getattr(torch, case['params'])
        # every channel has its own size and offset, as a block's activations have
        x = (normal(rows, cols, to=torch.float32) * torch.exp(normal(cols, scale=0.5, to=torch.float32)) + normal(cols, scale=0.5, to=torch.float32)).to(dtype)
        return {'case': case, 'x': x, 'gamma': normal(cols, scale=0.1, to=params) + 1, 'beta': normal(cols, scale=0.1, to=params),
                'gy': normal(rows, cols) if case['train'] else None}
    if case['kind'] == 'adamw':
        eight, sizes = case['bits'] == 8, _arrays(case)
        state = {'case': case, 't': 10 + seed % 1000, 'seed': seed, 'p': [], 'g': [], 'm': [], 'v': [], 'm_scale': [], 'v_scale': [], 'master': []}
        if eight:
            state['m_values'], state['r_values'] = torch.from_numpy(_M_VALUES).cuda(), torch.from_numpy(_R_VALUES).cuda()
        for n in sizes:
            size = torch.exp(normal((n + 63) // 64, 1, scale=1.0, to=torch.float32)).expand(-1, 64).reshape(-1)[:n] * 1e-3  # gradients of some 64 elements are alike in size
            p = normal(n, scale=0.05, to=torch.float32)
            state['g'].append((normal(n, to=torch.float32) * size).to(dtype))
            m, v = normal(n, to=torch.float32) * size * 0.3, size * size * torch.exp(normal(n, scale=0.3, to=torch.float32))
            if eight:
                m, m_scale = _stored(m, 16, torch.zeros(n, device='cuda'))
                v, v_scale = _stored(v.sqrt(), 32, torch.zeros(n, device='cuda'))
            state['m'].append(m)
            state['v'].append(v)
            state['m_scale'].append(m_scale if eight else None)
            state['v_scale'].append(v_scale if eight else None)
            state['master'].append(p if case['master'] and dtype != torch.float32 else None)
            state['p'].append(p.to(dtype) if dtype != torch.float32 else p)
        return state

    b, l, h, kh, dk, dv = case['batch'], case['length'], case['heads'], case['heads'] // case['shared'], case['keys'], case['values']
    lengths = _lengths(case, gen) if case['ragged'] else None

    def clean(x):  # what lies behind a sequence's end is not to be looked at
        return x if lengths is None else x.masked_fill_(~_inside(lengths, l), math.nan)

    # parts of one projection, as a block makes them
    wide = clean(normal(b, l, 1, 2 * kh * dk + h * dv))[:, :, 0]
    q, k, v = wide[..., :kh * dk].unflatten(2, (kh, dk)), wide[..., kh * dk:2 * kh * dk].unflatten(2, (kh, dk)), wide[..., 2 * kh * dk:].unflatten(2, (h, dv))
    decay = None
    if case['decay'] == 'heads':  # half-lives from some 20 to some thousand rows
        decay = torch.log1p(-torch.exp2(-5 - torch.arange(h, device='cuda', dtype=torch.float32) % 8))
    elif case['decay'] == 'rows':  # gates that depend on the row
        decay = clean(-torch.exp(normal(b, l, h, 1, scale=1.5, to=torch.float32) - 3))[..., 0]
    return {'case': case, 'q': q, 'k': k, 'v': v, 'decay': decay, 'scale': 1 / math.sqrt(dk), 'state': normal(b, h, dk, dv, to=torch.float32), 'lengths': lengths,
            'gy': clean(normal(b, l, h, dv)) if case['train'] else None, 'gnew': normal(b, h, dk, dv, scale=0.1, to=torch.float32) if case['train'] else None}


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
_EPS = 2e-5


def _norm_plain(s):
    x, dtype = s['x'].float(), s['x'].dtype
    gamma, params = s['gamma'].float(), s['gamma'].dtype
    mean = x.mean(1, keepdim=True)
    d = x - mean
    inv = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + _EPS)
    xh = d * inv
    out = {'y': (xh * gamma + s['beta'].float()).to(dtype), 'mean': mean[:, 0], 'inv_std': inv[:, 0]}
    if s['gy'] is not None:
        gy = s['gy'].float()
        g = gy * gamma
        gx = inv * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        out.update(gx=gx.to(dtype), ggamma=(gy * xh).sum(0, dtype=torch.float64).to(params), gbeta=gy.sum(0, dtype=torch.float64).to(params))
    return out


_CHUNK = 64


def _attend(q, k, v, decay, state, scale):
    """y[t] = q[t] S[t] with S[t] = exp(decay[t]) S[t-1] + scale k[t] v[t]^T, and the last S.  q, k, v [batch, heads, length, ...] in 32 bits, decay [batch, heads, length] in 64."""
    b, h, l, dk = q.shape
    dv, c = v.shape[3], min(_CHUNK, l)
    n = (l + c - 1) // c
    fill = lambda x: torch.nn.functional.pad(x, (0, 0, 0, n * c - l)).view(b, h, n, c, x.shape[3])  # noqa: E731
    q, k, v = fill(q), fill(k) * scale, fill(v)
    g = fill(decay[..., None])[..., 0].cumsum(3)  # of a chunk's rows, from its start
    apart = g[..., :, None] - g[..., None, :]
    before = torch.ones(c, c, device='cuda', dtype=torch.bool).tril()
    p = (q @ k.transpose(3, 4)) * torch.exp(torch.where(before, apart, -math.inf)).float()
    end = g[..., -1:]
    gathered = (k * torch.exp(end - g).float()[..., None]).transpose(3, 4) @ v  # what a chunk adds to the state
    # the states that the chunks begin with: all earlier ones' shares
    ends = end[..., 0].cumsum(2)
    since = torch.nn.functional.pad(ends, (1, 0))[..., :-1]
    apart = since[..., :, None] - ends[..., None, :]
    earlier = torch.ones(n, n, device='cuda', dtype=torch.bool).tril(-1)
    weights = torch.exp(torch.where(earlier, apart, -math.inf)).float()
    start = (weights @ gathered.reshape(b, h, n, dk * dv)).view(b, h, n, dk, dv) + torch.exp(since).float()[..., None, None] * state[:, :, None]
    y = p @ v + torch.exp(g).float()[..., None] * (q @ start)
    last = torch.exp(end[:, :, -1, 0]).float()[..., None, None] * start[:, :, -1] + gathered[:, :, -1]
    return y.reshape(b, h, n * c, dv)[:, :, :l], last


def _read(x, lengths):
    """[batch, heads, length, ...] in 32 bits, with zeros behind the sequences' ends."""
    x = x.float()
    return (x if lengths is None else torch.where(_inside(lengths, x.shape[1]), x, 0.0)).transpose(1, 2)


def _per_head(x, shared):
    return x.repeat_interleave(shared, 1) if shared > 1 else x


def _log_decay(s):
    """[batch, heads, length] in 64 bits, 0 behind the sequences' ends."""
    b, l, h = s['case']['batch'], s['case']['length'], s['case']['heads']
    if s['decay'] is None:
        return torch.zeros(b, h, l, device='cuda', dtype=torch.float64)
    d = s['decay'].double().expand(b, l, h) if s['decay'].ndim == 1 else s['decay'].double()
    return (d if s['lengths'] is None else torch.where(_inside(s['lengths'], l)[..., 0], d, 0.0)).transpose(1, 2)


def _attend_plain(s):
    lengths, dtype, shared, scale = s['lengths'], s['q'].dtype, s['case']['shared'], s['scale']
    q, k, v, g = _per_head(_read(s['q'], lengths), shared), _per_head(_read(s['k'], lengths), shared), _read(s['v'], lengths), _log_decay(s)
    inside = 1.0 if lengths is None else _inside(lengths, q.shape[2]).transpose(1, 2).float()
    y, last = _attend(q, k, v, g, s['state'], 1.0)
    out = {'y': (y * scale * inside).transpose(1, 2).to(dtype), 'state': last}
    if s['gy'] is None:
        return out
    gy = _read(s['gy'], lengths)
    # backwards a state takes the decay of the row that follows; rows behind the end do nothing
    after = torch.nn.functional.pad(g[..., 1:], (0, 1))
    back = lambda x: x.flip(2)  # noqa: E731
    gq, _ = _attend(gy, v, k, g, s['state'].transpose(2, 3), 1.0)
    gq = gq * scale * inside
    gk, _ = _attend(back(v), back(gy), back(q), back(after), s['gnew'].transpose(2, 3), scale)
    gv, gstate = _attend(back(k), back(q), back(gy), back(after), s['gnew'], scale)
    gk, gv = back(gk) * inside, back(gv) * inside
    # log decays: what every pair of rows around a row, and the last state, have of it
    gg = (q * gq - k * gk).sum(3, dtype=torch.float64).flip(2).cumsum(2).flip(2) + (last.double() * s['gnew']).sum((2, 3))[..., None]
    gg = gg * inside[..., 0] if lengths is not None else gg
    fold = lambda x: x.unflatten(1, (-1, shared)).sum(2) if shared > 1 else x  # noqa: E731
    out.update(gq=fold(gq).transpose(1, 2).to(dtype), gk=fold(gk).transpose(1, 2).to(dtype), gv=gv.transpose(1, 2).to(dtype),
               gstate=torch.exp(g[..., :1]).float()[..., None] * gstate)
    if s['decay'] is not None:
        out['gdecay'] = (gg.sum((0, 2)) if s['decay'].ndim == 1 else gg.transpose(1, 2)).float()
    return out


_ALPHA, _BETA1, _BETA2, _ADAM_EPS, _WEIGHT_DECAY = 0.001, 0.9, 0.999, 1e-8, 0.01
_LOW = 0xFFFFFFFF


def _philox(n, site, step, seed):
    """n words of 32 bits from Philox4x32-10, four to a counter."""
    c0 = torch.arange((n + 3) // 4, device='cuda')
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    c1, c2, c3 = torch.full_like(c0, site), torch.full_like(c0, step & _LOW), torch.full_like(c0, step >> 32 & _LOW)
    for _ in range(10):  # the generator's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _of_blocks(scale, n):
    return scale.repeat_interleave(_BLOCK)[:n]


def _power_of_two(e):
    return (e + 127 << 23).view(torch.float32)


def _stored(x, exponents, up):
    """(codes, scales of blocks) of x: its part of the scale, which is the power of two that no value of the block exceeds, to a number of steps of an eighth of its
    power of two, rounded down after `up` in [0, 1) of a step has been added."""
    n = x.numel()
    top = torch.nn.functional.pad(x.abs(), (0, -n % _BLOCK)).view(-1, _BLOCK).amax(1)
    f, e = torch.frexp(top)
    scale = _power_of_two(torch.where(top > 0, e - (f == 0.5).int(), -100).clamp(-100, 100).int())
    y = x.abs() / _of_blocks(scale, n)
    power = torch.where(y > 0, torch.frexp(y)[1] - 1 + exponents - 1, 1).clamp(min=1).int()
    steps = torch.floor(y * _power_of_two(exponents - 1 - power + 3) + up).int()
    code = (8 * power + steps - 8).clamp(max=8 * exponents - 1)
    if exponents == 32:  # a square root that is not zero does not become zero
        code = torch.where(x > 0, code.clamp(min=1), code)
    else:
        code = torch.where(torch.signbit(x), code + 8 * exponents, code)
    return code.to(torch.uint8), scale


def _adamw_plain(s):
    """In place, one rounding for each operation in 32 bits."""
    case, t = s['case'], s['t']
    step = _ALPHA * math.sqrt(1 - _BETA2 ** t) / (1 - _BETA1 ** t)
    f32 = lambda x: float(np.float32(x))  # noqa: E731
    step, c1, c2, eps, decay = f32(step), f32(1 - _BETA1), f32(1 - _BETA2), f32(_ADAM_EPS), f32(_WEIGHT_DECAY)

    def update(i):
        p, g, m, v, master = (s[k][i] for k in ('p', 'g', 'm', 'v', 'master'))
        weights, g, n = (p if master is None else master).float(), g.float(), p.numel()
        if case['bits'] == 8:
            old_m, r = s['m_values'][m.int()] * _of_blocks(s['m_scale'][i], n), s['r_values'][v.int()] * _of_blocks(s['v_scale'][i], n)
            old_v = r * r
        else:
            old_m, old_v = m, v
        new_m = old_m + c1 * (g - old_m)
        new_v = old_v + c2 * (g * g - old_v)
        root = torch.sqrt(new_v)
        new = weights - (step * (new_m / (root + eps)) + decay * weights)
        if case['bits'] == 8:
            words = _philox(n, i, t, s['seed'])
            up = lambda w: (w.float() + 0.5) * 2.0 ** -16  # noqa: E731
            m_code, m_scale = _stored(new_m, 16, up(words & 0xFFFF))
            v_code, v_scale = _stored(root, 32, up(words >> 16))
            m.copy_(m_code), v.copy_(v_code), s['m_scale'][i].copy_(m_scale), s['v_scale'][i].copy_(v_scale)
        else:
            m.copy_(new_m), v.copy_(new_v)
        p.copy_(new)
        if master is not None:
            master.copy_(new)

    [update(i) for i in range(len(s['p']))]
    return _adamw_outputs(s)


def _adamw_outputs(s):
    """All arrays' elements one after another; 8 bits as the values they stand for."""
    case = s['case']
    out = {'p': torch.cat(s['p'])}
    if case['bits'] == 8:
        scales = lambda k: torch.cat([_of_blocks(x, p.numel()) for x, p in zip(s[k], s['p'])])  # noqa: E731
        out.update(m=s['m_values'][torch.cat(s['m']).int()] * scales('m_scale'), root_v=s['r_values'][torch.cat(s['v']).int()] * scales('v_scale'))
    else:
        out.update(m=torch.cat(s['m']), v=torch.cat(s['v']))
    if s['master'][0] is not None:
        out['master'] = torch.cat(s['master'])
    return out


# ---------------------------------------------------------------------------------------------
# the calls
# ---------------------------------------------------------------------------------------------
class _Exported(object):
    """Device memory of an array, described for torch."""

    def __init__(self, a):
        self.array = a  # keeps the memory
        self.__cuda_array_interface__ = {'shape': a.shape, 'typestr': a.dtype.str, 'data': (a.data_ptr, False), 'version': 2}


def _named(**arrays):
    return {k: torch.as_tensor(_Exported(a), device='cuda') for k, a in arrays.items() if a is not None}


_NUMPY = {torch.float16: np.dtype('float16'), torch.float32: np.dtype('float32'), torch.int32: np.dtype('int32'), torch.uint8: np.dtype('uint8')}


def _array(chx, t):
    if t is None:
        return None
    dt = _NUMPY[t.dtype]
    return chx.ndarray(t, 0, tuple(t.shape), tuple(n * dt.itemsize for n in t.stride()), dt)


def _own(s):
    import chainer_amd as chx

    case, of = s['case'], lambda name: _array(chx, s[name])
    if case['kind'] == 'norm':
        x, gamma, beta = of('x'), of('gamma'), of('beta')
        y, norm = chx.layer_norm(x, gamma, beta, _EPS)
        out = _named(y=y, mean=norm.mean, inv_std=norm.inv_std)
        if s['gy'] is not None:
            gx, ggamma, gbeta = chx.layer_norm_grad(x, gamma, of('gy'), norm)
            out.update(_named(gx=gx, ggamma=ggamma, gbeta=gbeta))
        return out
    if case['kind'] == 'adamw':
        arrays = {k: [_array(chx, t) for t in s[k]] for k in ('p', 'g', 'm', 'v', 'm_scale', 'v_scale', 'master')}
        states = [chx.AdamWState(*x) for x in zip(*(arrays[k] for k in ('m', 'v', 'm_scale', 'v_scale', 'master')))]
        chx.adamw_update(arrays['p'], arrays['g'], states, s['t'], alpha=_ALPHA, beta1=_BETA1, beta2=_BETA2, eps=_ADAM_EPS, weight_decay_rate=_WEIGHT_DECAY, seed=s['seed'])
        return _adamw_outputs(s)
    args = [of(name) for name in ('q', 'k', 'v')]
    more = dict(log_decay=of('decay'), scale=s['scale'], state=of('state'), lengths=of('lengths'))
    y, new = chx.linear_attention(*args, **more)
    if s['gy'] is None:
        return _named(y=y, state=new)
    g = chx.linear_attention_grad(*args, of('gy'), gnew_state=of('gnew'), **more)
    return _named(y=y, state=new, gq=g.q, gk=g.k, gv=g.v, gdecay=g.log_decay, gstate=g.state)


def run(state):
    if own:
        return _own(state)
    return {'norm': _norm_plain, 'attend': _attend_plain, 'adamw': _adamw_plain}[state['case']['kind']](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and what it should give
# ---------------------------------------------------------------------------------------------
def work(case):
    it = np.dtype(case['dtype']).itemsize
    if case['kind'] == 'norm':
        n, params, train = case['rows'] * case['cols'], case['cols'] * np.dtype(case['params']).itemsize, case['train']
        return {'bytes': it * n * (4 if train else 2) + (4 if train else 2) * params + 8 * case['rows'], 'flops': n * (20 if train else 8)}
    if case['kind'] == 'adamw':
        n = sum(_arrays(case))
        weights = 8 + it if case['master'] and it == 2 else 2 * it
        return {'bytes': n * (weights + it + (16 if case['bits'] == 32 else 4)), 'flops': 14 * n}
    b, l, h, kh, dk, dv, train = case['batch'], case['length'], case['heads'], case['heads'] // case['shared'], case['keys'], case['values'], case['train']
    rows = b * l * (2 * kh * dk + h * dv)
    decay = {'rows': b * l * h, 'heads': h, 'none': 0}[case['decay']] * 4
    nbytes = it * (rows + b * l * h * dv) + decay + 2 * 4 * b * h * dk * dv
    if train:  # gy; the gradients
        nbytes += it * (b * l * h * dv + rows) + decay + 2 * 4 * b * h * dk * dv
    # the recurrence: decay, product and sum of the state, the row's product with it; three such products back, and a state of their own
    return {'bytes': nbytes, 'flops': b * l * h * dk * dv * (5 + (11 if train else 0))}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case['kind'] == 'norm':
        return _exact_norm(wide, case)
    if case['kind'] == 'adamw':
        return _exact_adamw(s, case)
    return _exact_attend(wide, case)


def _exact_norm(s, case):
    leaves = [s[k].requires_grad_(case['train']) for k in ('x', 'gamma', 'beta')]
    x, gamma, beta = leaves
    var, mean = torch.var_mean(x, 1, correction=0)
    inv = (var + _EPS).rsqrt()
    y = (x - mean[:, None]) * inv[:, None] * gamma + beta
    out = {'y': y.detach(), 'mean': mean.detach(), 'inv_std': inv.detach()}
    if case['train']:
        out.update(zip(('gx', 'ggamma', 'gbeta'), torch.autograd.grad(y, leaves, s['gy'])))
    return out


def _exact_adamw(s, case):
    """States of 8 bits come from draws next to a border between two codes: they have no such value."""
    t, cat = s['t'], lambda k: torch.cat(s[k]).double()
    eight = case['bits'] == 8
    g = cat('g')
    if eight:
        of = lambda k, scale, values: torch.cat([torch.from_numpy(values.astype(np.float64)).cuda()[c.long()] * x.double().repeat_interleave(_BLOCK)[:c.numel()]  # noqa: E731
                                                 for c, x in zip(s[k], s[scale])])
        m, v = of('m', 'm_scale', _M_VALUES), of('v', 'v_scale', _R_VALUES).square()
    else:
        m, v = cat('m'), cat('v')
    masters = s['master'][0] is not None
    p = cat('master') if masters else cat('p')
    m = _BETA1 * m + (1 - _BETA1) * g
    v = _BETA2 * v + (1 - _BETA2) * g * g
    p = p - _ALPHA * math.sqrt(1 - _BETA2 ** t) / (1 - _BETA1 ** t) * m / (v.sqrt() + _ADAM_EPS) - _WEIGHT_DECAY * p
    out = {'p': p, 'm': None if eight else m}
    out['root_v' if eight else 'v'] = None if eight else v
    if masters:
        out['master'] = p
    return out


def _exact_attend(s, case):
    """Row by row: the states forwards, for y and gq, and their gradients backwards, for gk, gv and the log decays' gradients."""
    b, l, h, shared, train = case['batch'], case['length'], case['heads'], case['shared'], case['train']
    if l * (2 if train else 1) * b * h * case['keys'] * case['values'] > 1.5e11:
        return None
    ends = torch.full((b,), l, device='cuda') if s['lengths'] is None else s['lengths'].long()
    live = (torch.arange(l, device='cuda')[:, None] < ends)  # [length, batch]
    rows = lambda x: torch.where(live[:, :, None, None], x.transpose(0, 1), 0.0)  # noqa: E731
    q, k = (rows(s[n]).repeat_interleave(shared, 2) for n in ('q', 'k'))
    v = rows(s['v'])
    decay = torch.ones(l, b, h, device='cuda', dtype=torch.float64)
    if s['decay'] is not None:
        decay = torch.where(live[..., None], torch.exp(s['decay'] if s['decay'].ndim == 1 else s['decay'].transpose(0, 1)), 1.0)
    gy = rows(s['gy']) if train else None
    state, ys, gqs = s['state'], [], []
    for t in range(l):
        state = torch.addcmul(state * decay[t, :, :, None, None], k[t].unsqueeze(3), v[t].unsqueeze(2))
        ys.append(torch.matmul(q[t].unsqueeze(2), state)[:, :, 0] * s['scale'])
        if train:
            gqs.append(torch.matmul(state, gy[t].unsqueeze(3))[..., 0] * s['scale'])
    out = {'y': torch.stack(ys, 1), 'state': state}
    if not train:
        return out
    r, gk, gv = s['gnew'], [None] * l, [None] * l
    for t in reversed(range(l)):
        r = torch.addcmul(r, q[t].unsqueeze(3) * s['scale'], gy[t].unsqueeze(2))
        gk[t] = torch.matmul(r, v[t].unsqueeze(3))[..., 0]
        gv[t] = torch.matmul(k[t].unsqueeze(2), r)[:, :, 0]
        r = r * decay[t, :, :, None, None]
    gq, gk, gv = (torch.where(live[..., None, None], torch.stack(x), 0.0) for x in (gqs, gk, gv))
    gg = (q * gq - k * gk).sum(3).flip(0).cumsum(0).flip(0) + (state * s['gnew']).sum((2, 3))
    gg = torch.where(live[..., None], gg, 0.0)
    fold = lambda x: x.unflatten(2, (h // shared, shared)).sum(3).transpose(0, 1)  # noqa: E731
    out.update(gq=fold(gq), gk=fold(gk), gv=gv.transpose(0, 1), gstate=r)
    if s['decay'] is not None:
        out['gdecay'] = gg.sum((0, 1)) if s['decay'].ndim == 1 else gg.transpose(0, 1)
    return out

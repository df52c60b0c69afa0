"""Cases for the training and serving operators around the contextualizer:

* ``linear``:  ``layers.residual_linear``, y = act(x W^T + b) + r, and its gradients;
* ``experts``: ``experts.expert_linear``, the same product grouped by expert with ragged row
  counts (no residual), and its gradients;
* ``adamw``:   ``optim.adamw_step``, one AdamW step over many tensors with 32-bit or 8-bit states.

``run`` computes them in plain torch operations in 32 bits (``own`` false) or through the
package's public entry points (``own`` true); ``exact`` computes them in 64 bits.
"""

import functools
import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
_ACTS = ('identity', 'relu', 'relu2', 'silu', 'gelu')
_BLOCK = 256  # elements that share a scale of the 8-bit states


def listed():
    return [
        # One token of one sequence through a dense layer: the latency of serving.
        dict(name='linear_token', op='linear', rows=1, d_in=768, d_out=1536, dtype='bf16',
             act='silu', residual=True, train=False),
        # One token each of a batch of sequences.
        dict(name='linear_batch', op='linear', rows=48, d_in=2048, d_out=1024, dtype='f16',
             act='relu2', residual=True, train=False),
        # A prompt of odd length through odd widths (rows that are not whole 16-byte units).
        dict(name='linear_odd', op='linear', rows=1037, d_in=389, d_out=771, dtype='bf16',
             act='gelu', residual=False, train=False),
        # Training step of a layer at 2 x 2048 tokens.
        dict(name='linear_train', op='linear', rows=4096, d_in=1024, d_out=1024, dtype='f16',
             act='gelu', residual=True, train=True),
        # Training step of a widening layer at 64 x 512 tokens.
        dict(name='linear_train_large', op='linear', rows=32768, d_in=768, d_out=1536,
             dtype='bf16', act='silu', residual=True, train=True),
        # Eight tokens, two experts each: most experts have one row or none.
        dict(name='experts_token', op='experts', rows=16, experts=16, spread=0.3, d_in=1024,
             d_out=2048, dtype='bf16', act='silu', train=False),
        # A prompt over many experts, unevenly loaded, some of them empty.
        dict(name='experts_prompt', op='experts', rows=8192, experts=32, spread=1.5, d_in=768,
             d_out=1536, dtype='f16', act='gelu', train=False),
        # Training step of a few experts on odd row counts.
        dict(name='experts_train_ragged', op='experts', rows=1999, experts=7, spread=1.0,
             d_in=392, d_out=520, dtype='f16', act='relu2', train=True),
        # Training step of a mixture at 64 x 512 tokens.
        dict(name='experts_train_large', op='experts', rows=32768, experts=8, spread=0.5,
             d_in=768, d_out=1536, dtype='bf16', act='silu', train=True),
        # A small model in fp32: many small tensors, so launches and host work count.
        dict(name='adamw_small', op='adamw', layers=6, width=128, context=256, dtype='f32',
             bits=32, master=False),
        # bf16 weights with fp32 master copies and fp32 states.
        dict(name='adamw_master', op='adamw', layers=24, width=1024, context=512, dtype='bf16',
             bits=32, master=True),
        # bf16 weights with 8-bit states.
        dict(name='adamw_8bit', op='adamw', layers=48, width=1536, context=2048, dtype='bf16',
             bits=8, master=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('linear', 'experts', 'adamw'))
    if op == 'adamw':
        bits = rng.choice((8, 32))
        dtype = rng.choice(('f32', 'bf16', 'f16'))
        return dict(op=op, layers=_log(rng, 1, 24), width=_log(rng, 64, 1536),
                    context=_log(rng, 64, 2048), dtype=dtype, bits=bits,
                    master=dtype != 'f32' and rng.random() < 0.5)
    train = rng.random() < 0.5
    case = dict(op=op, rows=_log(rng, 1, 32768), d_in=_log(rng, 64, 1536),
                d_out=_log(rng, 64, 1536), dtype=rng.choice(('bf16', 'f16')),
                act=rng.choice(_ACTS), train=train)
    if rng.random() < 0.6:  # most models' widths are whole multiples of a vector
        case['d_in'], case['d_out'] = 8 * (-(-case['d_in'] // 8)), 8 * (-(-case['d_out'] // 8))
    case['rows'] = min(case['rows'], 32768 * 768 * 1536 // (case['d_in'] * case['d_out']))
    if op == 'linear':
        case['residual'] = rng.random() < 0.5
    else:
        case['experts'] = _log(rng, 2, 64)
        case['spread'] = round(rng.uniform(0.0, 2.0), 2)
    return case


def _sizes(case):
    """Rows of each expert: a multinomial over log-normal loads, the same for every seed."""
    rng = random.Random(case['rows'] * 1000 + case['experts'])
    loads = [math.exp(rng.gauss(0.0, case['spread'])) for _ in range(case['experts'])]
    sizes = [0] * case['experts']
    for e in rng.choices(range(case['experts']), weights=loads, k=case['rows']):
        sizes[e] += 1
    return sizes


def _shapes(case):
    """Parameter shapes of a stack of Avey blocks: enricher, mixing matrix, fuser, norm."""
    d, c = case['width'], case['context']
    block = [(2 * d, d), (2 * d,), (c, c), (d,), (d, d), (d,), (d,)]
    return block * case['layers']


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dt = _DTYPES[case['dtype']]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device='cuda') * scale).to(dtype)

    state = dict(case)
    if case['op'] == 'adamw':
        shapes = _shapes(case)
        starts, total = [], 0
        for s in shapes:
            starts.append(total)
            total += -(-math.prod(s) // _BLOCK) * _BLOCK
        real = torch.zeros(total, device='cuda', dtype=torch.bool)
        for s, o in zip(shapes, starts):
            real[o:o + math.prod(s)] = True
        flat = {'p32': randn(total, scale=0.02, dtype=torch.float32) * real,
                'grad': randn(total, scale=1e-3) * real}
        m = randn(total, scale=5e-4, dtype=torch.float32) * real
        v = (1e-6 * (0.05 + torch.rand(total, generator=gen, device='cuda'))) * real
        flat['param'] = flat['p32'].to(dt)
        if case['master']:
            flat['master'] = flat['p32']
        del flat['p32']
        if case['bits'] == 8:
            for name, x in (('exp_avg', m), ('exp_avg_sq', v.sqrt())):
                scale = x.view(-1, _BLOCK).abs().amax(1).mul(1 / 448).clamp(min=2.0 ** -126)
                flat[name] = (x.view(-1, _BLOCK) / scale[:, None]).clamp(-448, 448).to(
                    torch.float8_e4m3fn).view(-1)
                flat[name + '_scale'] = scale
        else:
            flat['exp_avg'], flat['exp_avg_sq'] = m, v

        def views(name):
            if name not in flat:
                return None
            if name.endswith('scale'):
                return [flat[name][o // _BLOCK:o // _BLOCK + -(-math.prod(s) // _BLOCK)]
                        for s, o in zip(shapes, starts)]
            return [flat[name][o:o + math.prod(s)].view(s) for s, o in zip(shapes, starts)]

        state.update(flat=flat, step=100, seed=seed, lists={
            n: views(n) for n in ('param', 'grad', 'exp_avg', 'exp_avg_sq', 'master',
                                  'exp_avg_scale', 'exp_avg_sq_scale')})
        return state
    rows, d_in, d_out = case['rows'], case['d_in'], case['d_out']
    grad = case['train']
    groups = (case['experts'],) if case['op'] == 'experts' else ()
    state['x'] = randn(rows, d_in).requires_grad_(grad)
    state['weight'] = randn(*groups, d_out, d_in, scale=d_in ** -0.5).requires_grad_(grad)
    state['bias'] = randn(*groups, d_out, scale=0.1).requires_grad_(grad)
    if case.get('residual'):
        state['residual'] = randn(rows, d_out).requires_grad_(grad)
    if grad:
        state['dy'] = randn(rows, d_out)
    if groups:
        state['sizes'] = _sizes(case)
        ends = torch.tensor([0] + state['sizes'], device='cuda').cumsum(0)
        state['offsets'] = ends.to(torch.int32)
    return state


# ------------------------------------------------------------------ plain forms

def _act(x, act):
    """act(x) and its derivative."""
    if act == 'relu':
        return x.clamp(min=0), (x > 0).to(x.dtype)
    if act == 'relu2':
        r = x.clamp(min=0)
        return r * r, 2 * r
    if act == 'silu':
        s = 1 / (1 + torch.exp(-x))
        return x * s, s * (1 + x * (1 - s))
    if act == 'gelu':
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 0.134145 * x * x)
    return x, torch.ones_like(x)


def _plain_linear(x, w, b, r, dy, act):
    """y and, with dy, (dx, dw, db) of act(x w^T + b) + r, in fp32."""
    x, w = x.float(), w.float()
    y, d = _act(x @ w.t() + b.float(), act)
    if r is not None:
        y = y + r.float()
    if dy is None:
        return (y,)
    dpre = dy.float() * d
    return y, dpre @ w, dpre.t() @ x, dpre.sum(0)


def _hash(x):
    """32-bit integer hash of whole numbers below 2^32 (held in 64 bits)."""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _encode(x, noise):
    """x [blocks, 256] in fp32 as e4m3 codes and the blocks' scales; noise: 20-bit numbers."""
    scale = (x.abs().amax(1, keepdim=True) * (1 / 448)).clamp(min=2.0 ** -126)
    r = x.abs() * (1 / scale)
    small = r < 2.0 ** -6
    bits = torch.where(small, r + 2.0 ** -6, r).view(torch.int32)
    code = ((bits + noise) >> 20) - 960 - 8 * small.to(torch.int32)
    code = code.clamp(max=126) + 128 * (x < 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _plain_adamw(s):
    f = s['flat']
    s['step'] += 1
    step, lr, b1, b2, eps, wd = s['step'], 1e-3, 0.9, 0.95, 1e-8, 0.1
    quant = s['bits'] == 8
    g = f['grad'].float()
    p = (f['master'] if s['master'] else f['param']).float()
    m, v = f['exp_avg'], f['exp_avg_sq']
    if quant:
        m = m.float().view(-1, _BLOCK) * f['exp_avg_scale'][:, None]
        v = v.float().view(-1, _BLOCK) * f['exp_avg_sq_scale'][:, None]
        m, v = m.view(-1), (v * v).view(-1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = torch.sqrt(v)
    update = m / (root * (1 / math.sqrt(1 - b2 ** step)) + eps)
    p = p * (1 - lr * wd) - update * (lr / (1 - b1 ** step))
    if quant:
        key = (s['seed'] + 0x9e3779b9 * step) & 0xffffffff
        for mul in (0x7feb352d, 0x846ca68b):
            key = ((key ^ (key >> 16)) * mul) & 0xffffffff
        h = _hash(torch.arange(m.numel(), device=m.device) ^ key).view(-1, _BLOCK)
        low = (((h & 0xffff) << 4) + 8).to(torch.int32)
        high = (((h >> 16) << 4) + 8).to(torch.int32)
        for name, x, noise in (('exp_avg', m, low), ('exp_avg_sq', root, high)):
            code, scale = _encode(x.view(-1, _BLOCK), noise)
            f[name].copy_(code.view(-1))
            f[name + '_scale'].copy_(scale.view(-1))
    else:
        f['exp_avg'].copy_(m)
        f['exp_avg_sq'].copy_(v)
    f['param'].copy_(p)
    if s['master']:
        f['master'].copy_(p)


def _plain(s):
    op = s['op']
    if op == 'adamw':
        _plain_adamw(s)
        return _written(s)
    dt = s['x'].dtype
    x, w, b = s['x'].detach(), s['weight'].detach(), s['bias'].detach()
    dy = s.get('dy')
    if op == 'linear':
        r = s['residual'].detach() if s['residual'] is not False else None
        out = [t.to(dt) for t in _plain_linear(x, w, b, r, dy, s['act'])]
    else:
        dys = [None] * len(s['sizes']) if dy is None else dy.split(s['sizes'])
        parts = [_plain_linear(xe, w[e], b[e], None, dye, s['act'])
                 for e, (xe, dye) in enumerate(zip(x.split(s['sizes']), dys))]
        out = [(torch.cat if i < 2 else torch.stack)([p[i] for p in parts]).to(dt)
               for i in range(len(parts[0]))]
    if dy is not None and s.get('residual') is not None and s.get('residual') is not False:
        out.append(dy)
    return out


# ------------------------------------------------------------------ the package's calls

@functools.cache
def _package():
    from avey_kernel_b200 import experts, layers, optim
    return experts, layers, optim


def _own(s):
    experts, layers, optim = _package()
    op = s['op']
    if op == 'adamw':
        s['step'] += 1
        t = s['lists']
        optim.adamw_step(t['param'], t['grad'], t['exp_avg'], t['exp_avg_sq'], step=s['step'],
                         lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1,
                         masters=t['master'], exp_avg_scales=t['exp_avg_scale'],
                         exp_avg_sq_scales=t['exp_avg_sq_scale'], seed=s['seed'])
        return _written(s)
    leaves = [s['x'], s['weight'], s['bias']]
    if op == 'linear':
        r = s['residual'] if s['residual'] is not False else None
        y = layers.residual_linear(*leaves, activation=s['act'], residual=r)
        leaves += [] if r is None else [r]
    else:
        y = experts.expert_linear(s['x'], s['weight'], s['offsets'], s['bias'],
                                  activation=s['act'])
    if not s['train']:
        return [y]
    return [y, *torch.autograd.grad(y, leaves, s['dy'])]


def _written(s):
    """The buffers that an AdamW step writes."""
    return {k: v for k, v in s['flat'].items() if k != 'grad'}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ work and 64-bit results

def work(case):
    es = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'adamw':
        n = sum(math.prod(s) for s in _shapes(case))
        per = es + es + (8 if case['master'] else es)  # gradient, weight written, weight read
        per += 4 + 8 / _BLOCK * 2 if case['bits'] == 8 else 16
        return {'bytes': n * per, 'flops': n * 14}
    rows, k, n = case['rows'], case['d_in'], case['d_out']
    weights = n * k + n
    if case['op'] == 'experts':
        weights *= sum(1 for c in _sizes(case) if c)
    moved = rows * k + weights + rows * n + (rows * n if case.get('residual') else 0)
    flops = 2 * rows * n * k
    if case['train']:
        written = n * k + n  # every expert's gradient is written, empty ones among them
        if case['op'] == 'experts':
            written *= case['experts']
        moved += rows * n + rows * k + written
        flops *= 3
    return {'bytes': moved * es, 'flops': flops}


def _exact_act(x, act):
    """act(x) and its derivative in 64 bits, through autograd of torch's double functions."""
    x = x.detach().requires_grad_(True)
    f = {'identity': lambda t: t * 1.0, 'relu': torch.relu,
         'relu2': lambda t: torch.relu(t).square(), 'silu': torch.nn.functional.silu,
         'gelu': lambda t: torch.nn.functional.gelu(t, approximate='tanh')}[act]
    y = f(x)
    return y.detach(), torch.autograd.grad(y.sum(), x)[0]


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'adamw':
        f, t = s['flat'], s['step'] + 1
        grad = f['grad'].double()
        weight = (f['master'] if case['master'] else f['param']).double()
        first, second = f['exp_avg'].double(), f['exp_avg_sq'].double()
        if case['bits'] == 8:
            first = first * f['exp_avg_scale'].double().repeat_interleave(_BLOCK)
            second = (second * f['exp_avg_sq_scale'].double().repeat_interleave(_BLOCK)) ** 2
        first = torch.lerp(grad, first, 0.9)
        second = torch.lerp(grad.square(), second, 0.95)
        denom = (second / (1 - 0.95 ** t)).sqrt() + 1e-8
        weight = weight - 1e-3 * (0.1 * weight + first / (1 - 0.9 ** t) / denom)
        out = {k: None for k in _written(s)}
        out['param'] = weight
        if case['master']:
            out['master'] = weight
        if case['bits'] == 8:  # the codes depend on the rounding's random numbers
            out['exp_avg_scale'] = first.view(-1, _BLOCK).abs().amax(1) / 448
            out['exp_avg_sq_scale'] = second.view(-1, _BLOCK).amax(1).sqrt() / 448
        else:
            out['exp_avg'], out['exp_avg_sq'] = first, second
        return out
    x, w, b = (s[k].detach().double() for k in ('x', 'weight', 'bias'))
    sizes = s.get('sizes', [case['rows']])
    w3, b2 = w.view(len(sizes), *w.shape[-2:]), b.view(len(sizes), -1)
    y = x.new_zeros(case['rows'], case['d_out'])
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w3), torch.zeros_like(b2)
    start = 0
    for e, count in enumerate(sizes):
        rows = slice(start, start + count)
        start += count
        y[rows], d = _exact_act(torch.einsum('tk,nk->tn', x[rows], w3[e]) + b2[e], case['act'])
        if case['train']:
            d = d * s['dy'][rows].double()
            dx[rows] = torch.einsum('tn,nk->tk', d, w3[e])
            dw[e] = torch.einsum('tn,tk->nk', d, x[rows])
            db[e] = d.sum(0)
    if case.get('residual'):
        y = y + s['residual'].detach().double()
    if not case['train']:
        return [y]
    out = [y, dx, dw.view(w.shape), db.view(b.shape)]
    return out + ([s['dy'].double()] if case.get('residual') else [])

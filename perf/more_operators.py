"""Cases for the operators at the two ends of a stack of Avey blocks and around its experts:

* ``loss``:      ``losses.linear_cross_entropy``, softmax cross entropy of ``x W^T`` over a
  vocabulary without keeping the logits, and its gradients;
* ``route``:     ``experts.route``, the choice of experts for every token and their weights, and
  the gradient of the logits;
* ``experts``:   ``experts.arrange``, ``experts.dispatch`` and ``experts.combine``: sort the
  choices by expert, bring the tokens there and add the weighted results up, and their gradients;
* ``embedding``: ``layers.embedding``, rows of a table with a scale, and the table's gradient.

``run`` computes them in plain torch operations in 32 bits (``own`` false) or through the
package's public entry points (``own`` true); ``exact`` computes them in 64 bits.
"""

import functools
import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
_IGNORED = -100


def listed():
    return [
        # The likelihood of one token of one sequence: scoring while serving.
        dict(name='loss_token', op='loss', rows=1, width=768, vocab=32768, dtype='bf16',
             reduction='none', z_loss=0.0, ignored=0.0, train=False),
        # A few sequences of odd length with padding, a weight for each token, odd widths.
        dict(name='loss_ragged_train', op='loss', rows=1037, width=389, vocab=10007, dtype='f16',
             reduction='none', z_loss=1e-4, ignored=0.2, train=True),
        # Training step at 8 x 512 tokens and a vocabulary that no tile divides.
        dict(name='loss_train', op='loss', rows=4096, width=1024, vocab=50021, dtype='bf16',
             reduction='mean', z_loss=1e-4, ignored=0.05, train=True),
        # Training step at 32 x 512 tokens and a large vocabulary.
        dict(name='loss_train_large', op='loss', rows=16384, width=768, vocab=131072,
             dtype='bf16', reduction='mean', z_loss=0.0, ignored=0.0, train=True),
        # One token of one sequence.
        dict(name='route_token', op='route', rows=1, experts=64, k=2, dtype='f32',
             score='softmax', bias=False, groups=1, top_groups=1, group_best=1,
             renormalize=True, scale=1.0, train=False),
        # A prompt over many experts in groups, with the bias that balances them.
        dict(name='route_prompt', op='route', rows=4093, experts=256, k=8, dtype='bf16',
             score='sigmoid', bias=True, groups=8, top_groups=4, group_best=2,
             renormalize=True, scale=2.5, train=False),
        # Training step at 128 x 512 tokens.
        dict(name='route_train', op='route', rows=65536, experts=128, k=4, dtype='f32',
             score='softmax', bias=False, groups=1, top_groups=1, group_best=1,
             renormalize=False, scale=1.0, train=True),
        # One token each of a batch of sequences.
        dict(name='experts_token', op='experts', rows=16, experts=16, k=2, width=1024,
             dtype='bf16', residual=True, train=False),
        # Training step at 64 x 512 tokens.
        dict(name='experts_train', op='experts', rows=32768, experts=64, k=4, width=768,
             dtype='bf16', residual=True, train=True),
        # One token each of a batch of sequences.
        dict(name='embedding_token', op='embedding', rows=8, vocab=32768, width=768,
             dtype='bf16', scale=1.0, padding=False, train=False),
        # A padded batch of odd length through an odd width in fp32, scaled by the root of it.
        dict(name='embedding_ragged_train', op='embedding', rows=2047, vocab=32003, width=389,
             dtype='f32', scale=19.723, padding=True, train=True),
        # Training step at 128 x 512 tokens and a large vocabulary.
        dict(name='embedding_train_large', op='embedding', rows=65536, vocab=131072, width=768,
             dtype='bf16', scale=1.0, padding=False, train=True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm, odd ones among them."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('loss', 'loss', 'route', 'experts', 'embedding'))
    train = rng.random() < 0.6
    if op == 'loss':
        case = dict(op=op, rows=_log(rng, 1, 16384), width=_log(rng, 64, 2048),
                    vocab=_log(rng, 500, 131072), dtype=rng.choice(('bf16', 'f16')),
                    reduction=rng.choice(('mean', 'sum', 'none')),
                    z_loss=rng.choice((0.0, 1e-4)), ignored=rng.choice((0.0, 0.1, 0.5)),
                    train=train)
        if rng.random() < 0.6:  # most models' widths are whole multiples of a vector
            case['width'] = 8 * (-(-case['width'] // 8))
        most = 16384 * 768 * 131072 // (case['width'] * case['vocab'])
        case['rows'] = max(1, min(case['rows'], most))
        return case
    if op == 'route':
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _log(rng, 2, 512 // groups)
        top = rng.randint(1, groups)
        return dict(op=op, rows=_log(rng, 1, 65536 * 128 // max(experts, 128)), experts=experts,
                    k=rng.randint(1, min(8, experts // groups * top)),
                    dtype=rng.choice(('f32', 'bf16', 'f16')),
                    score=rng.choice(('softmax', 'sigmoid')), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top, group_best=rng.choice((1, 2)),
                    renormalize=rng.random() < 0.5, scale=rng.choice((1.0, 2.5)), train=train)
    dtype = rng.choice(('f32', 'bf16', 'f16'))
    if op == 'experts':
        experts, width, k = _log(rng, 2, 256), _log(rng, 32, 2048), rng.randint(1, 8)
        most = 32768 * 4 * 768 // (k * width * (2 if dtype == 'f32' else 1))
        return dict(op=op, rows=min(_log(rng, 1, 32768), most), experts=experts,
                    k=min(k, experts), width=width, dtype=dtype, residual=rng.random() < 0.5,
                    train=train)
    width = _log(rng, 32, 1536)
    most = 65536 * 768 // (width * (2 if dtype == 'f32' else 1))
    return dict(op=op, rows=min(_log(rng, 1, 65536), most), width=width,
                vocab=min(_log(rng, 500, 131072), 2 * most), dtype=dtype,
                scale=rng.choice((1.0, round(math.sqrt(width), 3))), padding=rng.random() < 0.5,
                train=train)


def _tokens(n, vocab, gen):
    """Tokens as text has them: the r-th most frequent one about as often as 1 / r."""
    u = torch.rand(n, generator=gen, device='cuda', dtype=torch.float64)
    rank = torch.exp(u * math.log(vocab + 1.0)).long().clamp(1, vocab) - 1
    return (rank * 7919 + 1) % vocab


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dt, op, rows, train = _DTYPES[case['dtype']], case['op'], case['rows'], case['train']

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device='cuda') * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device='cuda')

    state = dict(case)
    if op == 'loss':
        # Normalised rows that lean towards their target, as a trained model's do.
        target = _tokens(rows, case['vocab'], gen)
        weight = randn(case['vocab'], case['width'], scale=2 * case['width'] ** -0.5)
        x = torch.randn(rows, case['width'], generator=gen, device='cuda')
        state['x'] = (x + weight[target].float()).to(dt).requires_grad_(train)
        state['weight'] = weight.requires_grad_(train)
        ignored = rand(rows) < case['ignored']
        ignored[0] = False
        state['target'] = torch.where(ignored, _IGNORED, target)
        if train:
            # What comes from behind: a weight for each token, or one; f16 is trained with the
            # loss scaled up.
            scale = 2048.0 if case['dtype'] == 'f16' and case['reduction'] == 'mean' else 1.0
            state['dy'] = (0.5 + rand(rows) if case['reduction'] == 'none'
                           else torch.full((), scale, device='cuda'))
    elif op == 'route':
        state['logits'] = randn(rows, case['experts'], scale=1.5).requires_grad_(train)
        if case['bias']:
            state['expert_bias'] = randn(case['experts'], scale=0.05, dtype=torch.float32)
        if train:
            state['dy'] = randn(rows, case['k'], dtype=torch.float32)
    elif op == 'experts':
        n, k = case['experts'], case['k']
        load = torch.randn(n, generator=gen, device='cuda') * 0.5  # some experts are liked better
        chosen = (load + torch.randn(rows, n, generator=gen, device='cuda')).argsort(dim=1)
        state['chosen'] = chosen[:, n - k:].to(torch.int32).contiguous()
        state['x'] = randn(rows, case['width']).requires_grad_(train)
        state['y'] = randn(rows * k, case['width']).requires_grad_(train)
        state['weights'] = torch.softmax(randn(rows, k, dtype=torch.float32), 1).requires_grad_(train)
        if case['residual']:
            state['res'] = randn(rows, case['width']).requires_grad_(train)
        if train:
            state['drows'] = randn(rows * k, case['width'])
            state['dout'] = randn(rows, case['width'])
    else:
        state['tokens'] = _tokens(rows, case['vocab'], gen)
        if case['padding']:  # the last tenth of the batch
            state['tokens'][rows - rows // 10:] = 0
        state['weight'] = randn(case['vocab'], case['width'], scale=0.02).requires_grad_(train)
        if train:
            state['dy'] = randn(rows, case['width'])
    return state


# ------------------------------------------------------------------ plain forms

def _plain_loss(s):
    dt = s['x'].dtype
    x, w, t = s['x'].detach().float(), s['weight'].detach().float(), s['target']
    z = x @ w.t()
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    used = t != _IGNORED
    index = torch.where(used, t, 0)[:, None]
    picked = z.gather(1, index)[:, 0]
    each = (lse - picked + s['z_loss'] * lse * lse) * used
    count = used.sum()
    loss = {'none': each, 'sum': each.sum(), 'mean': each.sum() / count}[s['reduction']]
    if not s['train']:
        return [loss]
    g = s['dy'].expand_as(each) * used
    if s['reduction'] == 'mean':
        g = g / count.clamp(min=1)
    dz = e.div_(total).mul_((1 + 2 * s['z_loss'] * lse)[:, None])
    dz.scatter_add_(1, index, -torch.ones_like(picked)[:, None])
    dz.mul_(g[:, None])
    return [loss, (dz @ w).to(dt), (dz.t() @ x).to(dt)]


def _scores(z, kind):
    if kind == 'sigmoid':
        return 1 / (1 + torch.exp(-z))
    e = torch.exp(z - z.max(dim=1, keepdim=True).values)
    return e / e.sum(dim=1, keepdim=True)


def _choose(s):
    """The k experts of every token: by 64-bit scores, so that near ones keep their order."""
    z = s['logits'].detach().double()
    rows, n = z.shape
    score = _scores(z, s['score'])
    rank = score + s['expert_bias'].double() if s['bias'] else z
    if s['groups'] > 1:
        by = rank if s['bias'] or s['group_best'] == 1 else score
        best = by.view(rows, s['groups'], -1).sort(dim=2, descending=True).values
        group = best[:, :, :s['group_best']].sum(dim=2)
        order = torch.sort(-group, dim=1, stable=True).indices[:, :s['top_groups']]
        keep = torch.zeros_like(group, dtype=torch.bool).scatter_(1, order, True)
        keep = keep.repeat_interleave(n // s['groups'], dim=1)
        rank = torch.where(keep, rank, -math.inf)
    return torch.sort(-rank, dim=1, stable=True).indices[:, :s['k']]


def _plain_route(s):
    z = s['logits'].detach().float()
    chosen = _choose(s)
    score = _scores(z, s['score'])
    w = score.gather(1, chosen)
    total = w.sum(dim=1, keepdim=True) if s['renormalize'] else 1.0
    weights = w / total * s['scale']
    out = [weights, chosen.to(torch.int32)]
    if s['train']:
        g = s['dy'] * s['scale']
        if s['renormalize']:
            g = (g - (g * (w / total)).sum(dim=1, keepdim=True)) / total
        dscore = torch.zeros_like(score).scatter_(1, chosen, g)
        if s['score'] == 'sigmoid':
            dz = dscore * score * (1 - score)
        else:
            dz = score * (dscore - (dscore * score).sum(dim=1, keepdim=True))
        out.append(dz.to(s['logits'].dtype))
    return out


def _plain_experts(s):
    chosen, k = s['chosen'].reshape(-1).long(), s['k']
    x, y, w = s['x'].detach(), s['y'].detach(), s['weights'].detach()
    order = torch.sort(chosen, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    bounds = torch.arange(s['experts'] + 1, device=order.device)
    offsets = (chosen[:, None] < bounds).sum(dim=0)
    rows = x[order // k]
    slots = slots.view(-1, k)
    mine = y.float()[slots]  # [rows, k, width]
    out = (w[:, :, None] * mine).sum(dim=1)
    if s['residual']:
        out = out + s['res'].detach().float()
    out = [slots.to(torch.int32), offsets.to(torch.int32), rows, out.to(x.dtype)]
    if s['train']:
        dout = s['dout'].float()
        dx = s['drows'].float()[slots].sum(dim=1)
        dy = torch.empty_like(y)
        dy[slots] = (w[:, :, None] * dout[:, None, :]).to(y.dtype)
        out += [dx.to(x.dtype), dy, (mine * dout[:, None, :]).sum(dim=2)]
        if s['residual']:
            out.append(s['dout'])
    return out


def _plain_embedding(s):
    w, t = s['weight'].detach(), s['tokens']
    out = [(w[t].float() * s['scale']).to(w.dtype)]
    if s['train']:
        dw = torch.zeros(w.shape, device=w.device)
        dw.index_add_(0, t, s['dy'].float() * s['scale'])
        if s['padding']:
            dw[0] = 0
        out.append(dw.to(w.dtype))
    return out


_PLAIN = {'loss': _plain_loss, 'route': _plain_route, 'experts': _plain_experts,
          'embedding': _plain_embedding}


# ------------------------------------------------------------------ the package's calls

@functools.cache
def _package():
    from avey_kernel_b200 import experts, layers, losses
    return experts, layers, losses


def _own(s):
    experts, layers, losses = _package()
    op = s['op']
    if op == 'loss':
        loss = losses.linear_cross_entropy(s['x'], s['weight'], s['target'],
                                           ignore_index=_IGNORED, reduction=s['reduction'],
                                           z_loss=s['z_loss'])
        if not s['train']:
            return [loss]
        return [loss, *torch.autograd.grad(loss, (s['x'], s['weight']), s['dy'])]
    if op == 'route':
        weights, chosen = experts.route(s['logits'], s['k'], bias=s.get('expert_bias'),
                                        score=s['score'], groups=s['groups'],
                                        top_groups=s['top_groups'], group_best=s['group_best'],
                                        renormalize=s['renormalize'], scale=s['scale'])
        if not s['train']:
            return [weights, chosen]
        return [weights, chosen, *torch.autograd.grad(weights, s['logits'], s['dy'])]
    if op == 'experts':
        slots, offsets = experts.arrange(s['chosen'], s['experts'])
        rows = experts.dispatch(s['x'], slots)
        out = experts.combine(s['y'], slots, s['weights'], residual=s.get('res'))
        if not s['train']:
            return [slots, offsets, rows, out]
        leaves = [s['x'], s['y'], s['weights']] + ([s['res']] if s['residual'] else [])
        return [slots, offsets, rows, out,
                *torch.autograd.grad((rows, out), leaves, (s['drows'], s['dout']))]
    out = layers.embedding(s['tokens'], s['weight'], scale=s['scale'],
                           padding_idx=0 if s['padding'] else None)
    if not s['train']:
        return [out]
    return [out, *torch.autograd.grad(out, s['weight'], s['dy'])]


def run(state):
    return _own(state) if own else _PLAIN[state['op']](state)


# ------------------------------------------------------------------ work and 64-bit results

def work(case):
    es = 4 if case['dtype'] == 'f32' else 2
    rows, train = case['rows'], case['train']
    if case['op'] == 'loss':
        # The logits once and, in training, the two products of the gradients.
        size = (rows + case['vocab']) * case['width'] * es
        moved = size * (2 if train else 1) + rows * 8
        moved += 4 * rows * (2 if train else 1) if case['reduction'] == 'none' else 4
        return {'bytes': moved, 'flops': 2 * rows * case['width'] * case['vocab'] * (3 if train else 1)}
    if case['op'] == 'route':
        n, k = case['experts'], case['k']
        moved = rows * (n * es * (2 if train else 1) + k * (12 if train else 8))
        return {'bytes': moved, 'flops': rows * n * (10 if train else 5)}
    if case['op'] == 'experts':
        k, width = case['k'], case['width'] * es
        # choices, slots, weights; x to its rows, and the rows back to the tokens
        moved = rows * k * 12 + rows * width * (2 + 2 * k + (1 if case['residual'] else 0))
        flops = 2 * rows * k * case['width']
        if train:  # rows' gradients to x; the tokens' to the rows and weights
            moved += rows * k * 4 + rows * width * (2 + 2 * k)
            flops *= 3
        return {'bytes': moved, 'flops': flops}
    width = case['width'] * es
    # Rows of the table that the tokens name, as _tokens draws them.
    name = rows / math.log(case['vocab'] + 1.0)
    distinct = sum(1 - math.exp(-name * math.log1p(1 / r)) for r in range(1, case['vocab'] + 1))
    moved = rows * 8 + (distinct + rows) * width
    if train:
        moved += (rows + case['vocab']) * width
    return {'bytes': moved, 'flops': rows * case['width'] * (2 if train else 1)}


def _exact_loss(case, s):
    x, w, t = s['x'].detach().double(), s['weight'].detach().double(), s['target']
    valid = t.ne(_IGNORED)
    if case['train']:
        factor = s['dy'].double().expand(case['rows']).clone()
        if case['reduction'] == 'mean':
            factor /= max(int(valid.sum()), 1)
        dw = torch.zeros_like(w)
    losses, dx = [], []
    step = max(1, (1 << 28) // case['vocab'])
    for a in range(0, case['rows'], step):
        part = slice(a, a + step)
        logits = torch.einsum('rd,vd->rv', x[part], w)
        logp = torch.log_softmax(logits, dim=1)
        norm = logits[:, 0] - logp[:, 0]
        pick = torch.arange(logits.shape[0], device=x.device), t[part].clamp(min=0)
        each = case['z_loss'] * norm.square() - logp[pick]
        losses.append(each.masked_fill(~valid[part], 0.0))
        if case['train']:
            grad = logp.exp()
            grad *= (1 + 2 * case['z_loss'] * norm)[:, None]
            grad[pick] -= 1
            grad *= (factor[part] * valid[part])[:, None]
            dx.append(torch.einsum('rv,vd->rd', grad, w))
            dw += torch.einsum('rv,rd->vd', grad, x[part])
    each = torch.cat(losses)
    total = each if case['reduction'] == 'none' else each.sum()
    if case['reduction'] == 'mean':
        total = total / valid.sum()
    return [total, torch.cat(dx), dw] if case['train'] else [total]


def _exact_route(case, s):
    z = s['logits'].detach().double().requires_grad_(case['train'])
    score = torch.sigmoid(z) if case['score'] == 'sigmoid' else torch.softmax(z, dim=1)
    base = score.detach() + s['expert_bias'].double() if case['bias'] else z.detach()
    left = base.clone()
    size = case['experts'] // case['groups']
    if case['groups'] > 1:
        value = base if case['bias'] or case['group_best'] == 1 else score.detach()
        value = value.reshape(case['rows'], case['groups'], size)
        first = value.max(dim=2)
        merit = first.values
        if case['group_best'] == 2 and size > 1:
            rest = value.scatter(2, first.indices[:, :, None], -math.inf)
            merit = merit + rest.max(dim=2).values
        taken = torch.zeros_like(merit, dtype=torch.bool)
        for _ in range(case['top_groups']):
            open_merit = merit.masked_fill(taken, -math.inf)
            top = open_merit.max(dim=1, keepdim=True).values
            best = (open_merit == top) & ~taken
            taken |= best & best.int().cumsum(1).eq(1)  # the first of them, as ties go
        left = left.masked_fill(~taken.repeat_interleave(size, 1), -math.inf)
    chosen = []
    for _ in range(case['k']):
        top = left.max(dim=1, keepdim=True).values
        index = torch.where(left == top, torch.arange(case['experts'], device=z.device),
                            case['experts']).min(dim=1, keepdim=True).values
        chosen.append(index)
        left = left.scatter(1, index, -math.inf)
    chosen = torch.cat(chosen, dim=1)
    weights = torch.take_along_dim(score, chosen, dim=1)
    if case['renormalize']:
        weights = weights / weights.sum(dim=1, keepdim=True)
    weights = weights * case['scale']
    out = [weights.detach(), chosen.to(torch.int32)]
    if case['train']:
        out.append(torch.autograd.grad(weights, z, s['dy'].double())[0])
    return out


def _exact_experts(case, s):
    k, n = case['k'], case['rows'] * case['k']
    flat = s['chosen'].reshape(-1).long()
    # The place of a choice: those of lower experts, then those before it of its own.
    counts = torch.bincount(flat, minlength=case['experts'])
    ends = torch.cumsum(counts, 0)
    place = torch.argsort(flat * n + torch.arange(n, device=flat.device))
    slots = torch.argsort(place)
    offsets = torch.cat([ends.new_zeros(1), ends])
    x, w = s['x'].detach().double(), s['weights'].detach().double()
    y, at = s['y'].detach().double(), slots.view(-1, k)
    rows = torch.empty_like(y)
    out = s['res'].detach().double() if case['residual'] else torch.zeros_like(x)
    for j in range(k):
        rows[at[:, j]] = x
        out = out + w[:, j, None] * y[at[:, j]]
    result = [at.to(torch.int32), offsets.to(torch.int32), rows, out]
    if case['train']:
        drows, dout = s['drows'].double(), s['dout'].double()
        dx, dy, dw = torch.zeros_like(x), torch.empty_like(y), torch.empty_like(w)
        for j in range(k):
            dx += drows[at[:, j]]
            dy[at[:, j]] = w[:, j, None] * dout
            dw[:, j] = (y[at[:, j]] * dout).sum(dim=1)
        result += [dx, dy, dw] + ([dout] if case['residual'] else [])
    return result


def _exact_embedding(case, s):
    w, t = s['weight'].detach().double(), s['tokens']
    out = [torch.index_select(w, 0, t) * case['scale']]
    if case['train']:
        dy = s['dy'].double() * case['scale']
        if case['padding']:
            dy = dy * (t != 0)[:, None]
        order = torch.argsort(t)
        sums = torch.cumsum(torch.bincount(t, minlength=case['vocab']), 0)
        edges = torch.cat([sums.new_zeros(1), sums])
        dw = torch.segment_reduce(dy[order], 'sum', offsets=edges, axis=0, initial=0.0)
        out.append(dw)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {'loss': _exact_loss, 'route': _exact_route, 'experts': _exact_experts,
            'embedding': _exact_embedding}[case['op']](case, s)

"""``experts.route``, ``arrange``, ``dispatch`` and ``combine`` against their formulas in 64
bits, written apart from the package's PyTorch form.

Tolerances: with u = 2^-24 (fp32), 2^-11 (f16) or 2^-8 (bf16), weights are off by 2^-20 of
themselves (an exponential and a division of two units in the last place each, a sum of up
to 37 additions) and in the last place of what underflows (2^-120); a gradient of the logits
by 2^-18 of the sum of its terms' sizes, rounded once (u; f16 2^-25); a combined row by (k +
1) 2^-23 of the sum of its terms' sizes, rounded once; a weight's gradient by (width + 1)
2^-23 of the sum of its terms' sizes."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from avey_kernel_b200 import _native, experts

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -120, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -120}
DTYPES = list(UNIT)
INF = math.inf


# ------------------------------------------------------------------ the choice

def scores64(z, score):
    z = z.double()
    if score == 'sigmoid':
        return torch.sigmoid(z)
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - torch.where(top == -INF, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return torch.where(total == 0, 0.0, e / total)


def choose64(z, k, bias, score, groups, top_groups, group_best):
    """The k experts of each token, one token at a time in Python's own ordering."""
    s = scores64(z, score).tolist()
    z = z.double().tolist()
    b = None if bias is None else bias.double().tolist()
    out = []
    for zt, st in zip(z, s):
        n = len(zt)

        def rank(e, use_score):
            r = zt[e] if b is None and not use_score else st[e] + (0.0 if b is None else b[e])
            if math.isnan(zt[e]) or math.isnan(r):
                return -2, 0.0
            return (-1, 0.0) if zt[e] == -INF else (0, r)

        size = n // groups
        merits = []
        for g in range(groups):
            best = sorted((rank(e, group_best == 2 and b is None) for e in range(g * size, (g + 1) * size)),
                          reverse=True)[:group_best]
            good = [r for tier, r in best if tier == 0]
            merits.append(sum(good) if good else -INF)
        kept = sorted(range(groups), key=lambda g: (-merits[g], g))[:top_groups]
        pool = [e for e in range(n) if e // size in kept]
        out.append(sorted(pool, key=lambda e: (-rank(e, False)[0], -rank(e, False)[1], e))[:k])
    return torch.tensor(out, dtype=torch.int32).view(-1, k)


def reference(z, chosen, dy, score, renormalize, scale):
    """Weights and dlogits with their bounds. Scores over their sum are the softmax of their
    logarithms, in which what does not depend on a logit does not cancel either."""
    dt, z = z.dtype, z.double().requires_grad_(True)
    s = torch.sigmoid(z) if score == 'sigmoid' else torch.softmax(z, -1)
    if renormalize:
        logs = torch.nn.functional.logsigmoid(z) if score == 'sigmoid' else z
        w = torch.softmax(logs.gather(-1, chosen.long()), -1)
    else:
        w = s.gather(-1, chosen.long())
    w = w * scale
    out = [(w.detach(), 2.0 ** -20 * w.detach().abs() + 2.0 ** -120)]
    if dy is not None:
        dz = torch.autograd.grad(w, z, dy.double())[0]
        # |dz_e| is a sum of terms up to |score| (|g_e| + sum |g| w).
        g = torch.zeros_like(dz).scatter_(-1, chosen.long(), dy.double().abs() * scale)
        if renormalize:
            q = torch.zeros_like(dz).scatter_(-1, chosen.long(), w.detach() / scale)
        else:
            q = s.detach()
        size = q * (g + (g * q).sum(-1, keepdim=True))
        out.append((dz, 2.0 ** -18 * size + UNIT[dt] * dz.abs() * (1 + 2.0 ** -8) + TINY[dt]))
    return out


def close(got, want, name):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} outside, worst '
                           f'{float(((got - value).abs() / bound.clamp(min=1e-300)).max()):.3g} of the bound')


def check_route(rows, n, k, dt, device, score='softmax', bias=False, groups=1, top_groups=1, group_best=1,
                renormalize=True, scale=1.0, seed=0, spread=1.5):
    g = torch.Generator(device=device).manual_seed(seed)
    z = (torch.randn(rows, n, generator=g, device=device) * spread).to(dt)
    b = torch.randn(n, generator=g, device=device) * 0.05 if bias else None
    dy = torch.randn(rows, k, generator=g, device=device)
    want = choose64(z.cpu(), k, None if b is None else b.cpu(), score, groups, top_groups, group_best)
    leaf = z.clone().requires_grad_(True)
    kw = dict(bias=b, score=score, groups=groups, top_groups=top_groups, group_best=group_best,
              renormalize=renormalize, scale=scale)
    w, chosen = experts.route(leaf, k, **kw)
    assert chosen.dtype == torch.int32 and w.dtype == torch.float32 and not chosen.requires_grad
    assert torch.equal(chosen.cpu(), want)
    dz, = torch.autograd.grad(w, leaf, dy)
    assert dz.dtype == dt
    (ww, wz) = reference(z, chosen, dy, score, renormalize, scale)
    close(w, ww, 'weights')
    close(dz, wz, 'dlogits')
    with torch.no_grad():
        again = experts.route(z, k, **kw)
    assert torch.equal(again[0], w) and torch.equal(again[1], chosen)


DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
CHOICES = [dict(), dict(bias=True), dict(score='sigmoid', bias=True), dict(score='sigmoid', renormalize=False, scale=2.5),
           dict(renormalize=False), dict(bias=True, renormalize=False, scale=0.5)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('kw', CHOICES)
@pytest.mark.parametrize('dt', DTYPES)
def test_routing_and_its_gradient(kw, dt, device):
    check_route(300, 64, 6, dt, device, **kw)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('rows,n,k', [(1, 1, 1), (1, 64, 2), (9, 3, 3), (50, 33, 32), (70, 100, 7), (65, 129, 5),
                                      (40, 256, 8), (33, 511, 9), (20, 1000, 4), (17, 1024, 32)])
def test_routing_sizes(rows, n, k, device):
    for dt in (torch.float32, torch.bfloat16):
        check_route(rows, n, k, dt, device, score='sigmoid', bias=True, scale=2.0)
        check_route(rows, n, k, dt, device, renormalize=False)


GROUPS = [(64, 8, 4, 2, 6), (64, 8, 4, 1, 6), (96, 3, 1, 2, 20), (60, 12, 5, 2, 8), (8, 8, 3, 2, 3), (32, 32, 32, 1, 4),
          (320, 10, 2, 2, 8), (1024, 32, 7, 2, 16)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score,bias', [('softmax', False), ('softmax', True), ('sigmoid', False), ('sigmoid', True)])
@pytest.mark.parametrize('n,groups,top,best,k', GROUPS)
def test_routing_in_groups(n, groups, top, best, k, score, bias, device):
    check_route(60, n, k, torch.float32, device, score=score, bias=bias, groups=groups, top_groups=top, group_best=best)
    check_route(60, n, k, torch.bfloat16, device, score=score, bias=bias, groups=groups, top_groups=top,
                group_best=best, renormalize=False)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('groups', [1, 4])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_near_scores_keep_the_order_of_exact_arithmetic(score, groups, device):
    """Ranks a few 10^-8 apart, below fp32's steps at their size; and equal ones, in the
    order of their numbers."""
    n = 32
    g = torch.Generator().manual_seed(5)
    z = 0.5 + 2.0 ** -22 * torch.randint(-4, 5, (400, n), generator=g).float()
    bias = 0.25 + 2.0 ** -24 * torch.randint(-4, 5, (n,), generator=g).float()
    z[::7] = 0.5  # rows that the bias alone orders
    bias[3::5] = 0.25
    for b in (bias, None):
        want = choose64(z, 5, b, score, groups, 2 if groups > 1 else 1, 2)
        _, chosen = experts.route(z.to(device), 5, bias=None if b is None else b.to(device), score=score, groups=groups,
                                  top_groups=2 if groups > 1 else 1, group_best=2)
        assert torch.equal(chosen.cpu(), want)
    _, chosen = experts.route(torch.zeros(5, n, device=device), 4, bias=torch.zeros(n, device=device), groups=groups,
                              top_groups=1)
    assert chosen.tolist() == [[0, 1, 2, 3]] * 5


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('n,groups,k', [(16, 1, 4), (64, 1, 5), (256, 1, 8), (512, 1, 32), (1000, 1, 3), (64, 4, 6),
                                        (256, 8, 8), (60, 6, 7), (512, 16, 8)])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_clusters_of_near_scores_at_the_border(score, n, groups, k, device):
    """Rows with a cluster of two to six near ranks, some of them alike, among others that are far
    apart: inside the chosen ones, over their last place and behind it, and between groups."""
    g = torch.Generator().manual_seed(n + k)
    rows = 300
    z = torch.randn(rows, n, generator=g)
    bias = torch.randint(0, 3, (n,), generator=g).float() * 2.0 ** -24
    order = z.argsort(1, descending=True)
    for t in range(rows):
        size = 2 + t % 5
        first = max(0, min(n - size, (k - 4 if groups == 1 else 0) + t // 5 % 8))
        at = order[t, first:first + size]
        z[t, at] = z[t, at[0]] * (1 + 2.0 ** -23 * torch.randint(0, 2, (size,), generator=g).float())
    want = choose64(z, k, bias, score, groups, max(1, groups // 2), 2)
    _, chosen = experts.route(z.to(device), k, bias=bias.to(device), score=score, groups=groups,
                              top_groups=max(1, groups // 2), group_best=2)
    assert torch.equal(chosen.cpu(), want)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('depth', [(88.0, 104.0), (64.0, 88.0), (100.0, 140.0)])
@pytest.mark.parametrize('n,groups', [(32, 8), (24, 8), (256, 16), (60, 10)])
def test_small_scores_keep_the_order_of_exact_arithmetic(n, groups, depth, score, device):
    """Scores that fp32 holds with a few bits, or as 0, and those whose distance to the largest logit it rounds by
    some 10^-6: groups (and with a bias of zeros experts) whose ranks are alike or near."""
    g = torch.Generator().manual_seed(n)
    rows, size = 1500, n // groups
    base = -depth[0] - (depth[1] - depth[0]) * torch.rand(rows, 1, size, generator=g)
    near = torch.where(torch.rand(rows, groups, 1, generator=g) < 0.5, 2.0 ** -18, 2.0 ** -2)
    z = base + near * torch.randn(rows, groups, size, generator=g)
    swap = torch.rand(rows, groups, generator=g).argsort(1)  # which group is how near
    z = z.gather(1, swap.unsqueeze(-1).expand_as(z)).reshape(rows, n)
    if score == 'softmax':
        z[:, 0] = 0.0
        z = z + 13.37
    for bias, best in ((None, 2), (torch.zeros(n), 2), (torch.zeros(n), 1)):
        kw = dict(score=score, groups=groups, top_groups=2, group_best=best)
        want = choose64(z, min(3, 2 * size), bias, **kw)
        _, chosen = experts.route(z.to(device), min(3, 2 * size), bias=None if bias is None else bias.to(device), **kw)
        assert torch.equal(chosen.cpu(), want), int((chosen.cpu() != want).any(1).sum())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('groups', [1, 4])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('renormalize', [True, False])
@pytest.mark.parametrize('biased', [True, False])
def test_infinities_and_nan(score, renormalize, groups, biased, device):
    """-inf takes an expert out, a row of them gives zeros; a NaN or +inf makes the softmax
    NaN and stays with its own sigmoid. No index leaves the range, gradients follow."""
    n, k = 16, 5
    z = torch.randn(9, n, generator=torch.Generator().manual_seed(1))
    z[0, ::2] = -INF
    z[1] = -INF
    z[2, 3:] = -INF            # fewer left than are chosen
    z[3, 7] = math.nan
    z[4] = math.nan
    z[5, 2] = INF
    z[6] = torch.finfo(torch.float32).min
    z[7, 4:] = -INF
    z[7, 0] = math.nan
    bias = torch.linspace(1, -1, n) if biased else None
    kw = dict(score=score, groups=groups, top_groups=2 if groups > 1 else 1, group_best=2)
    leaf = z.to(device).requires_grad_(True)
    w, chosen = experts.route(leaf, k, bias=None if bias is None else bias.to(device), renormalize=renormalize, **kw)
    want = choose64(z, k, bias, score, **{a: b for a, b in kw.items() if a != 'score'})
    rows = [0, 1, 2, 6, 8] if score == 'softmax' else [0, 1, 2, 3, 4, 5, 6, 7, 8]
    assert torch.equal(chosen.cpu()[rows], want[rows])
    assert ((chosen >= 0) & (chosen < n)).all()
    assert all(len(set(row)) == k for row in chosen.tolist())
    dz, = torch.autograd.grad(w.sum(), leaf)
    w, dz = w.detach().cpu(), dz.cpu()
    assert (w[1] == 0).all() and (dz[1] == 0).all()
    assert (w[2][torch.isneginf(z[2].gather(0, want[2].long()))] == 0).all() and w[2].isfinite().all()
    assert w[[0, 2, 6, 8]].isfinite().all() and dz[[0, 2, 6, 8]].isfinite().all()
    if score == 'softmax':
        assert w[[3, 4, 5, 7]].isnan().all()
    else:
        assert w[4].isnan().all()
        if 7 not in chosen.tolist()[3]:
            assert w[3].isfinite().all()


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('groups', [1, 4])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('renormalize', [True, False])
def test_gradients_of_nan_and_infinite_logits(score, renormalize, groups, device):
    """A softmax over a row with NaN or +inf is NaN, and so are its gradients: those of the chosen
    ones' with renormalised weights, else all. A sigmoid's NaN shows where it is chosen: in all that
    its sum divides, else in its own. It adds nothing where it is not chosen."""
    n, k = 16, 5
    z = torch.randn(7, n, generator=torch.Generator().manual_seed(2))
    z[0, 7] = math.nan          # not chosen: it ranks last
    z[1, 2] = INF
    z[2, 3:] = math.nan         # fewer others than are chosen
    z[3] = math.nan
    z[4, 1], z[4, 2:9] = math.nan, -INF
    z[5, ::2] = -INF
    leaf = z.to(device).requires_grad_(True)
    w, chosen = experts.route(leaf, k, score=score, renormalize=renormalize, groups=groups, group_best=2,
                              top_groups=2 if groups > 1 else 1)
    dz, = torch.autograd.grad(w, leaf, torch.randn(7, k, generator=torch.Generator().manual_seed(3)).to(device))
    w, dz, chosen = w.detach().cpu(), dz.cpu(), chosen.cpu().long()
    mine = torch.zeros_like(z, dtype=torch.bool).scatter_(1, chosen, True)
    if score == 'softmax':
        bad = (z.isnan() | (z == INF)).any(1, keepdim=True)
        want_w, want_z = bad.expand_as(w), bad & mine if renormalize else bad.expand_as(z)
    else:
        bad = z.gather(1, chosen).isnan()
        bad = bad.any(1, keepdim=True).expand_as(bad) if renormalize else bad
        want_w, want_z = bad, torch.zeros_like(mine).scatter_(1, chosen, bad)
    assert torch.equal(w.isnan(), want_w) and torch.equal(dz.isnan(), want_z)
    assert not dz[~mine & ~want_z].any() or (score == 'softmax' and not renormalize)


@pytest.mark.parametrize('device', DEVICES)
def test_renormalised_weights_where_scores_underflow(device):
    z = torch.full((2, 8), -200.0)
    z[1, 0] = 300.0
    z[0, 3] = -199.0
    w, chosen = experts.route(z.to(device), 2, score='sigmoid')
    assert chosen[0].tolist() == [3, 0] and torch.allclose(w[0].cpu(), torch.tensor([0.7310586, 0.2689414]), atol=1e-6)
    w, chosen = experts.route(z.to(device), 2, bias=torch.tensor([-9.0] + [0.0] * 7).to(device))
    assert chosen[1].tolist() == [1, 2] and torch.allclose(w[1].cpu(), torch.tensor([0.5, 0.5]), atol=1e-6)


@pytest.mark.parametrize('device', DEVICES)
def test_leading_dimensions_strides_and_alignment(device):
    base = torch.randn(6, 5, 80, generator=torch.Generator().manual_seed(2)).to(device)
    for view in (base[..., 1:41], base[..., ::2], base.transpose(0, 1)[..., :40], base[0, 0, :40],
                 base[:0, :, :40], base[:1, :1, :40].expand(4, 3, 40)):
        leaf = view.detach().requires_grad_(True)
        w, chosen = experts.route(leaf, 3, renormalize=False)
        flat = view.contiguous().view(-1, 40).requires_grad_(True)
        w2, chosen2 = experts.route(flat, 3, renormalize=False)
        assert w.shape == (*view.shape[:-1], 3)
        assert torch.equal(chosen.reshape(-1, 3), chosen2) and torch.equal(w.reshape(-1, 3), w2)
        dy = torch.randn(w.shape, device=device)
        d1, = torch.autograd.grad(w, leaf, dy)
        d2, = torch.autograd.grad(w2, flat, dy.reshape(-1, 3))
        assert torch.equal(d1.reshape(-1, 40), d2)


def test_gradient_against_differences():
    z = torch.randn(7, 24, generator=torch.Generator().manual_seed(3), dtype=torch.float32)
    for kw in CHOICES:
        kw = dict(kw)
        if kw.pop('bias', False):
            kw['bias'] = torch.linspace(-0.1, 0.1, 24)
        dy = torch.randn(7, 4, generator=torch.Generator().manual_seed(4))
        step = torch.randn(7, 24, generator=torch.Generator().manual_seed(6))

        def f(t):
            s = scores64(t, kw.get('score', 'softmax')).gather(-1, chosen)
            s = s / s.sum(-1, keepdim=True) if kw.get('renormalize', True) else s
            return float((s * kw.get('scale', 1.0) * dy).sum())

        leaf = z.clone().requires_grad_(True)
        w, chosen = experts.route(leaf, 4, **kw)
        chosen = chosen.long()
        dz, = torch.autograd.grad(w, leaf, dy)
        h = 1e-5
        slope = (f(z.double() + h * step) - f(z.double() - h * step)) / (2 * h)
        # The quotient is off by its third derivative, h^2 times at most 100, and the
        # gradient by 2^-18 of the sizes of its 168 terms.
        assert abs(slope - float((dz.double() * step).sum())) <= 1e-8 + 168 * 2.0 ** -18


# ------------------------------------------------------------------ places and rows

@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.int32, torch.int64])
@pytest.mark.parametrize('rows,k,n', [(0, 2, 5), (1, 1, 1), (7, 3, 4), (500, 2, 64), (1365, 3, 7), (4097, 1, 1024),
                                      (9000, 8, 256), (100001, 1, 3)])
def test_places_are_a_stable_sort(rows, k, n, dt, device):
    g = torch.Generator().manual_seed(rows)
    chosen = torch.randint(-1 if rows > 10 else 0, n + (rows > 10), (rows, k), generator=g).to(dt)
    slots, offsets = experts.arrange(chosen.to(device), n)
    assert slots.dtype == offsets.dtype == torch.int32 and slots.shape == chosen.shape
    flat = chosen.reshape(-1).tolist()
    order = sorted(range(len(flat)), key=lambda i: flat[i] if 0 <= flat[i] < n else n)
    place = [0] * len(flat)
    for p, i in enumerate(order):
        place[i] = p
    assert slots.reshape(-1).tolist() == place
    counts = [0] * (n + 1)
    for e in flat:
        if 0 <= e < n:
            counts[e + 1] += 1
    assert offsets.tolist() == torch.tensor(counts).cumsum(0).tolist()


def test_places_agree_with_group_by_expert():
    chosen = torch.randint(0, 9, (200,), generator=torch.Generator().manual_seed(0))
    order, offsets = experts.group_by_expert(chosen, 9)
    slots, offsets2 = experts.arrange(chosen, 9)
    assert torch.equal(offsets, offsets2) and torch.equal(slots.long()[order], torch.arange(200))


def rows_data(tokens, k, width, dt, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*s, dtype=dt):
        return torch.randn(*s, generator=g, device=device).to(dtype)

    chosen = torch.randint(0, 5, (tokens, k), generator=g, device=device)
    slots, _ = experts.arrange(chosen, 5)
    return (randn(tokens, width), randn(tokens * k, width), slots, randn(tokens, k, dtype=torch.float32),
            randn(tokens, width), randn(tokens * k, width))


def check_rows(tokens, k, width, dt, device, residual=True):
    x, y, slots, w, dout, drows = rows_data(tokens, k, width, dt, device)
    leaves = [t.requires_grad_(True) for t in (x, y, w)]
    at = slots.long()
    rows = experts.dispatch(x, slots)
    out = experts.combine(y, slots, w, residual=x.detach() if residual else None)
    assert rows.dtype == out.dtype == dt
    want = torch.empty_like(y)
    for j in range(k):
        want[at[:, j]] = x.detach()
    assert torch.equal(rows.detach(), want)
    mine, u, tiny = y.detach().double()[at], UNIT[dt], TINY[dt]
    terms = w.detach().double().unsqueeze(-1) * mine
    value, size = terms.sum(1), terms.abs().sum(1)
    if residual:
        value, size = value + x.detach().double(), size + x.detach().double().abs()
    close(out, (value, (k + 1) * 2.0 ** -23 * size + u * value.abs() * (1 + 2.0 ** -7) + tiny), 'out')
    dx, dy, dw = torch.autograd.grad((rows, out), leaves, (drows, dout))
    d = drows.double()[at]
    close(dx, (d.sum(1), (k + 1) * 2.0 ** -23 * d.abs().sum(1) + u * d.sum(1).abs() * (1 + 2.0 ** -7) + tiny), 'dx')
    wd = w.detach().double().unsqueeze(-1) * dout.double().unsqueeze(1)
    value = torch.empty_like(y, dtype=torch.float64)
    value[at] = wd
    close(dy, (value, 2.0 ** -23 * value.abs() + u * value.abs() * (1 + 2.0 ** -7) + tiny), 'dy')
    p = mine * dout.double().unsqueeze(1)
    close(dw, (p.sum(2), (width + 1) * 2.0 ** -23 * p.abs().sum(2) + 2.0 ** -120), 'dw')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('tokens,k,width', [(1, 1, 1), (16, 2, 1024), (33, 4, 389), (100, 3, 66), (257, 8, 64), (9, 32, 40),
                                            (50, 5, 2500)])
def test_rows_to_the_experts_and_back(tokens, k, width, dt, device):
    check_rows(tokens, k, width, dt, device)


@pytest.mark.parametrize('device', DEVICES)
def test_rows_without_a_residual_and_without_tokens(device):
    check_rows(20, 2, 64, torch.float32, device, residual=False)
    x, y, slots, w, _, _ = rows_data(0, 2, 8, torch.float32, device)
    assert experts.dispatch(x, slots).shape == (0, 8) and experts.combine(y, slots, w).shape == (0, 8)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', [torch.float32, torch.bfloat16])
def test_rows_of_any_stride_and_alignment(dt, device):
    x, y, slots, w, dout, drows = rows_data(30, 3, 80, dt, device)
    for f in (lambda t: t[:, 1:41], lambda t: t[:, ::2], lambda t: t[:1, :40].expand(len(t), 40),
              lambda t: t[:, :40]):
        a, b = f(x), f(y)
        rows, out = experts.dispatch(a, slots), experts.combine(b, slots, w, residual=a)
        assert torch.equal(rows, experts.dispatch(a.contiguous(), slots))
        assert torch.equal(out, experts.combine(b.contiguous(), slots, w, residual=a.contiguous()))
        la, lb, lw = a.detach().requires_grad_(True), b.detach().requires_grad_(True), w.clone().requires_grad_(True)
        got = torch.autograd.grad((experts.dispatch(la, slots), experts.combine(lb, slots, lw)), (la, lb, lw),
                                  (f(drows), f(dout)))
        want = torch.autograd.grad((experts.dispatch(la, slots), experts.combine(lb, slots, lw)), (la, lb, lw),
                                   (f(drows).contiguous(), f(dout).contiguous()))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    wide = torch.empty(30, 6, device=device)[:, ::2].copy_(w)  # weights with a stride
    assert torch.equal(experts.combine(y, slots, wide), experts.combine(y, slots, w))
    assert torch.equal(experts.combine(y, slots.t().contiguous().t(), w), experts.combine(y, slots, w))


@pytest.mark.parametrize('device', DEVICES)
def test_slots_out_of_range_are_left_out(device):
    x, y, slots, w, dout, _ = rows_data(10, 2, 16, torch.float32, device)
    gone = slots.clone()
    gone[3, 1], gone[4, 0], gone[5, 0] = -1, 20, 1 << 30
    ly, lw = y.clone().requires_grad_(True), w.clone().requires_grad_(True)
    out = experts.combine(ly, gone, lw)
    keep = w.clone()
    keep[3, 1] = keep[4, 0] = keep[5, 0] = 0
    assert torch.equal(out, experts.combine(y, slots, keep))
    dw, = torch.autograd.grad(out, lw, dout)
    assert dw[3, 1] == dw[4, 0] == dw[5, 0] == 0
    rows = experts.dispatch(x, gone)
    named = [int(s) for s in gone.reshape(-1) if 0 <= s < 20]
    assert torch.equal(rows[named], experts.dispatch(x, slots)[named])


@pytest.mark.parametrize('device', DEVICES)
def test_a_choice_without_a_row_adds_nothing_whatever_its_weight(device):
    rows = torch.full((4, 8), math.nan, device=device)
    rows[1] = 2.0
    slots = torch.tensor([[1, -1], [4, 9]], dtype=torch.int32, device=device)
    w = torch.tensor([[0.5, math.inf], [math.nan, -math.inf]], device=device)
    res = torch.arange(16.0, device=device).view(2, 8)
    want = res + torch.tensor([[1.0], [0.0]], device=device)
    assert torch.equal(experts.combine(rows, slots, w, residual=res), want)


@pytest.mark.parametrize('device', DEVICES)
def test_a_choice_without_a_row_has_no_gradient_whatever_its_weight(device):
    rows = torch.full((4, 8), math.nan, device=device)
    rows[1] = 2.0
    slots = torch.tensor([[1, -1], [4, 9]], dtype=torch.int32, device=device)
    for filler in (math.nan, 3.0):
        rows[0] = filler
        for weight in (math.inf, math.nan, 1.0):
            leaves = [rows.clone().requires_grad_(True), torch.full((2, 2), weight, device=device)]
            leaves[1][0, 0] = 0.5
            leaves[1].requires_grad_(True)
            dy = torch.tensor([[1.0], [math.nan]], device=device).expand(2, 8)
            drows, dw = torch.autograd.grad(experts.combine(leaves[0], slots, leaves[1]), leaves, dy)
            assert torch.equal(drows, torch.tensor([0.0, 0.5, 0.0, 0.0], device=device).unsqueeze(1).expand(4, 8))
            assert torch.equal(dw, torch.tensor([[16.0, 0.0], [0.0, 0.0]], device=device))


@pytest.mark.parametrize('device', DEVICES)
def test_only_the_wanted_gradients(device):
    x, y, slots, w, dout, _ = rows_data(10, 2, 16, torch.float32, device)
    full = [t.clone().requires_grad_(True) for t in (y, w, x)]
    want = torch.autograd.grad(experts.combine(full[0], slots, full[1], residual=full[2]), full, dout)
    for i in range(3):
        leaves = [t.clone().requires_grad_(i == j) for j, t in enumerate((y, w, x))]
        out = experts.combine(leaves[0], slots, leaves[1], residual=leaves[2])
        if i != 1:
            leaves[0].data.zero_()  # the rows go into the weights' gradient only
        got, = torch.autograd.grad(out, leaves[i], dout)
        assert torch.equal(got, want[i])


def poison(*shapes, dt, device):
    """The allocator's next blocks of these sizes hold NaN."""
    if device == 'cuda':
        gone = [torch.full(shape, math.nan, dtype=dt, device=device) for shape in shapes for _ in range(3)]
        del gone


def check_dropped(tokens, k, width, dt, device, shift=0):
    """A tenth of the slots out of range (and with them as many places without a name): the rows of
    dispatch and the gradients are those of all slots where a place has a name, and zeros elsewhere."""
    x, y, slots, w, dout, _ = rows_data(tokens, k, width, dt, device)
    slots = torch.cat([slots.reshape(-1)[:shift], slots.reshape(-1)])[shift:].view(tokens, k)  # off 16 bytes
    g = torch.Generator(device=device).manual_seed(1)
    out = torch.rand(tokens, k, generator=g, device=device) < 0.1
    out[-1, -1] = True
    bad = torch.tensor([-1, tokens * k, 2 ** 31 - 1, -2 ** 31], device=device)[torch.arange(tokens * k, device=device) % 4]
    gone = torch.cat([bad[:shift], torch.where(out.view(-1), bad, slots.view(-1))]).int()[shift:].view(tokens, k)
    named = torch.zeros(tokens * k, dtype=torch.bool, device=device)
    named[gone[~out].long()] = True
    want = torch.where(named.unsqueeze(1), experts.dispatch(x, slots), 0)
    leaves = [y.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    wanted = torch.autograd.grad(experts.combine(*[leaves[0], slots, leaves[1]]), leaves, dout)
    poison((tokens * k, width), dt=dt, device=device)
    rows = experts.dispatch(x, gone)
    assert torch.equal(rows, want)
    got = experts.combine(leaves[0], gone, leaves[1])
    poison((tokens * k, width), dt=dt, device=device)
    dy, dw = torch.autograd.grad(got, leaves, dout)
    assert torch.equal(dy, torch.where(named.unsqueeze(1), wanted[0], 0))
    assert torch.equal(dw, torch.where(out, 0, wanted[1]))
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(experts.dispatch(leaf, gone), leaf, y)
    # (Sums of k terms in fp32 in any order, rounded once.)
    terms = y.double()[torch.where(out, 0, gone).long()].masked_fill(out.unsqueeze(2), 0)
    value, size = terms.sum(1), terms.abs().sum(1)
    close(dx, (value, (k + 1) * 2.0 ** -23 * size + UNIT[dt] * value.abs() * (1 + 2.0 ** -7) + TINY[dt]), 'dx')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('tokens,k,width,shift', [(1, 1, 8, 0), (10, 2, 16, 0), (3, 1, 5, 1), (33, 32, 40, 3), (700, 3, 389, 2),
                                                  (5000, 2, 64, 0)])
def test_places_that_no_slot_names_are_zeros(tokens, k, width, shift, dt, device):
    check_dropped(tokens, k, width, dt, device, shift)


@pytest.mark.gpu
@pytest.mark.parametrize('tokens,k,width,dt', [(33000, 4, 72, torch.float32), (140001, 8, 128, torch.bfloat16),
                                               (140001, 8, 24, torch.float16), (600001, 2, 1, torch.float32)])
def test_many_places_that_no_slot_names_are_zeros(tokens, k, width, dt):
    """Cleared by a launch of its own, with rows of every access size."""
    check_dropped(tokens, k, width, dt, 'cuda', 1)


@pytest.mark.parametrize('device', DEVICES)
def test_no_slot_names_a_place(device):
    x, y, slots, w, dout, _ = rows_data(40, 3, 24, torch.float32, device)
    leaf = y.clone().requires_grad_(True)
    poison((120, 24), dt=torch.float32, device=device)
    out = experts.combine(leaf, torch.full_like(slots, -1), w, residual=x)
    dy, = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(out, x) and not dy.any()
    poison((120, 24), dt=torch.float32, device=device)
    assert not experts.dispatch(x, torch.full_like(slots, 120)).any()


@pytest.mark.gpu
def test_dropped_choices_in_captured_steps():
    x, y, slots, w, dout, _ = rows_data(500, 4, 64, torch.bfloat16, 'cuda')
    leaf, at = y.clone().requires_grad_(True), slots.clone()

    def step():
        return experts.dispatch(x, at), torch.autograd.grad(experts.combine(leaf, at, w), leaf, dout)[0]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        at.copy_(torch.where(torch.arange(2000, device='cuda').view(500, 4) % (3 + i) == 0, -1, slots))
        for t in got:
            t.fill_(math.nan)
        graph.replay()
        assert all(torch.equal(a, b) and not a.isnan().any() for a, b in zip(got, step()))


# ------------------------------------------------------------------ refusals

def test_types_that_rows_may_have():
    slots, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    for bad in (torch.double, torch.long):
        with pytest.raises(ValueError, match='float'):
            experts.dispatch(torch.ones(4, 8).to(bad), slots)
        with pytest.raises(ValueError, match='float'):
            experts.combine(torch.ones(8, 8).to(bad), slots, w)
    with pytest.raises(ValueError, match='residual'):
        experts.combine(torch.ones(8, 8), slots, w, residual=torch.ones(4, 8).half())


def test_refusals_of_arguments():
    z = torch.randn(4, 12)
    for kw, match in ((dict(k=0), 'k must'), (dict(k=13), 'k must'), (dict(k=7, groups=2), 'k must'),
                      (dict(k=2, groups=5), 'groups'), (dict(k=2, groups=4, top_groups=5), 'groups'),
                      (dict(k=2, groups=0), 'groups'), (dict(k=2, top_groups=0), 'groups'),
                      (dict(k=2, group_best=3), 'group_best'), (dict(k=2, score='tanh'), 'score'),
                      (dict(k=2, bias=torch.zeros(11)), 'bias'), (dict(k=2, bias=torch.zeros(12).half()), 'bias'),
                      (dict(k=2, scale=math.inf), 'scale')):
        with pytest.raises(ValueError, match=match):
            experts.route(z, **kw)
    for bad in (z.double(), z.long(), torch.tensor(1.0), torch.randn(2, 1025), torch.randn(2, 0)):
        with pytest.raises(ValueError, match='logits'):
            experts.route(bad, 1)
    with pytest.raises(ValueError, match='chosen'):
        experts.arrange(z, 3)
    for n in (0, 1025):
        with pytest.raises(ValueError, match='num_experts'):
            experts.arrange(z.int(), n)
    slots, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    for bad in (slots.long(), slots[0], torch.zeros(4, 33, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match='slots'):
            experts.dispatch(z, bad)
    for args, match in (((z, slots, w), 'rows'), ((torch.randn(8, 0), slots, w), 'rows'), ((z.repeat(2, 1), slots, w.half()), 'weights'),
                        ((z.repeat(2, 1), slots, w[:3]), 'weights')):
        with pytest.raises(ValueError, match=match):
            experts.combine(*args)
    with pytest.raises(ValueError, match='residual'):
        experts.combine(z.repeat(2, 1), slots, w, residual=z[:3])


@pytest.mark.gpu
def test_refusals_of_cuda_tensors():
    z = torch.randn(4, 12, device='cuda')
    with pytest.raises(ValueError, match='bias'):
        experts.route(z, 2, bias=torch.zeros(12))
    slots, w = torch.zeros(4, 2, dtype=torch.int32), torch.ones(4, 2)
    with pytest.raises(ValueError, match='slots'):
        experts.dispatch(z, slots)
    with pytest.raises(ValueError, match='weights'):
        experts.combine(z.repeat(2, 1), slots.cuda(), w)
    with pytest.raises(ValueError, match='residual'):
        experts.combine(z.repeat(2, 1), slots.cuda(), w.cuda(), residual=z.half())
    with pytest.raises(ValueError, match='float'):
        experts.dispatch(z.double(), slots.cuda())


@pytest.mark.gpu
def test_tangents_traces_and_second_gradients_are_refused():
    z = torch.randn(4, 12, device='cuda', requires_grad=True)
    y, slots = torch.randn(8, 16, device='cuda', requires_grad=True), torch.arange(8, device='cuda').int().view(4, 2)
    w = torch.ones(4, 2, device='cuda')
    calls = ((lambda t: experts.route(t, 2)[0], z), (lambda t: experts.dispatch(t, slots), torch.randn(4, 16, device='cuda')),
             (lambda t: experts.combine(t, slots, w), y))
    for f, t in calls:
        t = t.detach().requires_grad_(True)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
            f(forward_ad.make_dual(t.detach(), torch.ones_like(t)))
        with pytest.raises(RuntimeError, match='traced'):
            make_fx(f)(t.detach())
        with pytest.raises(RuntimeError, match='again'):
            torch.autograd.grad(f(t).sum(), t, create_graph=True)


# ------------------------------------------------------------------ streams, graphs and a mixture's layer

def mixture(x, route_w, up, down, bias, k=2):
    """Router, experts and back, as a block of a model calls them."""
    logits = x @ route_w.t()
    weights, chosen = experts.route(logits, k, bias=bias, score='sigmoid', scale=2.0)
    slots, offsets = experts.arrange(chosen, route_w.shape[0])
    h = experts.expert_linear(experts.dispatch(x, slots), up, offsets, activation='relu2')
    return experts.combine(experts.expert_linear(h, down, offsets), slots, weights, residual=x)


def mixture_data(device, dt, tokens=300, n=8, width=64):
    g = torch.Generator(device=device).manual_seed(0)

    def randn(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device=device) * scale).to(dt)

    leaves = [randn(tokens, width), randn(n, width, scale=0.1), randn(n, 2 * width, width, scale=width ** -0.5),
              randn(n, width, 2 * width, scale=0.1)]
    return [t.requires_grad_(True) for t in leaves], 0.1 * torch.randn(n, generator=g, device=device)


@pytest.mark.parametrize('device,dt', [('cpu', torch.float32), pytest.param('cuda', torch.bfloat16, marks=pytest.mark.gpu),
                                       pytest.param('cuda', torch.float16, marks=pytest.mark.gpu)])
def test_a_mixture_of_experts_together(device, dt):
    """Against the same layer written token by token in 64 bits, norm-wise: the error is that of
    four roundings of the operands' type (x h y out) in sums of independent terms, each
    below u of the result's norm."""
    (x, route_w, up, down), bias = mixture_data(device, dt)
    dy = torch.randn(x.shape, generator=torch.Generator(device=device).manual_seed(1), device=device).to(dt)
    out = mixture(x, route_w, up, down, bias)
    grads = torch.autograd.grad(out, (x, route_w, up, down), dy)
    with torch.no_grad():
        logits = x @ route_w.t()
        _, chosen = experts.route(logits, 2, bias=bias, score='sigmoid', scale=2.0)
    ref = [t.detach().double().requires_grad_(True) for t in (x, route_w, up, down)]
    s = torch.sigmoid(ref[0] @ ref[1].t()).gather(1, chosen.long())
    s = 2.0 * s / s.sum(1, keepdim=True)
    want = ref[0]
    for e in range(8):
        h = torch.relu(ref[0] @ ref[2][e].t()).square() @ ref[3][e].t()
        want = want + h * (s * (chosen == e)).sum(1, keepdim=True)
    wanted = torch.autograd.grad(want, ref, dy.double())
    for name, a, b in zip(('out', 'dx', 'droute', 'dup', 'ddown'), (out, *grads), (want, *wanted)):
        off = float((a.double() - b).norm() / b.norm())
        assert off <= 4 * UNIT[dt] + (2.0 ** -18 if dt == torch.float32 else 0), (name, off)


@pytest.mark.gpu
def test_streams_and_captured_steps():
    leaves, bias = mixture_data('cuda', torch.bfloat16)
    dy = torch.randn_like(leaves[0])

    def step():
        out = mixture(*leaves, bias)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = step()
    with torch.cuda.graph(other):
        second = step()
    for scale in (1.0, -0.5, 3.0):
        leaves[0].data.mul_(scale)
        dy.mul_(scale)
        graph.replay()
        other.replay()
        want = step()
        assert all(torch.equal(p, q) and torch.equal(r, q) for p, q, r in zip(first, want, second))
    assert _native.device_status(clear=True) == 0


# ------------------------------------------------------------------ C entries

def _route(**kw):
    p = _native.AveyRouteParams(struct_size=ctypes.sizeof(_native.AveyRouteParams), dtype=0, k=2, groups=1, top_groups=1,
                                group_best=1, tokens=4, experts=8, scale=1.0, logits=1 << 20, logits_ld=8,
                                weights=1 << 20, chosen=1 << 20)
    for a, b in kw.items():
        setattr(p, a, b)
    return p


@pytest.mark.parametrize('change,match', [
    (dict(struct_size=8), 'struct_size'), (dict(dtype=3), 'f32'), (dict(score=2), 'score'), (dict(k=9), 'k must'),
    (dict(k=0), 'k must'), (dict(experts=1025), 'experts'), (dict(tokens=-1), 'tokens'), (dict(groups=3), 'groups'),
    (dict(top_groups=2), 'groups'), (dict(group_best=0), 'groups'), (dict(logits=0), 'required'),
    (dict(weights=0), 'required'), (dict(chosen=0), 'required'), (dict(logits_ld=7), 'strides'),
    (dict(logits=(1 << 20) + 2), 'aligned'), (dict(scale=math.inf), 'scale')])
def test_c_route_rejects_bad_arguments_before_any_launch(change, match):
    lib = _native.lib()
    assert lib.avey_route_fwd_v1(ctypes.byref(_route(**change)), None) == -1
    assert match in lib.avey_last_error().decode()
    assert lib.avey_route_bwd_v1(ctypes.byref(_route()), None) == -1
    assert 'dweights' in lib.avey_last_error().decode()
    assert lib.avey_route_fwd_v1(None, None) == -1


@pytest.mark.parametrize('change,match', [
    (dict(struct_size=8), 'struct_size'), (dict(index_bits=16), 'bits'), (dict(count=-1), 'count'),
    (dict(experts=0), 'experts'), (dict(offsets=0), 'required'), (dict(slots=0), 'required'), (dict(chosen=0), 'required'),
    (dict(slots=(1 << 20) + 2), 'aligned'), (dict(chosen=(1 << 20) + 4), 'aligned')])
def test_c_arrange_rejects_bad_arguments_before_any_launch(change, match):
    p = _native.AveyArrangeParams(struct_size=ctypes.sizeof(_native.AveyArrangeParams), index_bits=64, count=9, experts=3,
                                  chosen=1 << 20, slots=1 << 20, offsets=1 << 20)
    for a, b in change.items():
        setattr(p, a, b)
    lib = _native.lib()
    assert lib.avey_arrange_v1(ctypes.byref(p), None) == -1
    assert match in lib.avey_last_error().decode()


@pytest.mark.parametrize('call,change,match', [
    ('dispatch', dict(struct_size=8), 'struct_size'), ('dispatch', dict(dtype=3), 'f32'), ('dispatch', dict(k=33), 'k must'),
    ('dispatch', dict(k=0), 'k must'), ('dispatch', dict(tokens=1 << 30), 'k must'), ('dispatch', dict(width=0), 'width'),
    ('dispatch', dict(slots=0), 'slots'), ('dispatch', dict(x=0), 'x and rows'), ('dispatch', dict(rows=0), 'x and rows'),
    ('dispatch', dict(x_ld=7), 'strides'), ('combine', dict(rows_ld=7), 'strides'), ('combine', dict(out=0), 'out'),
    ('combine_bwd', dict(weights=0), 'weights'), ('combine_bwd', dict(x=0), 'x'),
    ('combine_bwd', dict(rows=0, dweights=1 << 20), 'rows'), ('combine', dict(weights=(1 << 20) + 2), 'aligned')])
def test_c_rows_reject_bad_arguments_before_any_launch(call, change, match):
    at = 1 << 20
    p = _native.AveyRowsParams(struct_size=ctypes.sizeof(_native.AveyRowsParams), dtype=0, k=2, tokens=4, width=8, slots=at,
                               x=at, x_ld=8, rows=at, rows_ld=8, weights=at, out=at)
    for a, b in change.items():
        setattr(p, a, b)
    lib = _native.lib()
    assert getattr(lib, f'avey_{call}_v1')(ctypes.byref(p), None) == -1
    assert match in lib.avey_last_error().decode()


def test_c_rows_workspace():
    at, lib = 1 << 20, _native.lib()

    def rows(**kw):
        p = _native.AveyRowsParams(struct_size=ctypes.sizeof(_native.AveyRowsParams), dtype=0, k=2, tokens=4096, width=8, slots=at,
                                   x=at, x_ld=8, rows=at, rows_ld=8, weights=at, out=at, drows=at, clear=1)
        for a, b in kw.items():
            setattr(p, a, b)
        return p

    size = ctypes.c_uint64()
    for kw, want in ((dict(), 0), (dict(tokens=4097), 4 * 8194), (dict(tokens=4097, clear=0), 0), (dict(tokens=0), 0),
                     (dict(tokens=1 << 29), 1 << 32)):
        assert lib.avey_rows_workspace_size(ctypes.byref(rows(**kw)), ctypes.byref(size)) == 0 and size.value == want
    assert lib.avey_rows_workspace_size(None, ctypes.byref(size)) == -1
    assert lib.avey_rows_workspace_size(ctypes.byref(rows(k=33)), ctypes.byref(size)) == -1
    short = _native.AveyRowsParams.workspace.offset  # a block that ends before its workspace
    for call in (lib.avey_dispatch_v1, lib.avey_combine_bwd_v1):
        for kw, match in ((dict(tokens=4097), b'workspace'), (dict(tokens=4097, workspace=at, workspace_bytes=8), b'smaller'),
                          (dict(tokens=4097, workspace=at + 4, workspace_bytes=1 << 20), b'aligned'),
                          (dict(struct_size=short - 8), b'struct_size')):
            assert call(ctypes.byref(rows(**kw)), None) == -1 and match in lib.avey_last_error()
    assert lib.avey_rows_workspace_size(ctypes.byref(rows(tokens=4097, struct_size=short)), ctypes.byref(size)) == 0
    assert size.value == 0  # what stands where `clear` is now had no meaning there

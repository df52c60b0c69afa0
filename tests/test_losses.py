"""``losses.linear_cross_entropy`` against the formula in 64 bits, forward and backward.

Tolerances are bounds of the rounding that the operator states. With u = 2^-8
(bf16) or 2^-11 (f16), V the vocabulary, and fp32 sums of n products bounded by
a = (n + 1) 2^-23 sum |terms|:

  lse   the largest a of its row, e = 2^-23 (3 |lse| + 256 + V / 256) for the powers (two units
        in the last place each), the running sums (136 additions a unit of columns, then one a
        unit) and the two changes of base;
  loss  that of lse, a of the target's z, z_loss 2 |lse| err(lse), 2^-22 (|lse| + |z_t|);
  dz    |coefficient| p (a + err(lse) + e) + u |dz|, in f16 also 2^-37 of the largest
        coefficient of all rows (half a step of the scaled dz's subnormals, 2^-25, where that
        one stands at 2^12 or more); and |coefficient| 2^-126, as fp32 powers below that
        are zero (a logit 88 below the log sum), with 2^-126 for results below it;
  dx, dW  those errors carried through the sums, plus the sums' own a, plus u of the result.

Beside these bounds, which grow with the sums' lengths, the error's norm stays below 2 u of the
result's: dz's roundings are independent, so their sum's norm is below u of it, and the result's
own rounding adds less than u. A block of 64 columns or rows that is lost or doubled shows there."""

import ctypes
import math
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from avey_kernel_b200 import _native, losses

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16]
IGNORE = -100


def reference(x, w, t, dy=None, reduction='mean', z_loss=0.0, ignore=IGNORE):
    """{name: (value, bound)} in 64 bits; x, w in the operands' type."""
    dt, u = x.dtype, UNIT[x.dtype]
    used = t != ignore
    x, w = x.double().masked_fill(~used[:, None], 0), w.double()
    n, vocab = x.shape[1], w.shape[0]
    z = x @ w.t()
    a = (n + 1) * 2.0 ** -23 * (x.abs() @ w.abs().t())
    lse = torch.logsumexp(z, 1)
    e = 2.0 ** -23 * (3 * lse.abs() + 256 + vocab / 256)
    elog = a.amax(1) + e
    at = (torch.arange(len(t), device=t.device), torch.where(used, t, 0).long())
    each = torch.where(used, lse - z[at] + z_loss * lse ** 2, 0.0)
    err = elog * (1 + 2 * abs(z_loss) * lse.abs()) + a[at] + 2.0 ** -22 * (lse.abs() + z[at].abs() + each.abs())
    err = torch.where(used, err, 0.0)
    count = used.sum()
    if reduction == 'none':
        loss = (each, err)
    else:
        k = count if reduction == 'mean' else 1
        loss = (each.sum() / k, err.sum() / k + 2.0 ** -24 * (each.sum() / k).abs())
    out = {'loss': loss}
    if dy is None:
        return out
    g = dy.double().expand(len(t)) * used
    if reduction == 'mean':
        g = g / count
    b = g[:, None]
    c = b * (1 + 2 * z_loss * lse[:, None])
    p = torch.exp(z - lse[:, None])
    hit = torch.zeros_like(p)
    hit[at] = 1.0
    dz = c * p - b * hit
    edz = c.abs() * p * (a + elog[:, None] * (1 + 2 * abs(z_loss)) + e[:, None]) + 2.0 ** -22 * (c.abs() * p + b.abs() * hit)
    top = torch.maximum(b.abs(), c.abs()).max()
    edz = edz + 2.0 ** -126 * c.abs()
    edz = edz + u * (dz.abs() + edz) + (2.0 ** -37 * top if dt == torch.float16 else 0) * used[:, None]
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126

    def product(q, eq, r, terms):
        v, s = q @ r, q.abs() @ r.abs()
        err = eq @ r.abs() + terms * 2.0 ** -23 * s
        return v, err + u * (v.abs() + err) + tiny

    out['dx'] = product(dz, edz, w, vocab)
    out['dw'] = product(dz.t(), edz.t(), x, len(t))
    return out


def close(got, want, name, unit=None):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} outside, worst '
                           f'{float(((got - value).abs() / bound.clamp(min=1e-300)).max()):.3g} of the bound')
    if unit is not None and value.norm() > 1e-2 * value.numel() ** 0.5 * (2.0 ** -14 if unit < 2.0 ** -9 else 0):
        off = float((got - value).norm() / value.norm().clamp(min=1e-300))
        assert off <= 2 * unit, f'{name}: off by {off:.3g} of its norm'


def data(rows, width, vocab, dt, seed=0, ignored=0.0, device='cuda', wide=torch.int64):
    g = torch.Generator(device=device).manual_seed(seed)
    w = (torch.randn(vocab, width, generator=g, device=device) * 2 * width ** -0.5).to(dt)
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    x = torch.randn(rows, width, generator=g, device=device) + w[t].float()
    out = torch.rand(rows, generator=g, device=device) < ignored
    return x.to(dt), w, torch.where(out, IGNORE, t).to(wide), 0.5 + torch.rand(rows, generator=g, device=device)


def run(x, w, t, dy, **kw):
    leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
    loss = losses.linear_cross_entropy(*leaves, t, **kw)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, dy)]


def check(rows, width, vocab, dt, reduction='none', seed=0, ignored=0.0, wide=torch.int64, **kw):
    x, w, t, g = data(rows, width, vocab, dt, seed, ignored, wide=wide)
    dy = g if reduction == 'none' else torch.tensor(1.5 if dt == torch.bfloat16 else 1024.0, device='cuda')
    want = reference(x, w, t, dy, reduction, **kw)
    loss, dx, dw = run(x, w, t, dy, reduction=reduction, **kw)
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == dt
    close(loss, want['loss'], 'loss')
    close(dx, want['dx'], 'dx', UNIT[dt])
    close(dw, want['dw'], 'dw', UNIT[dt])
    with torch.no_grad():
        assert torch.equal(losses.linear_cross_entropy(x, w, t, reduction=reduction, **kw), loss)
    assert _native.device_status(clear=True) == 0


SHAPES = [(1, 64, 1000), (7, 64, 33), (100, 72, 1), (255, 128, 257), (256, 64, 256), (257, 200, 5000), (1000, 520, 3001),
          (3000, 64, 700), (513, 1032, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('rows,width,vocab', SHAPES)
def test_losses_and_gradients(rows, width, vocab, dt):
    check(rows, width, vocab, dt)


@pytest.mark.gpu
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('ignored,z_loss', [(0.0, 0.0), (0.3, 1e-2), (0.95, 0.0)])
@pytest.mark.parametrize('dt', DTYPES)
def test_reductions_ignored_rows_and_z_loss(reduction, ignored, z_loss, dt):
    check(700, 136, 1500, dt, reduction, seed=3, ignored=ignored, z_loss=z_loss, wide=torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [1, 2, 5, 8, 9, 16, 127, 128, 129])
def test_row_counts_of_both_kernels(rows):
    for width, vocab in ((200, 3000), (389, 1003), (72, 16)):
        check(rows, width, vocab, torch.bfloat16, seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize('width,vocab', [(1, 1), (1, 300), (7, 129), (63, 65), (65, 513), (389, 2049), (130, 31)])
def test_odd_widths_and_vocabularies(width, vocab):
    check(300, width, vocab, torch.float16, seed=width)
    check(300, width, vocab, torch.bfloat16, 'mean', seed=vocab, ignored=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,width,vocab', [(16384, 64, 20000), (300, 2100, 300000)])
def test_vocabularies_in_pieces(rows, width, vocab):
    """More than 512 MB of dz: dx's sums go over pieces of the vocabulary."""
    check(rows, width, vocab, torch.bfloat16, 'mean', seed=1, ignored=0.1, z_loss=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,width,vocab', [(5, 64, 4096), (700, 72, 4096), (2000, 520, 1024), (20000, 64, 8192)])
@pytest.mark.parametrize('dt', DTYPES)
def test_no_column_is_lost_or_doubled(rows, width, vocab, dt):
    """Rows of zeros: every probability is 1 / vocab, a power of two, and with whole numbers in W
    (zeros for the targets, whose 1 / vocab - 1 is rounded) every product and sum of dx is
    exact. And dW for rows that give one logit all the weight."""
    g = torch.Generator(device='cuda').manual_seed(0)
    w = torch.randint(-2, 3, (vocab, width), generator=g, device='cuda').to(dt)
    t = torch.randint(0, vocab, (rows,), generator=g, device='cuda')
    x = torch.zeros(rows, width, dtype=dt, device='cuda')
    w[::64] = 0
    _, dx, dw = run(x, w, t // 64 * 64, torch.ones((), device='cuda'), reduction='sum')
    assert torch.equal(dx, (w.double().sum(0) / vocab).to(dt).expand(rows, width)) and not dw.any()
    # One logit of 600 has the probability 1, and the targets lie elsewhere.
    x = torch.randint(-2, 3, (rows, width), generator=g, device='cuda').to(dt)
    x[:, 0] = 1
    w = torch.zeros(vocab, width, dtype=dt, device='cuda')
    w[vocab // 2, 0] = 600
    t = torch.where(t == vocab // 2, 0, t)
    _, dx, dw = run(x, w, t, torch.ones((), device='cuda'), reduction='sum')
    want = torch.zeros(vocab, width, dtype=torch.float64, device='cuda').index_add(0, t, -x.double())
    want[vocab // 2] = x.double().sum(0)
    assert torch.equal(dw, want.to(dt)) and torch.equal(dx[:, 0], torch.full_like(dx[:, 0], 600))


@pytest.mark.gpu
def test_leading_dimensions_strides_and_alignment():
    x, w, t, g = data(60, 80, 500, torch.bfloat16, 4)
    want = run(x[:, :40], w[:, :40], t, g, reduction='none')
    for fx, fw in ((lambda v: v[:, :40], lambda v: v[:, :40]),
                   (lambda v: v[:, 1:41], lambda v: v[:, 3:43]), (lambda v: v[:, ::2], lambda v: v[:, ::2]),
                   (lambda v: v.t()[:40].t(), lambda v: v.t()[:40].t())):
        a, b = fx(x), fw(w)
        got, plain = run(a, b, t, g, reduction='none'), run(a.contiguous(), b.contiguous(), t, g, reduction='none')
        assert all(torch.equal(p, q) for p, q in zip(got, plain))
    got = run(x[:, :40].view(3, 4, 5, 40), w[:, :40], t.view(3, 4, 5), g.view(3, 4, 5), reduction='none')
    assert got[0].shape == (3, 4, 5) and all(torch.equal(p.reshape(q.shape), q) for p, q in zip(got, want))
    one = run(x[0, :40], w[:, :40], t[0], g[0], reduction='none')
    assert one[0].shape == () and one[1].shape == (40,)
    a, b = x[:1, :40].expand(60, 40), w[:1, :40].expand(500, 40)  # broadcast rows
    twice = run(a, b, t, g, reduction='none')
    wanted = reference(a, b, t, g, 'none')
    for got, name in zip(twice, ('loss', 'dx', 'dw')):
        close(got, wanted[name], name)
    stride = torch.stack((t, t + 7), 1)[:, 0]
    every = torch.stack((g, -g), 1)[:, 0]
    assert all(torch.equal(p, q) for p, q in zip(run(x[:, :40], w[:, :40], stride, every, reduction='none'), want))
    same = run(x[:, :40], w[:, :40], t, torch.ones(1, device='cuda').expand(60), reduction='none')
    total = run(x[:, :40], w[:, :40], t, torch.ones((), device='cuda'), reduction='sum')
    assert torch.equal(same[1], total[1]) and torch.equal(same[2], total[2])


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('rows', [6, 300])
def test_ignored_rows_have_no_part_in_anything(rows, device):
    dt = torch.float32 if device == 'cpu' else torch.bfloat16
    x, w, t, g = data(rows, 72, 400, dt, 5, device=device)
    out = torch.arange(rows, device=device) % 3 == 1
    t = torch.where(out, IGNORE, t)
    clean = run(x.masked_fill(out[:, None], 0), w, t, g, reduction='none')
    for bad in (math.nan, math.inf, -math.inf):
        x[out] = bad
        g[out] = bad
        got = run(x, w, t, torch.where(out, 0, g) if device == 'cpu' else g, reduction='none')
        assert all(torch.equal(p, q) for p, q in zip(got, clean))
        assert not got[0][out].any() and not got[1][out].any()
    t[:] = IGNORE
    loss, dx, dw = run(x, w, t, torch.ones((), device=device), reduction='sum')
    assert loss == 0 and not dx.any() and not dw.any()
    loss, dx, dw = run(x, w, t, torch.ones((), device=device), reduction='mean') if device == 'cuda' else (math.nan, x * 0, w * 0)
    assert math.isnan(loss) and (device == 'cpu' or not (dx.any() or dw.any()))


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('rows', [8, 300])
def test_bad_targets_and_bad_rows_show_in_their_own_loss(rows, device):
    dt = torch.float32 if device == 'cpu' else torch.bfloat16
    x, w, t, _ = data(rows, 72, 400, dt, 6, device=device)
    want = losses.linear_cross_entropy(x, w, t, reduction='none')
    t[1], t[2], t[3] = 400, -1, 1 << 40
    x[4, 5], x[5, 0] = math.nan, math.inf
    got = losses.linear_cross_entropy(x, w, t, reduction='none')
    assert got[1:6].isnan().all() and torch.equal(got[6:], want[6:]) and got[0] == want[0]
    assert losses.linear_cross_entropy(x, w, t).isnan()
    got = losses.linear_cross_entropy(x, w, t, reduction='none', ignore_index=400)
    assert got[1] == 0 and got[2].isnan()


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('rows', [8, 300])
def test_bad_targets_show_in_the_gradients(rows, reduction, device):
    """NaN in the rows' own dx and in all of dw, which sums over them; the other rows' dx is that of a
    call that ignores them (but for the mean's count)."""
    dt = torch.float32 if device == 'cpu' else torch.bfloat16
    x, w, t, _ = data(rows, 72, 400, dt, 6, ignored=0.2, device=device)
    t[0], t[5:8] = 3, IGNORE
    for bad in (400, -1, 1 << 40):
        t[2], t[rows - 2] = bad, IGNORE
        dy = torch.ones((rows,) if reduction == 'none' else (), device=device)
        loss, dx, dw = run(x, w, t, dy, reduction=reduction)
        _, want, finite = run(x, w, torch.where(t == bad, IGNORE, t), dy, reduction=reduction)
        assert (loss[2] if reduction == 'none' else loss).isnan()
        assert dx[2].isnan().all() and dw.isnan().all() and finite.isfinite().all()
        dx[2] = 0
        assert torch.equal(dx, want) if reduction != 'mean' else dx.isfinite().all()
        assert not dx[t == IGNORE].any() and dx[0].any()


def sure(rows, top, device, dt, vocab=512, far=10.0, seed=0):
    """Rows whose target's logit is about `top` and all others' about `far` below it or lower; logits
    are x itself, bit for bit (the weight is the identity)."""
    g = torch.Generator(device=device).manual_seed(seed)
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    x = top - far - 4 * torch.rand(rows, vocab, generator=g, device=device)
    x = x.masked_fill(torch.rand(rows, vocab, generator=g, device=device) < 0.7, 0.0)
    x[torch.arange(rows, device=device), t] = top
    return x.to(dt), torch.eye(vocab, device=device, dtype=dt), t


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('top', [30, 96, 416, 4096])
@pytest.mark.parametrize('rows', [8, 300])
def test_losses_of_sure_rows_keep_their_digits_whatever_the_logits_size(rows, top, device):
    """The sum of the powers is 1 and a little: its terms are off by 2^-22 of themselves, and
    some 40 additions at its size by 2^-24 each (16 of a chunk of 32 columns, one for each further one,
    two for each of the four column parts and eight warps that are joined); the logarithm, the difference and
    ln 2 by 2^-22 in all. No term grows with the logits."""
    x, w, t = sure(rows, top, device, torch.float32 if device == 'cpu' else torch.bfloat16)
    z = x.double()
    want = torch.logsumexp(z - z.gather(1, t[:, None]), 1)
    assert float(want.min()) < 2.0 ** -6  # (bf16 rounds the logits' distances)
    got = losses.linear_cross_entropy(x, w, t, reduction='none')
    assert (got >= 0).all()
    bound = 2.0 ** -22 * (1 + want) + 40 * 2.0 ** -24 * (1 + want) + 2.0 ** -22 * (1 + want)
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('top', [30, 96, 416, 4096])
@pytest.mark.parametrize('rows', [8, 300])
def test_gradients_of_sure_rows_keep_their_digits_whatever_the_logits_size(rows, top, device):
    """dx is dz itself (the weight is the identity), rounded to the operands' type twice. A probability is off by
    the power's and the coefficient's rounding, 3 2^-22, and by that of the sum of powers that the
    test of the losses counts, 2^-22 + 40 2^-24; p - 1 by as much of 1."""
    dt = torch.float32 if device == 'cpu' else torch.bfloat16
    x, w, t = sure(rows, top, device, dt)
    _, dx, _ = run(x, w, t, torch.ones((), device=device), reduction='sum')
    z = x.double()
    p = torch.softmax(z, 1)
    hit = torch.nn.functional.one_hot(t, 512).bool()
    want = torch.where(hit, -p.masked_fill(hit, 0).sum(1, keepdim=True), p)
    unit = 2.0 ** -24 if device == 'cpu' else UNIT[dt]
    bound = (4 * 2.0 ** -22 + 40 * 2.0 ** -24) * torch.where(hit, 1.0, p) + 2.1 * unit * want.abs() + 2.0 ** -126
    off = (dx.double() - want).abs() / bound
    assert float(off.max()) <= 1, float(off.max())


def test_c_blocks_that_end_before_the_low_parts_are_taken():
    short = _native.AveyLossParams.saved_low.offset
    size = _native.loss_workspace_size(_params(), backward=False)
    assert _native.loss_workspace_size(_params(struct_size=short), backward=False) == size
    lib = _native.lib()
    assert lib.avey_loss_fwd_v1(ctypes.byref(_params(saved_low=(1 << 20) + 2)), None) == -1
    assert b'aligned' in lib.avey_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('rows', [5, 400])
def test_large_logits_and_small_and_uneven_gradients(rows, dt):
    """Logits up to some thousands; gradients that come in from 2^-30 to 1, which f16 keeps
    relative to the largest."""
    x, w, t, g = data(rows, 64, 600, dt, 7)
    w = w * 64
    dy = torch.where(torch.arange(rows, device='cuda') % 2 == 0, g, g * 2.0 ** -30)
    want = reference(x, w, t, dy, 'none')
    loss, dx, dw = run(x, w, t, dy, reduction='none')
    close(loss, want['loss'], 'loss')
    close(dx, want['dx'], 'dx')
    close(dw, want['dw'], 'dw')
    plain = run(x, w, t, g, reduction='none')
    for scale in (2.0 ** -60, 2.0 ** 60, 0.0):
        # Powers of two change nothing but the exponent, where both stay in the range: a result of
        # 2^-80 and more loses less than 2^-40 of itself to terms below 2^-126 (of 600 or 400).
        if dt == torch.bfloat16:
            got = run(x, w, t, g * scale, reduction='none')
            for a, b in zip(got[1:], plain[1:]):
                there = (b.abs() >= 2.0 ** -80) & ((b * scale).abs() >= 2.0 ** -80)
                assert torch.equal(a[there], (b * scale)[there]) and (scale != 0 or not a.any())


@pytest.mark.gpu
def test_only_the_wanted_gradients():
    x, w, t, g = data(300, 72, 700, torch.bfloat16, 8, ignored=0.1)
    _, dx, dw = run(x, w, t, g, reduction='none')
    for wx, ww in ((True, False), (False, True)):
        a, b = x.clone().requires_grad_(wx), w.clone().requires_grad_(ww)
        loss = losses.linear_cross_entropy(a, b, t, reduction='none')
        got, = torch.autograd.grad(loss, a if wx else b, g)
        assert torch.equal(got, dx if wx else dw)


@pytest.mark.gpu
def test_no_rows():
    x, w, t, _ = data(0, 72, 40, torch.bfloat16)
    for reduction, want in (('none', None), ('sum', 0.0), ('mean', math.nan)):
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = losses.linear_cross_entropy(a, b, t, reduction=reduction)
        assert loss.shape == ((0,) if want is None else ())
        assert want is None or (math.isnan(loss) if math.isnan(want) else loss == want)
        dx, dw = torch.autograd.grad(loss, (a, b), torch.ones_like(loss))
        assert dx.shape == x.shape and dw.shape == w.shape and not dw.any()


@pytest.mark.gpu
def test_weights_past_2_to_the_31_elements():
    """A vocabulary whose rows are zero but for the last three: the log sum and the gradients by
    the formula with its equal logits counted."""
    vocab, width, rows = (1 << 21) + 50, 1032, 12
    w = torch.zeros(vocab, width, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(0)
    w[-3:] = torch.randn(3, width, generator=g, device='cuda').bfloat16()
    x = torch.randn(rows, width, generator=g, device='cuda').bfloat16() * 0.25
    t = torch.arange(rows, device='cuda') % 5 - 2
    t = torch.where(t < 0, vocab + t, t)
    z = x.double() @ w[-3:].double().t()
    lse = torch.log(vocab - 3 + z.exp().sum(1))
    picked = torch.where((t >= vocab - 3).unsqueeze(1), z, 0).gather(1, (t - (vocab - 3)).clamp(min=0).unsqueeze(1)).squeeze(1)
    loss, dx, dw = run(x, w, t, torch.ones((), device='cuda'), reduction='sum')
    total = (lse - picked).sum()
    assert abs(float(loss - total)) <= 2.0 ** -12 * float(total)  # 2^13 additions of 2^-24, rows of |z| < 64
    few = torch.no_grad()(losses.linear_cross_entropy)(x[:4], w, t[:4], reduction='none')
    assert (few.double() - (lse - picked)[:4]).abs().max() <= 2.0 ** -12 * float(lse.max())
    p = torch.exp(-lse).unsqueeze(1)
    flat = (p * x.double()).sum(0)  # dW of a row without a target
    assert (dw[1000].double() - flat).abs().max() <= 2.0 ** -7 * flat.abs().max()
    assert (dw[vocab // 2] == dw[1000]).all() and (dw[5:-3] == dw[1000]).all()
    dz = torch.exp(z - lse.unsqueeze(1))
    dz[torch.arange(rows, device='cuda')[t >= vocab - 3], (t - (vocab - 3))[t >= vocab - 3]] -= 1
    close(dx, (dz @ w[-3:].double(), 2.0 ** -7 * (dz.abs() @ w[-3:].double().abs()) + 1e-6), 'dx')
    close(dw[-3:], (dz.t() @ x.double(), 2.0 ** -7 * (dz.abs().t() @ x.double().abs()) + 1e-6), 'dw')


@pytest.mark.gpu
def test_results_are_bitwise_reproducible_on_any_stream():
    x, w, t, g = data(3000, 264, 9000, torch.bfloat16, 9, ignored=0.1)
    a = run(x, w, t, g, reduction='none')
    b = run(x, w, t, g, reduction='none')
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = run(x, w, t, g, reduction='none')
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.gpu
@pytest.mark.parametrize('rows,width', [(5, 72), (700, 389), (700, 72)])
def test_captured_training_steps(rows, width):
    """All launches of both directions in graphs: replays with new inputs, of two graphs in turn,
    against calls as they come."""
    x, w, t, _ = data(rows, width, 1300, torch.float16, 10, ignored=0.2)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    dy = torch.full((), 512.0, device='cuda')

    def step():
        loss = losses.linear_cross_entropy(*leaves, t, z_loss=1e-3)
        return [loss.detach() + 0, *(v + 0 for v in torch.autograd.grad(loss, leaves, dy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for scale in (1.0, 0.5, -2.0):
        leaves[0].data.mul_(scale)
        t.copy_(torch.randint(0, 1300, t.shape, device='cuda'))
        for graph in graphs * 2:
            graph.replay()
        want = step()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.gpu
def test_a_wait_that_runs_out_sets_the_flag_and_the_next_call_is_right():
    x, w, t, g = data(700, 256, 900, torch.bfloat16, 11)
    want = run(x, w, t, g, reduction='none')
    assert _native.device_status(clear=True) == 0
    try:
        _native.test_hooks(100_000, stall=True)
        run(x, w, t, g, reduction='none')
        assert _native.device_status(clear=True) & 1
    finally:
        _native.test_hooks()
    got = run(x, w, t, g, reduction='none')
    assert _native.device_status(clear=True) == 0
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_the_plain_form_on_the_cpu():
    x, w, t, g = data(40, 24, 60, torch.float32, 12, 0.2, device='cpu')
    for kw in (dict(), dict(z_loss=1e-2), dict(reduction='sum'), dict(reduction='none', z_loss=0.1)):
        reduction = kw.get('reduction', 'mean')
        dy = g if reduction == 'none' else torch.tensor(1.5)
        got = run(x, w, t, dy, **kw)
        wanted = [v.double().requires_grad_(True) for v in (x, w)]
        z = wanted[0] @ wanted[1].t()
        lse, used = torch.logsumexp(z, 1), t != IGNORE
        each = (lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0] + kw.get('z_loss', 0.0) * lse ** 2) * used
        want = each if reduction == 'none' else each.sum() / (used.sum() if reduction == 'mean' else 1)
        grads = torch.autograd.grad(want, wanted, dy.double())
        for a, b in zip(got, (want.detach(), *grads)):
            assert (a.double() - b).abs().max() <= 2.0 ** -18 * (1 + b.abs().max())  # sums of 60 terms in fp32


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
def test_the_plain_form_keeps_the_logits_in_fp32(dt):
    x, w, t, _ = data(40, 24, 60, dt, 14, 0.2, device='cpu')
    want = losses.linear_cross_entropy(x.float(), w.float(), t)
    assert torch.equal(losses.linear_cross_entropy(x, w, t), want)


def test_gradient_against_differences():
    """The formula of the gradient that the GPU tests hold the kernels to (``reference``), against
    differences of its loss."""
    x, w, t, g = data(9, 16, 40, torch.bfloat16, 13, 0.2, device='cpu')
    for reduction in ('none', 'sum', 'mean'):
        dy = g if reduction == 'none' else torch.tensor(1.5)
        want = reference(x, w, t, dy, reduction, z_loss=0.05)
        gen = torch.Generator().manual_seed(1)
        for name, base in (('dx', x), ('dw', w)):
            step = torch.randn(base.shape, generator=gen, dtype=torch.float64)

            def f(h):
                a, b = x.double(), w.double()
                a, b = (a + h * step, b) if name == 'dx' else (a, b + h * step)
                z = a @ b.t()
                lse, used = torch.logsumexp(z, 1), t != IGNORE
                each = (lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0] + 0.05 * lse ** 2) * used
                return float(((each if reduction == 'none' else each.sum() / (used.sum() if reduction == 'mean' else 1))
                              * dy.double()).sum())

            h = 1e-5
            slope, exact = (f(h) - f(-h)) / (2 * h), float((want[name][0] * step).sum())
            # Rounding: 2^-52 of sums below 100, over 2 h; the quotient's own error h^2 times the
            # third derivative, below (|step| |w|)^3 = 10^5.
            assert abs(slope - exact) <= 1e-5 + 1e-9 * abs(exact)


def test_types_that_rows_may_have():
    t = torch.zeros(4, dtype=torch.int64)
    for x, w in ((torch.ones(4, 8).double(), torch.ones(9, 8).double()), (torch.ones(4, 8), torch.ones(9, 8).half())):
        with pytest.raises(ValueError, match='float'):
            losses.linear_cross_entropy(x, w, t)


def test_refusals_of_arguments():
    x, w, t = torch.randn(4, 8), torch.randn(10, 8), torch.zeros(4, dtype=torch.int64)
    for args, kw, match in (((x, w[:, :7], t), {}, 'weight'), ((x, w[0], t), {}, 'weight'), ((x, w[:0], t), {}, 'weight'),
                            ((x, w, t[:3]), {}, 'targets'), ((x, w, t.float()), {}, 'targets'),
                            ((x, w, t), dict(reduction='max'), 'reduction'), ((x, w, t), dict(z_loss=math.inf), 'z_loss')):
        with pytest.raises(ValueError, match=match):
            losses.linear_cross_entropy(*args, **kw)


@pytest.mark.gpu
def test_refusals_of_cuda_tensors_tangents_and_traces():
    x, w, t, _ = data(12, 64, 50, torch.bfloat16)
    for a, b, c, match in ((x.float(), w.float(), t, 'bf16'), (x, w.half(), t, 'one dtype'), (x, w.cpu(), t, 'one dtype'),
                           (x, w, t.cpu(), 'targets')):
        with pytest.raises(ValueError, match=match):
            losses.linear_cross_entropy(a, b, c)
    with forward_ad.dual_level():
        for i in range(2):
            args = [x, w]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(RuntimeError, match='forward-mode'):
                losses.linear_cross_entropy(*args, t)
    with pytest.raises(RuntimeError, match='traced'):
        make_fx(lambda v: losses.linear_cross_entropy(v, w, t))(x)
    with pytest.raises(RuntimeError, match='again'):
        x.requires_grad_(True)
        torch.autograd.grad(losses.linear_cross_entropy(x, w, t), x, create_graph=True)


# ------------------------------------------------------------------ C entries

def _params(**kw):
    at = 1 << 20
    p = _native.AveyLossParams(struct_size=ctypes.sizeof(_native.AveyLossParams), dtype=2, target_bits=64, reduction=2,
                               rows=300, width=64, vocab=1000, x=at, x_ld=64, weight=at, weight_ld=64, targets=at,
                               target_stride=1, ignore_index=-100, loss=at, saved=at)
    for a, b in kw.items():
        setattr(p, a, b)
    return p


@pytest.mark.parametrize('change,match', [
    (dict(struct_size=8), 'struct_size'), (dict(dtype=0), 'bf16'), (dict(target_bits=16), 'bits'),
    (dict(reduction=3), 'reduction'), (dict(rows=-1), 'rows'), (dict(width=0), 'width'), (dict(vocab=0), 'vocab'),
    (dict(vocab=(1 << 30) + 1), 'vocab'), (dict(rows=1 << 30, vocab=1 << 30), 'too many'), (dict(loss=0), 'loss'),
    (dict(x=0), 'x and targets'), (dict(targets=0), 'x and targets'), (dict(weight=0), 'weight'), (dict(x_ld=63), 'strides'),
    (dict(weight_ld=63), 'strides'), (dict(target_stride=-1), 'strides'), (dict(x=(1 << 20) + 1), 'aligned'),
    (dict(targets=(1 << 20) + 4), 'aligned'), (dict(loss=(1 << 20) + 2), 'aligned'), (dict(z_loss=math.nan), 'z_loss')])
def test_c_entry_rejects_bad_arguments_before_any_launch(change, match):
    lib = _native.lib()
    assert lib.avey_loss_fwd_v1(ctypes.byref(_params(**change)), None) == -1
    assert match in lib.avey_last_error().decode()
    assert lib.avey_loss_fwd_v1(None, None) == -1


@pytest.mark.parametrize('change,match', [(dict(saved=0), 'saved'), (dict(dloss=0), 'dloss'), (dict(dx_ld=63), 'strides'),
                                          (dict(dloss_stride=-1), 'strides'), (dict(dx=(1 << 20) + 1), 'aligned')])
def test_c_backward_entry_rejects_bad_arguments(change, match):
    at, lib = 1 << 20, _native.lib()
    p = _params(**{**dict(dloss=at, dx=at, dx_ld=64, dweight=at), **change})
    assert lib.avey_loss_bwd_v1(ctypes.byref(p), None) == -1
    assert match in lib.avey_last_error().decode()


def test_workspace_stays_small_whatever_the_logits_take():
    at = 1 << 20
    back = dict(dloss=at, dx=at, dx_ld=768, dweight=at, width=768, x_ld=768, weight_ld=768)
    for rows, vocab in ((16384, 131072), (65536, 131072), (4096, 50021), (1, 1 << 20)):
        size = _native.loss_workspace_size(_params(rows=rows, vocab=vocab, **back), backward=True)
        # dz by pieces of 256 MB, or 4096 columns, twice, in whole tiles of 256 columns; x's copy and
        # dx's sums; a few words a row; sums of tiles that are shared, eight at most for each of 148 SMs.
        pieces = 2 * max(256 << 20, rows * 4096 * 2) + 2 * rows * 256 * 2
        assert size <= pieces + rows * 768 * (2 + 4) + 16 * rows + (1 << 20) + 8 * 148 * 256 * 256 * 4
    assert _native.loss_workspace_size(_params(rows=0)) == 0


@pytest.mark.parametrize('width', [768, 769, 64])
@pytest.mark.parametrize('rows,vocab', [(1, 131072), (8, 50000), (33, 32768), (100, 131072), (4096, 50021), (16384, 131072),
                                        (40000, 131072), (262144, 131072), (8192, 1 << 20), (1 << 20, 1000)])
def test_workspace_is_what_the_header_says(rows, vocab, width):
    at, mb, sms = 1 << 20, 1 << 20, 148
    whole = -(-width // 8) * 8
    copies = 0 if whole == width else 2 * whole * (rows + vocab)
    kw = dict(rows=rows, vocab=vocab, width=width, x_ld=width, weight_ld=width)
    room = 256 * 16  # each part begins at a multiple of 256
    size = _native.loss_workspace_size(_params(**kw), backward=False)
    few = 0 if rows > 8 else copies  # up to 8 rows are read as they are
    assert size <= max(8 * rows * (vocab / 1024 + 1), 5 * mb) + 8 * rows + copies - few + room
    for dweight, share in ((at, mb / 2), (0, 2 * mb)):
        size = _native.loss_workspace_size(_params(dloss=at, dx=at, dx_ld=width, dweight=dweight, **kw), backward=True)
        dz = max(512 * mb, 16384 * rows if rows > 32768 else 0) + 1024 * rows
        assert size <= dz + 6 * whole * rows + 32 * rows + sms * share + copies + room


def test_operands_are_read_after_the_wait_for_the_grid_before():
    """Every kernel that may be launched while the step before it runs waits for it, in all of its
    threads, before it reads anything."""
    source = (Path(_native.__file__).parent / 'csrc' / 'tc_loss.cuh').read_text()
    for name in source.split('__global__')[1:]:
        body = name[name.index('{'):]
        wait = body.index('griddep_wait();')
        for read in ('__ldg(', '__ldcg(', '__ldcs(', 'ce_load_unit', 'atomicAdd', 'ce_target'):
            assert read not in body[:wait]

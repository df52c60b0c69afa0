"""``losses.linear_cross_entropy`` against the formula in 64 bits, forward and backward.

Tolerances are bounds of the rounding that the operator states. With u = 2^-8
(bf16) or 2^-11 (f16), V the vocabulary, and fp32 sums of n products bounded by
a = (n + 1) 2^-23 sum |terms|:

  lse   the largest a of its row, e = 2^-23 (3 |lse| + 256 + V / 256) for the powers (two units
        in the last place each), the running sums (136 additions a unit of columns, then one a
        unit) and the two changes of base;
  loss  that of lse, a of the target's z, z_loss 2 |lse| err(lse), 2^-22 (|lse| + |z_t|);
  dz    |coefficient| p (a + err(lse) + e) + u |dz|, in f16 also 2^-39 of the row's largest
        coefficient (half a step of the scaled dz's subnormals, where the largest
        coefficient stands at 2^13 or more);
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
    edz = edz + u * (dz.abs() + edz) + (2.0 ** -39 * top if dt == torch.float16 else 0) * used[:, None]
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0

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

"""``layers.residual_linear`` and ``experts.expert_linear`` against the formula in
64 bits, forward and backward.

Tolerances are elementwise bounds of the rounding that the operators state.
With u = 2^-8 (bf16) or 2^-11 (f16) and fp32 sums of n products bounded by
a = n 2^-23 sum |terms|:

  pre   a                      y    |act'| a (+ act'' a^2) + 2^-19 |y| + u |y|
  act'  |act''| a + its code's half step (2^-15; relu2: 2^-10 or 2^-12 of itself)
  dpre  |dy| err(act') + u |dpre|;   dx, dW, db: those errors carried through
        the sums, plus the sums' own a, plus u of the result.
A relu's derivative may also flip where |pre| <= a. f16 adds 2^-25 to each
rounding (half the spacing near zero)."""

import ctypes
import re
import threading
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from avey_kernel_b200 import _binding, _native, experts, layers

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16]
ACTS = ['identity', 'relu', 'relu2', 'silu', 'gelu']


def act64(x, act):
    x = x.detach().requires_grad_(True)
    y = {'identity': lambda t: t * 1.0, 'relu': torch.relu, 'relu2': lambda t: torch.relu(t) ** 2,
         'silu': F.silu, 'gelu': lambda t: F.gelu(t, approximate='tanh')}[act](x)
    return y.detach(), torch.autograd.grad(y.sum(), x)[0]


def reference(x, w, b, r, dy, act, dt):
    """{name: (value, bound)} in 64 bits for one group."""
    x, w = x.double(), w.double()
    n, k = w.shape
    pre = x @ w.t()
    a = (k + 1) * 2.0 ** -23 * (x.abs() @ w.abs().t())
    if b is not None:
        pre = pre + b.double()
        a = a + 2.0 ** -23 * b.double().abs()
    y, d = act64(pre, act)
    second = 2.0 if act == 'relu2' else 1.2  # |act''| at most (away from relu's kink)
    ey = (d.abs() + second * a) * a + 2.0 ** -19 * y.abs()
    if act in ('relu', 'relu2'):
        ey = ey + a * (pre.abs() <= a)
    if r is not None:
        y = y + r.double()
        ey = ey + 2.0 ** -23 * (y.abs() + r.double().abs())
    out = {'y': (y, ey + UNIT[dt] * (y.abs() + ey) + TINY[dt])}
    if dy is None:
        return out
    dy = dy.double()
    if act == 'identity':
        ed = torch.zeros_like(d)
    elif act == 'relu':
        ed = (pre.abs() <= a).double()
    elif act == 'relu2':
        ed = 2 * a + (2.0 ** -10 if dt == torch.bfloat16 else 2.0 ** -12) * (d + 2 * a) + 2.0 ** -14 * (d < 2.0 ** -13)
    else:
        ed = second * a + 2.0 ** -15 + 2.0 ** -18
    g = dy * d
    eb = dy.abs() * ed + 2.0 ** -23 * g.abs()  # the bias's terms are not rounded to 16 bits
    eg = eb + UNIT[dt] * (g.abs() + eb) + TINY[dt] if act != 'identity' else eb
    rows = max(x.shape[0], 1)

    def product(p, ep, q, terms):
        v, s = p @ q, p.abs() @ q.abs()
        e = ep @ q.abs() + terms * 2.0 ** -23 * (s + ep @ q.abs())
        return v, e + UNIT[dt] * (v.abs() + e) + TINY[dt]

    out['dx'] = product(g, eg, w, n)
    out['dw'] = product(g.t(), eg.t(), x, rows)
    v, e = g.sum(0), eb.sum(0) + rows * 2.0 ** -23 * g.abs().sum(0)
    out['db'] = (v, e + UNIT[dt] * (v.abs() + e) + TINY[dt])
    return out


def close(got, want, name):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} outside, worst '
                           f'{float(((got - value).abs() / bound.clamp(min=1e-300)).max()):.3g} of the bound')


def data(rows, k, n, dt, seed=0, groups=()):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def randn(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device='cuda') * scale).to(dt)

    return (randn(rows, k), randn(*groups, n, k, scale=max(k, 1) ** -0.5), randn(*groups, n, scale=0.3),
            randn(rows, n), randn(rows, n))


def run_linear(x, w, b, r, dy, act, kernel=_native.LINEAR_AUTO):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = _binding.module().linear(leaves[0], leaves[1], leaves[2], leaves[3], None,
                                 layers._ACT_IDS[act], kernel)
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, wanted, dy))
    return y, [next(grads) if t is not None else None for t in leaves]


def check_linear(rows, k, n, dt, act, bias=True, residual=True, kernel=_native.LINEAR_AUTO, seed=0):
    x, w, b, r, dy = data(rows, k, n, dt, seed)
    b, r = (b if bias else None), (r if residual else None)
    want = reference(x, w, b, r, dy, act, dt)
    y, (dx, dw, db, dr) = run_linear(x, w, b, r, dy, act, kernel)
    close(y, want['y'], 'y')
    close(dx, want['dx'], 'dx')
    close(dw, want['dw'], 'dw')
    if bias:
        close(db, want['db'], 'db')
    if residual:
        assert torch.equal(dr, dy)
    with torch.no_grad():
        assert torch.equal(_binding.module().linear(x, w, b, r, None, layers._ACT_IDS[act], kernel), y)
    assert _native.device_status(clear=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('rows,k,n', [(1, 64, 64), (8, 72, 40), (64, 256, 96), (65, 128, 264), (300, 392, 520)])
def test_linear_and_its_gradients(rows, k, n, dt, act):
    check_linear(rows, k, n, dt, act)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('rows,k,n', [(65, 128, 264), (150, 520, 72), (33, 1032, 40), (250, 72, 4200)])
@pytest.mark.parametrize('kernel', [_native.LINEAR_TCGEN05, _native.LINEAR_FEW])
def test_both_kernels_between_few_rows_and_many(rows, k, n, dt, act, kernel):
    """Clusters that share K, and rows shared by CTAs; many CTAs of few rows."""
    check_linear(rows, k, n, dt, act, kernel=kernel, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize('kernel', [_native.LINEAR_TCGEN05, _native.LINEAR_FEW])
@pytest.mark.parametrize('rows', [1, 7, 8, 9, 16, 31, 33, 63, 64, 65, 127, 128, 129, 257])
def test_row_counts_on_both_kernels(rows, kernel):
    check_linear(rows, 136, 88, torch.bfloat16, 'silu', kernel=kernel, seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize('kernel', [_native.LINEAR_TCGEN05, _native.LINEAR_FEW])
@pytest.mark.parametrize('k,n', [(1, 1), (1, 17), (7, 9), (8, 8), (31, 33), (63, 65), (64, 127), (129, 255),
                                 (389, 771), (1027, 129)])
def test_odd_widths(k, n, kernel):
    check_linear(70, k, n, torch.float16, 'gelu', kernel=kernel, seed=k)
    check_linear(70, k, n, torch.bfloat16, 'identity', bias=False, residual=False, kernel=kernel, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,n,act', [(4096, 192, 136, 'relu'), (3001, 64, 768, 'gelu'), (2500, 1024, 64, 'relu2'),
                                          (20000, 128, 128, 'silu'), (150, 2056, 1544, 'gelu')])
def test_long_and_wide_shapes(rows, k, n, act):
    """Many row tiles, dW split over rows, several waves of tiles."""
    check_linear(rows, k, n, torch.bfloat16, act, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [40, 300])
def test_leading_dimensions_strides_and_alignment(rows):
    k, n = 72, 48
    x, w, b, r, dy = data(rows, k, n, torch.bfloat16, 3)
    want, (gx, gw, gb, _) = run_linear(x, w, b, r, dy, 'silu')

    def same(x2, w2, r2, dy2, shape):
        y, (dx, dw, db, dr) = run_linear(x2, w2, b, r2, dy2, 'silu')
        assert y.shape == torch.Size(shape) and dx.shape == x2.shape
        assert torch.equal(y.reshape(-1, n), want) and torch.equal(dx.reshape(-1, k), gx)
        assert torch.equal(dw, gw) and torch.equal(db, gb)

    same(x.view(2, rows // 2, k), w, r.view(2, rows // 2, n), dy.view(2, rows // 2, n), (2, rows // 2, n))
    for pad, shift in ((8, 0), (8, 8), (5, 0), (5, 3), (0, 1)):  # row strides and starts, 16-byte aligned or not
        big = torch.empty(rows * (k + pad) + shift, device='cuda', dtype=x.dtype)
        xs = big.as_strided((rows, k), (k + pad, 1), shift)
        xs.copy_(x)
        bigr = torch.empty(rows * (n + pad) + shift, device='cuda', dtype=x.dtype)
        rs = bigr.as_strided((rows, n), (n + pad, 1), shift)
        rs.copy_(r)
        bigd = torch.empty(rows * (n + pad) + shift, device='cuda', dtype=x.dtype)
        ds = bigd.as_strided((rows, n), (n + pad, 1), shift)
        ds.copy_(dy)
        bigw = torch.empty(n * (k + pad) + shift, device='cuda', dtype=x.dtype)
        ws = bigw.as_strided((n, k), (k + pad, 1), shift)
        ws.copy_(w)
        same(xs, ws, rs, ds, (rows, n))
    same(x.t().contiguous().t(), w.t().contiguous().t(), r.t().contiguous().t(), dy.t().contiguous().t(), (rows, n))


@pytest.mark.gpu
def test_expanded_gradients_and_inputs():
    x, w, b, r, _ = data(96, 64, 40, torch.bfloat16, 4)
    ones = torch.ones(96, 40, device='cuda', dtype=x.dtype)
    _, want = run_linear(x, w, b, r, ones, 'gelu')
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    layers.residual_linear(*leaves[:3], activation='gelu', residual=leaves[3]).sum().backward()
    for t, g in zip(leaves, want):
        assert torch.equal(t.grad, g)
    row = x[:1].detach().requires_grad_(True)  # one row broadcast to 96: its gradients add up
    layers.residual_linear(row.expand(96, 64), w, b, activation='silu').sum().backward()
    full = x[:1].expand(96, 64).contiguous().requires_grad_(True)
    layers.residual_linear(full, w, b, activation='silu').sum().backward()
    torch.testing.assert_close(row.grad.float(), full.grad.float().sum(0, keepdim=True), rtol=2.0 ** -7, atol=1e-3)


@pytest.mark.gpu
def test_only_the_wanted_gradients():
    x, w, b, r, dy = data(130, 64, 72, torch.float16, 6)
    _, full = run_linear(x, w, b, r, dy, 'silu')
    for i in range(4):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b, r))]
        y = layers.residual_linear(*leaves[:3], activation='silu', residual=leaves[3])
        (g,) = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(g, full[i])


@pytest.mark.gpu
@pytest.mark.parametrize('grouped', [False, True])
@pytest.mark.parametrize('act,k', [('silu', 520), ('identity', 520), ('gelu', 389)])
def test_passes_in_a_row_give_what_each_gives_alone(grouped, act, k):
    """dX is set up beside the step before it and dW starts beside dX: calls in a
    row, each on the workspace of the one before it, against single gradients."""
    rows, n, f = 9000, 712, torch.bfloat16
    x = torch.randn(rows, k, generator=torch.Generator('cuda').manual_seed(4), device='cuda').to(f)
    w = (torch.randn(5, n, k, device='cuda') * k ** -0.5).to(f)
    offsets = torch.tensor([0, 3000, 3000, 3100, 8000, 8990], dtype=torch.int32, device='cuda')
    x, w = x.requires_grad_(True), (w if grouped else w[0]).requires_grad_(True)
    b = torch.randn(w.shape[:-1], device='cuda').to(f).requires_grad_(True)

    def layer():
        if grouped:
            return experts.expert_linear(x, w, offsets, b, activation=act)
        return layers.residual_linear(x, w, b, activation=act)

    dys = [torch.randn(rows, n, device='cuda').to(f) for _ in range(3)]
    alone = []
    for dy in dys:
        grads = []
        for t in (x, w, b):
            grads += torch.autograd.grad(layer(), t, dy)
            torch.cuda.synchronize()
        alone.append(grads)
    for i in [0, 1, 2] * 10:
        got = torch.autograd.grad(layer(), (x, w, b), dys[i])
        assert all(torch.equal(a, c) for a, c in zip(got, alone[i]))


@pytest.mark.gpu
def test_gradients_against_differences_of_the_formula():
    """A step h along a direction moves <dy, y> by h <grad, direction> + O(h^3)."""
    x, w, b, r, dy = data(150, 48, 56, torch.bfloat16, 7)
    for act in ('silu', 'gelu', 'identity'):
        _, grads = run_linear(x, w, b, r, dy, act)
        bounds = reference(x, w, b, r, dy, act, x.dtype)

        def f(x, w, b):
            return (act64(x @ w.t() + b, act)[0] * dy.double()).sum()

        base = [t.double() for t in (x, w, b)]
        for i, name in enumerate(('dx', 'dw', 'db')):
            g = torch.Generator(device='cuda').manual_seed(i)
            v = torch.randn(base[i].shape, generator=g, device='cuda', dtype=torch.float64)
            h = 1e-5
            up, down = ([t + s * h * v if j == i else t for j, t in enumerate(base)] for s in (1, -1))
            diff = (f(*up) - f(*down)) / (2 * h)
            got = (grads[i].double() * v).sum()
            assert (got - diff).abs() <= (bounds[name][1] * v.abs()).sum() + 1e-4 * diff.abs() + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
def test_large_and_non_finite_values_stay_in_their_rows(act):
    x, w, b, _, dy = data(140, 64, 72, torch.bfloat16, 8)
    x[3], x[70, 5], x[71, 5] = 1e4, float('inf'), float('nan')
    y, (dx, _, _, _) = run_linear(x, w, b, None, dy, act)
    clean = torch.ones(140, dtype=torch.bool, device='cuda')
    clean[[70, 71]] = False
    want = reference(x[clean], w, b, None, dy[clean], act, x.dtype)
    close(y[clean], want['y'], 'y')
    close(dx[clean], want['dx'], 'dx')
    assert torch.isnan(y[71]).all() and not torch.isfinite(y[70]).all()


@pytest.mark.gpu
def test_results_are_bitwise_reproducible():
    x, w, b, r, dy = data(5000, 136, 72, torch.bfloat16, 9)
    a = run_linear(x, w, b, r, dy, 'gelu')
    c = run_linear(x, w, b, r, dy, 'gelu')
    assert torch.equal(a[0], c[0]) and all(torch.equal(p, q) for p, q in zip(a[1], c[1]))


@pytest.mark.gpu
def test_streams_and_graphs():
    x, w, b, r, dy = data(200, 64, 72, torch.bfloat16, 10)
    want, grads = run_linear(x, w, b, r, dy, 'silu')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, got = run_linear(x, w, b, r, dy, 'silu')
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(got, grads))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        z = layers.residual_linear(x, w, b, activation='silu', residual=r)
    x.mul_(2)
    graph.replay()
    with torch.no_grad():
        assert torch.equal(z, layers.residual_linear(x, w, b, activation='silu', residual=r))


@pytest.mark.gpu
@pytest.mark.parametrize('k', [389, 520])
def test_a_captured_training_step(k):
    """All steps of both directions, with what follows them on the stream, in a
    graph: replays with new inputs against calls as they come."""
    x, w, b, r, dy = data(3000, k, 712, torch.bfloat16, 24)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layers.residual_linear(*leaves, activation='gelu', residual=r)
        return [y.detach()] + [g + 1 for g in torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for scale in (1.0, 0.5, -2.0, 0.25):
        dy.mul_(scale)
        leaves[0].data.mul_(scale)
        for _ in range(3):
            graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


@pytest.mark.gpu
def test_arrays_past_2_to_the_31_elements():
    rows, k, n = (1 << 21) + 77, 1032, 64  # x and dx hold 2^31 + 1.7 10^7 elements
    w, b, dt = data(1, k, n, torch.bfloat16, 15)[1], None, torch.bfloat16
    x = torch.zeros(rows, k, dtype=dt, device='cuda')
    dy = torch.zeros(rows, n, dtype=dt, device='cuda')
    last = data(200, k, n, dt, 16)
    x[-200:], dy[-200:] = last[0], last[4]
    y, (dx, dw, _, _) = run_linear(x, w, b, None, dy, 'silu')
    want = reference(last[0], w, b, None, last[4], 'silu', dt)
    close(y[-200:], want['y'], 'y')
    close(dx[-200:], want['dx'], 'dx')
    close(dw, want['dw'], 'dw')  # the other rows add nothing
    assert not y[:-200].any() and not dx[:-200].any()


@pytest.mark.gpu
def test_compiled_functions_call_the_operators():
    x, w, b, r, _ = data(100, 64, 72, torch.bfloat16, 17)

    def f(x):
        return layers.residual_linear(x * 2, w, b, activation='silu', residual=r) + 1

    assert torch.equal(torch.compile(f)(x), f(x))


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [100, 700])
def test_a_wait_that_runs_out_sets_the_flag_and_the_next_call_is_right(rows):
    """With the TMA lanes issuing nothing and a limit of 10^5 cycles, the products'
    first wait runs out in every kernel (100 rows: the cluster kernel forward); the
    calls return, the status word tells, and nothing is left behind."""
    x, w, b, r, dy = data(rows, 256, 72, torch.bfloat16, 18)
    off = torch.tensor([0, 30, rows - 10], device='cuda', dtype=torch.int32)
    w2, b2 = torch.stack((w, w)), torch.stack((b, b))
    tiles = _native.LINEAR_TCGEN05
    want = run_linear(x, w, b, r, dy, 'silu', tiles)
    want2 = run_experts(x, w2, off, b2, dy, 'silu', tiles)
    assert _native.device_status(clear=True) == 0
    try:
        _native.test_hooks(100_000, stall=True)
        run_linear(x, w, b, r, dy, 'silu', tiles)
        assert _native.device_status(clear=True) & 1
        run_experts(x, w2, off, b2, dy, 'silu', tiles)
        assert _native.device_status(clear=True) & 1
    finally:
        _native.test_hooks()
        _native.device_status(clear=True)
    got, got2 = run_linear(x, w, b, r, dy, 'silu', tiles), run_experts(x, w2, off, b2, dy, 'silu', tiles)
    assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))
    assert all(torch.equal(p, q) for p, q in zip(got2, want2))
    assert _native.device_status() == 0


@pytest.mark.gpu
def test_the_first_call_of_a_thread():
    """A layer without epilogue starts with tensor maps, a driver call, in a thread
    that has no CUDA context yet; backward passes run in autograd's own threads."""
    x, w, _, _, dy = data(200, 64, 72, torch.bfloat16, 19)
    want, (dx, dw, _, _) = run_linear(x, w, None, None, dy, 'identity')
    got = []

    def call():
        try:
            got.append(run_linear(x, w, None, None, dy, 'identity'))
        except Exception as e:  # seen by the assertions below
            got.append(e)

    t = threading.Thread(target=call)
    t.start()
    t.join()
    y, grads = got[0]
    assert torch.equal(y, want) and torch.equal(grads[0], dx) and torch.equal(grads[1], dw)


@pytest.mark.gpu
def test_wide_layers_take_tiles_in_blocks_of_rows():
    """More than 16 column tiles of 256 forward and in dX, with row tiles that do and
    do not fill a block of 12."""
    check_linear(1700, 72, 4200, torch.bfloat16, 'silu', seed=20)
    check_linear(3000, 4200, 72, torch.bfloat16, 'identity', bias=False, residual=False, seed=21)
    check_experts([1600, 0, 1541, 100], 40, 4360, torch.bfloat16, 'gelu', 50, seed=22)


@pytest.mark.gpu
def test_empty_batches():
    x, w, b, r, dy = data(0, 64, 72, torch.bfloat16)
    y, (dx, dw, db, dr) = run_linear(x, w, b, r, dy, 'silu')
    assert y.shape == (0, 72) and dx.shape == (0, 64) and dr.shape == (0, 72)
    assert not dw.any() and not db.any()


# ------------------------------------------------------------------ experts

def run_experts(x, w, off, b, dy, act, kernel=_native.LINEAR_AUTO):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = _binding.module().linear(*leaves, None, off, layers._ACT_IDS[act], kernel)
    return (y, *torch.autograd.grad(y, leaves, dy))


def check_experts(sizes, k, n, dt, act, tail=0, kernel=_native.LINEAR_AUTO, seed=0, poison=True):
    rows, e = sum(sizes) + tail, len(sizes)
    x, w, b, _, dy = data(rows, k, n, dt, seed, (e,))
    off = torch.tensor([0] + sizes, device='cuda').cumsum(0).to(torch.int32)
    if tail and poison:  # rows of no expert reach nothing
        x[-tail:], dy[-tail:] = float('nan'), float('inf')
    y, dx, dw, db = run_experts(x, w, off, b, dy, act, kernel)
    start = 0
    for i, c in enumerate(sizes):
        s = slice(start, start + c)
        start += c
        want = reference(x[s], w[i], b[i], None, dy[s], act, dt)
        for name, got in (('y', y[s]), ('dx', dx[s]), ('dw', dw[i]), ('db', db[i])):
            close(got, want[name], f'expert {i} {name}')
        if c == 0:
            assert not dw[i].any() and not db[i].any()
    assert not y[start:].any() and not dx[start:].any()
    assert _native.device_status(clear=True) == 0


SIZES = [[5], [0, 0, 3], [1, 0, 2, 1, 0, 0, 4, 0], [64, 64, 64], [128, 1, 127, 129], [0, 200, 0, 0, 333, 17],
         [63, 65, 16, 15, 17, 48, 100], [700, 0, 0, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize('tail', [0, 1, 77])
@pytest.mark.parametrize('sizes', SIZES, ids=str)
def test_experts_and_their_gradients(sizes, tail):
    check_experts(sizes, 72, 136, torch.bfloat16, 'silu', tail, seed=len(sizes))


@pytest.mark.gpu
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('dt', DTYPES)
def test_experts_types_and_activations(dt, act):
    check_experts([100, 0, 37, 64], 64, 264, dt, act, 9)
    check_experts([3, 0, 1, 8], 64, 264, dt, act, 2)


@pytest.mark.gpu
@pytest.mark.parametrize('kernel', [_native.LINEAR_TCGEN05, _native.LINEAR_FEW])
@pytest.mark.parametrize('k,n', [(7, 9), (65, 31), (129, 257), (200, 328)])
def test_experts_odd_widths(k, n, kernel):
    check_experts([3, 40, 0, 21], k, n, torch.float16, 'gelu', 5, kernel)


@pytest.mark.gpu
@pytest.mark.parametrize('kernel', [_native.LINEAR_TCGEN05, _native.LINEAR_FEW])
@pytest.mark.parametrize('count', [31, 32, 33, 64, 130])
def test_many_experts(count, kernel):
    g = torch.Generator().manual_seed(count)
    sizes = torch.randint(0, 4, (count,), generator=g).tolist()
    check_experts(sizes, 40, 48, torch.bfloat16, 'relu', 3, kernel)


@pytest.mark.gpu
def test_large_experts_run_several_tiles_per_sm():
    check_experts([3000, 10, 5001, 1], 64, 520, torch.bfloat16, 'gelu', 100)


@pytest.mark.gpu
def test_a_non_finite_expert_leaves_the_others_alone():
    """Rows of the next expert share K blocks with the end of the one before."""
    for bad in (float('inf'), float('nan')):
        sizes, k, n = [70, 33, 90], 64, 72
        x, w, b, _, dy = data(193, k, n, torch.bfloat16, 11, (3,))
        off = torch.tensor([0, 70, 103, 193], device='cuda', dtype=torch.int32)
        x[70:103], dy[70:103] = bad, bad
        y, dx, dw, db = run_experts(x, w, off, b, dy, 'silu')
        for i, s in ((0, slice(0, 70)), (2, slice(103, 193))):
            want = reference(x[s], w[i], b[i], None, dy[s], 'silu', x.dtype)
            for name, got in (('y', y[s]), ('dx', dx[s]), ('dw', dw[i]), ('db', db[i])):
                close(got, want[name], f'expert {i} {name}')
        assert not torch.isfinite(dw[1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize('rows', [50, 300])
@pytest.mark.parametrize('raw,used', [
    ([0, 20, 10, 40], [0, 20, 20, 40]), ([0, 20, 4000, 30], [0, 20, -1, -1]), ([0, -5, 30, 2 ** 31 - 1], [0, 0, 30, -1]),
    ([7, 20, 30, 40], [0, 20, 30, 40]), ([0, -2 ** 31, -1, 0], [0, 0, 0, 0])])
def test_offsets_out_of_order_or_range_are_pulled_into_range(raw, used, rows):
    x, w, b, _, dy = data(rows, 64, 72, torch.bfloat16, 12, (3,))
    used = [rows if u == -1 else u for u in used]
    got = run_experts(x, w, torch.tensor(raw, device='cuda', dtype=torch.int32), b, dy, 'gelu')
    want = run_experts(x, w, torch.tensor(used, device='cuda', dtype=torch.int32), b, dy, 'gelu')
    for p, q in zip(got, want):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_group_sizes_may_change_under_a_captured_graph():
    x, w, b, _, _ = data(300, 64, 72, torch.bfloat16, 13, (4,))
    off = torch.tensor([0, 100, 150, 150, 300], device='cuda', dtype=torch.int32)
    with torch.no_grad():
        experts.expert_linear(x, w, off, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = experts.expert_linear(x, w, off, b, activation='silu')
        for new in ([0, 10, 20, 290, 295], [0, 0, 0, 0, 0], [0, 300, 300, 300, 300]):
            off.copy_(torch.tensor(new))
            graph.replay()
            assert torch.equal(y, experts.expert_linear(x, w, off, b, activation='silu'))


@pytest.mark.gpu
def test_shared_and_strided_expert_weights():
    x, w, b, _, dy = data(120, 64, 72, torch.bfloat16, 14, (3,))
    off = torch.tensor([0, 50, 50, 120], device='cuda', dtype=torch.int32)
    want = run_experts(x, w, off, b, dy, 'silu')
    wide = torch.empty(3, 80, 72, device='cuda', dtype=x.dtype)
    wide[:, :72, :64] = w
    for other in (wide[:, :72, :64], w.transpose(1, 2).contiguous().transpose(1, 2)):
        for p, q in zip(run_experts(x, other, off, b, dy, 'silu'), want):
            assert torch.equal(p, q)
    one = w[:1].detach().requires_grad_(True)  # one expert's weights for all three: gradients add up
    y = experts.expert_linear(x, one.expand(3, 72, 64), off, b, activation='silu')
    (g,) = torch.autograd.grad(y, one, dy)
    full = run_experts(x, w[:1].expand(3, 72, 64).contiguous(), off, b, dy, 'silu')[2]
    torch.testing.assert_close(g.float(), full.float().sum(0, keepdim=True), rtol=2.0 ** -7, atol=1e-3)


DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


@pytest.mark.parametrize('device', DEVICES)
def test_group_by_expert_sorts_stably_and_bounds_the_runs(device):
    ids = torch.tensor([3, 0, 3, 1, 0, 5, 3], device=device)
    order, off = experts.group_by_expert(ids, 7)
    assert order.tolist() == [1, 4, 3, 0, 2, 6, 5]
    assert off.tolist() == [0, 2, 3, 3, 6, 6, 7, 7] and off.dtype == torch.int32
    order, off = experts.group_by_expert(ids[:0], 2)
    assert order.numel() == 0 and off.tolist() == [0, 0, 0]


def test_cpu_tensors_take_pytorch():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((9, 5), (3, 4, 5), (3, 4)))
    off = torch.tensor([0, 4, 4, 8], dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    assert torch.autograd.gradcheck(lambda x, w, b: experts.expert_linear(x, w, off, b, activation='silu'), leaves)
    y = experts.expert_linear(x, w, off, b, activation='silu')
    torch.testing.assert_close(y[4:8], F.silu(x[4:8] @ w[2].t() + b[2]))
    assert not y[8:].any()
    r = torch.randn(9, 4, generator=g, dtype=torch.float64)
    torch.testing.assert_close(layers.residual_linear(x, w[0], b[0], activation='gelu', residual=r),
                               F.gelu(x @ w[0].t() + b[0], approximate='tanh') + r)
    with pytest.raises(ValueError, match='residual'):
        layers.residual_linear(x, w[0], residual=r[:3])
    with pytest.raises(ValueError, match='offsets'):
        experts.expert_linear(x, w, off[:3])
    with pytest.raises(ValueError, match='activation'):
        experts.expert_linear(x, w, off, activation='tanh')


@pytest.mark.gpu
def test_bad_tensors_raise_before_any_launch():
    x, w, b, r, _ = data(20, 64, 72, torch.bfloat16)
    w3, b3 = w.expand(2, 72, 64), b.expand(2, 72)
    off = torch.tensor([0, 5, 20], device='cuda', dtype=torch.int32)
    before = _native.launch_count()
    for call, match in [
            (lambda: layers.residual_linear(x.float(), w.float()), 'bf16 / f16'),
            (lambda: layers.residual_linear(x, w.half()), 'one dtype'),
            (lambda: layers.residual_linear(x, w.cpu()), 'one dtype'),
            (lambda: layers.residual_linear(x, w[:, :32]), 'weight'),
            (lambda: layers.residual_linear(x, w3), 'weight'),
            (lambda: layers.residual_linear(x, w, b[:5]), 'bias must have shape'),
            (lambda: layers.residual_linear(x, w, b, residual=r[:5]), 'residual must have shape'),
            (lambda: layers.residual_linear(x, w, activation='tanh'), 'activation'),
            (lambda: experts.expert_linear(x, w, off), 'weight'),
            (lambda: experts.expert_linear(x, w3, off, b), 'bias must have shape'),
            (lambda: experts.expert_linear(x, w3, off.long(), b3), 'int32'),
            (lambda: experts.expert_linear(x, w3, off[:2], b3), 'offsets must be 3'),
            (lambda: experts.expert_linear(x, w3, off.cpu(), b3), 'offsets'),
            (lambda: experts.expert_linear(x[None], w3, off, b3), 'rows, d_in')]:
        with pytest.raises(ValueError, match=match):
            call()
    assert _native.launch_count() == before
    y = layers.residual_linear(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match='create_graph'):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def _params(**kw):
    p = _native.AveyLinearParams()
    p.struct_size = ctypes.sizeof(p)
    p.dtype, p.rows, p.d_in, p.d_out, p.groups = _native.AVEY_BF16, 300, 64, 72, 1
    p.x, p.x_ld, p.weight, p.weight_ld, p.y, p.y_ld = 1 << 20, 64, 2 << 20, 64, 3 << 20, 72
    p.dy, p.dy_ld, p.dx, p.dx_ld = 4 << 20, 72, 5 << 20, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize('field,value,match', [
    ('struct_size', 8, 'struct_size'), ('dtype', _native.AVEY_F32, 'bf16 or f16'), ('activation', 5, 'activation'),
    ('kernel', 3, 'kernel'), ('rows', -1, 'rows must'), ('d_in', 0, 'rows must'), ('groups', 0, 'rows must'),
    ('groups', 2, 'needs offsets'), ('x', 0, 'x is required'), ('weight', 0, 'weight is required'),
    ('x_ld', 63, 'strides'), ('weight_ld', 8, 'strides'), ('y', 0, 'y is required'), ('y_ld', 71, 'y is required'),
    ('deriv', 1 << 21, 'identity has no derivative'), ('rows', 1 << 31, 'rows must'),
    ('x', (1 << 20) + 1, 'aligned to their elements'), ('offsets', (1 << 20) + 2, 'aligned to their elements')])
def test_c_entry_rejects_bad_arguments_before_any_launch(field, value, match):
    p = _params(**{field: value})
    before = _native.launch_count()
    with pytest.raises(_native.NativeError, match=match) as info:
        _native.linear(p, 0)
    assert info.value.status == -1 and _native.launch_count() == before


@pytest.mark.parametrize('change,match', [
    (dict(dy=0), 'dy is required'), (dict(dx_ld=10), 'dy is required'),
    (dict(activation=3), 'needs deriv'), (dict(activation=3, deriv=(1 << 21) + 2), '32-byte aligned'),
    (dict(dweight=(1 << 21) + 1), 'aligned to their elements')])
def test_c_backward_entry_rejects_bad_arguments(change, match):
    with pytest.raises(_native.NativeError, match=match):
        _native.linear(_params(**change), 0, backward=True)


def test_few_row_kernel_refuses_more_groups_than_its_grid_has():
    p = _params(kernel=_native.LINEAR_FEW, rows=65535, groups=65535, offsets=1 << 20, weight_group_stride=64 * 72)
    with pytest.raises(_native.NativeError, match='up to 65534 groups'):
        _native.linear(p, 0)


@pytest.mark.gpu
@pytest.mark.parametrize('change,match', [
    (dict(workspace=(1 << 21) + 128, workspace_bytes=1 << 20), '256-byte aligned'),
    (dict(workspace=1 << 21, workspace_bytes=64), 'workspace is smaller'), (dict(), 'workspace is smaller')])
def test_c_entry_rejects_a_workspace_before_any_launch(change, match):
    p = _params(x=(1 << 20) + 2, **change)
    before = _native.launch_count()
    with pytest.raises(_native.NativeError, match=match):
        _native.linear(p, 0)
    assert _native.launch_count() == before


@pytest.mark.gpu
@pytest.mark.parametrize('offset', [1, 2, 4])
def test_c_backward_entry_takes_a_weight_gradient_at_any_alignment(offset):
    """2000 rows split dW's contraction: the sums of its parts go to the array
    as well as a whole tile's would."""
    x, w, _, _, dy = data(2000, 64, 72, torch.bfloat16, 23)
    _, (_, want, _, _) = run_linear(x, w, None, None, dy, 'identity')
    room = torch.empty(72 * 64 + 8, dtype=torch.bfloat16, device='cuda')
    p = _params(rows=2000, x=x.data_ptr(), weight=w.data_ptr(), dy=dy.data_ptr(), y=0, dx=0,
                dweight=room.data_ptr() + 2 * offset)
    ws = torch.empty(_native.linear_workspace_size(p, backward=True), dtype=torch.uint8, device='cuda')
    p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
    _native.linear(p, torch.cuda.current_stream().cuda_stream, backward=True)
    assert torch.equal(room[offset:offset + 72 * 64].view(72, 64), want)


def test_workspace_sizes():
    """Nothing for aligned forward calls; copies of unaligned rows; dpre and bias
    sums in the backward pass."""
    assert _native.linear_workspace_size(_params()) == 0
    assert _native.linear_workspace_size(_params(x=(1 << 20) + 2)) == 300 * 64 * 2  # x, to whole 256 bytes
    assert _native.linear_workspace_size(_params(rows=10, x=(1 << 20) + 2)) == 0  # the few-row kernel reads any
    p = _params(activation=3, deriv=1 << 21, dbias=6 << 20)
    sums = 5 * 72 * 4
    assert _native.linear_workspace_size(p, backward=True) == 43264 + (sums + 255) // 256 * 256  # dpre: 300 x 72 x 2
    assert _native.linear_workspace_size(_params(), backward=True) == 0


def test_operands_are_loaded_after_the_wait_for_the_grid_before():
    """The kernels of the products may be launched while the step before them runs:
    in each, the wait for it stands before the first load, under no condition."""
    source = (Path(_native.__file__).parent / 'csrc' / 'tc_linear.cuh').read_text()
    kernels = source.split('__global__')[1:]
    assert len(kernels) == 2
    for body in kernels:
        before = body[:body.index('tma_load_3d_hint(')]
        assert re.search(r'^ *griddep_wait\(\);', before, re.M)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,kernel', [(5, _native.LINEAR_FEW), (70, _native.LINEAR_FEW), (70, _native.LINEAR_TCGEN05),
                                         (3000, _native.LINEAR_TCGEN05)])
def test_f16_relu2_has_its_gradient_wherever_y_is_finite(rows, kernel):
    """Squares past f16's range that a residual brings back into it, and without one
    the last pre-activation whose square rounds to 65504; rows without a gradient."""
    k, n = 16, 40
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = torch.full((rows, k), 1.0, device='cuda').half()
    x[:, 1:] = 0
    x[:, 0] = (16 + 6.5 * torch.rand(rows, generator=g, device='cuda')).half()  # 16 x: 256 to 360
    w = (0.1 * torch.randn(n, k, generator=g, device='cuda')).half()
    w[:, 0] = 16
    pre = x.double() @ w.double().t()
    r = (200 * torch.rand(rows, n, generator=g, device='cuda').double() - pre ** 2).clamp(min=-65504).half()
    dy = (2.0 ** -6 * torch.randn(rows, n, generator=g, device='cuda')).half()
    dy[::3] = 0
    b = torch.zeros(n, device='cuda').half()
    want = reference(x, w, b, r, dy, 'relu2', x.dtype)
    y, (dx, dw, db, _) = run_linear(x, w, b, r, dy, 'relu2', kernel)
    assert pre.max() > 300 and y.isfinite().all()  # act' past 600
    for name, got in (('y', y), ('dx', dx), ('dw', dw), ('db', db)):
        close(got, want[name], name)
    assert not dx[::3].any()
    x[:, 0], x[:, 1], w[:, 1:] = 15.9921875, 1, 0
    w[:, 1] = 0.078125  # the pre-activation is 255.953125
    want = reference(x, w, None, None, dy, 'relu2', x.dtype)
    y, (dx, dw, _, _) = run_linear(x, w, None, None, dy, 'relu2', kernel)
    assert y.isfinite().all()
    for name, got in (('y', y), ('dx', dx), ('dw', dw)):
        close(got, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize('which', range(5))
def test_a_tangent_is_refused(which):
    """Forward-mode derivatives of x, weight, bias, residual and dy would be lost."""
    tensors = list(data(20, 64, 72, torch.bfloat16, 25))
    x, w, b, r, dy = tensors
    y = layers.residual_linear(x.detach().requires_grad_(True), w, b, residual=r)
    with forward_ad.dual_level():
        layers.residual_linear(x, w, b, residual=r)  # a level without a tangent takes nothing away
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        x, w, b, r, dy = tensors
        with pytest.raises(RuntimeError, match='forward-mode'):
            if which == 4:
                y.backward(dy)
            else:
                layers.residual_linear(x, w, b, residual=r)
    off = torch.tensor([0, 5, 20], device='cuda', dtype=torch.int32)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
        experts.expert_linear(forward_ad.make_dual(tensors[0].detach(), tensors[0].detach()), tensors[1].expand(2, 72, 64), off)


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('trace', [lambda f, x: make_fx(f)(x), lambda f, x: make_fx(f, pre_dispatch=True)(x),
                                   lambda f, x: torch.jit.trace(f, (x,), check_trace=False)])
def test_a_trace_is_refused(trace, grad):
    """It would hold the output as it was allocated."""
    x, w, b, _, _ = data(20, 64, 72, torch.bfloat16, 26)
    w.requires_grad_(grad)
    with pytest.raises(RuntimeError, match='traced'):
        trace(lambda t: layers.residual_linear(t, w, b, activation='silu'), x)
    layers.residual_linear(x, w, b)


# ------------------------------------------------------------------ exact sums

# Whole numbers from -2 to 2: every product and sum is exact in fp32, in any order,
# and each result is the exact sum rounded once. A lost or doubled row shows where a
# bound on rounding errors, which grows with the rows, would not see it.

def whole_numbers(rows, k, n, dt, device, seed=0, groups=()):
    g = torch.Generator(device=device).manual_seed(seed)

    def draw(*s):
        return torch.randint(-2, 3, s, generator=g, device=device).to(dt)

    return draw(rows, k), draw(*groups, n, k), draw(*groups, n), draw(rows, n)


def exact_gradients(x, w, b, dy, act):
    x, w, dy = x.double(), w.double(), dy.double()
    pre = x @ w.t() + b.double()
    if act == 'relu':
        dy = dy * (pre > 0)
    return [pre.clamp(min=0) if act == 'relu' else pre, dy @ w, dy.t() @ x, dy.sum(0)]


@pytest.mark.gpu
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('act', ['identity', 'relu'])
@pytest.mark.parametrize('rows,k,n', [(20000, 128, 128), (3001, 72, 264), (65537, 64, 40), (9000, 389, 77)])
def test_no_row_is_lost_or_doubled_in_long_sums(rows, k, n, act, dt):
    x, w, b, dy = whole_numbers(rows, k, n, dt, 'cuda', rows)
    y, (dx, dw, db, _) = run_linear(x, w, b, None, dy, act)
    for name, got, want in zip(('y', 'dx', 'dw', 'db'), (y, dx, dw, db), exact_gradients(x, w, b, dy, act)):
        assert torch.equal(got, want.to(dt)), name


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['identity', 'relu'])
@pytest.mark.parametrize('sizes', [[5000, 1, 63, 64, 65, 9000, 0, 127, 2000], [15, 17, 4000, 4033, 33], [66000, 500]], ids=str)
def test_no_row_is_lost_or_doubled_between_experts(sizes, act):
    k, n, tail = 72, 136, 50
    x, w, b, dy = whole_numbers(sum(sizes) + tail, k, n, torch.bfloat16, 'cuda', len(sizes), (len(sizes),))
    off = torch.tensor([0] + sizes, device='cuda').cumsum(0).to(torch.int32)
    y, dx, dw, db = run_experts(x, w, off, b, dy, act)
    start = 0
    for i, c in enumerate(sizes):
        s = slice(start, start + c)
        start += c
        want = exact_gradients(x[s], w[i], b[i], dy[s], act)
        for name, got, v in zip(('y', 'dx', 'dw', 'db'), (y[s], dx[s], dw[i], db[i]), want):
            assert torch.equal(got, v.to(x.dtype)), f'expert {i} {name}'
    assert not y[start:].any() and not dx[start:].any()


@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,n,count,alone', [
    (64, 64, 4096, 0, 1), (64, 64, 1536, 64, 1), (300, 40, 300, 300, 1), (20000, 64, 72, 0, 1), (1024, 1024, 1024, 0, 0),
    (300, 392, 520, 7, 0), (16384, 256, 256, 0, 1), (9000, 64, 20000, 0, 0)])
def test_bias_sums_go_where_they_take_least(rows, k, n, count, alone):
    """An idle warp of the dX kernel takes them where they hide behind its products;
    elsewhere (one CTA would take 128 of them in turn, say) they are a launch."""
    x, w, b, dy = whole_numbers(rows, k, n, torch.bfloat16, 'cuda', rows + n, (count,) if count else ())
    off = None
    if count:
        sizes = [rows // count + (i < rows % count) for i in range(count)]
        off = torch.tensor([0] + sizes, device='cuda').cumsum(0).to(torch.int32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def grads(wanted):
        y = _binding.module().linear(*leaves, None, off, layers._ACT_IDS['relu'], _native.LINEAR_AUTO)
        before = _native.launch_count()
        out = torch.autograd.grad(y, wanted, dy)
        return out, _native.launch_count() - before

    (dx, dw, db), with_bias = grads(leaves)
    (dx2, dw2), without = grads(leaves[:2])
    (alone_db,), _ = grads(leaves[2:])
    assert with_bias - without == alone
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, alone_db)
    if not count:
        pre = x.detach().double() @ w.detach().double().t() + b.detach().double()
        assert torch.equal(db, (dy.double() * (pre > 0)).sum(0).to(db.dtype))
    else:
        for i in range(0, count, 7):
            s = slice(off[i].item(), off[i + 1].item())
            want = exact_gradients(x.detach()[s], w.detach()[i], b.detach()[i], dy[s], 'relu')[3]
            assert torch.equal(db[i], want.to(db.dtype))


def test_exact_sums_show_a_lost_row():
    """One row less in the 64-bit sums, or a block of rows twice, changes dW and db
    as they are compared above."""
    x, w, b, dy = whole_numbers(20000, 128, 128, torch.bfloat16, 'cpu', 1)
    _, _, dw, db = exact_gradients(x, w, b, dy, 'identity')
    for first, rows, sign in [(0, 1, -1), (77, 1, -1), (19999, 1, 1), (64 * 100, 64, -1), (64 * 200, 64, 1), (19968, 32, -1)]:
        s = slice(first, first + rows)
        _, _, part_w, part_b = exact_gradients(x[s], w, b, dy[s], 'identity')
        assert not torch.equal((dw + sign * part_w).bfloat16(), dw.bfloat16())
        assert not torch.equal((db + sign * part_b).bfloat16(), db.bfloat16())


@pytest.mark.parametrize('rows,groups,k,n,few', [
    (64, 2, 4096, 14336, False), (64, 4, 2048, 8192, False), (32, 2, 2048, 8192, False), (64, 4, 2048, 2048, True),
    (64, 8, 4096, 14336, True), (16, 2, 4096, 14336, True), (64, 16, 4096, 14336, True), (8, 1, 4096, 14336, True),
    (65, 16, 64, 64, False)])
def test_grouped_rows_go_by_the_size_of_the_product(rows, groups, k, n, few):
    """Only the kernel of tiles needs a workspace, for rows that it cannot read in place."""
    p = _params(rows=rows, groups=groups, d_in=k, d_out=n, offsets=1 << 20, x=(1 << 20) + 2, x_ld=k, weight_ld=k,
                weight_group_stride=n * k, y_ld=n)
    assert (_native.linear_workspace_size(p) == 0) == few


@pytest.mark.gpu
@pytest.mark.parametrize('grouped', [False, True])
def test_only_what_a_gradient_needs_has_to_stay_as_it_was(grouped):
    """Frozen weights need no x for the backward pass, constant inputs no weights, a
    bias neither: those may change in place in between, as with torch's layers."""
    x, w, b, _, dy = data(130, 64, 72, torch.bfloat16, 27, (2,) if grouped else ())
    off = torch.tensor([0, 50, 130], device='cuda', dtype=torch.int32)

    def layer(x, w, b):
        return (experts.expert_linear(x, w, off, b, activation='silu') if grouped else
                layers.residual_linear(x, w, b, activation='silu'))

    full = [t.detach().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(layer(*full), full, dy)
    for i, spoiled in ((0, (0, 2)), (1, (1, 2)), (2, (0, 1, 2))):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        y = layer(*leaves)
        with torch.no_grad():
            for j in spoiled:
                leaves[j].zero_()
        (got,) = torch.autograd.grad(y, leaves[i], dy)
        assert torch.equal(got, want[i])
    for i, needed in ((0, 1), (1, 0)):  # and what is needed is still guarded
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        y = layer(*leaves)
        with torch.no_grad():
            leaves[needed].zero_()
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y, leaves[i], dy)


@pytest.mark.parametrize('change,match', [
    (dict(x=0, dweight=6 << 20), 'x is required'), (dict(weight=0), 'weight is required')])
def test_c_backward_entry_wants_the_operands_of_what_is_wanted(change, match):
    with pytest.raises(_native.NativeError, match=match):
        _native.linear(_params(**change), 0, backward=True)
    _native.linear_workspace_size(_params(x=0), backward=True)
    _native.linear_workspace_size(_params(weight=0, dx=0, dweight=6 << 20), backward=True)

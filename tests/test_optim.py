"""AdamW (``optim.adamw_step``, ``optim.AdamW``, ``avey_adamw_v1``) against the
formula in 64 bits, and the 8-bit states against the plain PyTorch form.

Tolerances, with u = 2^-24 (fp32 rounding): m is two products and a sum, so its
error is at most 4u (|b1 m| + |c1 g|); v likewise with one product more, 6u v;
the update's numerator, root, denominator and quotient add 16u; a 16-bit
parameter adds half a unit in its last place."""

import ctypes
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from avey_kernel_b200 import _native, optim

U = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def make(shapes, dtype, device, bits=32, master=False, seed=0):
    """Lists of parameters, gradients and mid-training states."""
    g = torch.Generator().manual_seed(seed)
    s = {'params': [], 'grads': [], 'exp_avgs': [], 'exp_avg_sqs': [], 'masters': [] if master else None,
         'exp_avg_scales': [] if bits == 8 else None, 'exp_avg_sq_scales': [] if bits == 8 else None}
    for shape in shapes:
        w = torch.randn(shape, generator=g) * 0.05
        m = torch.randn(shape, generator=g) * 1e-3
        v = torch.rand(shape, generator=g) * 1e-6 + 1e-9
        s['params'].append(w.to(dtype).to(device))
        s['grads'].append((torch.randn(shape, generator=g) * 1e-3).to(dtype).to(device))
        if master:
            s['masters'].append(w.to(device))
        if bits == 8:
            for name, x in (('exp_avg', m), ('exp_avg_sq', v.sqrt())):
                mid = torch.full((x.numel(),), 1 << 19)
                codes, scales = optim._quantize(x.reshape(-1), mid)
                s[name + 's'].append(codes.view(shape).to(device))
                s[name + '_scales'].append(scales.to(device))
        else:
            s['exp_avgs'].append(m.to(device))
            s['exp_avg_sqs'].append(v.to(device))
    return s


def clone(s, device=None):
    return {k: None if v is None else [t.clone() if device is None else t.to(device, copy=True) for t in v]
            for k, v in s.items()}


def call(s, step=10, **kw):
    args = dict(HYPER, **kw)
    optim.adamw_step(s['params'], s['grads'], s['exp_avgs'], s['exp_avg_sqs'], step=step,
                     masters=s['masters'], exp_avg_scales=s['exp_avg_scales'],
                     exp_avg_sq_scales=s['exp_avg_sq_scales'], **args)


def f64(t):
    return t.detach().cpu().double().numpy()


def state64(s, i):
    m, v = s['exp_avgs'][i], s['exp_avg_sqs'][i]
    if s['exp_avg_scales'] is None:
        return f64(m), f64(v)
    return (f64(optim.dequantize(m.cpu(), s['exp_avg_scales'][i].cpu())),
            f64(optim.dequantize(v.cpu(), s['exp_avg_sq_scales'][i].cpu())) ** 2)


def expected(s, i, step, lr, betas, eps, weight_decay, gscale=1.0):
    """(p, m, v) after the step in 64 bits, and the error bounds of their fp32 forms."""
    b1, b2 = betas
    g = f64(s['grads'][i]) * gscale
    m0, v0 = state64(s, i)
    p0 = f64((s['masters'] or s['params'])[i])
    m = b1 * m0 + (1 - b1) * g
    v = b2 * v0 + (1 - b2) * g * g
    denom = np.sqrt(v) / math.sqrt(1 - b2 ** step) + eps
    size = lr / (1 - b1 ** step)
    p = p0 * (1 - lr * weight_decay) - size * m / denom
    spread = np.abs(b1 * m0) + np.abs((1 - b1) * g)
    bounds = (3 * U * np.abs(p0) + 16 * U * size * spread / denom, 5 * U * spread, 6 * U * v)
    return (p, m, v), bounds


def check(before, after, i, dtype, step, exact_states=True, **kw):
    (p, m, v), (ep, em, ev) = expected(before, i, step, **dict(HYPER, **kw))
    if before['masters'] is not None:
        assert np.all(np.abs(f64(after['masters'][i]) - p) <= ep)
        assert torch.equal(after['params'][i].cpu(), after['masters'][i].to(dtype).cpu())
    else:
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half the spacing of f16 near zero
        assert np.all(np.abs(f64(after['params'][i]) - p) <= ep + HALF_ULP[dtype] * (np.abs(p) + ep) + tiny)
    if exact_states:
        assert np.all(np.abs(f64(after['exp_avgs'][i]) - m) <= em)
        assert np.all(np.abs(f64(after['exp_avg_sqs'][i]) - v) <= ev)


SHAPES = [(1,), (7,), (0,), (16, 16), (257,), (3, 5, 41), (2048,), (2049,), (129, 131)]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('master', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_step_with_fp32_states_matches_the_formula(dtype, master, device):
    s = make(SHAPES, dtype, device, master=master)
    before = clone(s)
    call(s)
    for i in range(len(SHAPES)):
        check(before, s, i, dtype, 10)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_first_step_from_zero_states(dtype, device):
    s = make([(300,)], dtype, device)
    for name in ('exp_avgs', 'exp_avg_sqs'):
        s[name][0].zero_()
    s['grads'][0][:5] = 0  # no gradient, no state: only the decay moves these
    before = clone(s)
    call(s, step=1)
    check(before, s, 0, dtype, 1)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('master', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_step_with_8bit_states(dtype, master, device):
    s = make(SHAPES, dtype, device, bits=8, master=master)
    before = clone(s)
    call(s, seed=5)
    for i, shape in enumerate(SHAPES):
        n = math.prod(shape)
        check(before, s, i, dtype, 10, exact_states=False)
        # A stored state is one of the two codes around its exact value (steps of at
        # most 1/8 of the value, or 2^-9 of the scale where the grid is even).
        (_, m, v), (_, em, ev) = expected(before, i, 10, **HYPER)
        for name, x in (('exp_avg', m), ('exp_avg_sq', np.sqrt(v))):
            got = f64(optim.dequantize(s[name + 's'][i].cpu(), s[name + '_scales'][i].cpu())).reshape(-1)
            x = x.reshape(-1)
            scale = f64(s[name + '_scales'][i]).repeat(256)[:n]
            assert np.all(np.abs(got - x) <= np.maximum(np.abs(x) / 8, scale * 2.0 ** -9) * (1 + 64 * U))
            if n:
                top = np.array([np.abs(x[k:k + 256]).max() for k in range(0, n, 256)])
                np.testing.assert_allclose(f64(s[name + '_scales'][i]) * 448, top, rtol=64 * U)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_8bit_codes_follow_the_stated_rule(dtype):
    """Codes equal the plain form's; an fp32 difference of a few units in the last
    place moves one in 2^20 / 4 of them, so 2 x 10^5 give about one (8 allowed)."""
    shapes = [(100003,), (257, 389)]
    s = make(shapes, dtype, 'cpu', bits=8)
    s['grads'][0][1000:1300] *= 1e-7  # values far below their block's maximum
    s['exp_avgs'][0].view(torch.uint8)[1000:1300] = 1
    gpu = clone(s, 'cuda')
    call(s, step=77, seed=123456789)
    call(gpu, step=77, seed=123456789)
    moved = 0
    for i in range(2):
        for name in ('exp_avgs', 'exp_avg_sqs'):
            a, b = gpu[name][i].cpu().float(), s[name][i].float()
            moved += int((a != b).sum())
        for name in ('exp_avg_scales', 'exp_avg_sq_scales'):
            torch.testing.assert_close(gpu[name][i].cpu(), s[name][i], rtol=8 * U, atol=0)
    assert moved <= 8


@pytest.mark.parametrize('device', DEVICES)
def test_8bit_rounding_is_unbiased_over_steps(device):
    """The mean of n stochastic roundings of x has a standard deviation of at most
    half a step / sqrt(n): 6 of them bound the error (steps of x / 8)."""
    n = 1 << 14
    s = make([(n,)], torch.float32, device, bits=8)
    s['params'][0].zero_()
    s['grads'][0].fill_(0.37e-3)
    s['grads'][0][::256] = 1e-3  # the blocks' maxima
    for name in ('exp_avgs', 'exp_avg_sqs'):
        s[name][0].view(torch.uint8).zero_()
    call(s, step=1, seed=3)
    keep = torch.arange(n) % 256 != 0
    for codes, scales, x in ((s['exp_avgs'][0], s['exp_avg_scales'][0], 0.1 * 0.37e-3),
                             (s['exp_avg_sqs'][0], s['exp_avg_sq_scales'][0], math.sqrt(0.05) * 0.37e-3)):
        got = optim.dequantize(codes.cpu(), scales.cpu())[keep].double()
        assert len(torch.unique(got)) == 2
        assert abs(got.mean().item() / x - 1) <= 6 * (1 / 8) / 2 / math.sqrt(len(got))


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_unaligned_views_and_permuted_layouts(bits):
    base = make([(4001,), (64, 48)], torch.bfloat16, 'cuda', bits=bits)
    s = clone(base)

    def shifted(t):  # the same values one element into a larger buffer
        big = torch.empty(t.numel() + 1, dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device='cuda')
        big = big.view(t.dtype)
        big[1:].copy_(t.reshape(-1))
        return big[1:].view(t.shape)

    for name in ('params', 'grads', 'exp_avgs', 'exp_avg_sqs'):
        s[name] = [shifted(s[name][0]), s[name][1].t().contiguous().t()]
    # A permuted parameter counts its blocks in memory order: compare it with its transpose.
    ref = clone(base)
    for name in ('params', 'grads', 'exp_avgs', 'exp_avg_sqs'):
        ref[name][1] = ref[name][1].t().contiguous()
    call(s, seed=1)
    call(ref, seed=1)
    for name in ('params', 'exp_avgs', 'exp_avg_sqs'):
        assert torch.equal(s[name][0].float(), ref[name][0].float())
        assert torch.equal(s[name][1].t().float(), ref[name][1].float())
    if bits == 32:  # a gradient laid out differently from its parameter
        t = clone(base)
        t['grads'][1] = t['grads'][1].t().contiguous().t()
        want = clone(base)
        call(t)
        call(want)
        assert torch.equal(t['params'][1], want['params'][1])


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_more_tensors_than_one_launch_takes(bits):
    shapes = [(3 + i % 700,) for i in range(901)]
    s = make(shapes, torch.float32, 'cuda', bits=bits)
    before = clone(s)
    cpu = clone(s, 'cpu')
    n0 = _native.launch_count()
    call(s, seed=9)
    assert _native.launch_count() - n0 == 3  # 400 + 400 + 101
    for i in (0, 1, 399, 400, 401, 799, 800, 900):
        check(before, s, i, torch.float32, 10, exact_states=bits == 32)
    if bits == 8:
        call(cpu, seed=9)
        moved = sum(int((a.cpu().float() != b.float()).sum()) for name in ('exp_avgs', 'exp_avg_sqs')
                    for a, b in zip(s[name], cpu[name]))
        assert moved <= 12  # 6 x 10^5 codes, about 2 expected to differ


@pytest.mark.parametrize('device', DEVICES)
def test_non_finite_gradients_stay_where_they_are(device):
    for bits in (32, 8):
        s = make([(1024,)], torch.float32, device, bits=bits)
        clean = clone(s)
        s['grads'][0][300] = float('nan')
        s['grads'][0][301] = float('inf')
        call(s, seed=2)
        call(clean, seed=2)
        others = torch.ones(1024, dtype=torch.bool)
        others[300:302] = False
        p, q = s['params'][0].cpu(), clean['params'][0].cpu()
        assert torch.equal(p[others], q[others])
        assert torch.isnan(p[300]) and not torch.isfinite(p[301])
        if bits == 8:  # the states of that block are lost, no others
            scales = s['exp_avg_scales'][0].cpu()
            assert not torch.isfinite(scales[1]) and torch.isfinite(scales[[0, 2, 3]]).all()


@pytest.mark.parametrize('device', DEVICES)
def test_grad_scale_multiplies_the_gradients(device):
    for bits in (32, 8):
        a = make([(700,)], torch.float32, device, bits=bits)
        b = clone(a)
        call(a, grad_scale=torch.tensor(0.25, device=device))
        b['grads'][0] *= 0.25
        call(b)
        for name in ('params', 'exp_avgs', 'exp_avg_sqs'):
            assert torch.equal(a[name][0].float(), b[name][0].float())


@pytest.mark.gpu
def test_tensors_past_2_to_the_31_elements():
    n = (1 << 31) + 777
    p = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    g = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    m = torch.zeros(n, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    v = torch.zeros(n, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    scales = [torch.zeros(optim.state_scales(n), device='cuda') for _ in range(2)]
    g[-5:] = 1.0
    g[:3] = -1.0
    optim.adamw_step([p], [g], [m], [v], step=1, lr=0.5, betas=(0.9, 0.95), weight_decay=0.0,
                     exp_avg_scales=[scales[0]], exp_avg_sq_scales=[scales[1]])
    # The first step moves by lr g / |g|.
    assert torch.equal(p[-6:].float().cpu(), torch.tensor([0, -.5, -.5, -.5, -.5, -.5]))
    assert torch.equal(p[:4].float().cpu(), torch.tensor([.5, .5, .5, 0]))
    assert int(p.count_nonzero()) == 8
    assert scales[0][-1].item() == pytest.approx(0.1 / 448, rel=1e-6)
    assert int(scales[0].gt(1e-30).sum()) == 2


@pytest.mark.gpu
def test_runs_on_the_current_stream_and_in_a_graph():
    s = make([(5000,), (33,)], torch.bfloat16, 'cuda')
    ref = clone(s)
    call(ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    t = clone(s)
    with torch.cuda.stream(side):
        call(t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(t['params'][0], ref['params'][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(s)
    graph.replay()
    assert torch.equal(s['params'][0], ref['params'][0]) and torch.equal(s['exp_avgs'][1], ref['exp_avgs'][1])


@pytest.mark.parametrize('device', DEVICES)
def test_autograd_notices_that_parameters_changed(device):
    w = torch.nn.Parameter(torch.ones(4, device=device))
    loss = (w * w).sum()
    loss.backward(retain_graph=True)
    optim.AdamW([w], lr=0.1).step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def _train(device, steps, **kw):
    """A small least-squares fit; its loss after `steps` steps."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(512, 32, generator=g).to(device)
    y = (x @ torch.randn(32, 8, generator=g).to(device)).tanh()
    w1 = torch.nn.Parameter((torch.randn(32, 64, generator=g) * 0.2).to(device))
    w2 = torch.nn.Parameter((torch.randn(64, 8, generator=g) * 0.2).to(device))
    opt = optim.AdamW([w1, w2], lr=1e-2, betas=(0.9, 0.99), weight_decay=0.0, **kw)
    for _ in range(steps):
        opt.zero_grad()
        loss = ((x @ w1).relu() @ w2 - y).square().mean()
        loss.backward()
        opt.step()
    return loss.item(), opt, (w1, w2)


@pytest.mark.parametrize('device', DEVICES)
def test_optimizer_class_trains_as_torch_does(device):
    loss, opt, (w1, w2) = _train(device, 60)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(512, 32, generator=g).to(device)
    y = (x @ torch.randn(32, 8, generator=g).to(device)).tanh()
    v1 = torch.nn.Parameter((torch.randn(32, 64, generator=g) * 0.2).to(device))
    v2 = torch.nn.Parameter((torch.randn(64, 8, generator=g) * 0.2).to(device))
    ref = torch.optim.AdamW([v1, v2], lr=1e-2, betas=(0.9, 0.99), weight_decay=0.0)
    for _ in range(60):
        ref.zero_grad()
        want = ((x @ v1).relu() @ v2 - y).square().mean()
        want.backward()
        ref.step()
    assert loss == pytest.approx(want.item(), rel=1e-2)
    start, _, _ = _train(device, 1)
    eight, _, _ = _train(device, 60, state_bits=8, seed=1)
    assert eight < 0.25 * start and eight < 2 * loss  # 8-bit states fit as well, within noise


@pytest.mark.parametrize('bits,master,dtype', [(32, False, torch.float32), (8, True, torch.bfloat16)])
def test_state_dict_round_trip_keeps_types_and_steps(bits, master, dtype):
    def params():
        g = torch.Generator().manual_seed(1)
        return [torch.nn.Parameter(torch.randn(40, 30, generator=g).to(dtype)),
                torch.nn.Parameter(torch.randn(11, generator=g).to(dtype))]

    def grads(ps, k):
        for p in ps:
            p.grad = torch.full_like(p, 0.01 * k)

    a = params()
    kw = dict(lr=1e-2, state_bits=bits, master_weights=master, seed=4)
    oa = optim.AdamW(a, **kw)
    for k in range(3):
        grads(a, k + 1)
        oa.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = optim.AdamW(b, **kw)
    ob.load_state_dict(oa.state_dict())
    for p, q in zip(a, b):
        for name, t in oa.state[p].items():
            if isinstance(t, torch.Tensor):
                assert ob.state[q][name].dtype == t.dtype
                assert ob.state[q][name].data_ptr() != t.data_ptr()
    for ps, o in ((a, oa), (b, ob)):
        grads(ps, 7)
        o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        assert oa.state[p]['step'] == ob.state[q]['step'] == 4


@pytest.mark.parametrize('bits', [32, 8])
def test_state_dict_of_another_layout_follows_the_parameter(bits):
    """8-bit values move by half a code at most: the codes of a block are 2^-3 of
    their value or less apart, and 2^-9 of the block's maximum / 448 below 2^-6."""
    g = torch.Generator().manual_seed(8)
    w = torch.randn(40, 30, generator=g)
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.t().contiguous().t())
    oa, ob = (optim.AdamW([p], lr=1e-2, state_bits=bits, seed=4) for p in (a, b))
    a.grad = torch.randn(40, 30, generator=g)
    oa.step()
    ob.load_state_dict(oa.state_dict())
    for name in ('exp_avg', 'exp_avg_sq'):
        old, new = oa.state[a][name], ob.state[b][name]
        assert new.dtype == old.dtype and new.stride() == b.stride()
        if bits == 32:
            assert torch.equal(new, old)
            continue
        want = optim.dequantize(old, oa.state[a][name + '_scale'])
        got = optim.dequantize(new, ob.state[b][name + '_scale'])
        top = want.abs().max() / 448
        assert ((got - want).abs() <= want.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + top * 2.0 ** -10).all()
    b.grad = a.grad.clone()
    ob.step()


def test_parameters_without_a_gradient_are_left_alone():
    p, q = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    o = optim.AdamW([p, q], lr=0.1)
    p.grad = torch.ones(4)
    o.step()
    assert torch.equal(q, torch.ones(4)) and not o.state[q]
    q.grad = torch.ones(4)
    o.step()
    assert o.state[p]['step'] == 2 and o.state[q]['step'] == 1


@pytest.mark.parametrize('kw,match', [
    (dict(state_bits=16), 'state_bits'), (dict(lr=-1.0), 'lr'), (dict(betas=(1.0, 0.9)), 'betas'),
    (dict(eps=float('nan')), 'eps')])
def test_optimizer_rejects_bad_settings(kw, match):
    with pytest.raises(ValueError, match=match):
        optim.AdamW([torch.nn.Parameter(torch.ones(2))], **kw)


@pytest.mark.gpu
@pytest.mark.parametrize('change,match', [
    (dict(grads=lambda t: [t[0].float(), t[1]]), 'one type'),
    (dict(grads=lambda t: [t[0].cpu(), t[1]]), 'one device'),
    (dict(grads=lambda t: t[:1]), 'one tensor for each parameter'),
    (dict(grads=lambda t: [t[0][:5], t[1]]), 'shape of its parameter'),
    (dict(exp_avgs=lambda t: [t[0].half(), t[1]]), 'one type|float32 or float8'),
    (dict(exp_avg_sqs=lambda t: [t[0], t[1].t().contiguous().t()]), 'shape and strides'),
    (dict(params=lambda t: [t[0][::2], t[1]], grads=lambda t: [t[0][::2], t[1]]), 'dense in memory'),
    (dict(params=lambda t: [t[0].double(), t[1].double()], grads=lambda t: [x.double() for x in t]),
     'float32, float16 or bfloat16'),
    (dict(params=lambda t: [t[0], t[0]], grads=lambda t: [t[0], t[0]], exp_avgs=lambda t: [t[0], t[0]],
          exp_avg_sqs=lambda t: [t[0], t[0]]), 'more than once'),
    (dict(exp_avg_scales=lambda t: [torch.zeros(1, device='cuda')] * 2), 'go with float8'),
])
def test_step_rejects_what_it_cannot_take(change, match):
    s = make([(600,), (8, 12)], torch.bfloat16, 'cuda')
    for name, f in change.items():
        s[name] = f(s[name])
    before = _native.launch_count()
    with pytest.raises(ValueError, match=match):
        call(s)
    assert _native.launch_count() == before


@pytest.mark.parametrize('view', [lambda t: t[::2], lambda t: t[:, :3], lambda t: t[:1].expand(6, 8)])
def test_cpu_step_refuses_parameters_that_are_not_dense(view):
    p = view(torch.ones(6, 8))
    m, v = (torch.empty_strided(p.shape, p.stride()).zero_() for _ in range(2))
    with pytest.raises(ValueError, match='dense in memory'):
        optim.adamw_step([p], [torch.ones(p.shape)], [m], [v], step=1, lr=0.1)


@pytest.mark.gpu
def test_8bit_states_need_the_right_scales():
    s = make([(600,)], torch.bfloat16, 'cuda', bits=8)
    s['exp_avg_scales'] = [s['exp_avg_scales'][0][:2]]
    with pytest.raises(ValueError, match='must be 3 contiguous'):
        call(s)


def _params(**kw):
    t = (_native.AveyAdamWTensor * 1)()
    t[0] = _native.AveyAdamWTensor(1 << 20, 2 << 20, 3 << 20, 4 << 20, 0, 0, 0, 100)
    p = _native.AveyAdamWParams()
    p.struct_size = ctypes.sizeof(p)
    p.dtype, p.state_bits, p.count, p.tensors = _native.AVEY_BF16, 32, 1, t
    p.lr, p.beta1, p.beta2, p.eps, p.weight_decay, p.step = 1e-3, 0.9, 0.95, 1e-8, 0.0, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return p, t


@pytest.mark.parametrize('field,value,match', [
    ('struct_size', 8, 'struct_size'), ('dtype', _native.AVEY_F64, 'f32, f16 or bf16'),
    ('state_bits', 16, 'state_bits'), ('count', -1, 'tensors'), ('lr', float('inf'), 'lr'),
    ('beta1', 1.0, 'beta1'), ('beta2', -0.1, 'beta2'), ('step', 0, 'step'),
    ('state_bits', 8, 'exp_avg_scale')])
def test_c_entry_rejects_bad_arguments_before_any_launch(field, value, match):
    p, _keep = _params(**{field: value})
    before = _native.launch_count()
    with pytest.raises(_native.NativeError, match=match) as info:
        _native.adamw(p, 0)
    assert info.value.status == -1 and _native.launch_count() == before


@pytest.mark.parametrize('field,value,bits', [
    ('param', (1 << 20) + 1, 32), ('grad', (2 << 20) + 1, 8), ('exp_avg', (3 << 20) + 2, 32),
    ('exp_avg_scale', (5 << 20) + 2, 8), ('master', (6 << 20) + 2, 32)])
def test_c_entry_wants_arrays_aligned_to_their_elements(field, value, bits):
    p, t = _params(state_bits=bits)
    t[0].exp_avg_scale = t[0].exp_avg_sq_scale = 5 << 20
    setattr(t[0], field, value)
    with pytest.raises(_native.NativeError, match='aligned to their elements'):
        _native.adamw(p, 0)


def test_c_entry_wants_masters_for_all_or_none():
    p, t = _params(count=2)
    two = (_native.AveyAdamWTensor * 2)(t[0], t[0])
    two[1].master = 5 << 20
    p.tensors = two
    with pytest.raises(_native.NativeError, match='for all tensors or for none'):
        _native.adamw(p, 0)


@pytest.mark.gpu
@pytest.mark.parametrize('name', ['params', 'grads', 'exp_avgs', 'exp_avg_sqs', 'masters'])
def test_native_step_refuses_tangents(name):
    """The step would leave the tangents as they were."""
    s = make([(40,), (8, 12)], torch.bfloat16, 'cuda', master=True)
    with forward_ad.dual_level():
        call(s)
        before = clone(s)
        s[name][1] = forward_ad.make_dual(s[name][1], torch.ones_like(s[name][1]))
        with pytest.raises(RuntimeError, match='forward-mode'):
            call(s)
    assert torch.equal(s['params'][0], before['params'][0])


@pytest.mark.gpu
@pytest.mark.parametrize('trace', [lambda f, x: make_fx(f)(x), lambda f, x: torch.jit.trace(f, (x,), check_trace=False)])
def test_native_step_refuses_to_be_traced(trace):
    s = make([(40,)], torch.float32, 'cuda')

    def step(g):
        call(dict(s, grads=[g]))
        return s['params'][0] + 1

    with pytest.raises(RuntimeError, match='traced'):
        trace(step, s['grads'][0])


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('default', [torch.bfloat16, torch.float64])
def test_8bit_states_do_not_go_by_the_default_type(default, device):
    """Their scales are fp32, and exact, under any default type."""
    def run():
        p = torch.nn.Parameter(torch.ones(700, device=device, dtype=torch.float32))
        p.grad = torch.linspace(-1, 1, 700, device=device, dtype=torch.float32)
        opt = optim.AdamW([p], lr=0.1, state_bits=8, seed=3)
        for _ in range(2):
            opt.step()
        return p.detach(), opt.state[p]

    want, state = run()
    torch.set_default_dtype(default)
    try:
        got, other = run()
    finally:
        torch.set_default_dtype(torch.float32)
    assert torch.equal(got, want)
    for name in ('exp_avg_scale', 'exp_avg_sq_scale'):
        assert other[name].dtype == torch.float32 and torch.equal(other[name], state[name])


@pytest.mark.parametrize('bits,change,match', [
    (32, dict(exp_avgs=torch.Tensor.bfloat16), 'float32 or float8'),
    (32, dict(exp_avg_sqs=torch.Tensor.double), 'float32 or float8'),
    (32, dict(masters=torch.Tensor.bfloat16), 'masters.1. must be float32'),
    (8, dict(exp_avg_scales=torch.Tensor.bfloat16), 'scales of parameter 1 must be 1 contiguous'),
    (8, dict(exp_avg_sq_scales=lambda t: torch.cat((t, t))), 'scales of parameter 1 must be 1 contiguous'),
    (8, dict(exp_avg_scales=lambda t: t[:0]), 'scales of parameter 1 must be 1 contiguous')])
@pytest.mark.parametrize('device', DEVICES)
def test_states_of_another_type_or_size_are_refused_before_any_change(bits, change, match, device):
    s = make([(600,), (8, 12)], torch.bfloat16, device, bits=bits, master=True)
    for name, f in change.items():
        s[name][1] = f(s[name][1])
    before = clone(s)
    with pytest.raises(ValueError, match=match + '|one type'):
        call(s)
    assert torch.equal(s['params'][0], before['params'][0])


def test_cpu_step_does_not_go_by_the_default_device():
    a = make([(600,), (8, 12)], torch.bfloat16, 'cpu', bits=8)
    b = clone(a)
    call(a, seed=7)
    torch.set_default_device('meta')
    try:
        call(b, seed=7)
    finally:
        torch.set_default_device(None)
    for name in ('params', 'exp_avgs', 'exp_avg_sqs'):
        assert all(torch.equal(p.float(), q.float()) for p, q in zip(a[name], b[name]))


@pytest.mark.parametrize('device', DEVICES)
def test_a_step_that_raises_is_not_counted(device):
    """Neither for the parameters before the bad one nor for it; the next step is
    what it would have been."""
    p, q, r = (torch.nn.Parameter(torch.full((4,), 2.0, device=device)) for _ in range(3))
    opt, ref = optim.AdamW([p, q], lr=0.1), optim.AdamW([r], lr=0.1)
    for t in (p, q, r):
        t.grad = torch.ones_like(t)
    opt.step()
    ref.step()
    good, q.grad = q.grad, torch.ones(4, device=device).to_sparse()
    with pytest.raises(ValueError, match='sparse'):
        opt.step()
    with pytest.raises(ValueError, match='lr'):
        q.grad = good
        opt.param_groups[0]['lr'] = float('nan')
        opt.step()
    opt.param_groups[0]['lr'] = 0.1
    p.grad.mul_(-1)
    r.grad.mul_(-1)
    opt.step()
    ref.step()
    assert opt.state[p]['step'] == opt.state[q]['step'] == 2
    assert torch.equal(p, r)

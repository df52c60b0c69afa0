"""The example's model, from tokens to the loss and back to all of its weights, against the same
model written in plain torch in 64 bits."""

import importlib.util
import re
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from avey_kernel_b200 import _native, experts, layers, losses

PATH = Path(__file__).resolve().parents[1] / 'examples' / 'train_block.py'
spec = importlib.util.spec_from_file_location('train_block', PATH)
train_block = importlib.util.module_from_spec(spec)
spec.loader.exec_module(train_block)


def plain(p, tokens, targets, chosen):
    """The loss of the model with the parameters p (by name), whose every token takes all experts
    (`chosen` of them: the renormalised weights are the softmax of the router's logits)."""
    x = p['embed'][tokens]
    blocks = 1 + max(int(name.split('.')[1]) for name in p if name.startswith('blocks'))
    for i in range(blocks):
        q = {name.split('.')[2]: t for name, t in p.items() if name.startswith(f'blocks.{i}.')}
        width, context = x.shape[-1], x.shape[1]
        e = F.silu(F.layer_norm(x, (width,)) @ q['enrich_w'].t() + q['enrich_b'])
        head, tail = e[..., :width], e[..., width:]
        unit = F.normalize(tail, dim=-1)
        s = (unit @ unit.transpose(1, 2)) * q['mix'].tril()
        assert s.shape[-1] == context
        x = (s @ tail) * head @ q['fuse_w'].t() + q['fuse_b'] + x
        h = F.layer_norm(x, (width,))
        weights = torch.softmax(h @ q['route_w'].t(), -1)
        assert chosen == weights.shape[-1]
        for k in range(chosen):
            up = torch.relu(h @ q['up_w'][k].t() + q['up_b'][k]).square()
            x = x + weights[..., k:k + 1] * (up @ q['down_w'][k].t() + q['down_b'][k])
    z = F.layer_norm(x, (x.shape[-1],)) @ p['head'].t()
    return F.cross_entropy(z.flatten(0, 1), targets.flatten())


@pytest.mark.parametrize('device,dt', [('cpu', torch.float32), pytest.param('cuda', torch.bfloat16, marks=pytest.mark.gpu),
                                       pytest.param('cuda', torch.float16, marks=pytest.mark.gpu)])
def test_gradients_of_the_example_model(device, dt):
    """On the way to a weight's gradient some 24 tensors are rounded to the operands' type, each by
    at most u = 2^-24, 2^-8 or 2^-11 of itself, and a layer passes on relative errors of its
    inputs at about their size (norms and weights of the order of one): 24 u of the norm. (fp32: 2^-15, as
    sums of some hundred terms add 2^-17 each.)"""
    torch.manual_seed(0)
    model = train_block.Model(vocab=50, context=24, width=64, num_experts=2, chosen=2, blocks=2)
    for name, t in model.named_parameters():
        if name.endswith('_b'):
            torch.nn.init.normal_(t, std=0.1)
    model = model.to(device, dt)
    gen = torch.Generator().manual_seed(1)
    seq = torch.randint(0, 50, (6, 25), generator=gen).to(device)
    loss = model(seq[:, :-1], seq[:, 1:])
    loss.backward()
    p = {name: t.detach().double().requires_grad_(True) for name, t in model.named_parameters()}
    want = plain(p, seq[:, :-1], seq[:, 1:], 2)
    want.backward()
    u = {torch.float32: 2.0 ** -15 / 24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dt]
    assert abs(float(loss.detach() - want.detach())) <= 24 * u * float(want.detach())
    for name, t in model.named_parameters():
        off = float((t.grad.double() - p[name].grad).norm() / p[name].grad.norm())
        assert off <= 24 * u, (name, off)
    if device == 'cuda':
        first = [t.grad.clone() for t in model.parameters()]
        model.zero_grad()
        model(seq[:, :-1], seq[:, 1:]).backward()
        assert all(torch.equal(a, t.grad) for a, t in zip(first, model.parameters()))
        assert _native.device_status(clear=True) == 0


def ends(dt, seed, tokens=300, width=72, vocab=700, num=4):
    """Tokens in, two experts each, the loss: inputs, and a step that returns it and its gradients."""
    gen = torch.Generator().manual_seed(seed)
    new = lambda *shape: (torch.randn(*shape, generator=gen) / shape[-1] ** 0.5).cuda().to(dt).requires_grad_(True)  # noqa: E731
    leaves = [new(vocab, width), new(num, width), new(num, width, width)]
    ids = torch.randint(0, vocab, (tokens,), generator=gen).cuda()

    def step(table, router, w):
        h = layers.embedding(ids, table, scale=4.0)
        weights, chosen = experts.route(h @ router.t(), 2)
        slots, offsets = experts.arrange(chosen, num)
        y = experts.expert_linear(experts.dispatch(h, slots), w, offsets, activation='silu')
        h = experts.combine(y, slots, weights, residual=h)
        return losses.linear_cross_entropy(h, table, ids.roll(-1), z_loss=1e-3)

    def train():
        loss = step(*leaves)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    return ids, leaves, step, train


@pytest.mark.gpu
def test_two_captured_steps_replayed_at_once():
    (ids1, _, _, one), (ids2, _, _, two) = ends(torch.bfloat16, 0), ends(torch.float16, 1, tokens=9000, vocab=5000)
    one(), two()
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, train in zip(graphs, (one, two)):
        with torch.cuda.graph(graph):
            got.append(train())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(3):
        ids1.copy_(ids1.flip(0).roll(i))
        ids2.copy_(ids2 % (5000 >> i))
        for stream, graph in zip(streams, graphs):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for _ in range(4):
                    graph.replay()
        for stream in streams:
            torch.cuda.current_stream().wait_stream(stream)
        for values, train in zip(got, (one, two)):
            assert all(torch.equal(p, q) for p, q in zip(values, train()))
    assert _native.device_status(clear=True) == 0


@pytest.mark.gpu
def test_compiled_functions_call_the_operators():
    _, leaves, step, train = ends(torch.bfloat16, 2)
    compiled = torch.compile(step, backend='eager')
    loss = compiled(*leaves)
    got = [loss.detach(), *torch.autograd.grad(loss, leaves)]
    assert all(torch.equal(p, q) for p, q in zip(got, train()))


def test_chained_kernels_wait_for_the_one_before_ahead_of_their_reads():
    """Every kernel that a chain of launches (launch_chain.h) names waits before anything that reads: what
    its body calls ahead of the wait is none of the functions that load."""
    csrc = Path(_native.__file__).parent / 'csrc'
    launched = set()
    for name in ('avey_loss.cu', 'avey_tokens.cu'):
        source = (csrc / name).read_text()
        calls = re.findall(r'chain\.launch\(\s*"[^"]*",\s*([\w:<>, ]+?)[,(]', source)
        assert len(calls) == source.count('chain.launch(') and calls
        launched |= {re.sub(r'<.*', '', call).split('::')[-1] for call in calls}
    launched = {'ce_product' if name == 'K' else name for name in launched}  # launch_product's argument
    seen = set()
    for name in ('tc_loss.cuh', 'route_kernels.cuh', 'sort_kernels.cuh', 'rows_kernels.cuh', 'linear_steps.cuh'):
        for part in (csrc / name).read_text().split('__global__')[1:]:
            kernel = re.search(r'(\w+)\((?:const|CeMaps|float)', part[part.index(')'):] if '__launch_bounds__' in part[:40] else part)
            if kernel.group(1) not in launched:
                continue
            seen.add(kernel.group(1))
            body = part[part.index('{'):]
            assert 'griddep_wait();' in body, kernel.group(1)
            ahead = body[:body.index('griddep_wait();')]
            for read in ('__ld', 'load', 'atomic', 'ce_target', 'ce_scale', 'st_key', 'st_count', 'st_place_block', 'st_zero', 'rw_blank',
                         'rw_slots', 'rt_choose', 'q.keys', 'q.ids', 'q.edges', 'q.partial', 'q.each'):
                assert read not in ahead, (kernel.group(1), read)
    assert seen == launched, seen ^ launched

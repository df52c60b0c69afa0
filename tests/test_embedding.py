"""``layers.embedding`` against its formula in 64 bits.

Tolerances, with u = 2^-24 (fp32), 2^-11 (f16) or 2^-8 (bf16): a row is scaled in fp32 and
rounded once (2^-23 + u of itself; without a scale it is the table's, bit for bit); a
gradient is a sum of n rows in fp32 ((n + 1) 2^-23 of the sum of its terms' sizes), scaled
and rounded once; f16 adds 2^-25."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from avey_kernel_b200 import _native, layers

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -120, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -120}
DTYPES = list(UNIT)
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def close(got, want, name):
    value, bound = want
    got = got.detach().double()
    assert got.shape == value.shape, name
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} outside, worst '
                           f'{float(((got - value).abs() / bound.clamp(min=1e-300)).max()):.3g} of the bound')


def gradient(tokens, dy, vocab, scale, padding):
    """The table's gradient and its bound."""
    t, d = tokens.reshape(-1).long(), dy.reshape(-1, dy.shape[-1]).double()
    keep = (t >= 0) & (t < vocab) & (t != (-1 if padding is None else padding))
    t, d = t[keep], d[keep]
    value = torch.zeros(vocab, dy.shape[-1], dtype=torch.float64, device=dy.device).index_add(0, t, d) * scale
    size = torch.zeros_like(value).index_add(0, t, d.abs()) * abs(scale)
    count = torch.bincount(t, minlength=vocab).double().unsqueeze(1)
    return value, (count + 1) * 2.0 ** -23 * size + UNIT[dy.dtype] * value.abs() * (1 + 2.0 ** -7) + TINY[dy.dtype]


def check(tokens, vocab, width, dt, scale=1.0, padding=None, seed=0):
    device = tokens.device
    g = torch.Generator(device=device).manual_seed(seed)
    w = torch.randn(vocab, width, generator=g, device=device).to(dt).requires_grad_(True)
    dy = torch.randn(*tokens.shape, width, generator=g, device=device).to(dt)
    out = layers.embedding(tokens, w, scale=scale, padding_idx=padding)
    assert out.dtype == dt and out.shape == (*tokens.shape, width)
    rows = w.detach()[tokens.clamp(0, vocab - 1).long()]
    inside = ((tokens >= 0) & (tokens < vocab)).unsqueeze(-1)
    if scale == 1.0:
        assert torch.equal(torch.where(inside, out.detach(), 0), torch.where(inside, rows, 0))
    else:
        value = torch.where(inside, rows.double() * scale, 0)
        close(torch.where(inside, out.detach(), 0),
              (value, (2.0 ** -23 + UNIT[dt] * (1 + 2.0 ** -7)) * value.abs() + TINY[dt]), 'out')
    assert out.detach()[~inside.squeeze(-1)].isnan().all()
    dw, = torch.autograd.grad(out, w, dy)
    assert dw.dtype == dt
    value, bound = gradient(tokens, dy, vocab, scale, padding)
    close(dw, (value, bound), 'dw')
    assert not dw[value.abs().sum(1) == 0].any()
    return out, dw


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dt', DTYPES)
@pytest.mark.parametrize('shape,vocab,width', [((1,), 1, 1), ((3, 5), 7, 8), ((33,), 1023, 389), ((64,), 1024, 64),
                                               ((2, 100), 50, 768), ((4096,), 1025, 40), ((5000,), 300, 24),
                                               ((70, 100), 33000, 66)])
def test_rows_and_their_gradient(shape, vocab, width, dt, device):
    g = torch.Generator().manual_seed(vocab)
    tokens = torch.randint(0, vocab, shape, generator=g).to(device)
    check(tokens, vocab, width, dt)
    check(tokens.int(), vocab, width, dt, scale=0.37, padding=vocab // 2)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('lengths', [[1] * 40, [32], [31, 33], [64, 1, 31, 32], [100, 28, 5, 200, 1, 1, 62], [4097],
                                     [1000, 1, 3000, 96]])
def test_runs_of_one_token_that_end_anywhere(lengths, device):
    """Sorted, shuffled and reversed: runs over many edges of the pieces that blocks take."""
    t = torch.cat([torch.full((n,), 3 * i + 1) for i, n in enumerate(lengths)])
    perm = torch.randperm(len(t), generator=torch.Generator().manual_seed(0))
    for order in (t, t[perm], t.flip(0)):
        check(order.to(device), 3 * len(lengths) + 2, 40, torch.float32)
        check(order.to(device), 3 * len(lengths) + 2, 33, torch.bfloat16, scale=2.0)


@pytest.mark.parametrize('device', DEVICES)
def test_tokens_outside_and_padding(device):
    t = torch.tensor([[0, 5, -1, 9], [9, 10, 2 ** 40, -2 ** 40]], device=device)
    check(t, 10, 12, torch.float32, padding=9)
    check(t.clamp(-5, 50).int(), 10, 12, torch.bfloat16, scale=3.0)
    check(torch.full((300,), 4, device=device), 6, 8, torch.float32, padding=4)  # nothing but padding
    check(torch.full((300,), 77, device=device), 6, 8, torch.float32)            # nothing inside


@pytest.mark.parametrize('device', DEVICES)
def test_no_tokens_strides_and_alignment(device):
    w = torch.randn(20, 48, device=device, requires_grad=True)
    empty = torch.zeros(0, 3, dtype=torch.int64, device=device)
    out = layers.embedding(empty, w)
    assert out.shape == (0, 3, 48)
    dw, = torch.autograd.grad(out, w, torch.zeros(0, 3, 48, device=device))
    assert dw.shape == w.shape and not dw.any()
    tokens = torch.randint(0, 20, (6, 8), device=device)
    for view in (w[:, 1:33], w[:, ::2], w.t()[:20, :20], w[:1].expand(20, 48)):
        leaf = view.detach().requires_grad_(True)
        for t in (tokens.t(), tokens[:, ::2], tokens[0, 0]):
            a, b = layers.embedding(t, leaf, scale=0.5), layers.embedding(t.contiguous(), leaf.detach().contiguous(), scale=0.5)
            assert torch.equal(a, b)
            dy = torch.randn(*t.shape, 2 * leaf.shape[1], device=device)[..., 1:leaf.shape[1] + 1]
            d1, = torch.autograd.grad(a, leaf, dy)
            value, bound = gradient(t, dy, 20, 0.5, None)
            close(d1, (value, bound), 'dw')


@pytest.mark.gpu
def test_results_are_bitwise_reproducible_and_whole_numbers_exact():
    g = torch.Generator(device='cuda').manual_seed(0)
    t = (torch.rand(50000, generator=g, device='cuda') ** 4 * 3000).long()
    dy = torch.randint(-2, 3, (50000, 72), generator=g, device='cuda').float()
    w = torch.zeros(3000, 72, device='cuda', requires_grad=True)
    a, = torch.autograd.grad(layers.embedding(t, w), w, dy)
    assert torch.equal(a.double(), gradient(t, dy, 3000, 1.0, None)[0])  # no row is lost or doubled
    dy = torch.randn(50000, 72, generator=g, device='cuda')
    a, = torch.autograd.grad(layers.embedding(t, w), w, dy)
    b, = torch.autograd.grad(layers.embedding(t, w), w, dy)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('n,vocab,width', [(8192, 1000, 24), (8193, 1000, 24), (9500, 1 << 20, 4), (20000, 1 << 20, 1),
                                           (38000, 777, 300), (40000, (1 << 20) + 7, 2)])
def test_all_pieces_and_numbers_of_passes(n, vocab, width):
    """The sort of one launch and that of many, of one to three digits, with pieces of 8 to 32 places;
    tokens from both ends of the vocabulary, one of them a quarter of all."""
    g = torch.Generator(device='cuda').manual_seed(n)
    t = torch.randint(0, vocab, (n,), generator=g, device='cuda')
    t[::4] = vocab - 3
    t[1:100] = torch.arange(99, device='cuda') - 1
    check(t, vocab, width, torch.float32, padding=5)


@pytest.mark.gpu
def test_tables_past_2_to_the_31_elements():
    vocab, width = (1 << 21) + 50, 1032  # 2.16 10^9 elements
    w = torch.zeros(vocab, width, dtype=torch.bfloat16, device='cuda')
    w[-3:] = torch.arange(1, 4, device='cuda').unsqueeze(1)
    t = torch.tensor([vocab - 1, 0, vocab - 3, vocab - 1], device='cuda')
    w.requires_grad_(True)
    out = layers.embedding(t, w)
    assert out[:, -1].tolist() == [3, 0, 1, 3]
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw[-1, 5] == 2 and dw[-3, -1] == 1 and dw[0, 0] == 1 and not dw[1:-3].any() and not dw[-2].any()


@pytest.mark.gpu
def test_streams_and_captured_steps():
    w = torch.randn(500, 72, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    t = torch.randint(0, 500, (40, 200), device='cuda')
    dy = torch.randn(40, 200, 72, device='cuda').bfloat16()

    def step():
        out = layers.embedding(t, w, scale=2.0)
        return [out.detach(), *torch.autograd.grad(out, w, dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        t.copy_(torch.randint(0, 500 >> i, (40, 200), device='cuda'))
        for _ in range(3):
            graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_types_that_a_table_may_have():
    for bad in (torch.double, torch.long):
        with pytest.raises(ValueError, match='float'):
            layers.embedding(torch.zeros(3, dtype=torch.int64), torch.ones(5, 4).to(bad))


def test_refusals_of_arguments():
    w, t = torch.randn(5, 4), torch.zeros(3, dtype=torch.int64)
    for args, kw, match in (((t.float(), w), {}, 'tokens'), ((t, w[0]), {}, 'weight'), ((t, w[:0]), {}, 'weight'),
                            ((t, w), dict(padding_idx=5), 'padding'), ((t, w), dict(padding_idx=-1), 'padding'),
                            ((t, w), dict(scale=math.nan), 'scale')):
        with pytest.raises(ValueError, match=match):
            layers.embedding(*args, **kw)


@pytest.mark.gpu
def test_refusals_of_cuda_tensors_tangents_and_traces():
    w, t = torch.randn(5, 4, device='cuda', requires_grad=True), torch.zeros(3, dtype=torch.int64, device='cuda')
    with pytest.raises(ValueError, match='tokens'):
        layers.embedding(t.cpu(), w)
    with pytest.raises(ValueError, match='float'):
        layers.embedding(t, w.double())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
        layers.embedding(t, forward_ad.make_dual(w.detach(), torch.ones_like(w)))
    with pytest.raises(RuntimeError, match='traced'):
        make_fx(lambda u: layers.embedding(t, u))(w.detach())
    with pytest.raises(RuntimeError, match='again'):
        torch.autograd.grad(layers.embedding(t, w).sum(), w, create_graph=True)


@pytest.mark.parametrize('change,match', [
    (dict(struct_size=8), 'struct_size'), (dict(dtype=3), 'f32'), (dict(index_bits=8), 'bits'), (dict(count=-1), 'count'),
    (dict(width=0), 'width'), (dict(vocab=0), 'vocab'), (dict(vocab=(1 << 30) + 1), 'vocab'), (dict(tokens=0), 'tokens'),
    (dict(table=0), 'table'), (dict(out=0), 'out'), (dict(table_ld=7), 'strides'), (dict(scale=math.inf), 'scale'),
    (dict(out=(1 << 20) + 2), 'aligned'), (dict(tokens=(1 << 20) + 4), 'aligned')])
def test_c_entry_rejects_bad_arguments_before_any_launch(change, match):
    at = 1 << 20
    p = _native.AveyEmbeddingParams(struct_size=ctypes.sizeof(_native.AveyEmbeddingParams), dtype=0, index_bits=64, count=4,
                                    width=8, vocab=9, padding=-1, scale=1.0, tokens=at, table=at, table_ld=8, out=at)
    for a, b in change.items():
        setattr(p, a, b)
    lib = _native.lib()
    assert lib.avey_embedding_fwd_v1(ctypes.byref(p), None) == -1
    assert match in lib.avey_last_error().decode()


def test_c_workspace_sizes():
    at = 1 << 20
    p = _native.AveyEmbeddingParams(struct_size=ctypes.sizeof(_native.AveyEmbeddingParams), dtype=2, index_bits=64,
                                    count=100, width=8, vocab=1000, scale=1.0, tokens=at, dy=at, dy_ld=8, dtable=at)
    size, lib = ctypes.c_uint64(), _native.lib()
    assert lib.avey_embedding_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    # Keys and numbers of 100 tokens twice, 14 words of edges, two parts of 13 pieces of 8.
    assert size.value == 4 * 512 + 256 + 1024
    p.dy = 0
    assert lib.avey_embedding_bwd_v1(ctypes.byref(p), None) == -1 and b'dy' in lib.avey_last_error()


@pytest.mark.parametrize('count,width,vocab', [(1, 1, 1), (64, 64, 1000), (8192, 768, 32768), (8193, 1, 1000), (9471, 389, 1 << 30),
                                               (18943, 5, 1 << 21), (18944, 768, 131072), (65536, 768, 131072), (1 << 20, 64, 1 << 20)])
def test_workspace_is_what_the_header_says(count, width, vocab):
    at, size = 1 << 20, ctypes.c_uint64()
    p = _native.AveyEmbeddingParams(struct_size=ctypes.sizeof(_native.AveyEmbeddingParams), dtype=2, index_bits=64, count=count,
                                    width=width, vocab=vocab, scale=1.0, tokens=at, dy=at, dy_ld=width, dtable=at)
    assert _native.lib().avey_embedding_workspace_size(ctypes.byref(p), ctypes.byref(size)) == 0
    # (The last piece of 8 to 32 places may be short: 8 bytes a column.)
    assert size.value <= 32 * count + count * width / (4 if count >= 18944 else 1) + 8 * width + 4096

"""Train a small Avey model end to end on this package's operators.

A block is the enricher (``layers.residual_linear`` with its activation), the
contextualizer (``avey``), the fuser (``layers.residual_linear`` with the
residual in its epilogue) and a mixture of experts (``experts.expert_linear``
on tokens sorted by ``experts.group_by_expert``); the weights are updated by
``optim.AdamW``. The data are synthetic: sequences that follow a fixed
permutation of the tokens, of which one in eight is replaced by a random one; the
model tells the next token.

    python examples/train_block.py --steps 100 --state-bits 8

On a B200 it trains in bf16 on the native kernels; without a GPU it runs the
package's PyTorch path in fp32.
"""

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from avey_kernel_b200 import avey, experts, layers, optim  # noqa: E402


def _weight(*shape):
    return nn.Parameter(torch.randn(*shape) * shape[-1] ** -0.5)


class Block(nn.Module):
    """Enricher, contextualizer and fuser with a residual, then experts with a residual."""

    def __init__(self, context, width, num_experts):
        super().__init__()
        self.enrich_w, self.enrich_b = _weight(2 * width, width), nn.Parameter(torch.zeros(2 * width))
        self.mix = nn.Parameter(torch.randn(context, context) * 0.1)
        self.fuse_w, self.fuse_b = _weight(width, width), nn.Parameter(torch.zeros(width))
        self.route_w = _weight(num_experts, width)
        self.up_w, self.up_b = _weight(num_experts, 2 * width, width), nn.Parameter(torch.zeros(num_experts, 2 * width))
        self.down_w, self.down_b = _weight(num_experts, width, 2 * width), nn.Parameter(torch.zeros(num_experts, width))

    def forward(self, x):
        width = x.shape[-1]
        h = F.layer_norm(x, (width,))
        e = layers.residual_linear(h, self.enrich_w, self.enrich_b, activation='silu')
        mixed = avey(e[..., width:], self.mix, z_tl=e[..., :width])
        x = layers.residual_linear(mixed, self.fuse_w, self.fuse_b, residual=x)
        # Each token goes to its likeliest expert, weighted by the router's probability.
        h = F.layer_norm(x, (width,)).reshape(-1, width)
        probs = torch.softmax(layers.residual_linear(h, self.route_w).float(), dim=-1)
        weight, expert = probs.max(dim=-1)
        order, offsets = experts.group_by_expert(expert, self.route_w.shape[0])
        y = experts.expert_linear(h[order], self.up_w, offsets, self.up_b, activation='relu2')
        y = experts.expert_linear(y, self.down_w, offsets, self.down_b)
        y = torch.zeros_like(h).index_copy(0, order, y) * weight.to(x.dtype).unsqueeze(-1)
        return x + y.view_as(x)


class Model(nn.Module):
    def __init__(self, vocab, context, width, num_experts, blocks):
        super().__init__()
        self.embed = _weight(vocab, width)
        self.blocks = nn.ModuleList(Block(context, width, num_experts) for _ in range(blocks))
        self.head = _weight(vocab, width)

    def forward(self, tokens):
        x = self.embed[tokens]
        for block in self.blocks:
            x = block(x)
        return layers.residual_linear(F.layer_norm(x, (x.shape[-1],)), self.head)


def train(steps=100, batch=8, context=64, width=64, vocab=32, num_experts=4, blocks=1, state_bits=32,
          lr=3e-3, device=None, seed=0, log=None):
    """Train and return the loss of every step."""
    device = device or ('cuda' if torch.cuda.is_available() else 'cpu')
    torch.manual_seed(seed)
    dtype = torch.bfloat16 if device == 'cuda' else torch.float32
    model = Model(vocab, context, width, num_experts, blocks).to(device, dtype)
    opt = optim.AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.01,
                      state_bits=state_bits, master_weights=dtype != torch.float32, seed=seed)
    gen = torch.Generator().manual_seed(seed)
    follow = torch.randperm(vocab, generator=gen)
    losses = []
    for step in range(steps):
        seq = [torch.randint(0, vocab, (batch,), generator=gen)]
        for _ in range(context):
            seq.append(torch.where(torch.rand(batch, generator=gen) < 0.125,
                                   torch.randint(0, vocab, (batch,), generator=gen), follow[seq[-1]]))
        seq = torch.stack(seq, dim=1).to(device)
        logits = model(seq[:, :-1])
        loss = F.cross_entropy(logits.float().reshape(-1, vocab), seq[:, 1:].reshape(-1))
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if log and step % log == 0:
            print(f'step {step:4d}  loss {loss.item():.4f}', flush=True)
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--steps', type=int, default=100)
    ap.add_argument('--batch', type=int, default=8)
    ap.add_argument('--context', type=int, default=64)
    ap.add_argument('--width', type=int, default=64)
    ap.add_argument('--experts', type=int, default=4)
    ap.add_argument('--blocks', type=int, default=1)
    ap.add_argument('--state-bits', type=int, default=32, choices=(8, 32))
    ap.add_argument('--lr', type=float, default=3e-3)
    a = ap.parse_args()
    losses = train(a.steps, a.batch, a.context, a.width, num_experts=a.experts, blocks=a.blocks,
                   state_bits=a.state_bits, lr=a.lr, log=10)
    print(f'loss {losses[0]:.4f} -> {losses[-1]:.4f}')


if __name__ == '__main__':
    main()

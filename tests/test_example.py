"""The example runs the operators together and learns."""

import importlib.util
from pathlib import Path

import pytest
import torch

from avey_kernel_b200 import _native

PATH = Path(__file__).resolve().parents[1] / 'examples' / 'train_block.py'
spec = importlib.util.spec_from_file_location('train_block', PATH)
train_block = importlib.util.module_from_spec(spec)
spec.loader.exec_module(train_block)


@pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('bits', [32, 8])
def test_example_learns(bits, device):
    """One token in eight is random: the loss falls from above ln 32 = 3.5 to well
    below it (0.7 is the entropy of the sequences)."""
    losses = train_block.train(steps=60, batch=8, state_bits=bits, device=device)
    assert all(torch.isfinite(torch.tensor(losses)))
    assert losses[0] > 3.0 and sum(losses[-5:]) / 5 < 2.0
    if device == 'cuda':
        assert _native.device_status(clear=True) == 0

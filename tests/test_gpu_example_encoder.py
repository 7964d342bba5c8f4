"""examples/train_encoder.py: the network learns, in 8-bit states as in 32-bit
ones, and what it trains stays channels last with the states it should have."""
from __future__ import annotations

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _module():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_encoder
    finally:
        sys.path.pop(0)
    return train_encoder


@pytest.mark.gpu
def test_the_encoder_learns_with_8_and_32_bit_states():
    example = _module()
    last = {}
    for bits in (8, 32):
        print(f"[encoder] {bits}-bit states", flush=True)
        encoder, opt, losses = example.train(steps=60, size=64, batch=2, width=16, state_bits=bits)
        first, last[bits] = losses[:5].mean().item(), losses[-10:].mean().item()
        # A third of the loss at least is the discs' place and colour, which is
        # what there is to learn in so few steps.
        assert last[bits] < first * 2 / 3, (bits, first, last[bits])
        assert 0.0 < opt.grad_norm.item() < float("inf")
        big = encoder.blocks[3].conv2.weight
        assert ("exp_avg_8bit" in opt.state[big]) == (bits == 8)
        assert "exp_avg" in opt.state[encoder.norm.weight]
        assert big.is_contiguous(memory_format=torch.channels_last)
    # The rounding of the states is noise about the same path.
    assert abs(last[8] - last[32]) <= 0.15 * last[32], last


def test_the_encoders_shapes_without_a_gpu():
    """Its answers for an odd image size, with the norms replaced by torch's (they
    have the same parameters)."""
    example = _module()
    net = example.Encoder(width=8, per_cell=3)
    for name, m in list(net.named_modules()):
        if isinstance(m, example.GroupNorm):
            ref = torch.nn.GroupNorm(m.num_groups, m.num_channels)
            ref.load_state_dict(m.state_dict())
            parent = net.get_submodule(name.rpartition(".")[0])
            setattr(parent, name.rpartition(".")[2], ref)
    points, colours, opacities = net(torch.rand(2, 3, 70, 50))
    paths = 5 * 4 * 3
    assert points.shape == (2, paths, 10, 2)
    assert colours.shape == (2, paths, 3) and opacities.shape == (2, paths)

"""Pins of oracle/network64.py: the gradients of group norm against differences
and torch's float64 autograd, the AdamW step against torch's float64 one, and
the 8-bit states' rounding."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import network64 as O


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("groups,c", [(1, 3), (4, 4), (2, 6)])
def test_group_norm_against_torch_and_differences(act, groups, c):
    rng = np.random.default_rng(0)
    x, w, b = rng.normal(size=(2, c, 3, 5)), rng.normal(size=c), rng.normal(size=c)
    dy = rng.normal(size=x.shape)
    y, dx, dw, db = O.group_norm64(x, groups, w, b, act=act, dy=dy)
    t = [torch.from_numpy(a).requires_grad_(True) for a in (x, w, b)]
    z = torch.nn.functional.group_norm(t[0], groups, t[1], t[2], 1e-5)
    f = {None: lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu}[act]
    out = f(z)
    grads = torch.autograd.grad(out, t, torch.from_numpy(dy))
    for got, want in zip((y, dx, dw, db), (out, *grads)):
        assert np.allclose(got, want.detach().numpy(), rtol=1e-9, atol=1e-11)
    if act == "relu":
        return  # differences across the kink say nothing
    h = 1e-6
    for arr, grad, k in ((x, dx, 7), (x, dx, 31), (w, dw, 1), (b, db, 2)):
        vals = []
        for sign in (1, -1):
            moved = arr.copy()
            moved.ravel()[k] += sign * h
            args = [moved if a is arr else a for a in (x, w, b)]
            vals.append((O.group_norm64(args[0], groups, args[1], args[2], act=act) * dy).sum())
        # Central differences: h^2 times third derivatives and 1e-16 / h.
        assert abs((vals[0] - vals[1]) / (2 * h) - grad.ravel()[k]) <= 1e-6 * max(1, abs(grad.ravel()[k]))


def test_adamw_against_torch():
    rng = np.random.default_rng(1)
    p = torch.from_numpy(rng.normal(size=50)).requires_grad_(True)
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    m = v = np.zeros(50)
    for step in range(1, 5):
        g, old = rng.normal(size=50), p.detach().numpy().copy()
        p.grad = torch.from_numpy(g)
        opt.step()
        want, m, v = O.adamw_step64(old, g, m, v, step=step, lr=1e-2, betas=(0.8, 0.95), eps=1e-6,
                                    weight_decay=0.1)
        assert np.allclose(p.detach().numpy(), want, rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("mantissa", [3, 4])
def test_hold8_rounds_to_neighbours_without_bias(mantissa):
    rng = np.random.default_rng(2)
    x = rng.normal(size=BLOCKS * O.BLOCK) * np.exp2(rng.integers(-20, 3, size=BLOCKS * O.BLOCK))
    low, e = O.hold8(x, mantissa, 0)
    high, _ = O.hold8(x, mantissa, 65535)
    near, _ = O.hold8(x, mantissa, 0x8000)
    assert np.all(np.abs(low) <= np.abs(x)) and np.all(np.abs(high) >= np.abs(low))
    # The spacing in a value's binade, or in the least one.
    top = np.repeat(np.exp2(e - 127.0), O.BLOCK)
    spacing = np.exp2(np.maximum(np.floor(np.log2(np.abs(x))), np.log2(top) - 13) - mantissa)
    assert np.all(np.abs(x - low) <= spacing) and np.all(np.abs(near - x) <= spacing / 2 * 1.0001)
    # What is held is held again unchanged, however it is rounded.
    for r in (0, 0x8000, 65535):
        assert np.array_equal(O.hold8(low, mantissa, r)[0], low)
    # Over all 65536 random numbers the mean is the value, to the numbers' own
    # granularity.
    one = np.full(65536, 1.2345)
    mean = O.hold8(one, mantissa, np.arange(65536))[0].mean()
    assert abs(mean - 1.2345) <= 2.0 ** -mantissa / 65536


BLOCKS = 20


def test_hold8_zero_floor_and_values_that_are_not_finite():
    x = np.zeros(300)
    assert not O.hold8(x, 4, 65535, floor=True)[0].any()
    x[:4] = [1.0, 1e-30, np.inf, np.nan]
    got = O.hold8(x, 4, 0, floor=True)[0]
    assert got[0] == 1.0 and got[1] == 2.0 ** -17 and np.isnan(got[2:4]).all() and not got[4:].any()
    assert O.hold8(x, 4, 0)[0][1] == 0.0


def test_rounding_numbers_are_even_and_uncorrelated():
    """2^18 numbers in 256 cells: chi-square of 255 degrees of freedom has mean
    255 and deviation 22.6; neighbours, the two halves, steps and tensors are
    uncorrelated to 6 standard errors."""
    n = 1 << 18
    a, b = O.rounding_numbers(3, 17, 5, n)
    for r in (a, b):
        count = np.bincount(r >> 8, minlength=256)
        assert abs(((count - n / 256) ** 2 / (n / 256)).sum() - 255) <= 6 * 22.6
    others = [b, np.roll(a, 1), np.roll(a, 128), O.rounding_numbers(3, 18, 5, n)[0],
              O.rounding_numbers(3, 17, 6, n)[0], O.rounding_numbers(4, 17, 5, n)[0]]
    for o in others:
        assert abs(np.corrcoef(a, o)[0, 1]) <= 6 / np.sqrt(n)

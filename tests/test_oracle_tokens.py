"""The float64 restatements of Newton-Schulz steps, the Muon step, tokens'
log-probabilities and the policy loss (oracle/network64.py), pinned by torch's
float64, by singular values and by differences."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import network64 as O


@pytest.mark.parametrize("shape", [(5, 9), (9, 5), (4, 4), (1, 7), (2, 3, 6)])
def test_newton_schulz_acts_on_the_singular_values(shape):
    x = np.random.default_rng(0).standard_normal(shape)
    a, b, c = 3.4445, -4.7750, 2.0315
    u, s, vt = np.linalg.svd(x, full_matrices=False)
    s = s / np.sqrt((s * s).sum(-1, keepdims=True))
    for _ in range(3):
        s = a * s + b * s ** 3 + c * s ** 5
    np.testing.assert_allclose(O.newton_schulz64(x, 3), (u * s[..., None, :]) @ vt, atol=1e-12)


def test_muon_step_is_torchs():
    """torch.optim.Muon computes its products in bfloat16: the directions agree to that."""
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("this torch has no Muon")
    g = torch.Generator().manual_seed(1)
    for shape, adjust in (((24, 16), None), ((16, 24), "match_rms_adamw")):
        p = torch.nn.Parameter(torch.randn(shape, generator=g))
        opt = torch.optim.Muon([p], lr=0.1, weight_decay=0.1, adjust_lr_fn=adjust)
        want, m = p.detach().numpy(), np.zeros(shape)
        for _ in range(3):
            p.grad = torch.randn(shape, generator=g)
            want, m = O.muon_step64(want, p.grad.numpy(), m, lr=0.1, adjust=adjust)
            opt.step()
        np.testing.assert_allclose(opt.state[p]["momentum_buffer"].numpy(), m, atol=1e-6)
        moved = np.abs(p.detach().numpy() - want).max()
        assert moved < 0.1 * 3 * 0.1 * (1 if adjust is None else 0.2 * 24 ** 0.5), moved


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs_are_torchs(temperature):
    rng = np.random.default_rng(2)
    z = torch.tensor(rng.standard_normal((3, 4, 11)) * 3, requires_grad=True)
    tokens = torch.tensor(rng.integers(0, 11, (3, 4)))
    mask = torch.tensor(rng.random((3, 4)) < 0.7)
    up = torch.tensor(rng.standard_normal((3, 4)))
    lp = torch.log_softmax(z / temperature, -1).gather(-1, tokens[..., None])[..., 0] * mask
    dz, = torch.autograd.grad(lp, z, up)
    got = O.token_logprobs64(z.detach().numpy(), tokens.numpy(), mask.numpy(), temperature,
                             up.numpy())
    np.testing.assert_allclose(got[0], lp.detach().numpy(), atol=1e-13)
    np.testing.assert_allclose(got[1], dz.numpy(), atol=1e-13)


def test_policy_terms_by_differences_and_by_torch():
    rng = np.random.default_rng(3)
    lp, old, ref = rng.standard_normal((3, 400)) * 0.3 - 2.0
    adv = rng.standard_normal(400)
    kw = dict(clip=(0.2, 0.3), kl_weight=0.1)
    loss, slope, kl, clipped = O.policy_terms64(lp, old, adv, ref, **kw)
    h = 1e-6
    up, down = (O.policy_terms64(lp + s * h, old, adv, ref, **kw)[0] for s in (1, -1))
    far = (np.abs(np.exp(lp - old) - 0.8) > 1e-5) & (np.abs(np.exp(lp - old) - 1.3) > 1e-5)
    np.testing.assert_allclose(((up - down) / (2 * h))[far], slope[far], atol=1e-8)
    x = torch.tensor(lp, requires_grad=True)
    r = (x - torch.tensor(old)).exp()
    a, d = torch.tensor(adv), torch.tensor(ref) - x
    whole = -torch.minimum(r * a, r.clamp(0.8, 1.3) * a) + 0.1 * (d.exp() - d - 1)
    np.testing.assert_allclose(loss, whole.detach().numpy(), atol=1e-12)
    got, = torch.autograd.grad(whole.sum(), x)
    np.testing.assert_allclose(got.numpy()[far], slope[far], atol=1e-12)
    assert (kl >= 0).all() and 0 < clipped.mean() < 1


def test_policy_weights():
    mask = np.array([[1, 1, 0], [0, 0, 0], [0, 1, 0]], bool)
    np.testing.assert_allclose(O.policy_weights64(mask, "token"), mask / 3)
    np.testing.assert_allclose(O.policy_weights64(mask, "sequence"),
                               mask * np.array([[0.25], [0.0], [0.5]]))
    assert O.policy_weights64(mask * False, "token").sum() == 0
    assert O.policy_weights64(mask, "sum").sum() == 3

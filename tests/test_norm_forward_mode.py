"""Forward-mode derivatives of group_norm are refused, with and without the extension:
a result without a tangent would be a derivative of zero."""
from __future__ import annotations

from contextlib import nullcontext

import pytest
import torch
from torch.autograd import forward_ad


def _refused(device):
    from repo_amd.norm import group_norm
    for which in ("x", "weight", "bias"):
        for grad in (False, True):
            with forward_ad.dual_level():
                t = dict(x=torch.ones(2, 8, 3, 3, device=device),
                         weight=torch.ones(8, device=device), bias=torch.ones(8, device=device))
                t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
                with (nullcontext() if grad else torch.no_grad()):
                    with pytest.raises((RuntimeError, NotImplementedError), match="(?i)jvp"):
                        group_norm(t["x"], 2, t["weight"], t["bias"], activation="silu")
                # Nothing that has none is refused.
                plain = group_norm(torch.ones(2, 8, 3, 3, device=device), 2)
                assert forward_ad.unpack_dual(plain).tangent is None


def test_the_python_node_refuses_tangents(monkeypatch):
    """On host tensors, with the launch left out."""
    from repo_amd import _native as N
    from repo_amd import norm, torchcall
    monkeypatch.setattr(torchcall, "_MODULE", None)
    monkeypatch.setattr(N, "call", lambda name, *args: None)
    monkeypatch.setattr(N, "stream", lambda device=None: 0)
    monkeypatch.setattr(N, "require_gpu", lambda t, name: None)
    monkeypatch.setattr(norm, "_workspace_elems", lambda *args: 1)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None, raising=False)
    _refused("cpu")


@pytest.mark.gpu
def test_tangents_are_refused():
    from repo_amd import torchcall
    assert torchcall.module() is not None
    _refused("cuda")


@pytest.mark.gpu
def test_tangents_are_refused_without_the_extension(monkeypatch):
    from repo_amd import torchcall
    monkeypatch.setattr(torchcall, "_MODULE", None)
    _refused("cuda")

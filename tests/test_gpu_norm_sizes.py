"""repo_amd.norm.group_norm at sizes whose launches are of other forms: many samples
of many groups.  Tolerances as in test_gpu_norm."""
from __future__ import annotations

import os

import numpy as np
import pytest
import torch

import test_gpu_norm as T


def test_workspace_of_groups_with_nothing_to_join():
    """Each group's only partial result is read where it is applied: no launch in
    between, whose workgroups would be four groups each of all samples, and no
    room for what it would leave."""
    from repo_amd import _native as N
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")
    elems = N.lib().cs_group_norm_workspace_elems
    for n, s, c in ((32800, 3, 2048), (1 << 15, 4, 2048), (1 << 20, 1, 2048)):
        assert elems(n, s, c, c, 1, 0) == n * c * 2
        assert elems(n, s, c, c, 1, 1) == n * c * 4
    # Where there are several of each there is.
    assert elems(1, 4096, 2048, 2048, 1, 0) > 2048 * 4


def test_sizes_beyond_a_launch_are_refused():
    """On the host, before any launch (the addresses are not read)."""
    from repo_amd import _native as N
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("library not built (run __graft_entry__.build())")

    def forward(n, s, c, groups, dtype):
        return N.lib().cs_group_norm_forward(4096, n, s, c, groups, dtype, None, None, 0, 1e-5, 0,
                                             4096, None, None, 8192, None)

    def backward(n, s, c, groups, dtype):
        return N.lib().cs_group_norm_backward(4096, 8192, n, s, c, groups, dtype, None, None, 0, 0,
                                              4096, 4096, 4096, 4096, 4096, None, None)

    for run in (forward, backward):
        assert run((1 << 23) + 1, 4, 8, 8, 0) == N.CS_ERR_ARGS
        assert run((1 << 22) + 1, 1, 2048, 2048, 0) == N.CS_ERR_ARGS   # two slices in fp32
    assert backward(1, 64, 1 << 27, 1, 1) == N.CS_ERR_ARGS


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(32800, 2048, (3,), 2048), (33000, 1024, (4,), 512)],
                         ids=["32800x2048x3g2048", "33000x1024x4g512"])
def test_many_samples_of_many_groups(shape):
    """Samples are independent: the first, the middle and the last against float64; dw
    and db, sums over all of them, against float64 on the device."""
    n, c, space, groups = shape
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn((n, *space, c), generator=g, device="cuda").bfloat16().movedim(-1, 1)
    dy = torch.randn((n, *space, c), generator=g, device="cuda").bfloat16().movedim(-1, 1)
    w = (1 + 0.3 * torch.randn(c, generator=g, device="cuda")).bfloat16()
    b = (0.3 * torch.randn(c, generator=g, device="cuda")).bfloat16()
    y, dx, dw, db = T._run(x, w, b, dy, groups, None)
    for part in (slice(0, 8), slice(n // 2, n // 2 + 8), slice(n - 8, n)):
        T._check(x[part], w, b, dy[part], groups, None, y[part], dx[part])
    for k in range(0, n, 4096):   # every sample was computed
        assert not torch.isnan(dx[k:k + 4096]).any() and not torch.isnan(y[k:k + 4096]).any()
    ref_w, ref_b, sum_w, sum_b = (torch.zeros(c, dtype=torch.float64, device="cuda")
                                  for _ in range(4))
    for k in range(0, n, 1024):
        v = x[k:k + 1024].double().movedim(1, -1).reshape(-1, int(np.prod(space)), groups,
                                                          c // groups)
        mean = v.mean((1, 3), keepdim=True)
        r = 1 / torch.sqrt((v - mean).square().mean((1, 3), keepdim=True) + 1e-5)
        xh = ((v - mean) * r).reshape(-1, c)
        zs = (w.double().abs() * (xh.abs() + (mean.abs() * r).expand_as(v).reshape(-1, c) + 1)
              + b.double().abs())
        d = dy[k:k + 1024].double().movedim(1, -1).reshape(-1, c)
        ref_w += (d * xh).sum(0)
        ref_b += d.sum(0)
        sum_w += (d.abs() * (1 + zs) * (1 + xh.abs())).sum(0)
        sum_b += (d.abs() * (1 + zs)).sum(0)
    for got, ref, size in ((dw, ref_w, sum_w), (db, ref_b, sum_b)):
        err = (got.double() - ref).abs()
        assert bool((err <= 1.5 * T.K * T.U * size + 2.0 ** -8 * ref.abs()).all())

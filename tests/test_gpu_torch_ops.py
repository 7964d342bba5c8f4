"""The extension on torch's C++ tensors (repo_amd/csrc/torch_ops.cpp): what it does
is what the Python paths beside it do, bit for bit, and it refuses what it cannot
take."""
from __future__ import annotations

from contextlib import contextmanager

import numpy as np
import pytest
import torch


def _extension():
    from repo_amd import torchcall
    ext = torchcall.module()
    if ext is None:
        pytest.skip("extension not built (run __graft_entry__.build())")
    return ext


@pytest.mark.gpu
def test_the_extension_is_there():
    from repo_amd import torchcall
    assert torchcall.module() is not None


@pytest.mark.gpu
@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
@pytest.mark.parametrize("shape,groups", [((2, 24, 9, 7), 4), ((3, 10, 50), 5), ((6, 12), 3),
                                          ((1, 64, 70, 60), 16)])
def test_group_norm_with_and_without_it(shape, groups, affine):
    """A profiling factory brackets each launch from Python, which takes the
    Python node; labels and results."""
    from repo_amd import _native as N
    from repo_amd.norm import group_norm
    _extension()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g).cuda()
    w = torch.randn(shape[1], generator=g).cuda() if affine in ("both", "weight") else None
    b = torch.randn(shape[1], generator=g).cuda() if affine in ("both", "bias") else None
    dy = torch.randn(shape, generator=g).cuda()
    seen = []

    @contextmanager
    def factory(label):
        seen.append(label)
        yield

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b) if t is not None]
        it = iter(leaves)
        args = [None if t is None else next(it) for t in (x, w, b)]
        y = group_norm(args[0], groups, args[1], args[2], activation="silu")
        with torch.no_grad():
            z = group_norm(args[0], groups, args[1], args[2], activation="silu")
        return [y.detach(), z, *torch.autograd.grad(y, leaves, dy)]

    got = run()
    assert not seen
    N.set_profile_ctx_factory(factory)
    try:
        want = run()
    finally:
        N.set_profile_ctx_factory(None)
    assert seen == ["norm.fwd", "norm.fwd", "norm.bwd"]
    assert len(got) == len(want)
    for p, q in zip(got, want):
        assert torch.equal(p, q) and p.stride() == q.stride()


@pytest.mark.gpu
@pytest.mark.parametrize("need", ["x", "w", "b", "wb"])
@pytest.mark.parametrize("absent", ["", "w", "b"])
def test_group_norm_partial_gradients(need, absent):
    from repo_amd.norm import group_norm
    if set(need) & set(absent):
        return
    g = torch.Generator().manual_seed(2)
    t = dict(x=torch.randn(2, 8, 5, 5, generator=g).cuda(), w=torch.randn(8, generator=g).cuda(),
             b=torch.randn(8, generator=g).cuda())
    full = {k: v.clone().requires_grad_(True) for k, v in t.items() if k not in absent}
    part = {k: v.clone().requires_grad_(k in need) for k, v in t.items() if k not in absent}
    for d in (full, part):
        group_norm(d["x"], 2, d.get("w"), d.get("b"), activation="gelu").square().sum().backward()
    for k, v in part.items():
        assert (v.grad is not None) == (k in need)
        if k in need:
            assert torch.equal(v.grad, full[k].grad)


@pytest.mark.gpu
def test_group_norm_second_derivative_is_refused_not_dropped():
    from repo_amd.norm import group_norm
    x = torch.randn(2, 8, 5, 5, device="cuda", requires_grad=True)
    w = torch.randn(8, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(group_norm(x, 2, w, activation="silu").sum(), (x, w),
                                 create_graph=True)
    assert gx.requires_grad and gw.requires_grad
    with pytest.raises(RuntimeError, match="once"):
        # With a term of its own, so that a dropped one would go unnoticed.
        (gx.square().sum() + x.sum()).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_with_and_without_it(state_bits, dtype, monkeypatch):
    from repo_amd import torchcall
    from repo_amd.optim import AdamW
    _extension()

    def run():
        g = torch.Generator().manual_seed(3)
        ps = [torch.randn(s, generator=g).to(dtype).cuda().requires_grad_(True)
              for s in ((5000,), (33, 7), (4096,), (1,))]
        opt = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2, "weight_decay": 0.0}],
                    state_bits=state_bits, max_grad_norm=0.5, seed=4)
        for step in range(5):
            for k, p in enumerate(ps):
                p.grad = torch.randn(p.shape, generator=g).to(dtype).cuda()
                if step == 2 and k == 1:
                    p.grad = None   # from here on the step counts differ
            opt.step()
        return [p.detach() for p in ps] + [*opt.flat_state(), opt.grad_norm.clone()] + [
            opt.state[p]["step"] for p in ps]

    got = run()
    monkeypatch.setattr(torchcall, "_MODULE", None)
    want = run()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
def test_adamw_notices_what_changes_between_steps():
    """Each change takes the step out of the quick path and is honoured."""
    from repo_amd.optim import AdamW
    _extension()
    p, q = (torch.ones(64, 4, device="cuda", requires_grad=True) for _ in range(2))
    opt = AdamW([p, q], lr=0.1, weight_decay=0.0)

    def grads():
        for t in (p, q):
            t.grad = torch.ones_like(t)

    def moved(t, by=0.1):
        return torch.allclose(t.detach(), t_old[id(t)] - by, atol=1e-4)

    changes = [
        lambda: None, lambda: None,
        lambda: setattr(p, "data", p.detach().clone()),
        lambda: setattr(p, "grad", torch.ones(4, 64, device="cuda").t()),
        lambda: setattr(p, "grad", torch.ones((), device="cuda").expand(64, 4)),
        lambda: opt.state[q].update(exp_avg=opt.state[q]["exp_avg"].clone()),
        lambda: opt.state[q].update(step=opt.state[q]["step"].clone()),
        lambda: opt.load_state_dict(opt.state_dict()),
        lambda: setattr(p.grad, "data", torch.ones(64, 4, device="cuda")),
    ]
    for k, change in enumerate(changes):
        grads()
        change()
        t_old = {id(t): t.detach().clone() for t in (p, q)}
        opt.step()
        assert moved(p) and moved(q), k
        assert float(opt.state[p]["step"]) == float(opt.state[q]["step"]) == k + 1
    grads()
    q.grad = None
    t_old = {id(t): t.detach().clone() for t in (p, q)}
    opt.step()
    assert moved(p) and moved(q, 0.0)
    grads()
    p.grad.data = torch.ones(10, device="cuda")
    with pytest.raises(ValueError, match="a gradient of"):
        opt.step()
    grads()
    q.grad = torch.ones(64, 4, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_copied_optimizer_goes_on_by_itself(state_bits):
    """copy.deepcopy and pickle of an optimizer with its parameters: the copy takes
    the same steps, and neither moves the other's parameters."""
    import copy
    import pickle
    from repo_amd.optim import AdamW
    g = torch.Generator().manual_seed(5)
    ps = [torch.randn(s, generator=g).cuda().requires_grad_(True) for s in ((5000,), (40, 3))]
    opt = AdamW(ps, state_bits=state_bits, seed=6, max_grad_norm=1.0)

    def step(o):
        for group in o.param_groups:
            for k, p in enumerate(group["params"]):
                p.grad = torch.full_like(p, 0.01 * (k + 1))
        o.step()
        return [p.detach().clone() for group in o.param_groups for p in group["params"]]

    step(opt)
    step(opt)
    for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (twin.state_bits, twin.seed, twin.max_grad_norm) == (state_bits, 6, 1.0)
        before = [p.detach().clone() for p in ps]
        a = [step(twin) for _ in range(2)]
        assert all(torch.equal(p.detach(), q) for p, q in zip(ps, before))
        kept = copy.deepcopy(opt)
        b = [step(kept) for _ in range(2)]
        assert all(torch.equal(p, q) for x, y in zip(a, b) for p, q in zip(x, y))


def test_it_refuses_arguments():
    ext = _extension()
    x = torch.zeros(2, 8, 3, 3)
    with pytest.raises(TypeError):
        ext.group_norm(x, None, None, 2, 1e-5)
    with pytest.raises(TypeError):
        ext.group_norm(None, None, None, 2, 1e-5, 0)
    with pytest.raises(TypeError):
        ext.group_norm(x, 3, None, 2, 1e-5, 0)
    with pytest.raises(TypeError):
        ext.group_norm(x, None, None, "2", 1e-5, 0)
    with pytest.raises(ValueError, match="on the GPU"):
        ext.group_norm(x, None, None, 2, 1e-5, 0)
    with pytest.raises(TypeError):
        ext.adamw_current([x], [], [], [], 0, 0, False)
    with pytest.raises(TypeError):
        ext.adamw_current([x], [None], [()], [()], 0, 0, False)
    with pytest.raises(TypeError):
        ext.adamw_count(0, 0)


def test_adamw_current_on_host_tensors():
    """The checks read only tensors' properties, so they run on any device."""
    ext = _extension()
    p = torch.zeros(6, requires_grad=True)
    p.grad = torch.ones(6)
    st = {"a": torch.zeros(6), "step": torch.tensor(3.0)}
    table = np.array([[p.data_ptr(), 0, 0, 0, 0, 6, 16 | 1 << 8, 0]], np.int64)
    steps = np.array([st["step"].data_ptr()], np.int64)

    def now(gradients=True, keys=("a", "step"), held=None):
        held = tuple(st[k] for k in keys) if held is None else held
        return ext.adamw_current([p], [st], [keys], [held], table.ctypes.data, steps.ctypes.data,
                                 gradients)

    assert now() == 3.0 and table[0, 1] == p.grad.data_ptr()
    assert now(False) == 0.0
    assert now(held=(torch.zeros(6), st["step"])) == -1.0
    assert now(keys=("b",), held=(st["a"],)) == -1.0
    for col, value in ((0, 8), (5, 7), (6, 1)):
        kept = table[0, col]
        table[0, col] = value
        assert now() == -1.0 and now(False) == -1.0
        table[0, col] = kept
    for grad in (None, torch.ones(12)[::2], torch.ones(6).to_sparse()):
        p.grad = grad
        assert now() == -1.0 and now(False) == 0.0
    ext.adamw_count(steps.ctypes.data, 1, 9.0)
    assert float(st["step"]) == 9.0
    assert ext.adamw_current([], [], [], [], 0, 0, True) == 0.0

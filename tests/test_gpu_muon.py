"""repo_amd.optim's orthogonalize and Muon against float64 (oracle/network64.py): types, shapes
from one value to several tiles, odd sizes, both orientations, stacks, layouts, spectra, scales,
values that are not finite, other steps and coefficients, masters, streams and graphs.

Tolerance.  The steps amplify roundings by the input's spectrum, so the measure is the same steps
in numpy's float32 on the same input, E = |float32 - float64| (Frobenius).  There an element of a
product has operands as they are and a sum's roundings.  Here operands carry 2^-24 each (two
halves), what is left out of a product 2^-24 more: 4 roundings for 1.  Phases of several steps
make 1.4 of it: 5.6, taken as 8.  Where both are exact (one value) 32 roundings of each value of
the result remain: 32 2^-24 |result|.  A 16-bit result adds half a step of its type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import network64 as O

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [
    (1, 1), (1, 2), (2, 1), (1, 700), (700, 1), (2, 3), (5, 5), (31, 33), (63, 64), (64, 65),
    (96, 97), (127, 127), (128, 128), (129, 128), (128, 129), (130, 131), (64, 576), (576, 64),
    (40, 3001), (3001, 40), (32, 256), (33, 257), (16, 500), (700, 20), (31, 1030), (2048, 30),
    (2049, 30), (64, 512), (60, 768), (64, 769), (1024, 64), (64, 1025), (96, 256), (96, 257), (512, 90),
    (96, 513), (97, 96), (255, 257), (256, 512), (300, 1000), (1000, 130), (513, 520), (641, 2000),
]


def _np(t):
    return t.detach().double().cpu().numpy()


def newton_schulz32(x, steps, coefficients, eps):
    """The steps in numpy's float32."""
    x = np.asarray(x, np.float32)
    if x.shape[-2] > x.shape[-1]:
        return np.swapaxes(newton_schulz32(np.swapaxes(x, -1, -2), steps, coefficients, eps), -1, -2)
    a, b, c = (np.float32(v) for v in coefficients)
    norm = np.sqrt((x.astype(np.float64) ** 2).sum((-1, -2), keepdims=True))
    x = (x / np.maximum(norm, eps)).astype(np.float32)
    for _ in range(steps):
        g = x @ np.swapaxes(x, -1, -2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _bounds(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """The result in float64 and how far (Frobenius, each matrix) it may be off."""
    ref = O.newton_schulz64(x, steps, coefficients, eps)
    plain = newton_schulz32(x, steps, coefficients, eps).astype(np.float64)
    size = np.sqrt((ref ** 2).sum((-1, -2)))
    return ref, 8 * np.sqrt(((plain - ref) ** 2).sum((-1, -2))) + 32 * U * size, size


def _check(x, y, **kw):
    assert y.dtype is x.dtype and y.shape == x.shape and y.device == x.device
    ref, bound, size = _bounds(_np(x), **kw)
    off = np.sqrt(((_np(y) - ref) ** 2).sum((-1, -2)))
    least = (2.0 ** -25 if x.dtype is torch.float16 else 0.0) * np.sqrt(x.shape[-1] * x.shape[-2])
    assert np.all(off <= bound * (1 + HALF[x.dtype]) + HALF[x.dtype] * size + least), \
        (off / (bound + HALF[x.dtype] * size + 1e-300)).max()


def _random(shape, dtype=torch.float32, seed=0, kind="noise", by=1e-3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    m, n = shape[-2:]
    if kind != "noise":
        k = torch.arange(1, min(m, n) + 1).float()
        s = {"slow": 1 / k, "fast": 1 / k ** 2, "one": (k == 1).float(),
             "flat": torch.ones_like(k)}[kind]
        u, _, v = torch.linalg.svd(x, full_matrices=False)
        x = (u * s) @ v
    return (x * by).to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_matches_float64(shape, dtype):
    from repo_amd.optim import orthogonalize
    x = _random(shape, DTYPES[dtype], seed=shape[0])
    kept = x.clone()
    _check(x, orthogonalize(x))
    assert torch.equal(x, kept)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["slow", "fast", "one", "flat"])
@pytest.mark.parametrize("shape", [(150, 150), (140, 1300), (500, 60)])
def test_spectra(shape, kind):
    from repo_amd.optim import orthogonalize
    x = _random(shape, kind=kind, seed=3)
    _check(x, orthogonalize(x))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 9])
@pytest.mark.parametrize("coefficients", [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0),
                                          (1.875, -1.25, 0.375), (1.0, 0.0, 0.0)])
def test_steps_and_coefficients(steps, coefficients):
    from repo_amd.optim import orthogonalize
    for shape in ((70, 80), (100, 900)):
        x = _random(shape, seed=steps)
        _check(x, orthogonalize(x, steps, coefficients), steps=steps, coefficients=coefficients)


@pytest.mark.gpu
def test_many_plain_steps_end_in_the_orthogonal_factor():
    from repo_amd.optim import orthogonalize
    x = _random((90, 200), kind="flat")
    y = orthogonalize(x, 30, (1.5, -0.5, 0.0)).double()
    assert float((y @ y.mT - torch.eye(90, device="cuda").double()).abs().max()) < 1e-5
    u, _, v = torch.linalg.svd(x.double(), full_matrices=False)
    assert float((y - u @ v).abs().max()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(24, 96, 97), (3, 2, 130, 60), (5, 1, 1), (300, 3, 5), (2, 64, 700)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_stacks(shape, dtype):
    from repo_amd.optim import orthogonalize
    x = _random(shape, DTYPES[dtype], seed=5)
    x = x * (10.0 ** torch.arange(-2, x.shape[0] - 2).clamp(max=3).float().cuda()).view(
        -1, *(1,) * (x.dim() - 1)).to(x.dtype)
    y = orthogonalize(x)
    _check(x, y)
    flat, out = x.flatten(0, -3), y.flatten(0, -3)
    for k in (0, len(flat) // 2, len(flat) - 1):   # by itself a matrix's sums may be cut otherwise
        _check(flat[k], orthogonalize(flat[k]))
        _check(flat[k], out[k])


@pytest.mark.gpu
def test_more_matrices_than_a_call_takes():
    """16384 of up to 256 x 256 are as many as a call may have."""
    from repo_amd.optim import orthogonalize
    for shape in ((20000, 2, 3), (16400, 100, 40)):
        x = _random(shape, torch.bfloat16, seed=11)
        y = orthogonalize(x)
        for k in (0, 16383, 16384, shape[0] - 1):
            _check(x[k], y[k])


@pytest.mark.gpu
def test_layouts():
    from repo_amd.optim import orthogonalize
    wide = _random((5, 140, 150), seed=6)
    want = orthogonalize(wide[:, 3:133, 7:].contiguous())
    assert torch.equal(orthogonalize(wide[:, 3:133, 7:]), want)
    t = wide.mT
    y = orthogonalize(t)
    assert y.stride() == t.stride() and torch.equal(y, orthogonalize(wide).mT)
    _check(wide[1:2].expand(3, -1, -1), orthogonalize(wide[1:2].expand(3, -1, -1)))
    _check(wide.permute(1, 0, 2), orthogonalize(wide.permute(1, 0, 2)))
    off = _random((1, 65 * 66 + 1), torch.bfloat16)[0, 1:].view(65, 66)   # off 4 bytes
    _check(off, orthogonalize(off))


@pytest.mark.gpu
def test_scales_zeros_and_eps():
    from repo_amd.optim import orthogonalize
    x = _random((60, 130), by=1.0, seed=7)
    y = orthogonalize(x, eps=0.0)
    for by in (2.0 ** 100, 2.0 ** -60, 2.0 ** -100):
        assert torch.equal(orthogonalize(x * by, eps=0.0), y)
    assert torch.isnan(orthogonalize(torch.zeros(3, 4, device="cuda"), eps=0.0)).all()
    assert not orthogonalize(torch.zeros(3, 4, device="cuda")).any()
    # Where eps is the scale, values below 2^-25 of the halves' scale (2^13) are cut: 2^-38 an
    # element, once a step, and a step makes at most 3.4445 of what is there.
    small = x * 2.0 ** -60
    ref = O.newton_schulz64(_np(small))
    cut = sum(3.4445 ** k for k in range(1, 6)) * 2.0 ** -38
    assert np.abs(_np(orthogonalize(small)) - ref).max() <= cut
    _check(x, orthogonalize(x, eps=100.0), eps=100.0)


@pytest.mark.gpu
def test_no_matrices():
    from repo_amd.optim import orthogonalize
    for shape in ((0, 3), (3, 0), (0, 4, 5), (2, 0, 5)):
        assert orthogonalize(torch.zeros(shape, device="cuda")).shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_values_that_are_not_finite_stay_in_their_matrix(bad):
    from repo_amd.optim import orthogonalize
    for shape in ((4, 70, 200), (4, 200, 200)):
        x = _random(shape, seed=8)
        want = orthogonalize(x)   # a stack of the same sizes: the same sums
        x[1, 3, 5] = bad
        y = orthogonalize(x)
        assert torch.isnan(y[1]).any()
        for k in (0, 2, 3):
            assert torch.equal(y[k], want[k])


# ------------------------------------------------------------------------------- Muon


MIXED = [(70, 5, 3, 3), (64, 3, 7, 7), (300, 64), (64, 300), (1, 9), (9, 1), (40, 40, 1, 1), (2, 2)]


def _params(shapes, dtype, seed=0, layout=None):
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape in shapes:
        t = (0.05 * torch.randn(shape, generator=g)).to(dtype).cuda()
        if layout is not None:
            t = layout(t)
        out.append(torch.nn.Parameter(t))
    return out


def _grads(params, seed):
    g = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = torch.empty_like(p).copy_((1e-3 * torch.randn(p.shape, generator=g)).to(p.dtype))


def _check_steps(params, opt, steps=3, seed=1, order=None, **kw):
    """Steps of `opt` against float64, each from the state that the one before left."""
    args = dict(lr=0.02, weight_decay=0.1, momentum=0.95, nesterov=True, adjust=None)
    args.update(kw)
    for step in range(steps):
        _grads(params, seed + step)
        before = []
        for p in params:
            st = opt.state[p]
            w = st.get("master", p) if p.dtype is not torch.float32 else p
            m = st.get("momentum_buffer")
            before.append((_np(w), np.zeros(p.shape) if m is None else _np(m)))
        opt.step()
        for p, (w, m) in zip(params, before):
            g, st = _np(p.grad), opt.state[p]
            want, moved = O.muon_step64(w, g, m, **args)
            size = np.abs(m) + np.abs(g)
            assert np.all(np.abs(_np(st["momentum_buffer"]) - moved) <= 4 * U * size)
            u = (g + args["momentum"] * (moved - g) if args["nesterov"] else moved).reshape(p.shape[0], -1)
            rows, cols = u.shape
            _, bound, osize = _bounds(u)
            by = args["lr"] * (0.2 * max(rows, cols) ** 0.5 if args["adjust"] else max(1, rows / cols) ** 0.5)
            # u itself is rounded: 6 u (|m| + |g|), through steps that make at most 485 of it in
            # directions that the norm of one leaves small.
            spread = 6 * U * np.sqrt((size ** 2).sum()) / max(np.sqrt((u ** 2).sum()), 1e-7) * 4 * osize
            held = st["master"] if p.dtype is not torch.float32 else p
            off = np.sqrt(((_np(held) - want) ** 2).sum())
            assert off <= by * (bound + spread) + 4 * U * np.sqrt((want ** 2).sum()) + 4 * U * by * osize, \
                (tuple(p.shape), off)
            if p.dtype is not torch.float32:
                assert torch.equal(p, st["master"].to(p.dtype))
                assert st["master"].dtype is torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_steps_match_float64(dtype):
    from repo_amd.optim import Muon
    params = _params(MIXED, DTYPES[dtype])
    _check_steps(params, Muon(params, lr=0.02))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(nesterov=False), dict(momentum=0.0), dict(weight_decay=0.0),
                                dict(adjust="match_rms_adamw"), dict(lr=0.0)])
def test_options(kw):
    from repo_amd.optim import Muon
    params = _params(MIXED[:4], torch.float32)
    names = {"adjust": "adjust_lr_fn"}
    opt = Muon(params, **{"lr": 0.02, **{names.get(k, k): v for k, v in kw.items()}})
    _check_steps(params, opt, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layouts_of_parameters(dtype):
    from repo_amd.optim import Muon
    last = lambda t: t.contiguous(memory_format=torch.channels_last) if t.dim() == 4 else t.t().contiguous().t()  # noqa: E731
    params = _params(MIXED, DTYPES[dtype], layout=last)
    _check_steps(params, Muon(params, lr=0.02))
    # Gradients of another layout than their parameter's.
    params = _params([(33, 20, 3, 3), (50, 60)], DTYPES[dtype], seed=4)
    ours, theirs = (_params([(33, 20, 3, 3), (50, 60)], DTYPES[dtype], seed=4) for _ in range(2))
    a, b = Muon(ours, lr=0.02), Muon(theirs, lr=0.02)
    for _ in range(2):
        _grads(ours, 9)
        for p, q in zip(ours, theirs):
            q.grad = last(p.grad)
        a.step(), b.step()
    for p, q in zip(ours, theirs):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_refused_parameters_and_states():
    from repo_amd.optim import Muon
    base = torch.zeros(4, 5, 6, device="cuda")
    bad = [base.permute(1, 0, 2), base[:, :, :3], base.double()]
    for t in bad:
        p = torch.nn.Parameter(t)
        good = torch.nn.Parameter(torch.ones(3, 3, device="cuda"))
        opt = Muon([good, p], lr=1.0)
        good.grad, p.grad = torch.ones_like(good), torch.zeros_like(p)
        with pytest.raises(ValueError):
            opt.step()
        assert bool((good == 1).all())     # nothing was launched
    p = torch.nn.Parameter(torch.zeros(4, 5, device="cuda"))
    opt = Muon([p])
    p.grad = torch.zeros_like(p)
    opt.state[p]["momentum_buffer"] = torch.zeros(4, 5, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="does not fit"):
        opt.step()
    opt.state[p]["momentum_buffer"] = torch.zeros(5, 4, device="cuda").t()
    with pytest.raises(ValueError, match="does not fit"):
        opt.step()
    p.grad = torch.zeros(4, 5, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()


@pytest.mark.gpu
def test_more_parameters_than_a_launch_takes():
    from repo_amd.optim import Muon
    shapes = [(3 + k % 7, 2 + k) for k in range(45)] + [(0, 4), (4, 0)]
    params = _params(shapes, torch.float32, seed=2)
    _check_steps(params[:45], Muon(params, lr=0.02))


@pytest.mark.gpu
def test_groups_missing_gradients_and_hooks():
    from repo_amd.optim import Muon
    params = _params([(20, 30), (30, 20), (40, 10)], torch.bfloat16)
    opt = Muon([{"params": params[:1], "lr": 0.1, "ns_steps": 3}, {"params": params[1:]}], lr=0.02)
    _grads(params, 0)
    params[2].grad = None
    kept = params[2].clone()
    seen = []
    opt.register_step_pre_hook(lambda *_: seen.append("pre"))
    opt.register_step_post_hook(lambda *_: seen.append("post"))
    versions = [p._version for p in params]
    assert opt.step(lambda: 5.0) == 5.0 and seen == ["pre", "post"]
    assert torch.equal(params[2], kept) and params[2] not in opt.state
    assert params[0]._version > versions[0] and params[2]._version == versions[2]
    want, _ = O.muon_step64(np.zeros((20, 30)), _np(params[0].grad), np.zeros((20, 30)), lr=0.1, steps=3)
    other, _ = O.muon_step64(np.zeros((20, 30)), _np(params[0].grad), np.zeros((20, 30)), lr=0.1, steps=5)
    start = _np(_params([(20, 30)], torch.bfloat16)[0])
    moved = _np(opt.state[params[0]]["master"]) - start * (1 - 0.1 * 0.1)
    assert np.abs(moved - want).max() < 1e-5 < np.abs(moved - other).max()
    opt.zero_grad()
    assert all(p.grad is None for p in params)


@pytest.mark.gpu
def test_masters_follow_writes_and_checkpoints():
    from repo_amd.optim import Muon
    shapes = [(20, 30), (30, 20)]
    params = _params(shapes, torch.bfloat16)
    opt = Muon(params, lr=0.02)
    _check_steps(params, opt, steps=2)
    with torch.no_grad():
        params[0].mul_(2.0)                   # a write that autograd counts
    _grads(params, 7)
    twice = params[0].detach().float()
    kept = opt.state[params[1]]["master"].clone()
    opt.param_groups[0]["lr"] = 0.0
    opt.step()
    assert torch.equal(opt.state[params[0]]["master"], twice)
    assert torch.equal(opt.state[params[1]]["master"], kept)
    # A checkpoint goes on bit for bit, masters and all.
    opt.param_groups[0]["lr"] = 0.02
    sd = opt.state_dict()
    again = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = Muon(again, lr=1.0)
    other.load_state_dict(sd)
    for step in range(2):
        _grads(params, 20 + step)
        for p, q in zip(params, again):
            q.grad = p.grad.clone()
        opt.step(), other.step()
    for p, q in zip(params, again):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], other.state[q]["master"])


@pytest.mark.gpu
def test_results_repeat_and_streams():
    from repo_amd.optim import Muon, orthogonalize
    x = _random((3, 300, 200), torch.bfloat16, seed=9)
    y = orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)
    runs = []
    for _ in range(2):
        params = _params(MIXED, torch.bfloat16)
        opt = Muon(params, lr=0.02)
        for step in range(3):
            _grads(params, step)
            opt.step()
        runs.append([p.detach().clone() for p in params])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_graphs_follow_their_inputs():
    from repo_amd.optim import Muon, orthogonalize
    xs = [_random((2, 130, 300), torch.bfloat16, seed=s) for s in range(3)]
    want = [orthogonalize(x) for x in xs]
    graphs = []
    for _ in range(2):
        held = xs[0].clone()
        orthogonalize(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(held)
        graphs.append((graph, held, out))
    for first, second in ((0, 1), (2, 0), (1, 2), (1, 1)):
        for (graph, held, _), k in zip(graphs, (first, second)):
            held.copy_(xs[k])
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), k in zip(graphs, (first, second)):
            assert torch.equal(out, want[k])
    # A captured step: replays are steps.
    eager, captured = (_params(MIXED, torch.bfloat16) for _ in range(2))
    a, b = Muon(eager, lr=0.02), Muon(captured, lr=0.02)
    _grads(eager, 0), _grads(captured, 0)
    a.step(), b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for step in range(1, 4):
        _grads(eager, step)
        for p, q in zip(eager, captured):
            q.grad.copy_(p.grad)
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager, captured):
            assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_captured_step_makes_no_states(dtype, monkeypatch):
    """They would be made anew, momentum zero, in each replay."""
    from repo_amd.optim import Muon
    p = _random((70, 90), DTYPES[dtype]).requires_grad_()
    p.grad = _random((70, 90), DTYPES[dtype], seed=1)
    opt = Muon([p])
    kept = p.detach().clone()
    with monkeypatch.context() as m:
        m.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
        with pytest.raises(RuntimeError, match="make one step before"):
            opt.step()
    assert torch.equal(p, kept)
    opt.step()
    assert not torch.equal(p, kept)


@pytest.mark.gpu
def test_profile_labels():
    from contextlib import contextmanager
    from repo_amd import _native as N
    from repo_amd.optim import Muon, orthogonalize
    seen = []

    @contextmanager
    def factory(label):
        seen.append(label)
        yield
    N.set_profile_ctx_factory(factory)
    try:
        orthogonalize(torch.ones(3, 4, device="cuda"))
        params = _params([(3, 4)], torch.float32)
        _grads(params, 0)
        Muon(params).step()
    finally:
        N.set_profile_ctx_factory(None)
    assert seen == ["optim.orthogonalize", "optim.muon"]


@pytest.mark.gpu
def test_sparse_gradients_are_refused_by_name():
    from repo_amd.optim import Muon
    p = torch.nn.Parameter(torch.ones(4, 3, device="cuda"))
    opt = Muon([p])
    p.grad = torch.ones(4, 3, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="Muon does not support sparse gradients"):
        opt.step()
    assert torch.equal(p.detach(), torch.ones(4, 3, device="cuda"))


@pytest.mark.gpu
def test_copies_notice_writes_before_their_first_step():
    import copy
    import pickle
    from repo_amd.optim import Muon
    params = _params([(20, 30), (30, 20)], torch.bfloat16)
    opt = Muon(params, lr=0.0)
    _grads(params, 3)
    opt.step()
    for copied in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        p, q = copied.param_groups[0]["params"]
        with torch.no_grad():
            p.add_(1.0)
        want, kept = p.detach().clone(), copied.state[q]["master"].clone()
        _grads([p, q], 4)
        copied.param_groups[0]["weight_decay"] = 0.0
        copied.step()
        assert torch.equal(p, want) and torch.equal(copied.state[p]["master"], want.float())
        assert torch.equal(copied.state[q]["master"], kept)

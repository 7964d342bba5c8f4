"""repo_amd.policy: log-probabilities of tokens and the policy loss, and their gradients,
against float64 (oracle/network64.py): types, vocabularies of one to long ones, odd
sizes, strides, masks that leave a row or everything out, values that are not finite,
tokens outside the vocabulary, extreme ratios, other streams, graphs, far offsets.

Tolerances, with u = 2^-24.  A term 2^(z k - c) of the sum has a relative error of at most
  2 u |z - c| / T  (its argument's roundings) + 3 u  (the hardware's exponential, 1 ulp),
rescaled at most 40 times (2 u each) and added at most V / 64 + 40 times (u each); k is
rounded, which stands for another temperature: u (max z - min z) / T.  With R = (max z -
min z) / T over the finite logits
  |l error| <= u (2 R + V / 64 + 130 + |l|) =: e   (l is rounded to fp32 at the end)
A gradient element slope (delta - p) / T then is off by at most
  |slope| / T (e (delta + p) + 8 u (delta + p)) + |slope error| (delta + p) / T
and half a step of its type.  The slopes' errors: |A| r e + beta exp(d) e + 4 u |slope|."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import network64 as O

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Half a step: eps / 2 relative (bf16: 8 significant bits, eps 2^-7, so 2^-8), or half the least value.
HALF = {torch.float32: (2.0 ** -24, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
        torch.float16: (2.0 ** -11, 2.0 ** -25)}
# (tokens' shape, vocabulary)
SHAPES = [
    ((), 7), ((1,), 1), ((3,), 2), ((2, 3), 3), ((5, 7), 8), ((1, 1), 9), ((2, 2), 63), ((2, 2), 64),
    ((3, 2), 65), ((2, 3), 255), ((3, 5), 257), ((12, 33), 515), ((4, 9), 1037), ((2, 2, 3), 1024),
    ((2, 3), 2047), ((2, 3), 2048), ((2, 3), 2049), ((1, 3), 4097), ((3, 3), 8192), ((2, 3), 8200),
    ((1, 5), 16384), ((1, 3), 16391), ((2, 3), 20011), ((1, 3), 25003), ((1, 3), 32768), ((2, 2), 32771), ((1, 2), 65536),
    ((1, 2), 65543), ((1, 2), 131072), ((1, 2), 131075), ((1, 2), 200001), ((300, 2), 40),
]


@pytest.fixture(scope="module", autouse=True)
def _memory_given_back():
    """The tests behind these find the allocator as they would without them."""
    yield
    if torch.cuda.is_available():
        torch.cuda.synchronize()
        torch.cuda.empty_cache()


def _np(t):
    return t.detach().double().cpu().numpy()


def _inputs(shape, vocab, dtype, seed=0, spread=3.0, keep=0.75):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((*shape, vocab), generator=g) * spread
    tokens = torch.randint(0, vocab, shape, generator=g)
    z.scatter_add_(-1, tokens.unsqueeze(-1), 4 * torch.rand((*shape, 1), generator=g))
    mask = torch.rand(shape, generator=g) < keep
    up = torch.randn(shape, generator=g)
    return z.to(dtype).cuda(), tokens.cuda(), mask.cuda(), up.cuda()


def _lp_bound(z, lp, temperature):
    Z = _np(z)
    fin = np.isfinite(Z)
    r = (np.where(fin, Z, -np.inf).max(-1) - np.where(fin, Z, np.inf).min(-1)) / temperature
    return U * (2 * np.maximum(r, 0) + Z.shape[-1] / 64 + 130 + np.abs(lp))


def _check_grad(got, z, tokens, slope, slope_err, lp, temperature):
    """slope [...] of the log-probabilities (0 where masked)."""
    Z = _np(z) / temperature
    with np.errstate(invalid="ignore"):
        p = np.exp(Z - Z.max(-1, keepdims=True))
        p = p / p.sum(-1, keepdims=True)
    d = np.zeros_like(p)
    np.put_along_axis(d, tokens.cpu().numpy()[..., None], 1.0, -1)
    ref = np.where(slope[..., None] == 0, 0.0, slope[..., None] * (d - p) / temperature)
    e = _lp_bound(z, lp, temperature) + 8 * U
    rel, least = HALF[got.dtype]
    bound = ((np.abs(slope) * e + slope_err)[..., None] * (d + p) / temperature * (1 + rel)
             + rel * np.abs(ref) + least)
    bound = np.where(slope[..., None] == 0, 0.0, bound)
    err = np.abs(_np(got) - ref)
    assert np.all(err <= bound), float((err / np.maximum(bound, 1e-300)).max())


def _check_logprobs(z, tokens, mask, up, temperature=1.0):
    from repo_amd.policy import token_logprobs
    leaf = z.detach().requires_grad_()
    lp = token_logprobs(leaf, tokens, mask=mask, temperature=temperature)
    assert lp.dtype is torch.float32 and lp.shape == tokens.shape
    grad, = torch.autograd.grad(lp, leaf, up)
    assert grad.dtype is z.dtype and grad.shape == z.shape
    m = None if mask is None else mask.cpu().numpy()
    ref = O.token_logprobs64(_np(z), tokens.cpu().numpy(), m, temperature)
    counts = np.ones(ref.shape, bool) if m is None else m
    err = np.abs(_np(lp) - ref)
    assert np.all(err <= np.where(counts, _lp_bound(z, ref, temperature), 0.0)), err.max()
    _check_grad(grad, z, tokens, np.where(counts, _np(up), 0.0), 0.0, ref, temperature)
    with torch.no_grad():
        assert torch.equal(token_logprobs(z, tokens, mask=mask, temperature=temperature), lp)
    return lp, grad


@pytest.mark.gpu
@pytest.mark.parametrize("shape,vocab", SHAPES, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_logprobs_match_float64(shape, vocab, dtype):
    z, tokens, mask, up = _inputs(shape, vocab, DTYPES[dtype], seed=vocab)
    _check_logprobs(z, tokens, mask, up)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.3, 0.9, 2.5])
def test_temperatures(temperature):
    z, tokens, _, up = _inputs((3, 5), 1037, torch.bfloat16)
    _check_logprobs(z, tokens, None, up, temperature)


def _policy_inputs(shape, vocab, dtype, seed=0, temperature=1.0, borders=(0.2, 0.28)):
    z, tokens, mask, _ = _inputs(shape, vocab, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    lp = O.token_logprobs64(_np(z), tokens.cpu().numpy(), None, temperature)
    moved = 0.2 * torch.randn(shape, generator=g).double().numpy()
    for border in (np.log1p(-borders[0]), np.log1p(borders[1])):
        moved = np.where(np.abs(moved - border) < 2e-3, moved + 6e-3, moved)
    old = torch.tensor(lp - moved).float().cuda()
    ref = torch.tensor(lp).float().cuda() + 0.3 * torch.randn(shape, generator=g).cuda()
    adv = torch.randn(shape, generator=g).cuda()
    return z, tokens, mask, adv, old, ref


def _check_policy(z, tokens, mask, adv, old, ref, *, clip=(0.2, 0.28), kl_weight=0.05,
                  temperature=1.0, reduction="token", scale=1.0, factor=None):
    from repo_amd.policy import policy_loss
    leaf = z.detach().requires_grad_()
    got = policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask, clip=clip,
                      kl_weight=kl_weight, temperature=temperature, reduction=reduction,
                      scale=scale)
    loss = got.loss if factor is None else got.loss * factor
    grad, = torch.autograd.grad(loss, leaf)
    assert grad.dtype is z.dtype and grad.shape == z.shape
    assert got.loss.dtype is torch.float32 and got.loss.dim() == 0
    assert not (got.logprobs.requires_grad or got.kl.requires_grad or got.clipped.requires_grad)
    m = np.ones(tuple(tokens.shape), bool) if mask is None else mask.cpu().numpy()
    t = tokens.cpu().numpy()
    lp = O.token_logprobs64(_np(z), t, m, temperature)
    A = _np(adv)
    A = A[..., None] if A.ndim < m.ndim else A
    A = np.broadcast_to(A, m.shape)
    R = None if ref is None else _np(ref)
    with np.errstate(all="ignore"):
        terms, slope, kl, clipped = (np.where(m, v, 0.0) for v in O.policy_terms64(
            lp, _np(old), A, R, clip, kl_weight))
        ratio = np.where(m, np.exp(lp - _np(old)), 0.0)
        ed = np.where(m, np.exp((R if R is not None else lp) - lp), 0.0)
    w = O.policy_weights64(m, reduction)
    e = _lp_bound(z, lp, temperature)
    assert np.all(np.abs(_np(got.logprobs) - lp) <= np.where(m, e, 0.0))
    # Weights are rounded to fp32, terms and sums are in 64 bits.
    size = np.abs(terms) + np.abs(A) * ratio + kl_weight * kl
    derr = np.abs(A) * ratio * e + kl_weight * np.abs(np.expm1(np.where(m, (R if R is not None else lp) - lp, 0))) * e
    bound = abs(scale) * ((w * derr).sum() + 3 * U * (w * size).sum()) + U * abs(scale * (w * terms).sum())
    assert abs(float(got.loss) - scale * (w * terms).sum()) <= bound + 1e-37
    assert abs(float(got.kl) - (w * kl).sum()) <= (w * (np.abs(ed - 1) * e + e * e * ed)).sum() + 4 * U * (w * kl).sum() + 1e-37
    assert abs(float(got.clipped) - (w * clipped).sum()) <= 4 * U * (w * clipped).sum()
    f = 1.0 if factor is None else factor
    slopes = w * slope * scale * f
    serr = np.abs(w * scale * f) * ((np.abs(A) * ratio + kl_weight * ed) * e) + 6 * U * np.abs(slopes)
    _check_grad(grad, z, tokens, slopes, np.where(m, serr, 0.0), lp, temperature)
    return got, grad


@pytest.mark.gpu
@pytest.mark.parametrize("shape,vocab", SHAPES, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_policy_matches_float64(shape, vocab, dtype):
    _check_policy(*_policy_inputs(shape, vocab, DTYPES[dtype], seed=vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("shape", [(6, 10), (70, 3), (3, 130), (17,), (2, 3, 66)])
def test_reductions(shape, reduction):
    """Sequences shorter and longer than a wave, and one of which no token counts."""
    z, tokens, mask, adv, old, ref = _policy_inputs(shape, 97, torch.float32, seed=5)
    if len(shape) > 1:
        mask[..., -1, :] = False
    _check_policy(z, tokens, mask, adv, old, ref, reduction=reduction, scale=0.37)
    _check_policy(z, tokens, None, adv, old, ref, reduction=reduction, temperature=0.7)


@pytest.mark.gpu
def test_other_forms():
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 130, torch.float16, seed=9)
    _check_policy(z, tokens, mask, adv, old, None, kl_weight=0.0)
    _check_policy(z, tokens, mask, adv, old, ref, kl_weight=0.0)      # KL is told, not added
    _check_policy(z, tokens, mask, adv[:, 0], old, ref)               # one a sequence
    _check_policy(z, tokens, mask, adv[:, :1], old, ref, clip=(0.0, 1e9))
    _check_policy(z, tokens.int(), mask, adv.half(), old, ref)
    _check_policy(z, tokens, mask, torch.zeros_like(adv), old, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [1.0, 1.0 / 3, -2.5, 0.0, 65536.0])
def test_other_incoming_gradients_are_not_rounded_twice(factor):
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 517, torch.bfloat16, seed=11)
    _check_policy(z, tokens, mask, adv, old, ref, factor=factor)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(9001, 41), (2100, 5003), (1030, 16400), (530, 65600)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_rows_than_the_backward_launches_workgroups_for(rows, vocab, dtype):
    """It takes rows in turns where its factor most likely is one.  Half a gradient is half of every
    number that it is made of, as with a scale of a half."""
    from repo_amd.policy import policy_loss
    z, tokens, mask, _ = _inputs((rows, 1), vocab, DTYPES[dtype], seed=5)
    z.requires_grad_()
    adv = torch.randn(rows, 1, device="cuda")
    old = -torch.rand(rows, 1, device="cuda") * 3
    grads = []
    for scale, factor in ((0.5, 1.0), (1.0, 0.5)):
        loss = policy_loss(z, tokens, adv, old, mask=mask, reduction="sum", scale=scale).loss
        grads.append(torch.autograd.grad(loss * factor if factor != 1.0 else loss, z)[0])
    assert torch.equal(*grads) and bool(grads[0].any())


@pytest.mark.gpu
def test_backward_twice_and_accumulated():
    from repo_amd.policy import policy_loss
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 517, torch.bfloat16, seed=12)
    leaf = z.detach().requires_grad_()
    loss = policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1).loss
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss * 0.5, leaf, retain_graph=True)
    third, = torch.autograd.grad(loss, leaf)
    assert torch.equal(first, kept) and torch.equal(third, kept)
    assert torch.equal(second, kept * 0.5)   # a power of two: the same roundings
    a = policy_loss(leaf, tokens, adv, old, mask=mask).loss
    b = policy_loss(leaf, tokens, adv, old, mask=mask).loss
    (a + b).backward()
    alone, = torch.autograd.grad(policy_loss(leaf, tokens, adv, old, mask=mask).loss, leaf)
    assert torch.equal(leaf.grad, alone * 2)
    with pytest.raises(RuntimeError):   # the logits were written in place
        x = (leaf * 1.0)
        y = policy_loss(x, tokens, adv, old).loss
        x.mul_(2.0)
        y.backward()


@pytest.mark.gpu
def test_without_gradients_nothing_is_kept():
    from repo_amd.policy import policy_loss
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 517, torch.float32, seed=13)
    want, _ = _check_policy(z, tokens, mask, adv, old, ref)
    leaf = z.detach().requires_grad_()
    with torch.no_grad():
        got = policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask, clip=(0.2, 0.28),
                          kl_weight=0.05)
    assert not got.loss.requires_grad
    for x, y in zip(got, want):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_rows_are_not_looked_at(dtype):
    from repo_amd.policy import policy_loss, token_logprobs
    z, tokens, mask, adv, old, ref = _policy_inputs((5, 7), 203, DTYPES[dtype], seed=14)
    clean = policy_loss(z, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1)
    out = ~mask
    z2, t2 = z.clone(), tokens.clone()
    z2[out] = float("nan")
    z2[out & (torch.arange(7, device="cuda") % 2 == 0)] = float("inf")
    t2[out] = -100
    t2[0][out[0]] = 1 << 40
    bad = [torch.where(out, torch.full_like(t, v), t) for t, v in
           ((adv, float("nan")), (old, float("-inf")), (ref, float("inf")))]
    leaf = z2.requires_grad_()
    got = policy_loss(leaf, t2, bad[0], bad[1], ref_logprobs=bad[2], mask=mask, kl_weight=0.1)
    for x, y in zip(got, clean):
        assert torch.equal(x, y)
    grad, = torch.autograd.grad(got.loss, leaf)
    assert torch.isfinite(grad).all() and not grad[out].any() and grad[mask].any()
    lp = token_logprobs(leaf, t2, mask=mask)
    assert torch.equal(lp, clean.logprobs) and not lp[out].any()
    up = torch.where(out, torch.full_like(adv, float("nan")), adv)
    grad, = torch.autograd.grad(lp, leaf, up)
    assert torch.isfinite(grad).all() and not grad[out].any()


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
def test_nothing_counts(reduction):
    from repo_amd.policy import policy_loss
    z, tokens, mask, adv, old, ref = _policy_inputs((5, 7), 203, torch.float32, seed=15)
    leaf = z.requires_grad_()
    got = policy_loss(leaf, tokens, adv, old, mask=torch.zeros_like(mask), reduction=reduction)
    assert float(got.loss) == 0.0 and float(got.kl) == 0.0 and float(got.clipped) == 0.0
    assert not torch.autograd.grad(got.loss, leaf)[0].any()


@pytest.mark.gpu
def test_no_tokens_at_all():
    from repo_amd.policy import policy_loss, token_logprobs
    for shape in ((0,), (0, 4), (3, 0), (2, 0, 5)):
        z = torch.zeros(*shape, 11, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        t, f = torch.zeros(shape, dtype=torch.int64, device="cuda"), torch.zeros(shape, device="cuda")
        got = policy_loss(z, t, f, f)
        assert float(got.loss) == 0.0 and got.logprobs.shape == shape
        assert torch.autograd.grad(got.loss, z)[0].shape == z.shape
        lp = token_logprobs(z, t)
        assert lp.shape == shape and lp.dtype is torch.float32
        lp.sum().backward()
        assert z.grad.shape == z.shape


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 515, 3001, 70001])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_infinite_logits(vocab, dtype):
    """-inf takes a token out of the vocabulary; a row of them alone, +inf and NaN have no
    distribution; the rows beside them are not touched."""
    from repo_amd.policy import token_logprobs
    z, tokens, _, up = _inputs((7,), vocab, DTYPES[dtype], seed=16)
    at = tokens.tolist()
    z[0, : vocab // 2] = float("-inf")
    z[0, at[0]] = 1.0
    z[1] = float("-inf")
    z[2, (at[2] + 1) % vocab] = float("inf")
    z[3, (at[3] + 5) % vocab] = float("nan")
    z[4, at[4]] = float("-inf")
    z[5] = float("-inf")
    z[5, at[5]] = -3.0
    leaf = z.requires_grad_()
    lp = token_logprobs(leaf, tokens)
    grad, = torch.autograd.grad(lp, leaf, up)
    with np.errstate(all="ignore"):
        ref = O.token_logprobs64(_np(z), tokens.cpu().numpy())
    for r in (0, 6):
        assert abs(float(lp[r]) - ref[r]) <= _lp_bound(z[r:r + 1], ref[r:r + 1], 1.0)[0]
        assert torch.isfinite(grad[r]).all()
    assert not grad[0, : vocab // 2][torch.arange(vocab // 2, device="cuda") != at[0]].any()
    for r in (1, 2, 3):
        assert torch.isnan(lp[r]) and torch.isnan(grad[r]).any()
    assert float(lp[4]) == float("-inf")
    assert float(lp[5]) == 0.0 and not grad[5].any()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 515, 3001, 70001, 140001])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_types_lowest_values(dtype, vocab):
    """Masks of the vocabulary by the type's lowest value: those tokens have no probability, and a
    row of them alone has one distribution, the uniform."""
    from repo_amd.policy import token_logprobs
    z, tokens, _, up = _inputs((4,), vocab, DTYPES[dtype], seed=31)
    low = torch.finfo(DTYPES[dtype]).min
    z[0, 1::2] = low
    tokens[0] = 0
    z[1] = low
    z[2] = -low
    z[3, tokens[3]] = low
    for temperature in (1.0, 0.5):
        leaf = z.detach().requires_grad_()
        lp = token_logprobs(leaf, tokens, temperature=temperature)
        grad, = torch.autograd.grad(lp, leaf, up)
        assert torch.isfinite(grad).all() and torch.isfinite(lp[:3]).all()
        keep = z[:1, ::2].contiguous()
        want = O.token_logprobs64(_np(keep), np.zeros(1, np.int64), None, temperature)
        assert abs(float(lp[0]) - want[0]) <= _lp_bound(keep, want, temperature)[0]
        assert not grad[0, 1::2].any()
        even = -np.log(vocab)
        for r in (1, 2):
            assert abs(float(lp[r]) - even) <= U * (130 + vocab / 64 + abs(even))
        assert float(lp[3]) < -1e4


@pytest.mark.gpu
def test_tokens_outside_the_vocabulary_give_nan():
    from repo_amd.policy import policy_loss, token_logprobs
    z, tokens, _, adv, old, ref = _policy_inputs((2, 4), 515, torch.float32, seed=17)
    good = token_logprobs(z, tokens)
    bad = tokens.clone()
    bad[0, 1], bad[1, 2], bad[1, 3] = -1, 515, 1 << 40
    where = bad != tokens
    leaf = z.requires_grad_()
    lp = token_logprobs(leaf, bad)
    assert torch.isnan(lp[where]).all() and torch.equal(lp[~where], good[~where])
    grad, = torch.autograd.grad(lp, leaf, adv)
    assert torch.isnan(grad[where]).all() and torch.isfinite(grad[~where]).all()
    got = policy_loss(leaf, bad, adv, old, ref_logprobs=ref)
    grad, = torch.autograd.grad(got.loss, leaf)
    assert torch.isnan(got.loss) and torch.isnan(grad[where]).all()
    assert torch.isfinite(grad[~where]).all()


@pytest.mark.gpu
def test_far_ratios():
    """Old log-probabilities far off: ratios of 0 and beyond fp32, clipped and not."""
    from repo_amd.policy import policy_loss
    z, tokens, _, _, _, _ = _policy_inputs((4,), 64, torch.float32, seed=18)
    lp = O.token_logprobs64(_np(z), tokens.cpu().numpy())
    old = torch.tensor(lp + np.array([200.0, -200.0, 200.0, -60.0])).float().cuda()
    adv = torch.tensor([1.0, 1.0, -1.0, -1.0]).cuda()
    leaf = z.requires_grad_()
    got = policy_loss(leaf, tokens, adv, old, reduction="sum", clip=(0.2, 0.2))
    grad, = torch.autograd.grad(got.loss, leaf)
    r = np.exp(lp[3] - float(old[3]))
    want = -0.0 - 1.2 + 0.8 + r
    assert abs(float(got.loss) - want) <= 1e-4 * want
    assert not grad[1:3].any() and torch.isfinite(grad).all()
    assert float(got.clipped) == 2.0
    assert grad[3].abs().max() > 1e20 and grad[0].abs().max() < 1e-20


@pytest.mark.gpu
def test_strides_and_alignments():
    """Shifted slices, transposed and expanded leading dimensions, columns of a wider
    matrix, a vocabulary that is not contiguous, tensors that begin anywhere."""
    for dtype in DTYPES.values():
        for vocab in (64, 131, 3001):
            wide, _, _, _ = _inputs((3, 6), vocab + 5, dtype, seed=19)
            flat = wide.flatten()
            views = [wide[:, :-1, :vocab], wide[:, 1:, 3:3 + vocab], wide.transpose(0, 1)[..., :vocab],
                     wide[:1].expand(3, 6, -1)[..., 5:], flat[1:1 + 2 * vocab].view(2, vocab),
                     flat[7:7 + vocab], wide[..., ::2], wide.transpose(1, 2)]
            for v in views:
                g = torch.Generator().manual_seed(20)
                tokens = torch.randint(0, v.shape[-1], v.shape[:-1], generator=g).cuda()
                up = torch.randn(v.shape[:-1], generator=g).cuda()
                _check_logprobs(v, tokens, None, up)
                old = torch.tensor(O.token_logprobs64(_np(v), tokens.cpu().numpy())).float().cuda()
                _check_policy(v, tokens, up > -1, up, old + 0.05, old + 0.1)
    # Constants of any strides.
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 130, torch.float32, seed=21)
    t = lambda x: x.t().contiguous().t()  # noqa: E731
    _check_policy(z, t(tokens), t(mask), t(adv), t(old), t(ref))


@pytest.mark.gpu
def test_a_gradient_by_differences():
    z, tokens, mask, adv, old, ref = _policy_inputs((2, 3), 6, torch.float32, seed=22)
    from repo_amd.policy import policy_loss

    def loss(x):
        return policy_loss(x, tokens, adv, old, ref_logprobs=ref, kl_weight=0.2, clip=(0.2, 0.28),
                           reduction="sum").loss
    leaf = z.requires_grad_()
    grad, = torch.autograd.grad(loss(leaf), leaf)
    h = 2.0 ** -7
    for i in range(z.numel()):
        step = torch.zeros(z.numel(), device="cuda")
        step[i] = h
        step = step.view(z.shape)
        with torch.no_grad():
            slope = (float(loss(z + step)) - float(loss(z - step))) / (2 * h)
        # Central differences: h^2 / 6 times a third derivative below 40, and the losses' roundings.
        near = (torch.exp(torch.tensor(O.token_logprobs64(_np(z), tokens.cpu().numpy())).cuda() - old))
        edge = ((near - 0.8).abs() < 0.05) | ((near - 1.28).abs() < 0.05)
        if not edge.view(-1)[i // 6]:
            assert abs(slope - float(grad.view(-1)[i])) <= 40 * h * h / 6 + 4e-6 / h, i


@pytest.mark.gpu
def test_results_repeat_and_streams():
    from repo_amd.policy import policy_loss, token_logprobs
    z, tokens, mask, adv, old, ref = _policy_inputs((40, 9), 3001, torch.bfloat16, seed=23)
    leaf = z.requires_grad_()

    def once():
        got = policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1)
        return (*got, torch.autograd.grad(got.loss, leaf)[0], token_logprobs(leaf, tokens).detach())
    want = [t.clone() for t in once()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(want, once()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_graphs_follow_their_inputs():
    """Forward and backward in one graph, replayed with other inputs; two graphs at once."""
    from repo_amd.policy import policy_loss
    sets = [_policy_inputs((6, 5), 1037, torch.bfloat16, seed=s) for s in (24, 25, 26)]
    shape = sets[0]

    def once(z, tokens, mask, adv, old, ref):
        leaf = z.detach().requires_grad_()
        got = policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1)
        return (*got, torch.autograd.grad(got.loss * 1.5, leaf)[0])
    eager = [[t.clone() for t in once(*s)] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):
        held = [t.clone() for t in shape]
        with torch.cuda.stream(side):
            once(*held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = once(*held)
        graphs.append((graph, held, out))
    for first, second in ((0, 1), (2, 0), (1, 2), (1, 1)):
        for (graph, held, _), k in zip(graphs, (first, second)):
            for t, v in zip(held, sets[k]):
                t.copy_(v)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), k in zip(graphs, (first, second)):
            for a, b in zip(out, eager[k]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """5.4e9 bytes of logits: the last row, 2.7e9 elements in, is the same row by itself."""
    from repo_amd.policy import policy_loss, token_logprobs
    rows, vocab = 20600, 131075
    z = torch.empty(rows, vocab, dtype=torch.bfloat16, device="cuda")
    few, tokens, _, up = _inputs((4,), vocab, torch.bfloat16, seed=27)
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    at = torch.tensor([0, 1, rows // 2, rows - 1], device="cuda")
    z[at] = few
    mask[at] = True
    t = torch.full((rows,), -1, device="cuda")
    t[at] = tokens
    old, adv = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    small = few.detach().requires_grad_()
    want = token_logprobs(small, tokens)
    old[at], adv[at] = want.detach() + 0.1, up
    leaf = z.requires_grad_()
    got = policy_loss(leaf, t, adv, old, mask=mask)
    assert torch.equal(got.logprobs[at], want)
    grad, = torch.autograd.grad(got.loss, leaf)
    few_loss = policy_loss(small, tokens, up, want.detach() + 0.1).loss
    assert torch.equal(grad[at], torch.autograd.grad(few_loss, small)[0])
    assert not grad[2:at[2]].any() and not grad[at[2] + 1:-1].any()


@pytest.mark.gpu
def test_double_backward_and_forward_mode_are_refused():
    from repo_amd.policy import policy_loss, token_logprobs
    z, tokens, _, adv, old, _ = _policy_inputs((2, 3), 64, torch.float32, seed=28)
    leaf = z.requires_grad_()
    for make in (lambda x: policy_loss(x, tokens, adv, old).loss, lambda x: token_logprobs(x, tokens).sum()):
        grad, = torch.autograd.grad(make(leaf), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            grad.sum().backward()
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(z.detach(), torch.ones_like(z))
            with pytest.raises((RuntimeError, NotImplementedError)):
                make(dual)


@pytest.mark.gpu
def test_nodes_without_the_extension_give_the_same(monkeypatch):
    from repo_amd import policy
    assert policy._extension() is not None
    sets = [_policy_inputs(shape, 131, torch.bfloat16, seed=30) for shape in ((), (5,), (3, 4), (2, 3, 4))]

    def run():
        out = []
        for z, tokens, mask, adv, old, ref in sets:
            for factor in (1.0, 0.3):
                leaf = z.detach().requires_grad_()
                got = policy.policy_loss(leaf, tokens, adv, old, ref_logprobs=ref, mask=mask,
                                         kl_weight=0.1)
                lp = policy.token_logprobs(leaf, tokens.int(), temperature=0.7)
                assert got.logprobs.shape == lp.shape == tokens.shape
                out += [*got, *torch.autograd.grad(got.loss * factor, leaf, retain_graph=True),
                        *torch.autograd.grad(got.loss, leaf), lp,
                        *torch.autograd.grad(lp, leaf, adv)]
        with torch.no_grad():
            out += [*policy.policy_loss(leaf, tokens, adv, old), policy.token_logprobs(leaf, tokens)]
        return out
    want = run()
    monkeypatch.setattr(policy, "_extension", lambda: None)
    for a, b in zip(want, run()):
        assert torch.equal(a, b) and a.requires_grad == b.requires_grad


@pytest.mark.gpu
def test_profile_labels():
    from contextlib import contextmanager
    from repo_amd import _native as N
    from repo_amd.policy import policy_loss, token_logprobs
    z, tokens, _, adv, old, _ = _policy_inputs((2, 3), 64, torch.float32, seed=29)
    seen = []

    @contextmanager
    def factory(label):
        seen.append(label)
        yield
    N.set_profile_ctx_factory(factory)
    try:
        leaf = z.requires_grad_()
        policy_loss(leaf, tokens, adv, old).loss.backward()
        token_logprobs(leaf, tokens).sum().backward()
    finally:
        N.set_profile_ctx_factory(None)
    assert {"policy.loss", "policy.logprobs", "policy.logprobs_bwd"} <= set(seen)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [64, 3001, 70001])
def test_ratios_and_kl_terms_beyond_fp64(vocab):
    """Log-probabilities that differ by 700 and more: e^709.78 is the largest value of fp64.
    Clipped tokens, whatever their ratio: a finite loss and no gradient.  Others: infinity, not
    NaN.  e^d - d - 1 of a far negative d is -d - 1."""
    from repo_amd.policy import policy_loss, token_logprobs
    far = [700.0, 709.0, 709.7, 710.0, 710.9, 711.0, 720.0, 749.7, 750.0, 799.0, 801.0, 900.0, 1e4]
    z, tokens, _, _ = _inputs((len(far),), vocab, torch.float32, seed=31)
    lp = token_logprobs(z, tokens)
    off = torch.tensor(far, device="cuda")
    ones = torch.ones_like(lp)
    leaf = z.requires_grad_()
    for adv, old, each in ((ones, lp - off, -1.2), (-ones, lp + off, 0.8)):
        got = policy_loss(leaf, tokens, adv, old, reduction="sum")
        grad, = torch.autograd.grad(got.loss, leaf)
        # Of 64-bit terms, rounded once.
        assert abs(float(got.loss) - each * len(far)) <= 2 * U * abs(each) * len(far)
        assert float(got.clipped) == len(far) and not grad.any()
    for row, d in enumerate(far):
        one = slice(row, row + 1)
        args = (z.detach()[one], tokens[one])
        unclipped = policy_loss(*args, -ones[one], lp[one] - d).loss
        near = policy_loss(*args, ones[one], lp[one], ref_logprobs=lp[one] + d, reduction="sum")
        # An fp32 loss is infinite from e^88.8 on; the KL term has no part in it here.
        assert float(unclipped) == float(near.kl) == float("inf"), d
        assert abs(float(near.loss) + 1.0) <= 4 * float(_lp_bound(args[0], _np(lp[one]), 1.0).max())
        below = policy_loss(*args, ones[one], lp[one], ref_logprobs=lp[one] - d, reduction="sum").kl
        e = float(_lp_bound(args[0], _np(lp[one]), 1.0).max())
        # The reference's value is rounded to fp32 too, and so is the term.
        assert abs(float(below) - (d - 1.0)) <= 2 * e + 2 * U * (d + 20.0) + U * d, d


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_results_can_be_written_in_place(extension, monkeypatch):
    """As a training loop does (loss += other, loss /= n): each result is a tensor of its own."""
    from repo_amd import policy
    if not extension:
        monkeypatch.setattr(policy, "_extension", lambda: None)
    z, tokens, mask, adv, old, ref = _policy_inputs((4, 6), 131, torch.bfloat16, seed=32)

    def make(x):
        return policy.policy_loss(x, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1)
    leaf = z.detach().requires_grad_()
    plain = make(leaf)
    want, = torch.autograd.grad(plain.loss * 0.5, leaf)
    got = make(leaf)
    loss = got.loss
    loss += 1.0
    loss *= 0.5
    assert torch.equal(loss, (plain.loss + 1.0) * 0.5)
    for name in ("logprobs", "kl", "clipped"):
        assert torch.equal(getattr(got, name), getattr(plain, name))
        getattr(got, name).fill_(7.0)
    assert torch.equal(loss, (plain.loss + 1.0) * 0.5)
    loss.backward()
    assert torch.equal(leaf.grad, want)
    for x in (z, leaf, torch.zeros(0, 3, 5, device="cuda")):   # without gradients and without tokens too
        args = () if x.dim() == 3 and len(x) else (torch.zeros(0, 3),) * 2
        got = make(x) if args == () else policy.policy_loss(
            x, torch.zeros(0, 3, dtype=torch.int64, device="cuda"), *(a.cuda() for a in args))
        before = [t.detach().clone() for t in got]
        got.kl.add_(3.0)
        assert torch.equal(got.clipped, before[3]) and torch.equal(got.loss.detach(), before[0])
        got.clipped.add_(3.0)
        assert torch.equal(got.kl, before[2] + 3.0)


def _with_or_without_extension(extension, monkeypatch):
    from repo_amd import policy
    if not extension:
        monkeypatch.setattr(policy, "_extension", lambda: None)
    z, tokens, mask, adv, old, ref = _policy_inputs((6, 5), 1037, torch.bfloat16, seed=33)

    def make(x):
        return policy.policy_loss(x, tokens, adv, old, ref_logprobs=ref, mask=mask, kl_weight=0.1)
    return z, make


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_a_backward_pass_captured_by_itself(extension, monkeypatch):
    """The loss before the capture, or in a graph of its own: each replay writes the gradient of the
    incoming gradient as it is then, whatever became of the last one's."""
    z, make = _with_or_without_extension(extension, monkeypatch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = z.detach().requires_grad_()
        want = {f: torch.autograd.grad(make(leaf).loss * f, leaf)[0] for f in (1.0, 2.0)}
        for captured in (False, True):
            up = torch.ones((), device="cuda")
            first = torch.cuda.CUDAGraph()
            if captured:
                side.synchronize()
                with torch.cuda.graph(first, stream=side):
                    got = make(leaf)
                first.replay()
            else:
                got = make(leaf)
            side.synchronize()
            second = torch.cuda.CUDAGraph()
            with torch.cuda.graph(second, stream=side):
                grad, = torch.autograd.grad(got.loss, leaf, up, retain_graph=True)
            for f in (1.0, 2.0, 1.0, 1.0, 2.0):
                up.fill_(f)
                second.replay()
                assert torch.equal(grad, want[f])
                grad.zero_()
            side.synchronize()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_an_eager_gradient_of_a_captured_loss_is_its_own(extension, monkeypatch):
    """Replays make the loss anew; a gradient that was computed between them stays."""
    z, make = _with_or_without_extension(extension, monkeypatch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = z.detach().clone().requires_grad_()
        others = [z.detach().clone(), z.detach() * 0.5]
        want = [torch.autograd.grad(make(x.requires_grad_()).loss, x)[0] for x in others]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = make(leaf)
        found = []
        for x in others:
            leaf.data.copy_(x.detach())   # as a captured network's last launch would write them
            graph.replay()
            found.append(torch.autograd.grad(got.loss, leaf, retain_graph=True)[0])
        for a, b in zip(found, want):
            assert torch.equal(a, b)
        side.synchronize()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.gpu
@pytest.mark.parametrize("extension", [True, False])
def test_tangents_of_the_constants_are_refused(extension, monkeypatch):
    """A loss without a tangent would be a derivative of zero."""
    from repo_amd import policy
    from torch.autograd import forward_ad
    if not extension:
        monkeypatch.setattr(policy, "_extension", lambda: None)
    z, tokens, _, adv, old, ref = _policy_inputs((2, 3), 64, torch.float32, seed=34)
    for which in ("advantages", "old_logprobs", "ref_logprobs"):
        for leaf in (z, z.detach().requires_grad_()):
            with forward_ad.dual_level():
                c = dict(advantages=adv, old_logprobs=old, ref_logprobs=ref)
                c[which] = forward_ad.make_dual(c[which], torch.ones_like(c[which]))
                with pytest.raises(ValueError, match=f"no gradient for {which}: detach it"):
                    policy.policy_loss(leaf, tokens, **c)
                c[which] = c[which].detach()
                assert torch.isfinite(policy.policy_loss(leaf, tokens, **c).loss)

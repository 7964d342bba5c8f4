"""Training a network that writes paths as tokens: log-probabilities of the tokens it
chose, and the clipped policy loss with a KL term.

New beside the reference, which optimizes its primitives directly.  The choice of
a token has no gradient, so such a network learns from what the renderer makes of
its answers: their losses (``repo_amd.metric``, ``repo_amd.fused``) are the rewards,
and these operators, from the network's logits, what goes back into it.  Both run in
libcubicsplat_hip.so, in fp32 whatever the logits' type.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N
from . import torchcall

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_REDUCTIONS = {"token": 0, "sequence": 1, "sum": 2}


class PolicyLoss(NamedTuple):
    """loss: 0-d fp32, differentiable in the logits.  Without gradients: logprobs, of
    each token (0 where masked); kl, the weighted mean of the KL estimate (0 without
    ref_logprobs); clipped, the weighted share of tokens whose ratio was clipped."""
    loss: torch.Tensor
    logprobs: torch.Tensor
    kl: torch.Tensor
    clipped: torch.Tensor


def _check(logits, tokens, mask, temperature):
    if logits.dim() < 1 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be float32, bfloat16 or float16 [..., vocabulary], got "
                         f"{logits.dtype} {tuple(logits.shape)}")
    if logits.shape[-1] < 1:
        raise ValueError("an empty vocabulary has no tokens")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32, got {tokens.dtype}")
    _beside(tokens, "tokens", logits)
    if mask is not None:
        if mask.dtype is not torch.bool:
            raise ValueError(f"mask must be bool, got {mask.dtype}")
        _beside(mask, "mask", logits)
    if not 1e-20 < temperature < 1e20:
        raise ValueError(f"Invalid temperature: {temperature}")


def _beside(t, name, logits):
    if t.shape != logits.shape[:-1]:
        raise ValueError(f"{name} must have shape {tuple(logits.shape[:-1])}, got "
                         f"{tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"{name} is on {t.device}, logits on {logits.device}")


def _rows(logits):
    """logits as [batch, length, vocab] with the vocabulary contiguous."""
    if logits.dim() < 3:
        logits = logits.reshape((1,) * (3 - logits.dim()) + logits.shape)
    elif logits.dim() > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
    return logits if logits.shape[-1] == 1 or logits.stride(-1) == 1 else logits.contiguous()


def _head(z, tokens, mask, temperature):
    """The first ten arguments of the entry points."""
    batch, length, vocab = z.shape
    return (z.data_ptr(), batch, length, vocab, z.stride(0), z.stride(1), _DTYPES[z.dtype],
            tokens.data_ptr(), None if mask is None else mask.data_ptr(), temperature)


def _plain(t, dtype):
    return t.detach().to(dtype).contiguous()


def _inputs(logits, tokens, mask):
    return (_rows(logits.detach()), _plain(tokens, torch.int64),
            None if mask is None else mask.contiguous())


# The nodes below are for runs without the extension, and where each launch is bracketed by a
# context manager; the extension's do the same.

class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature):
        z, tokens, mask = _inputs(logits, tokens, mask)
        lp = torch.empty(tokens.shape, dtype=torch.float32, device=z.device)
        stats = torch.empty((*z.shape[:2], 2), dtype=torch.float32, device=z.device)
        with N.prof("policy.logprobs"):
            N.call("cs_token_logprobs_forward", *_head(z, tokens, mask, temperature),
                   stats.data_ptr(), lp.data_ptr(), N.stream(z.device))
        ctx.save_for_backward(z, tokens, mask, stats)
        ctx.temperature, ctx.shape = temperature, logits.shape
        return lp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        z, tokens, mask, stats = ctx.saved_tensors
        return (_gradient(z, tokens, mask, ctx.temperature, stats, upstream.contiguous(),
                          ctx.shape), None, None, None)


def _gradient(z, tokens, mask, temperature, stats, slopes, shape, factor=None, into=None):
    """The logits' gradient for slopes of the log-probabilities, times *factor; into
    `into`, which holds it for a factor of one, or a new tensor."""
    grad = torch.empty(shape, dtype=z.dtype, device=z.device) if into is None else into
    with N.prof("policy.logprobs_bwd"):
        N.call("cs_token_logprobs_backward", *_head(z, tokens, mask, temperature),
               stats.data_ptr(), slopes.data_ptr(), N.ptr(factor), 0 if into is None else 1,
               grad.data_ptr(), N.stream(z.device))
    return grad


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, need, advantages, old, ref, *numbers):
        z, tokens, mask = _inputs(logits, tokens, mask)
        batch, length, _ = z.shape
        dev = z.device
        advantages = advantages.detach().float().expand(tokens.shape).reshape(batch, length)
        old, ref = _plain(old, torch.float32), None if ref is None else _plain(ref, torch.float32)
        # A loss in a graph leaves its gradient to the backward pass, which may be in none or
        # in another one: replays of one without the other would find what the last has made of it.
        hold = need and not torch._C._cuda_isCurrentStreamCapturing()
        grad = torch.empty(logits.shape, dtype=z.dtype, device=dev) if hold else None
        lp = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        slopes = torch.empty((batch, length), dtype=torch.float32, device=dev)
        stats = torch.empty((batch, length, 2), dtype=torch.float32, device=dev)
        out = torch.empty(3, dtype=torch.float32, device=dev)
        work = torch.empty(int(N.lib().cs_policy_loss_workspace_elems(batch, length)),
                           dtype=torch.float32, device=dev)
        with N.prof("policy.loss"):
            N.call("cs_policy_loss", *_head(z, tokens, mask, temperature), advantages.data_ptr(),
                   advantages.stride(0), advantages.stride(1), old.data_ptr(), N.ptr(ref),
                   *numbers, work.data_ptr(), stats.data_ptr(), slopes.data_ptr(), lp.data_ptr(),
                   out.data_ptr(), N.ptr(grad), N.stream(dev))
        # Tensors of their own, which callers may write in place, and not views of one.
        loss, kl, clipped = (t.data for t in out.unbind())
        ctx.mark_non_differentiable(lp, kl, clipped)
        if need:
            ctx.save_for_backward(z, tokens, mask, stats, slopes)
            ctx.grad, ctx.temperature, ctx.shape = grad, temperature, logits.shape
        return loss, lp, kl, clipped

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, *_):
        # The gradient for an incoming one is there; another one's is computed from the
        # logits, not from that one's rounded values.  A second backward pass finds it given away,
        # and one in a graph leaves it.
        z, tokens, mask, stats, slopes = ctx.saved_tensors
        into, ctx.grad = ctx.grad, None
        if torch._C._cuda_isCurrentStreamCapturing():
            into = None
        factor = upstream.to(torch.float32).contiguous()
        return (_gradient(z, tokens, mask, ctx.temperature, stats, slopes, ctx.shape, factor,
                          into), *(None,) * 12)


def _extension():
    return torchcall.module() if N._PROFILE_CTX_FACTORY is None else None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *,
                   mask: Optional[torch.Tensor] = None, temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature) at the chosen tokens, without the softmax's
    other values ever in memory.

    logits: [..., V] fp32, bf16 or fp16 on the GPU; slices such as ``logits[:, :-1]``
    are read where they lie.  tokens: [...] int64 or int32.  mask: [...] bool; where
    it is False the logits and the token are not looked at (they may be anything), the
    result is 0 and the gradient zeros.  A token outside the vocabulary gives NaN.
    Returns [...] fp32.  Differentiable (once, in reverse mode) in the logits, whose
    gradient is of their type; sums are taken in a fixed order."""
    _check(logits, tokens, mask, temperature)
    N.require_gpu(logits, "logits")
    if tokens.numel() == 0:
        return logits.sum(-1, dtype=torch.float32)
    if logits.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, tokens, mask=mask, temperature=temperature)
    ext = _extension()
    return (ext.token_logprobs if ext is not None else _TokenLogprobs.apply)(
        logits, tokens, mask, float(temperature))


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, advantages: torch.Tensor,
                old_logprobs: torch.Tensor, *, ref_logprobs: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, clip: Tuple[float, float] = (0.2, 0.2),
                kl_weight: float = 0.0, temperature: float = 1.0, reduction: str = "token",
                scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss with a KL term, from logits:

        l = log softmax(logits / temperature)[token],  r = exp(l - old),  d = ref - l
        L = -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_weight (exp(d) - d - 1)

    summed over the tokens that ``mask`` leaves, with weights by ``reduction``:
    "token", the mean over all of them; "sequence", the mean over the sequences (the
    last dimension of ``tokens``) that have any of each one's mean; "sum".  The whole is
    multiplied with ``scale`` (for gradient accumulation: a backward pass whose incoming
    gradient is one has its work done already).

    logits, tokens, mask, temperature: as for token_logprobs.  advantages: [...] as the
    tokens, or one a sequence ([..., 1] or without the last dimension); old_logprobs and
    ref_logprobs: [...].  These three are constants: fp32, bf16 or fp16 without a gradient.
    Without tokens that count the loss is 0.  Differentiable (once, in reverse mode) in the
    logits."""
    _check(logits, tokens, mask, temperature)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'token', 'sequence' or 'sum', got {reduction!r}")
    low, high = clip
    for name, value in (("clip", low), ("clip", high), ("kl_weight", kl_weight)):
        if not 0.0 <= value < float("inf"):
            raise ValueError(f"Invalid {name}: {value}")
    if not abs(scale) < float("inf"):
        raise ValueError(f"Invalid scale: {scale}")
    if kl_weight > 0 and ref_logprobs is None:
        raise ValueError("kl_weight needs ref_logprobs")
    constants = {"advantages": advantages, "old_logprobs": old_logprobs,
                 "ref_logprobs": ref_logprobs}
    for name, t in constants.items():
        if t is None:
            continue
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
        if (t.requires_grad and torch.is_grad_enabled()) or N.has_tangent(t):
            raise ValueError(f"policy_loss has no gradient for {name}: detach it")
        if name != "advantages":
            _beside(t, name, logits)
    if advantages.device != logits.device:
        raise ValueError(f"advantages is on {advantages.device}, logits on {logits.device}")
    shape = tokens.shape
    if advantages.shape == shape[:-1] and advantages.shape != shape:
        advantages = advantages.unsqueeze(-1)
    if advantages.shape != shape and not (
            len(shape) > 0 and advantages.shape == (*shape[:-1], 1)):
        raise ValueError(f"advantages must have shape {tuple(shape)} or one value a sequence, got "
                         f"{tuple(advantages.shape)}")
    N.require_gpu(logits, "logits")
    if tokens.numel() == 0:
        return PolicyLoss(logits.sum(dtype=torch.float32), *(
            torch.zeros(s, dtype=torch.float32, device=logits.device) for s in (shape, (), ())))
    if logits.device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(logits.device):
            return policy_loss(logits, tokens, advantages, old_logprobs,
                               ref_logprobs=ref_logprobs, mask=mask, clip=clip,
                               kl_weight=kl_weight, temperature=temperature, reduction=reduction,
                               scale=scale)
    constants = (advantages, old_logprobs, ref_logprobs, float(low), float(high),
                 float(kl_weight), _REDUCTIONS[reduction], float(scale))
    ext = _extension()
    if ext is not None:
        return PolicyLoss(*ext.policy_loss(logits, tokens, mask, float(temperature), *constants))
    return PolicyLoss(*_PolicyLoss.apply(logits, tokens, mask, float(temperature),
                                         torch.is_grad_enabled() and logits.requires_grad,
                                         *constants))

"""Float64 restatements of the operators for networks in front of the renderer
(numpy, from the formulas): group norm with an activation and its gradients,
the AdamW step, what the 8-bit optimizer states hold, Newton-Schulz steps and the
Muon step, log-probabilities of tokens and the clipped policy loss."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 128


# ---------------------------------------------------------------- group norm


def _erf(x):
    from scipy.special import erf
    return erf(x)


def activation64(z, act):
    """act(z) and act'(z)."""
    if act in (None, "none"):
        return z, np.ones_like(z)
    if act == "relu":
        return np.where(z > 0, z, 0.0), (z > 0).astype(np.float64)
    if act == "silu":
        with np.errstate(over="ignore"):
            p = 1.0 / (1.0 + np.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        p = 0.5 * (1.0 + _erf(z / math.sqrt(2.0)))
        return z * p, p + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    raise ValueError(act)


def group_norm64(x, groups, weight=None, bias=None, eps=1e-5, act=None, dy=None):
    """x [N, C, S...]: y, or with dy (y, dx, dweight, dbias)."""
    x = np.asarray(x, np.float64)
    n, c = x.shape[:2]
    g = x.reshape(n, groups, -1)
    xc = g - g.mean(2, keepdims=True)
    r = 1.0 / np.sqrt((xc * xc).mean(2, keepdims=True) + eps)
    xh = (xc * r).reshape(n, c, -1)
    w = np.ones(c) if weight is None else np.asarray(weight, np.float64)
    b = np.zeros(c) if bias is None else np.asarray(bias, np.float64)
    y, slope = activation64(xh * w[:, None] + b[:, None], act)
    if dy is None:
        return y.reshape(x.shape)
    dz = np.asarray(dy, np.float64).reshape(n, c, -1) * slope
    t = (dz * w[:, None]).reshape(n, groups, -1)
    xg = xh.reshape(n, groups, -1)
    dx = r * (t - t.mean(2, keepdims=True) - xg * (t * xg).mean(2, keepdims=True))
    return (y.reshape(x.shape), dx.reshape(x.shape), (dz * xh).sum((0, 2)), dz.sum((0, 2)))


# --------------------------------------------------------------------- AdamW


def adamw_step64(p, g, m, v, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 clip=1.0):
    """(p, m, v) after one step, in float64."""
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    g = g * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    return adamw_move64(p, m, v, step=step, lr=lr, betas=betas, eps=eps,
                        weight_decay=weight_decay), m, v


def adamw_move64(p, m, v, *, step, lr, betas, eps, weight_decay):
    """The parameter after a step that left the moments m and v."""
    p, m, v = (np.asarray(a, np.float64) for a in (p, m, v))
    hat = (m / (1 - betas[0] ** step)) / (np.sqrt(v / (1 - betas[1] ** step)) + eps)
    return p * (1 - lr * weight_decay) - lr * hat


def mix32(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def rounding_numbers(seed, step, tensor, numel):
    """The two 16-bit numbers of each element (first moment, root)."""
    key = mix32(mix32((seed + step * 0x3C6EF372) & 0xFFFFFFFF) + np.uint64(tensor))
    i = np.arange(numel, dtype=np.uint64)
    r = mix32(key + (i & np.uint64(0xFFFFFFFF)) + (i >> np.uint64(32)) * np.uint64(0x3C6EF372))
    return (r & np.uint64(0xFFFF)).astype(np.int64), (r >> np.uint64(16)).astype(np.int64)


def hold8(x, mantissa, r, floor=False):
    """What the 8 bits hold of x (one tensor, in memory order): (values,
    signed codes without the NaN ones, block exponents).  r: 16-bit numbers,
    0x8000 everywhere for rounding to nearest.  floor: no value but zero
    becomes zero.  Values that are not finite become NaN."""
    x = np.asarray(x, np.float64).ravel()
    n = x.size
    rows = np.pad(x, (0, -n % BLOCK)).reshape(-1, BLOCK)
    r = np.pad(np.broadcast_to(np.asarray(r, np.float64), (n,)), (0, -n % BLOCK)).reshape(-1, BLOCK)
    finite = np.isfinite(rows)
    a = np.where(finite, np.abs(rows), 0.0)
    top = a.max(1, keepdims=True)
    # The biased fp32 exponent of the largest; 0 for subnormals and zero.
    e = np.where(top > 0, np.frexp(top)[1] - 1 + 127, 0).astype(np.int64)
    e = np.maximum(e, 0)
    # In units of the least binade's spacing, 2^(e - 127 - 13 - mantissa).
    unit = np.ldexp(1.0, (e - 127 - 13 - mantissa).astype(np.int64))
    u = a / unit
    binade = np.maximum(np.frexp(u)[1] - 1 - mantissa, 0)
    spacing = np.ldexp(1.0, binade)
    whole = np.floor(u / spacing)
    whole = whole + ((u / spacing - whole) * 65536.0 + r >= 65536.0)
    if floor:
        whole = np.where((a > 0) & (whole == 0), 1.0, whole)
    held = np.where(finite, np.copysign(whole * spacing * unit, rows), np.nan)
    return held.reshape(-1)[:n], e.reshape(-1)


# ---------------------------------------------------------------------- Muon


def newton_schulz64(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """x [..., m, n] after the steps x <- a x + (b g + c g^2) x, g = x x^T."""
    x = np.asarray(x, np.float64)
    if x.shape[-2] > x.shape[-1]:
        return np.swapaxes(newton_schulz64(np.swapaxes(x, -1, -2), steps, coefficients, eps), -1, -2)
    a, b, c = coefficients
    x = x / np.maximum(np.sqrt((x * x).sum((-1, -2), keepdims=True)), eps)
    for _ in range(steps):
        g = x @ np.swapaxes(x, -1, -2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def muon_step64(p, g, momentum_buffer, *, lr, weight_decay=0.1, momentum=0.95, nesterov=True,
                adjust=None, **newton_schulz):
    """(p, momentum_buffer) after one step."""
    p, g, m = (np.asarray(a, np.float64) for a in (p, g, momentum_buffer))
    m = m + (1 - momentum) * (g - m)
    u = (g + momentum * (m - g) if nesterov else m).reshape(p.shape[0], -1)
    rows, cols = u.shape
    by = (0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw"
          else math.sqrt(max(1.0, rows / cols)))
    o = newton_schulz64(u, **newton_schulz).reshape(p.shape)
    return p * (1 - lr * weight_decay) - lr * by * o, m


# -------------------------------------------------------------------- tokens


def token_logprobs64(z, tokens, mask=None, temperature=1.0, upstream=None):
    """z [..., V]: the chosen tokens' log-probabilities, or with upstream (they, dz)."""
    z = np.asarray(z, np.float64) / temperature
    mask = np.ones(tokens.shape, bool) if mask is None else np.asarray(mask, bool)
    z = np.where(mask[..., None], z, 0.0)
    at = np.where(mask, tokens, 0)[..., None]
    top = z.max(-1, keepdims=True)
    e = np.exp(z - top)
    total = e.sum(-1, keepdims=True)
    lp = np.where(mask, (np.take_along_axis(z - top, at, -1) - np.log(total))[..., 0], 0.0)
    if upstream is None:
        return lp
    slope = np.where(mask, upstream, 0.0)[..., None] / temperature
    dz = -slope * (e / total)
    np.put_along_axis(dz, at, np.take_along_axis(dz, at, -1) + slope, -1)
    return lp, dz


def policy_terms64(lp, old, adv, ref=None, clip=(0.2, 0.2), kl_weight=0.0):
    """(loss, derivative by lp, KL estimate, clipped) of each token."""
    r = np.exp(lp - old)
    low, high = 1 - clip[0], 1 + clip[1]
    gain = np.minimum(r * adv, np.clip(r, low, high) * adv)
    clipped = np.where(adv >= 0, r > high, r < low)
    slope = np.where(clipped, 0.0, -adv * r)
    d = np.zeros_like(lp) if ref is None else ref - lp
    kl = np.expm1(d) - d
    return -gain + kl_weight * kl, slope - kl_weight * np.expm1(d), kl, clipped & (adv != 0)


def policy_weights64(mask, reduction):
    """The weight of each token; the last dimension is a sequence's."""
    m = np.asarray(mask, np.float64)
    if reduction == "sum":
        return m
    if reduction == "token":
        return m / max(1.0, m.sum())
    n = m.sum(-1, keepdims=True)
    return m / np.maximum(n, 1.0) / max(1.0, float((n > 0).sum()))

"""Adam, Adan and AdamW with the step in one HIP launch for many parameters.

The reference optimizes its primitives with ``torch.optim.Adam`` over
per-group learning rates (gaussian_trace/model.py:172-189).  ``Adam`` here is
a drop-in for that class on fp32 device parameters: same constructor, param
groups, ``state`` entries (``step``, ``exp_avg``, ``exp_avg_sq``) and
``state_dict`` layout, so a checkpoint moves between the two.  The update is
torch's single-tensor Adam (amsgrad and maximize off); one ``cs_adam_step``
launch covers up to 16 tensors.  Optimizer step pre/post hooks (global and
per instance) run as for torch's optimizers; the profiler range torch wraps
around ``step`` is left out, since it costs more host time than the launch.

``Adan`` is the reference's own optimizer (manbo/optim.py:10-190, the default
of its training script) with the update of ops/optim.py:8-113 as one
``cs_adan_step`` launch per 16 tensors; ``adan_step_from_grad_tilelang`` is
the reference's functional single-tensor form.

``AdamW`` (new: the reference trains its primitives directly, without a
network) is for the weights of a network in front of the renderer: decoupled
weight decay, fp32, bf16 and fp16 parameters of any dense layout, a global-norm
clip without a host read, states in 32 or 8 bits, one launch for up to 56
tensors.  ``global_grad_norm`` is the norm by itself.
"""
from __future__ import annotations

import ctypes
import math
from itertools import chain
from operator import is_

import numpy as np
import torch
from torch.autograd.graph import increment_version
from torch.optim import optimizer as _torch_optimizer

from . import _native as N
from . import torchcall

MAX_TENSORS_PER_LAUNCH = 16


def _run_pre_hooks(opt, closure):
    """torch's step pre-hooks (global and of the instance): the (args, kwargs)
    of the step and its closure as they leave them."""
    args, kwargs = (opt,), {"closure": closure} if closure is not None else {}
    if _torch_optimizer._global_optimizer_pre_hooks or opt._optimizer_step_pre_hooks:
        for pre_hook in chain(_torch_optimizer._global_optimizer_pre_hooks.values(),
                              opt._optimizer_step_pre_hooks.values()):
            result = pre_hook(opt, args, kwargs)
            if result is not None:
                if isinstance(result, tuple) and len(result) == 2:
                    args, kwargs = result
                else:
                    raise RuntimeError(
                        "optimizer step pre-hooks must return None or (args, kwargs), got "
                        f"{result}")
        closure = kwargs.get("closure", closure)
    return args, kwargs, closure


def _run_post_hooks(opt, args, kwargs):
    if opt._optimizer_step_post_hooks or _torch_optimizer._global_optimizer_post_hooks:
        for post_hook in chain(opt._optimizer_step_post_hooks.values(),
                               _torch_optimizer._global_optimizer_post_hooks.values()):
            post_hook(opt, args, kwargs)


class _LaunchArgs:
    """ctypes argument arrays for one launch of n tensors, reused across steps."""

    def __init__(self, n):
        self.n = n
        self.params = (ctypes.c_void_p * n)()
        self.grads = (ctypes.c_void_p * n)()
        self.ms = (ctypes.c_void_p * n)()
        self.vs = (ctypes.c_void_p * n)()
        self.numels = (ctypes.c_int64 * n)()
        self.step_sizes = (ctypes.c_float * n)()
        self.bc2s = (ctypes.c_float * n)()
        self.wds = (ctypes.c_float * n)()


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
                 amsgrad=False, *, maximize=False, capturable=False, differentiable=False,
                 foreach=None, fused=None):
        if not 0.0 <= float(lr):
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= float(eps):
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad or maximize or capturable or differentiable:
            raise NotImplementedError(
                "repo_amd.optim.Adam implements amsgrad=False, maximize=False, "
                "capturable=False, differentiable=False")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False,
                        maximize=False, foreach=None, capturable=False, differentiable=False,
                        fused=None)
        super().__init__(params, defaults)
        self._launch_args = {}
        self._step_views = {}

    def zero_grad(self, set_to_none: bool = True) -> None:
        """torch.optim.Optimizer.zero_grad (foreach off), without the profiler
        range it opens around the loop."""
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    if set_to_none:
                        p.grad = None
                    else:
                        if p.grad.grad_fn is not None:
                            p.grad.detach_()
                        else:
                            p.grad.requires_grad_(False)
                        p.grad.zero_()

    def _step_count(self, st):
        """Increments the state's CPU ``step`` tensor through a cached numpy
        view of it (the tensor stays what torch's Adam stores) and returns the
        new count."""
        t = st["step"]
        if t.device.type != "cpu" or t.requires_grad:
            t += 1
            return float(t)
        c = self._step_views.get(id(t))
        if c is None or c[0] is not t:
            if len(self._step_views) > 4 * MAX_TENSORS_PER_LAUNCH + len(self.state):
                self._step_views.clear()
            c = self._step_views[id(t)] = (t, t.numpy())
        arr = c[1]
        arr += 1
        return float(arr)

    def step(self, closure=None):
        args, kwargs, closure = _run_pre_hooks(self, closure)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        batches = {}
        state = self.state
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            key = (float(beta1), float(beta2), float(group["eps"]))
            lr, wd = float(group["lr"]), float(group["weight_decay"])
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise RuntimeError("Adam does not support sparse gradients")
                if p.dtype is not torch.float32 or not p.is_contiguous() or not p.is_cuda:
                    raise ValueError(
                        "repo_amd.optim.Adam needs contiguous float32 CUDA (ROCm) parameters")
                st = state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                step = self._step_count(st)
                bc1 = 1.0 - beta1 ** step
                bc2 = 1.0 - beta2 ** step
                if not g.is_contiguous():
                    g = g.contiguous()
                batches.setdefault((p.device.index, key), []).append(
                    (p, g, st["exp_avg"], st["exp_avg_sq"], lr / bc1, math.sqrt(bc2), wd))
        for (dev, (beta1, beta2, eps)), items in batches.items():
            for k in range(0, len(items), MAX_TENSORS_PER_LAUNCH):
                self._launch(dev, items[k:k + MAX_TENSORS_PER_LAUNCH], beta1, beta2, eps)
        self._optimizer_step_code()
        _run_post_hooks(self, args, kwargs)
        return loss

    # torch's Optimizer wraps `step` of each subclass in a profiler range unless
    # the function is marked as already hooked; the hooks are called above.
    step.hooked = True

    def _launch(self, dev, items, beta1, beta2, eps):
        n = len(items)
        a = self._launch_args.get(n)
        if a is None:
            a = self._launch_args[n] = _LaunchArgs(n)
        for k, (p, g, m, v, step_size, bc2s, wd) in enumerate(items):
            a.params[k] = p.data_ptr()
            a.grads[k] = g.data_ptr()
            a.ms[k] = m.data_ptr()
            a.vs[k] = v.data_ptr()
            a.numels[k] = p.numel()
            a.step_sizes[k] = step_size
            a.bc2s[k] = bc2s
            a.wds[k] = wd
        with N.prof("optim.adam"):
            N.call("cs_adam_step", n, a.params, a.grads, a.ms, a.vs, a.numels, a.step_sizes,
                   a.bc2s, a.wds, beta1, beta2, eps, N.stream(dev))


DEFAULT_TILELANG_THREADS = 256


class _AdanLaunchArgs:
    """ctypes argument arrays for one cs_adan_step launch of n tensors."""

    def __init__(self, n):
        self.n = n
        self.params = (ctypes.c_void_p * n)()
        self.grads = (ctypes.c_void_p * n)()
        self.ms = (ctypes.c_void_p * n)()
        self.ns = (ctypes.c_void_p * n)()
        self.ds = (ctypes.c_void_p * n)()
        self.npgs = (ctypes.c_void_p * n)()
        self.numels = (ctypes.c_int64 * n)()
        self.scalars = (ctypes.c_float * (10 * n))()
        self.flags = (ctypes.c_int32 * (2 * n))()


def _adan_launch(dev, items, clip_ptr, cache=None):
    """items: (param, grad, exp_avg, exp_avg_sq, exp_avg_diff, neg_pre_grad,
    [10 scalars], first, no_prox) per tensor, at most CS_ADAM_MAX_TENSORS."""
    n = len(items)
    a = cache.get(n) if cache is not None else None
    if a is None:
        a = _AdanLaunchArgs(n)
        if cache is not None:
            cache[n] = a
    for k, (p, g, m, v, d, npg, sc, first, no_prox) in enumerate(items):
        a.params[k] = p.data_ptr()
        a.grads[k] = g.data_ptr()
        a.ms[k] = m.data_ptr()
        a.ns[k] = v.data_ptr()
        a.ds[k] = d.data_ptr()
        a.npgs[k] = npg.data_ptr()
        a.numels[k] = p.numel()
        for j in range(10):
            a.scalars[10 * k + j] = sc[j]
        a.flags[2 * k] = int(first)
        a.flags[2 * k + 1] = int(no_prox)
    with N.prof("optim.adan"):
        N.call("cs_adan_step", n, a.params, a.grads, a.ms, a.ns, a.ds, a.npgs, a.numels,
               a.scalars, a.flags, clip_ptr, N.stream(dev))


class Adan(torch.optim.Optimizer):
    """The reference's Adan (manbo/optim.py:10-190): same constructor checks,
    param groups, per-parameter state (exp_avg, exp_avg_sq, exp_avg_diff,
    neg_pre_grad) and per-group integer ``step``, with the update of
    adan_step_from_grad_kernel (ops/optim.py:8-113) run as one cs_adan_step
    launch for up to 16 tensors.  With max_grad_norm > 0 the global-norm clip
    factor clamp(max_norm / (norm + eps), max=1) is computed on the device and
    read there (the reference reads it on the host with .item()).
    tilelang_threads is accepted for the reference's signature."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.98, 0.92, 0.99), eps: float = 1e-8,
                 weight_decay: float = 0.0, max_grad_norm: float = 0.0, no_prox: bool = False,
                 tilelang_threads: int = DEFAULT_TILELANG_THREADS):
        if not 0.0 <= max_grad_norm:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= betas[2] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 2: {betas[2]}")
        if tilelang_threads <= 0:
            raise ValueError(f"Invalid tilelang_threads: {tilelang_threads}")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                        max_grad_norm=max_grad_norm, no_prox=no_prox,
                        tilelang_threads=tilelang_threads)
        super().__init__(params, defaults)
        self._launch_args = {}

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("no_prox", False)
            group.setdefault("tilelang_threads", DEFAULT_TILELANG_THREADS)
        self._launch_args = {}

    @torch.no_grad()
    def restart_opt(self):
        for group in self.param_groups:
            group["step"] = 0
            for p in group["params"]:
                if not p.requires_grad:
                    continue
                state = self.state[p]
                state["exp_avg"] = torch.zeros_like(p)
                state["exp_avg_sq"] = torch.zeros_like(p)
                state["exp_avg_diff"] = torch.zeros_like(p)
                state["neg_pre_grad"] = torch.zeros_like(p)

    def _clip_factor(self):
        """Device fp32 clamp(max_norm / (||g|| + eps), max=1) over every
        gradient (manbo/optim.py:78-96), or None when clipping is off."""
        max_norm = float(self.defaults["max_grad_norm"])
        if max_norm <= 0:
            return None
        device = self.param_groups[0]["params"][0].device
        total = torch.zeros(1, device=device)
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None:
                    total.add_(p.grad.pow(2).sum())
        norm = torch.sqrt(total)
        eps = self.param_groups[0]["eps"]
        return torch.clamp(torch.tensor(max_norm, device=device) / (norm + eps),
                           max=1.0).to(torch.float32).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        clip = self._clip_factor()
        batches = {}
        for group in self.param_groups:
            beta1, beta2, beta3 = group["betas"]
            group["step"] = group.get("step", 0) + 1
            step = int(group["step"])
            bc1 = 1.0 - beta1 ** step
            bc2 = 1.0 - beta2 ** step
            bc3_sqrt = math.sqrt(1.0 - beta3 ** step)
            no_prox = bool(group["no_prox"])
            scalars = (float(beta1), float(beta2), float(beta3), float(bc1), float(bc2),
                       float(bc3_sqrt), float(group["lr"]), float(group["weight_decay"]),
                       float(group["eps"]), 1.0)
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.dtype != torch.float32:
                    raise ValueError("Adan expects float32 params")
                if not p.is_contiguous():
                    raise ValueError("Adan expects contiguous params")
                N.require_gpu(p, "Adan parameter")
                state = self.state[p]
                if len(state) == 0:
                    state["exp_avg"] = torch.zeros_like(p)
                    state["exp_avg_sq"] = torch.zeros_like(p)
                    state["exp_avg_diff"] = torch.zeros_like(p)
                    state["neg_pre_grad"] = torch.zeros_like(p)
                bufs = (state["exp_avg"], state["exp_avg_sq"], state["exp_avg_diff"],
                        state["neg_pre_grad"])
                if any(b.dtype != torch.float32 or not b.is_contiguous() for b in bufs):
                    raise ValueError("Adan expects contiguous float32 states")
                grad = p.grad
                if not (grad.dtype == torch.float32 and grad.device == p.device
                        and grad.is_contiguous()):
                    buf = state.get("_grad_buf")
                    if buf is None or buf.shape != p.shape:
                        buf = state["_grad_buf"] = torch.empty_like(p)
                    buf.copy_(grad)
                    grad = buf
                batches.setdefault(p.device.index, []).append(
                    (p, grad, *bufs, scalars, step == 1, no_prox))
        for dev, items in batches.items():
            for k in range(0, len(items), MAX_TENSORS_PER_LAUNCH):
                _adan_launch(dev, items[k:k + MAX_TENSORS_PER_LAUNCH],
                             None if clip is None else clip.data_ptr(), self._launch_args)
        return loss


def adan_step_from_grad_tilelang(param, grad, exp_avg, exp_avg_sq, exp_avg_diff, neg_pre_grad, *,
                                 step: int, lr: float = 1e-3, betas=(0.98, 0.92, 0.99),
                                 eps: float = 1e-8, weight_decay: float = 0.0,
                                 no_prox: bool = False, clip_global_grad_norm: float = 1.0,
                                 threads: int = DEFAULT_TILELANG_THREADS) -> None:
    """ops/optim.py:116-172: one Adan step in place from an external gradient
    (threads is accepted for the reference's signature)."""
    _ = threads
    beta1, beta2, beta3 = betas
    bc1 = 1.0 - beta1 ** step
    bc2 = 1.0 - beta2 ** step
    bc3 = 1.0 - beta3 ** step
    g = grad if grad.is_contiguous() else grad.contiguous()
    scalars = (float(beta1), float(beta2), float(beta3), float(bc1), float(bc2),
               float(bc3 ** 0.5), float(lr), float(weight_decay), float(eps),
               float(clip_global_grad_norm))
    _adan_launch(param.device.index,
                 [(param, g, exp_avg, exp_avg_sq, exp_avg_diff, neg_pre_grad, scalars,
                   int(step) == 1, bool(no_prox))], None)


# ------------------------------------------------------------------- AdamW

_ADAMW_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_EIGHT = 16                 # the bit of a table row's type for 8-bit states
_SET_SHIFT = 8
_P, _G, _MASTER, _AVG, _SQ, _NUMEL, _META, _NUMBER = range(8)   # columns of the table
_AVG8, _SQ8, _ORDER8 = "exp_avg_8bit", "exp_avg_sq_8bit", "order_8bit"


def _mix32(x):
    x &= 0xFFFFFFFF
    x ^= x >> 16
    x = (x * 0x9E3779B9) & 0xFFFFFFFF
    x ^= x >> 15
    x = (x * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _is_dense(t):
    """Whether t's elements fill one range of memory, each of them once."""
    if t.is_contiguous():
        return True
    run = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != run:
            return False
        run *= size
    return True


def _same_layout(a, b):
    """Whether two dense tensors of one shape lie in memory in the same order."""
    if a.is_contiguous() and b.is_contiguous():
        return True
    return all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _memory_order(t):
    """The dimensions of a dense tensor from the outermost in memory to the innermost,
    without those of size one; () for the logical order."""
    if t.is_contiguous():
        return ()
    return tuple(sorted((d for d in range(t.dim()) if t.shape[d] != 1),
                        key=lambda d: -t.stride(d)))


def _in_order(flat, shape, order):
    """A flat tensor whose values lie in the memory order `order`, as one of `shape`."""
    dims = [*order, *(d for d in range(len(shape)) if d not in order)]
    return flat.view([shape[d] for d in dims]).permute(
        sorted(range(len(dims)), key=dims.__getitem__))


def _codes_numel(numel):
    """Bytes of an 8-bit state: whole blocks of codes and a byte for each."""
    return -(-numel // N.ADAMW_BLOCK) * (N.ADAMW_BLOCK + 1)


def _same(a, b):
    """Whether two lists hold the same objects."""
    return len(a) == len(b) and all(map(is_, a, b))


class _Held:
    """State tensors and where each lies: their storage may be replaced (t.data =
    ..., as a program does that moves states off the GPU and back) while the
    objects stay."""
    __slots__ = ("tensors", "places", "address", "held")

    def __init__(self, tensors):
        self.tensors, ext = tuple(tensors), torchcall.module()
        self.held = None if ext is None else ext.adamw_held
        if ext is None:
            self.places = [self.place(t) for t in self.tensors]
        else:
            self.places = (ctypes.c_int64 * (4 * len(self.tensors)))()
            self.address = ctypes.addressof(self.places)
            ext.adamw_place(self.tensors, self.address)

    @staticmethod
    def place(t):
        return t.data_ptr(), t.dtype, t.layout, t.shape, t.stride()

    def same(self):
        if self.held is not None:
            return self.held(self.tensors, self.address)
        return [self.place(t) for t in self.tensors] == self.places


def _version_of(t):
    """What autograd counts of t's writes in place; tensors of inference mode have no count."""
    return 0 if t.is_inference() else t._version


class _Versions:
    """The version counters of the parameters when their masters last agreed with them."""

    def __init__(self, params):
        self.params = params
        self.values = np.zeros(len(params), dtype=np.int64)
        self.address, self.ext = self.values.ctypes.data, torchcall.module()

    def unwritten(self):
        """Whether no 16-bit parameter was written since."""
        if self.ext is not None:
            return self.ext.adamw_unwritten(self.params, self.address)
        return all(p.dtype is torch.float32 or _version_of(p) == v
                   for p, v in zip(self.params, self.values.tolist()))

    def count(self, entries):
        """A step has written the entries' parameters, which autograd does not know of."""
        if self.ext is not None and len(entries) == len(self.params):
            self.ext.adamw_written(self.params, self.address)
        else:
            # Views of one buffer share their counter, also with those that take no part.
            before = [_version_of(p) for p in self.params]
            agreed = self.values == before
            agreed[[e.place[0] for e in entries]] = True
            increment_version([e.p for e in entries])
            self.values[agreed] = np.array([_version_of(p) for p in self.params])[agreed]


def _copied(value):
    return value.detach().clone() if isinstance(value, torch.Tensor) else value


def _refuse_options(groups):
    """Options of torch's AdamW that change its update, wherever a group has them from."""
    for group in groups:
        get = group.get
        if get("amsgrad") or get("maximize") or get("differentiable"):
            option = next(o for o in ("amsgrad", "maximize", "differentiable") if get(o))
            raise NotImplementedError(f"repo_amd.optim.AdamW implements {option}=False")


class _AdamWEntry:
    """What the launches need of one parameter; remade when a tensor of it is
    another one, or lies elsewhere."""
    __slots__ = ("p", "st", "avg_key", "sq_key", "avg", "sq", "master", "step_t", "step", "row",
                 "ptr", "numel", "dtype", "device", "shape", "stride", "contiguous", "place", "held")

    def fresh(self):
        p, st = self.p, self.st
        try:
            return (p.data_ptr() == self.ptr and p.numel() == self.numel
                    and p.dtype is self.dtype
                    and (p.is_contiguous() if self.contiguous else p.stride() == self.stride)
                    and st[self.avg_key] is self.avg and st[self.sq_key] is self.sq
                    and st["step"] is self.step_t
                    and (self.master is None or st["master"] is self.master)
                    and self.held.same())
        except KeyError:
            return False


class _AdamWPlan:
    """The table of one device's launches, reused while the same parameters take
    part.  Each group has a set of its own as long as its parameters' step counts
    agree."""

    def __init__(self, version, entries, ngroups):
        self.version, self.entries, self.ngroups = version, entries, ngroups
        self.groups = [e.place[1] for e in entries]
        self.table = np.array([e.row for e in entries], dtype=np.int64).reshape(-1, 8)
        self.table[:, _NUMBER] = [e.place[0] for e in entries]
        self.address = self.table.ctypes.data
        self.grads = self.table[:, _G]
        self.metas = self.table[:, _META]
        self.types = self.metas.copy()
        self.by_group = self.types | (np.array(self.groups, np.int64) << _SET_SHIFT)
        self.metas[:] = self.by_group
        self.regular = True   # the sets are the groups'
        self.make_sets(ngroups)

    def set_steps(self, steps, regular):
        """Gives each row its set: its group's, or where the step counts of a group
        differ its (group, step) pair's.  The pairs of the sets in use."""
        if regular:
            if not self.regular:
                self.metas[:] = self.by_group
                self.make_sets(self.ngroups)
            self.regular = True
            return list(dict(zip(self.groups, steps)).items())
        pairs = list(zip(self.groups, steps))
        numbers = {}
        for pair in pairs:
            numbers.setdefault(pair, len(numbers))
        self.metas[:] = self.types | np.array([numbers[pair] << _SET_SHIFT for pair in pairs],
                                              np.int64)
        self.make_sets(len(numbers))
        self.regular = False
        return list(numbers)

    def make_sets(self, n):
        self.sets = np.zeros((n, 8), dtype=np.float32)
        self.keys = np.zeros(n, dtype=np.uint32)
        self.sets_address, self.keys_address = self.sets.ctypes.data, self.keys.ctypes.data


class _AdamWBulk:
    """All parameters at once, where each has a state and is contiguous, and all
    are on one device: a few calls of the extension look at every parameter, state
    and gradient (a step of 53 of them: 12 us of host time, where 53 that are not
    contiguous take 98 by their entries' own checks)."""

    def __init__(self, version, entries, ngroups):
        self.version, self.device, self.n = version, entries[0].device, len(entries)
        self.plan = _AdamWPlan(version, entries, ngroups)
        self.groups = sorted(set(self.plan.groups))
        self.step_tensors = [e.step_t for e in entries]
        self.steps = np.array([t.data_ptr() for t in self.step_tensors], dtype=np.int64)
        keys = [(e.avg_key, e.sq_key, "step") + (() if e.master is None else ("master",))
                for e in entries]
        self.args = ([e.p for e in entries], [e.st for e in entries], keys,
                     [tuple(e.st[key] for key in ks) for e, ks in zip(entries, keys)],
                     self.plan.address, self.steps.ctypes.data)
        self._current = torchcall.module().adamw_current
        self.held = _Held(chain.from_iterable(self.args[3]))

    def current(self, gradients):
        """The common step count, or 0 without gradients; -1 where anything changed.
        The step counts are read by their addresses, so where they lie comes first."""
        return self._current(*self.args, gradients) if self.held.same() else -1.0

    @staticmethod
    def of(version, order, ngroups):
        if torchcall.module() is not None and all(
                e is not None and e.contiguous and e.device == order[0].device for e in order):
            return _AdamWBulk(version, list(order), ngroups)
        return None


def _check_grad(g, p):
    if g.layout is not torch.strided:
        raise RuntimeError("AdamW does not support sparse gradients")
    if g.dtype is not p.dtype or g.device != p.device or g.shape != p.shape:
        raise ValueError(f"a gradient of {g.dtype} {tuple(g.shape)} on {g.device} beside a "
                         f"parameter of {p.dtype} {tuple(p.shape)} on {p.device}")


def global_grad_norm(grads):
    """The 2-norm over all gradients together, as a 0-d fp32 device tensor:
    squares summed in fp32 within a thread and in fp64 across them, in a fixed
    order, without a host read.  grads: fp32, bf16 and fp16 tensors of one
    device, of any strides; None entries are passed over."""
    held = []
    for g in grads:
        if g is None:
            continue
        if g.layout is not torch.strided:
            raise RuntimeError("global_grad_norm does not support sparse gradients")
        if g.dtype not in _ADAMW_DTYPES:
            raise ValueError(f"global_grad_norm takes float32, bfloat16 and float16, got {g.dtype}")
        N.require_gpu(g, "a gradient of global_grad_norm")
        if held and g.device != held[0].device:
            raise ValueError("global_grad_norm takes gradients of one device")
        held.append(g.detach() if _is_dense(g) else g.detach().contiguous())
    if not held:
        raise ValueError("global_grad_norm needs a gradient")
    table = np.zeros((len(held), 8), dtype=np.int64)
    table[:, _G] = [g.data_ptr() for g in held]
    table[:, _NUMEL] = [g.numel() for g in held]
    table[:, _META] = [_ADAMW_DTYPES[g.dtype] for g in held]
    with torch.cuda.device(held[0].device):
        return _norm_launch(table.ctypes.data, len(held), held[0].device, 0.0)[0]


def _norm_launch(address, n, device, max_norm):
    """Device (norm, clip factor) of the table's gradients."""
    out = torch.empty(2, dtype=torch.float32, device=device)
    partials = torch.empty(N.GRAD_NORM_BLOCKS + n, dtype=torch.float64, device=device)
    with N.prof("optim.grad_norm"):
        N.call("cs_grad_norm", n, address, max_norm, partials.data_ptr(), out.data_ptr(),
               N.stream(device))
    return out


class AdamW(torch.optim.Optimizer):
    """AdamW over all of a network's tensors (torch.optim.AdamW's update,
    amsgrad and maximize off), for fp32, bf16 and fp16 device parameters of any
    dense layout.

    ``state`` holds ``step`` (a CPU tensor), ``exp_avg`` and ``exp_avg_sq`` in
    fp32, as torch's does for fp32 parameters, so those checkpoints move between
    the two.  A 16-bit parameter has an fp32 copy ``master`` in its state; the
    update moves the copy, and the parameter is the copy rounded to nearest.  A
    parameter that is written in place between steps (``load_state_dict`` of the
    model, for one) is noticed by its version counter: where it is not the copy
    rounded, the copy takes its values.  Writes that leave the counter alone
    (through ``p.data``) are not noticed; whoever makes such deletes
    ``state[p]["master"]``, and the next step makes it anew.

    ``state_bits=8`` keeps both moments of a tensor of at least
    ``min_8bit_numel`` elements in a byte each (``exp_avg_8bit``,
    ``exp_avg_sq_8bit``): 4 exponent bits below the largest of 128 neighbours'
    and 3 (first moment, signed) or 4 (root of the second) mantissa bits, rounded
    stochastically with numbers that depend on ``seed``, the step, the tensor's
    place among the parameters and the element alone, so a run repeats bit for
    bit.  The codes lie in the parameter's memory order, which stands beside them
    (``order_8bit``, the dimensions from the outermost) where it is not the logical
    one.  load_state_dict takes states of either width and converts them, also
    those of a parameter that lies in another order.

    ``max_grad_norm`` > 0 scales all gradients by min(1, max_grad_norm / (norm +
    1e-6)) within the step, from the norm over all of them (``grad_norm``, a
    device tensor); the gradients themselves stay as they are."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 amsgrad=False, *, maximize=False, capturable=False, differentiable=False,
                 foreach=None, fused=None, state_bits=32, min_8bit_numel=4096,
                 max_grad_norm=0.0, seed=0):
        if not 0.0 <= float(lr):
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= float(eps):
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad or maximize or capturable or differentiable:
            raise NotImplementedError(
                "repo_amd.optim.AdamW implements amsgrad=False, maximize=False, "
                "capturable=False, differentiable=False")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not 0 <= min_8bit_numel:
            raise ValueError(f"Invalid min_8bit_numel: {min_8bit_numel}")
        if not 0.0 <= max_grad_norm:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        self.state_bits, self.min_8bit_numel = int(state_bits), int(min_8bit_numel)
        self.max_grad_norm, self.seed = float(max_grad_norm), int(seed)
        self._reset()
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False,
                        maximize=False, foreach=None, capturable=False, differentiable=False,
                        fused=None)
        super().__init__(params, defaults)

    def _reset(self):
        # Entries in the parameters' order (None: no state yet), with the lists
        # that they were made from, to notice a change of any.
        self._order, self._params, self._sizes, self._keys, self._values = [], [], [], [], []
        self._version, self._bulk, self._plans, self._flat, self._norm = 0, None, {}, None, None
        self._versions = _Versions([])

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits,
                "min_8bit_numel": self.min_8bit_numel, "max_grad_norm": self.max_grad_norm,
                "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._reset()

    zero_grad = Adam.zero_grad

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _refuse_options([param_group])
        super().add_param_group(param_group)

    @property
    def grad_norm(self):
        """The norm over all gradients before the last step's clip, a 0-d
        device tensor (None without max_grad_norm or before the first step)."""
        return None if self._norm is None else self._norm[0]

    # ---- state

    def _eight(self, numel):
        return self.state_bits == 8 and numel >= self.min_8bit_numel

    def _check_param(self, p):
        if p.dtype not in _ADAMW_DTYPES or not p.is_cuda or p.layout is not torch.strided:
            raise ValueError("repo_amd.optim.AdamW needs float32, bfloat16 or float16 CUDA (ROCm) "
                             f"parameters, got {p.dtype} on {p.device}")
        if not _is_dense(p):
            raise ValueError("repo_amd.optim.AdamW needs parameters that fill their memory, got "
                             f"shape {tuple(p.shape)} with strides {p.stride()}")

    def _init_state(self, p, st):
        if "step" not in st:
            st["step"] = torch.tensor(0.0, dtype=torch.float32)
        if self._eight(p.numel()):
            if _AVG8 not in st and _SQ8 not in st:
                self._set_order(p, st)
            for name in (_AVG8, _SQ8):
                if name not in st:
                    st[name] = torch.zeros(_codes_numel(p.numel()), dtype=torch.uint8,
                                           device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                if name not in st:
                    st[name] = torch.zeros_like(p, dtype=torch.float32,
                                                memory_format=torch.preserve_format)
        if p.dtype is not torch.float32 and "master" not in st:
            st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)

    @staticmethod
    def _set_order(p, st):
        """Codes lie in their parameter's memory order, which they do not show: it
        stands beside them, where it is not the logical one."""
        order = _memory_order(p)
        if order:
            st[_ORDER8] = order
        else:
            st.pop(_ORDER8, None)

    def _entry(self, number, k):
        """A new entry of parameter `number`, which is of group k."""
        p = self._params[number]
        self._version += 1
        self._check_param(p)
        st = self.state[p]
        eight = self._eight(p.numel())
        self._init_state(p, st)
        e = _AdamWEntry()
        e.place = (number, k)
        e.p, e.st, e.dtype, e.device = p, st, p.dtype, p.device
        e.ptr, e.numel, e.contiguous = p.data_ptr(), p.numel(), p.is_contiguous()
        e.shape, e.stride = p.shape, p.stride()
        e.avg_key, e.sq_key = (_AVG8, _SQ8) if eight else ("exp_avg", "exp_avg_sq")
        e.avg, e.sq = st[e.avg_key], st[e.sq_key]
        e.master = st.get("master") if p.dtype is not torch.float32 else None
        for t in (e.avg, e.sq, e.master):
            if t is None:
                continue
            if eight and t is not e.master:
                good = (t.dtype is torch.uint8 and t.numel() == _codes_numel(p.numel())
                        and t.is_contiguous())
            else:
                good = (t.dtype is torch.float32 and t.shape == p.shape and _is_dense(t)
                        and _same_layout(t, p))
            if not good or t.device != p.device:
                raise ValueError("an AdamW state does not fit its parameter: "
                                 f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on "
                                 f"{t.device} beside {tuple(p.shape)} with strides {p.stride()} on "
                                 f"{p.device}")
        old = self._order[number]
        if (e.master is not None and old is not None and old.master is e.master
                and (old.ptr != e.ptr or self._versions.values[number] != _version_of(p))):
            self._follow(e)
        self._versions.values[number] = _version_of(p)
        # Codes have no shape of their own: that of the parameter which they last were of.
        if eight and (tuple(st.get(_ORDER8, ())) != _memory_order(p) or (
                old is not None and old.avg is e.avg and old.shape != p.shape)):
            raise ValueError("an 8-bit AdamW state does not fit its parameter: it is of another "
                             f"memory order or shape than {tuple(p.shape)} with strides "
                             f"{p.stride()} (load_state_dict(state_dict()) brings it into a new "
                             "order)")
        step = st["step"]
        if not (isinstance(step, torch.Tensor) and step.device.type == "cpu"
                and step.dtype is torch.float32 and step.numel() == 1):
            step = st["step"] = torch.tensor(float(step), dtype=torch.float32)
        e.step_t, e.step = step, ctypes.c_float.from_address(step.data_ptr())
        e.row = [p.data_ptr(), 0, 0 if e.master is None else e.master.data_ptr(),
                 e.avg.data_ptr(), e.sq.data_ptr(), p.numel(),
                 _ADAMW_DTYPES[p.dtype] | (_EIGHT if eight else 0), 0]
        e.held = _Held(t for t in (e.avg, e.sq, e.step_t, e.master) if t is not None)
        self._order[number] = e
        return e

    @staticmethod
    @torch.no_grad()
    def _follow(e):
        """Where a 16-bit parameter is not its master rounded it has been written since:
        the master takes its values there."""
        p = e.p.detach()
        e.master.copy_(torch.where(e.master.to(p.dtype) == p, e.master, p.float()))

    def _entries(self):
        """The entries in the parameters' order, None where a parameter has none.
        An entry that is there may still have to be remade (`fresh`)."""
        groups, ext = self.param_groups, torchcall.module()
        if ext is not None and ext.adamw_unchanged(groups, self._params, self._sizes, self.state,
                                                   self._keys, self._values):
            return self._order
        params = [p for group in groups for p in group["params"]]
        sizes = [len(group["params"]) for group in groups]
        keys, values = list(self.state), list(self.state.values())
        if not (sizes == self._sizes and _same(params, self._params) and _same(keys, self._keys)
                and _same(values, self._values)):
            old = {id(e.p): e for e in self._order if e is not None}
            versions = self._versions.values
            self._order, self._versions = [], _Versions(params)
            for k, group in enumerate(groups):
                for p in group["params"]:
                    e = old.get(id(p))
                    if e is not None and e.st is self.state.get(p):
                        self._versions.values[len(self._order)] = versions[e.place[0]]
                        e.place = (len(self._order), k)
                    else:
                        e = None
                    self._order.append(e)
            self._params, self._sizes, self._keys, self._values = params, sizes, keys, values
            self._version += 1
        return self._order

    # ---- the step

    def step(self, closure=None):
        args, kwargs, closure = _run_pre_hooks(self, closure)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._step()
        self._optimizer_step_code()
        _run_post_hooks(self, args, kwargs)
        return loss

    step.hooked = True   # as Adam's: the hooks are called above

    def _step(self):
        # Gathered first: nothing is launched or counted if a tensor is refused.
        _refuse_options(self.param_groups)
        order = self._entries()
        bulk = self._bulk
        if bulk is not None and bulk.version == self._version:
            step = bulk.current(True) + 1.0
            if step > 0.0 and self._versions.unwritten():
                self._on(bulk.device, self._launch, bulk.device, bulk.plan,
                         [(k, step) for k in bulk.groups])
                torchcall.module().adamw_count(bulk.args[-1], bulk.n, step)
                self._versions.count(bulk.plan.entries)
                return
        work, number, regular = {}, -1, True
        written = not self._versions.unwritten()
        last, w = None, None
        for k, group in enumerate(self.param_groups):
            first = None
            for p in group["params"]:
                number += 1
                g = p.grad
                if g is None:
                    continue
                e = order[number]
                if e is None or not e.fresh():
                    e = self._entry(number, k)
                elif (written and e.master is not None
                      and self._versions.values[number] != _version_of(p)):
                    self._follow(e)
                    self._versions.values[number] = _version_of(p)
                _check_grad(g, p)
                if not (e.contiguous and g.is_contiguous()) and not (
                        _is_dense(g) and _same_layout(g, p)):
                    g = torch.empty_like(p).copy_(g.detach())
                step = e.step.value + 1.0
                if step != first:
                    regular = regular and first is None
                    first = step
                if e.device is not last:
                    last = e.device
                    w = work.setdefault(last, ([], [], []))
                w[0].append(e)
                w[1].append(g)
                w[2].append(step)
        if not work:
            return
        if len(self.state) != len(self._keys):   # states made just now
            self._keys, self._values = list(self.state), list(self.state.values())
        if self.max_grad_norm > 0 and len(work) > 1:
            raise NotImplementedError("max_grad_norm needs all parameters on one device")
        if bulk is None or bulk.version != self._version:
            self._bulk = _AdamWBulk.of(self._version, order, len(self.param_groups))
        for device, (entries, grads, steps) in work.items():
            plan = self._plans.get(device)
            if plan is None or plan.version != self._version or not _same(plan.entries, entries):
                plan = self._plans[device] = _AdamWPlan(self._version, entries,
                                                        len(self.param_groups))
            plan.grads[:] = [g.data_ptr() for g in grads]
            pairs = plan.set_steps(steps, regular)
            self._on(device, self._launch, device, plan, pairs)
            for e, step in zip(entries, steps):
                e.step.value = step
            self._versions.count(entries)

    @staticmethod
    def _on(device, launch, *args):
        if torch._C._cuda_isCurrentStreamCapturing():
            raise RuntimeError("an AdamW step counts on the host and cannot be captured")
        if device.index == torch._C._cuda_getDevice():
            launch(*args)
        else:
            with torch.cuda.device(device):
                launch(*args)

    def _launch(self, device, plan, pairs):
        """pairs: the (group, step) of each set in use."""
        sets, keys, groups = plan.sets, plan.keys, self.param_groups
        for i, (k, step) in enumerate(pairs):
            group = groups[k]
            beta1, beta2 = group["betas"]
            lr = float(group["lr"])
            i = k if plan.regular else i
            sets[i] = (1.0 - lr * group["weight_decay"], lr / (1.0 - beta1 ** step),
                       1.0 / math.sqrt(1.0 - beta2 ** step), 1.0 - beta1, beta2, 1.0 - beta2,
                       group["eps"], 0.0)
            keys[i] = _mix32(self.seed + int(step) * 0x3C6EF372)
        n, clip = len(plan.entries), None
        if self.max_grad_norm > 0:
            self._norm = _norm_launch(plan.address, n, device, self.max_grad_norm)
            clip = self._norm.data_ptr() + 4
        with N.prof("optim.adamw"):
            N.call("cs_adamw_step", n, plan.address, len(keys), plan.sets_address,
                   plan.keys_address, clip, N.stream(device))

    # ---- reading and loading

    def flat_state(self, dtype=torch.float32, align=1):
        """Both moments of all parameters, (exp_avg, exp_avg_sq), each as one
        flat tensor of ``dtype``: the parameters one after the other in the order
        of the groups, each in the order in which it lies in memory and beginning
        at a multiple of ``align`` elements, with zeros between them and for
        parameters that have taken no step.  8-bit states give the values that
        they stand for."""
        if dtype not in _ADAMW_DTYPES:
            raise ValueError(f"flat_state gives float32, bfloat16 and float16, got {dtype}")
        if align < 1:
            raise ValueError(f"Invalid align: {align}")
        order, bulk = self._entries(), self._bulk
        if (bulk is None or bulk.version != self._version
                or bulk.current(False) < 0.0):
            number, bulk = -1, None
            for k, group in enumerate(self.param_groups):
                for p in group["params"]:
                    number += 1
                    e = order[number]
                    if e is None or not e.fresh():
                        st = self.state.get(p)
                        if st and ("exp_avg" in st or _AVG8 in st):
                            self._entry(number, k)
                        else:
                            order[number] = None
        flat = self._flat
        kind = (dtype, align, self._version, None if bulk is not None else
                [p.numel() for p, e in zip(self._params, order) if e is None])
        if flat is None or flat[0] != kind or not (
                flat[1] is bulk if bulk is not None else _same(flat[2], order)):
            flat = self._flat = (kind, bulk, list(order), *self._flat_table(order, dtype, align))
        _, _, _, device, table, address, begins, total, bare = flat
        make = torch.zeros if bare else torch.empty
        out = (make(total, dtype=dtype, device=device), make(total, dtype=dtype, device=device))
        if len(table):
            np.add(begins, out[0].data_ptr(), out=table[:, _P])
            np.add(begins, out[1].data_ptr(), out=table[:, _G])
            args = ("cs_adamw_unpack_state", len(table), address, _ADAMW_DTYPES[dtype],
                    N.stream(device))
            if device.index == torch._C._cuda_getDevice():
                N.call(*args)
            else:
                with torch.cuda.device(device):
                    N.call(*args)
        return out

    def _flat_table(self, order, dtype, align):
        """Where flat_state's launch reads, and where in its outputs, in bytes, it writes."""
        device = self._params[0].device
        if any(p.device != device for p in self._params):
            raise NotImplementedError("flat_state needs all parameters on one device")
        padded = [-(-p.numel() // align) * align for p in self._params]
        begins = np.cumsum([0] + padded)
        here = [i for i, e in enumerate(order) if e is not None]
        table = np.array([order[i].row for i in here], dtype=np.int64).reshape(-1, 8)
        table[:, _META] &= _EIGHT
        # Up to the alignment only: a parameter without a state may follow.
        table[:, _MASTER] = [padded[i] for i in here]
        return (device, table, table.ctypes.data, begins[here] * dtype.itemsize, int(begins[-1]),
                any(n and e is None for n, e in zip(padded, order)))

    def load_state_dict(self, state_dict):
        """Takes states of either width, and of bf16 or fp16 (as torch's
        optimizers keep them beside 16-bit parameters), and holds them as this
        optimizer does.  torch's own loading would cast every state to its
        parameter's type, so only the groups and step counts go through it."""
        pre, post = (self._optimizer_load_state_dict_pre_hooks,
                     self._optimizer_load_state_dict_post_hooks)
        state_dict = state_dict.copy()
        for hook in pre.values():
            got = hook(self, state_dict)
            if got is not None:
                state_dict = got
        _refuse_options(state_dict["param_groups"])
        # torch's loading would keep the very tensors of the step counts.
        slim = {**state_dict, "state": {k: {"step": _copied(s["step"])} if "step" in s else {}
                                        for k, s in state_dict["state"].items()}}
        self._optimizer_load_state_dict_pre_hooks = type(pre)()
        self._optimizer_load_state_dict_post_hooks = type(post)()
        try:
            super().load_state_dict(slim)
        finally:
            self._optimizer_load_state_dict_pre_hooks = pre
            self._optimizer_load_state_dict_post_hooks = post
        ids = [k for group in state_dict["param_groups"] for k in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for k, p in zip(ids, params):
            if k in state_dict["state"]:
                self._take_state(p, state_dict["state"][k])
        # From here on writes to a parameter are told from what its master was loaded for.
        self._entries()
        number = -1
        for k, group in enumerate(self.param_groups):
            for p in group["params"]:
                number += 1
                if "master" in self.state.get(p, ()):
                    self._entry(number, k)
        for hook in post.values():
            hook(self)

    @torch.no_grad()
    def _take_state(self, p, given):
        self._check_param(p)
        st = self.state[p]
        eight = self._eight(p.numel())

        def fp32(t):
            if t.shape != p.shape:   # copy_ would broadcast it
                raise ValueError(f"an AdamW state does not fit its parameter: {tuple(t.shape)} "
                                 f"beside {tuple(p.shape)}")
            return torch.empty_like(p, dtype=torch.float32,
                                    memory_format=torch.preserve_format).copy_(t)

        for name, value in given.items():
            if name not in ("step", "exp_avg", "exp_avg_sq", _AVG8, _SQ8, _ORDER8, "master"):
                st[name] = value
        if given.get("master") is not None and p.dtype is not torch.float32:
            st["master"] = fp32(given["master"])
        if _AVG8 in given:
            codes = [given[name].to(p.device, copy=True) for name in (_AVG8, _SQ8)]
            if any(c.dtype is not torch.uint8 or c.numel() != _codes_numel(p.numel())
                   for c in codes):
                raise ValueError("8-bit AdamW states of another size than the parameter's")
            order = given.get(_ORDER8) or ()
            if order and not (isinstance(order, (tuple, list)) and sorted(order) == [
                    d for d in range(p.dim()) if p.shape[d] != 1]):
                raise ValueError(f"8-bit AdamW states in an order {order} of the dimensions of "
                                 f"{tuple(p.shape)}")
            same = tuple(order) == _memory_order(p)
            if eight and same:
                st[_AVG8], st[_SQ8] = codes
                self._set_order(p, st)
                return
            if same:
                avg, sq = (torch.empty_like(p, dtype=torch.float32,
                                            memory_format=torch.preserve_format) for _ in range(2))
            else:
                avg, sq = (torch.empty(p.numel(), dtype=torch.float32, device=p.device)
                           for _ in range(2))
            row = [avg.data_ptr(), sq.data_ptr(), p.numel(), codes[0].data_ptr(),
                   codes[1].data_ptr(), p.numel(), _EIGHT, 0]
            self._convert("cs_adamw_unpack_state", p, row, 0)
            if not same:
                avg, sq = (fp32(_in_order(t, p.shape, order)) for t in (avg, sq))
        elif "exp_avg" in given:
            avg, sq = fp32(given["exp_avg"]), fp32(given["exp_avg_sq"])
        else:
            return
        if not eight:
            st["exp_avg"], st["exp_avg_sq"] = avg, sq
            return
        self._init_state(p, st)
        row = [st[_AVG8].data_ptr(), st[_SQ8].data_ptr(), 0, avg.data_ptr(), sq.data_ptr(),
               p.numel(), 0, 0]
        self._convert("cs_adamw_pack_state", p, row)

    @staticmethod
    def _convert(name, p, row, *args):
        table = np.array([row], dtype=np.int64)
        with torch.cuda.device(p.device):
            N.call(name, 1, table.ctypes.data, *args, N.stream(p.device))

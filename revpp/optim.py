"""AdamW with gradient clipping over a stage's flat buffers, and the StepLR schedule.

Matches torch.optim.AdamW(lr, betas=(0.9, 0.999), eps=1e-6, weight_decay=0.01) preceded by
clip_grad_norm_(max_norm=1.0) (BERT/experiment/base.py:303-304, BERT/src/engine.py:56-67).
By default the norm is the stage's own (the reference clips each pipeline stage locally);
``global_clip`` all-reduces the squared norm over the pipeline first.

On CUDA the update is two kernels: a squared-norm reduction and one fused pass that
applies the clip coefficient (read on the device), the AdamW update, refreshes the bf16
shadow weights and zeroes the gradients.
"""
from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence

import torch
import torch.distributed as dist

from revpp.models.params import FlatParams


class FlatAdamW:
    def __init__(self, flat: FlatParams, lr: float, betas=(0.9, 0.999), eps: float = 1e-6,
                 weight_decay: float = 0.01, max_grad_norm: float = 1.0):
        self.flat = flat
        self.lr = lr
        self.beta1, self.beta2 = betas
        self.eps = eps
        self.weight_decay = weight_decay
        self.max_grad_norm = max_grad_norm
        self.kernels = flat.device.type == "cuda"
        if self.kernels:
            from revpp.ops import ext

            self._C = ext()
        self._sumsq = torch.zeros(1, dtype=torch.float32, device=flat.device)

    def grad_sumsq(self) -> torch.Tensor:
        """Squared L2 norm of the stage gradient, as a 1-element device tensor."""
        self._sumsq.zero_()
        if self.kernels:
            self._C.grad_sumsq(self.flat.grad, self._sumsq)
        else:
            self._sumsq.add_(self.flat.grad.double().pow(2).sum().float())
        return self._sumsq

    def step(self, sumsq: Optional[torch.Tensor] = None, zero_grad: bool = True) -> None:
        f = self.flat
        f.step += 1
        if self.max_grad_norm > 0 and sumsq is None:
            sumsq = self.grad_sumsq()
        if self.kernels:
            self._C.adamw_step(f.data, f.grad, f.exp_avg, f.exp_avg_sq, shadow=f.shadow, lr=self.lr,
                               beta1=self.beta1, beta2=self.beta2, eps=self.eps, wd=self.weight_decay, step=f.step,
                               max_norm=self.max_grad_norm, sumsq=sumsq if self.max_grad_norm > 0 else None,
                               zero_grad=zero_grad)
            return
        with torch.no_grad():
            g = f.grad
            if self.max_grad_norm > 0:
                norm = float(sumsq.sqrt())
                coef = min(1.0, self.max_grad_norm / (norm + 1e-6))
                g = g * coef
            f.data.mul_(1.0 - self.lr * self.weight_decay)
            f.exp_avg.lerp_(g, 1.0 - self.beta1)
            f.exp_avg_sq.mul_(self.beta2).addcmul_(g, g, value=1.0 - self.beta2)
            bc1 = 1.0 - self.beta1 ** f.step
            bc2 = 1.0 - self.beta2 ** f.step
            denom = (f.exp_avg_sq.sqrt() / math.sqrt(bc2)).add_(self.eps)
            f.data.addcdiv_(f.exp_avg, denom, value=-self.lr / bc1)
            f.refresh_shadow()
            if zero_grad:
                f.grad.zero_()

    def state_dict(self) -> dict:
        return {"lr": self.lr, **self.flat.state_dict()}

    def load_state_dict(self, sd: dict) -> None:
        self.lr = float(sd.get("lr", self.lr))
        self.flat.load_state_dict(sd)


class StepLR:
    """lr <- lr * gamma every ``step_size`` epochs (torch.optim.lr_scheduler.StepLR, step_size=1)."""

    def __init__(self, opt: FlatAdamW, step_size: int = 1, gamma: float = 1.0):
        self.opt = opt
        self.step_size = step_size
        self.gamma = gamma
        self.epoch = 0

    def step(self) -> None:
        self.epoch += 1
        if self.epoch % self.step_size == 0:
            self.opt.lr *= self.gamma


def _values(t: torch.Tensor) -> torch.Tensor:
    """The strided tensor that holds the numbers of ``t``."""
    if t.layout == torch.strided:
        return t
    return t._values() if t.layout == torch.sparse_coo else t.values()


def _layout(t: torch.Tensor):
    """Strides and sizes that count, the shortest stride first."""
    return sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1)


def _pieces(t: torch.Tensor):
    """Where the contiguous pieces of ``t`` start (bytes, ascending), and how many bytes each has."""
    dims, length, starts = _layout(t), 1, torch.zeros(1, dtype=torch.int64, device="cpu")
    while dims and dims[0][0] == length:
        length *= dims.pop(0)[1]
    for st, n in dims:
        starts = (starts[:, None] + st * torch.arange(n, device="cpu")).flatten()
    return t.data_ptr() + t.element_size() * starts.sort().values, t.element_size() * length


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors whose spans overlap have a byte in common."""
    if a.is_contiguous() and b.is_contiguous():
        return True
    (x, m), (y, n) = _pieces(a), _pieces(b)
    at = torch.searchsorted(y, x + m)  # pieces of b that start before each piece of a ends
    return bool(((at > 0) & (y[(at - 1).clamp_(min=0)] + n > x)).any())


def _check_apart(grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor]) -> None:
    """Refuses outputs that share memory with another output, themselves or a gradient that is not their own."""
    spans = []  # first byte, end, what it is, the tensor
    for i, (g, o) in enumerate(zip(map(_values, grads), map(_values, outs))):
        own = g.data_ptr() == o.data_ptr() and g.dtype == o.dtype and g.shape == o.shape and all(
            a == b for a, b, n in zip(g.stride(), o.stride(), g.shape) if n > 1)
        for name, t in (("out", o),) if own else (("out", o), ("gradient", g)):
            if t.numel():
                last = sum(st * (n - 1) for n, st in zip(t.shape, t.stride()))
                spans.append((t.data_ptr(), t.data_ptr() + t.element_size() * (last + 1), (name, i), t))
        if not o.is_contiguous():
            starts, length = _pieces(o)
            if (starts.diff() < length).any():
                raise ValueError(f"out {i} shares memory with itself: make it contiguous")
    spans.sort(key=lambda s: s[:3])
    reach = []  # earlier ones that end behind the present start
    for s in spans:
        reach = [a for a in reach if a[1] > s[0]]
        for a in reach:
            if "out" in (a[2][0], s[2][0]) and _share(a[3], s[3]):
                raise ValueError("{} {} shares memory with {} {}: an output must be its own gradient, or lie apart from "
                                 "all other tensors".format(*a[2], *s[2]))
        reach.append(s)


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None,
               norm_type: float = 2.0) -> torch.Tensor:
    """Clip separate gradient tensors by their global norm, as ``FlatAdamW`` does for a flat buffer.

    For parameters that live outside ``FlatParams`` (modules split by ``parallel.tracer``): scales every
    gradient by min(1, max_norm / (norm + 1e-6)), in place or into ``out`` (for instance the
    ``FlatParams.grad_of`` views), and returns the norm (fp32 scalar).  An output that shares memory with
    another one, or with a gradient that is not its own, is refused, and so is a None in the lists
    (parameters without a gradient have to be left out).  CUDA tensors go through the
    kernels (``ops.clip_grads``: fp32, bf16 and fp16), CPU tensors through PyTorch (float64 too)."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    if isinstance(grads[0], torch.Tensor) and grads[0].is_cuda:
        from revpp import ops

        return ops.clip_grads(grads, max_norm, out, norm_type)
    if norm_type not in (2.0, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"out must have one tensor per gradient: {len(outs)} for {len(grads)}")
    for name, tensors in (("gradient", grads), ("out", outs)):
        for i, t in enumerate(tensors):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} {i} is not a tensor: {type(t).__name__}")
            if not t.is_floating_point():
                raise ValueError(f"{name} {i} must be a floating-point tensor, got {t.dtype}")
            if t.device != grads[0].device:
                raise ValueError(f"all tensors must be on one device: {name} {i} is on {t.device}, gradient 0 on "
                                 f"{grads[0].device}")
    if any(o.shape != g.shape for o, g in zip(outs, grads)):
        raise ValueError("out must have its gradients' sizes")
    if not grads[0].is_meta:
        _check_apart(grads, outs)
    with torch.no_grad():
        full = [g.double() for g in grads if g.numel()]
        if norm_type == 2.0:
            norm = sum((g.square().sum() for g in full), torch.zeros((), dtype=torch.float64)).sqrt()
        else:
            norm = torch.stack([g.abs().max() for g in full]).max() if full else torch.zeros((), dtype=torch.float64)
        coef = (max_norm / (norm + 1e-6)).clamp(max=1.0)
        for g, o in zip(grads, outs):  # float64 gradients are scaled in 64 bits, the others in 32
            o.copy_(g * coef if g.dtype == torch.float64 else g.float() * coef.float())
    return norm.float()


def allreduce_sumsq(sumsq: torch.Tensor, group=None) -> torch.Tensor:
    """Global gradient norm across pipeline stages (``--global-clip``)."""
    if dist.is_available() and dist.is_initialized():
        dist.all_reduce(sumsq, op=dist.ReduceOp.SUM, group=group)
    return sumsq

"""The policy and preference losses of the training tape on the kernels of ``csrc/policy.cu``: rows of logits in, loss, terms and the
logits' gradient out."""
from __future__ import annotations

from ctypes import c_double as D
from typing import Optional

import torch

from . import native as N

N.register("trl_policy_loss", [N.P, N.I, N.L, N.L, N.P, N.P, N.P, N.L, N.P, N.P, D, D, D, D] + [N.P] * 6)
N.register("trl_preference_loss", [N.P, N.I, N.L, N.L, N.L, N.P, N.P, N.P, D, D, N.I, D] + [N.P] * 6)
N.register("trl_loss_scale", [N.P, N.I, N.P, N.L, N.P])

TYPES = {torch.float32: 0, torch.bfloat16: 1}


def there() -> bool:
    return N.has("trl_policy_loss")


def _rows(logits: torch.Tensor):
    """The logits as contiguous rows, and a gradient that lies as they do: vectors of 16 bytes begin at the same columns of both."""
    x = logits.contiguous()
    off = x.data_ptr() % 16 // x.element_size()
    return x, off


def _like(x: torch.Tensor, off: int) -> torch.Tensor:
    if not off:
        return torch.empty_like(x)
    return torch.empty(x.numel() + off, dtype=x.dtype, device=x.device)[off:].view(x.shape)


def policy(logits, targets, mask, adv, old, ref, *, lo: float, hi: float, kl: float, scale: float, want_grad: bool):
    """Loss, terms ``[4, rows]`` (log-probability, ratio, KL, weight), clipped rows and the gradient (or None).  All on one device:
    targets int64, mask bool or None, the rest fp32, contiguous; ``adv`` one value for every ``rows / len(adv)`` rows."""
    x, off = _rows(logits)
    v, n, new = x.shape[-1], targets.numel(), dict(device=x.device)
    with torch.cuda.device(x.device):
        terms, clipped, loss = torch.empty(4, n, **new), torch.empty(n, dtype=torch.bool, **new), torch.empty((), **new)
        work = torch.empty(2 * n, dtype=torch.float64, **new)
        grad = _like(x, off) if want_grad else None
        N.check(N.lib().trl_policy_loss(x.data_ptr(), TYPES[x.dtype], n, v, targets.data_ptr(), N.ptr(mask), adv.data_ptr(), n // adv.numel(), N.ptr(old),
                                        N.ptr(ref), lo, hi, kl, scale, terms.data_ptr(), clipped.data_ptr(), loss.data_ptr(), N.ptr(grad),
                                        work.data_ptr(), N.stream()), "policy_loss")
    N.count(3 if want_grad else 2)
    return loss, terms, clipped, grad


def preference(logits, targets, mask, ref: Optional[torch.Tensor], *, beta: float, smooth: float, average: bool, scale: float, want_grad: bool):
    """Loss, log-probabilities of the sequences, margins of the pairs and the gradient (or None); tensors as for :func:`policy`."""
    x, off = _rows(logits)
    v, n, (seqs, t), new = x.shape[-1], targets.numel(), targets.shape, dict(device=x.device)
    with torch.cuda.device(x.device):
        totals, margins, loss = torch.empty(seqs, **new), torch.empty(seqs // 2, **new), torch.empty((), **new)
        work = torch.empty(2 * n + 2 * seqs, dtype=torch.float64, **new)
        grad = _like(x, off) if want_grad else None
        N.check(N.lib().trl_preference_loss(x.data_ptr(), TYPES[x.dtype], seqs // 2, t, v, targets.data_ptr(), N.ptr(mask), N.ptr(ref), beta, smooth,
                                            int(average), scale, totals.data_ptr(), margins.data_ptr(), loss.data_ptr(), N.ptr(grad), work.data_ptr(),
                                            N.stream()), "preference_loss")
    N.count(4 if want_grad else 3)
    return loss, totals, margins, grad


def scale_grad(grad: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """The gradient times the loss's own, a number on the device, in place (nothing is touched where it is 1)."""
    with torch.cuda.device(grad.device):
        N.check(N.lib().trl_loss_scale(grad.data_ptr(), TYPES[grad.dtype], up.reshape(1).float().data_ptr(), grad.numel(), N.stream()), "loss_scale")
    torch.autograd.graph.increment_version(grad)
    N.count()
    return grad

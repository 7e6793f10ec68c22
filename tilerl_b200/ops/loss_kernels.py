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


def _like(x: torch.Tensor) -> torch.Tensor:
    """A gradient that lies as the logits do: vectors of 16 bytes begin at the same columns of both."""
    off = x.data_ptr() % 16 // x.element_size()
    return torch.empty_like(x) if not off else torch.empty(x.numel() + off, dtype=x.dtype, device=x.device)[off:].view(x.shape)


def policy(logits, targets, mask, adv, old, ref, *, lo: float, hi: float, kl: float, scale: float, want_grad: bool):
    """Loss, (log-probabilities, ratios, KL, weights) and clipped rows in the targets' shape, and the gradient (or None).  All contiguous and
    on one device: targets int64, mask bool or None, the rest fp32; ``adv`` one value for every ``rows / len(adv)`` rows."""
    x, n = logits.contiguous(), targets.numel()
    with N.on(x.device):
        # one piece of memory: what the kernels keep (n doubles), the terms, the loss
        some, clipped = torch.empty(6 * n + 1, dtype=torch.float32, device=x.device), torch.empty_like(targets, dtype=torch.bool)
        grad, at = _like(x) if want_grad else None, some.data_ptr()
        N.check(N.lib().trl_policy_loss(x.data_ptr(), TYPES[x.dtype], n, x.shape[-1], targets.data_ptr(), N.ptr(mask), adv.data_ptr(), n // adv.numel(),
                                        N.ptr(old), N.ptr(ref), lo, hi, kl, scale, at + 8 * n, clipped.data_ptr(), at + 24 * n, N.ptr(grad), at,
                                        N.stream()), "policy_loss")
    v = x.shape[-1]
    N.count(1 if v <= 4096 and n <= 64 >> max(0, (v - 1).bit_length() - 9) else 2)      # (up to eight blocks of short rows sum their losses themselves)
    return some[6 * n], some.as_strided((4, *targets.shape), (n, *targets.stride()), 2 * n).unbind(0), clipped, grad


def preference(logits, targets, mask, ref: Optional[torch.Tensor], *, beta: float, smooth: float, average: bool, scale: float, want_grad: bool):
    """Loss, log-probabilities of the sequences, margins of the pairs and the gradient (or None); tensors as for :func:`policy`."""
    x, n, (seqs, t) = logits.contiguous(), targets.numel(), targets.shape
    keep = 6 * n + 2 * seqs                             # floats that the kernels keep: of a row four for its gradient and its log-probability (fp64), of a pair its loss (fp64) and weights
    with N.on(x.device):
        some = torch.empty(keep + seqs + seqs // 2 + 1, dtype=torch.float32, device=x.device)
        grad, at = _like(x) if want_grad else None, some.data_ptr()
        N.check(N.lib().trl_preference_loss(x.data_ptr(), TYPES[x.dtype], seqs // 2, t, x.shape[-1], targets.data_ptr(), N.ptr(mask), N.ptr(ref), beta, smooth,
                                            int(average), scale, at + 4 * keep, at + 4 * (keep + seqs), at + 4 * (keep + seqs + seqs // 2), N.ptr(grad), at,
                                            N.stream()), "preference_loss")
    N.count(2 + int(want_grad) + int(seqs > 16))
    return some[-1], some[keep:keep + seqs], some[keep + seqs:-1], grad


def scale_grad(grad: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """The gradient times the loss's own, a number on the device, in place (nothing is touched where it is 1)."""
    with N.on(grad.device):
        N.check(N.lib().trl_loss_scale(grad.data_ptr(), TYPES[grad.dtype], up.reshape(1).float().data_ptr(), grad.numel(), N.stream()), "loss_scale")
    torch.autograd.graph.increment_version(grad)
    N.count()
    return grad

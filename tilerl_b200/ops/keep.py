"""Activations kept in 8 bits between the passes of a training step: groups of 128 values of a row with one fp32 scale each.

``scale = amax * (1 / 127)`` and ``q = rint(x * ((1 / amax) * 127))``, every quotient and product rounded to fp32, so the kernels of
``csrc/keep.cu`` and the torch forms give the same bytes.  A group with an infinity or NaN in it stands for NaN as a whole; one
whose largest magnitude is below 2^-120 is kept as zeros.  A value is off by at most half a step, ``amax / 254``."""
from __future__ import annotations

from typing import Tuple

import torch

from . import native as N

N.register("trl_keep_pack", [N.P] * 3 + [N.L, N.I, N.P])
N.register("trl_keep_unpack", [N.P] * 3 + [N.L, N.I, N.P])
N.register("trl_keep_swiglu", [N.P] * 4 + [N.L, N.I, N.P])
N.register("trl_keep_swiglu_grad", [N.P] * 4 + [N.L, N.I, N.P])

GROUP = 128
PART = float(torch.tensor(1.0) / torch.tensor(127.0))
LEAST = 2.0 ** -120
MOST = float.fromhex("0x1.020406p+121")      # the largest scale 127 times which is finite in fp32


def _empty(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    like = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    return like, torch.empty(*x.shape[:-1], -(-x.shape[-1] // GROUP), dtype=torch.float32, device=x.device)


def pack(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Torch form: ``x [..., W]`` -> int8 of its shape and scales ``[..., ceil(W / 128)]``."""
    w = x.shape[-1]
    if not x.numel():
        return _empty(x)
    y = torch.nn.functional.pad(x, (0, -w % GROUP)).reshape(*x.shape[:-1], -1, GROUP)
    most = y.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(most) & (most >= LEAST)
    q = torch.where(fine, torch.round(y * (most.reciprocal() * 127.0)), 0.0).to(torch.int8)
    scale = torch.where(torch.isfinite(most), torch.where(fine, (most * PART).clamp(max=MOST), 0.0), float("nan"))
    return q.reshape(*x.shape[:-1], -1)[..., :w].contiguous(), scale[..., 0]


def unpack(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Torch form of what packed rows stand for."""
    w = q.shape[-1]
    if not q.numel():
        return torch.empty(q.shape, dtype=torch.float32, device=q.device)
    y = torch.nn.functional.pad(q, (0, -w % GROUP)).reshape(*q.shape[:-1], -1, GROUP).float()
    return (y * scale[..., None]).reshape(*q.shape[:-1], -1)[..., :w].contiguous()


def _takes(x: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype == torch.float32 and x.numel() > 0 and x.shape[-1] < 1 << 31 and N.has("trl_keep_pack")


class Kept8:
    """Rows in 8 bits: ``q`` int8 of the rows' shape, ``scale`` fp32 ``[..., groups]``; ``rows()`` gives back what they stand for, in fp32."""
    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        self.q, self.scale = q, scale

    def nbytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()

    def rows(self) -> torch.Tensor:
        q = self.q
        if not (q.is_cuda and q.numel() and N.has("trl_keep_unpack")):
            return unpack(q, self.scale)
        with N.on(q.device):
            out = torch.empty_like(q, dtype=torch.float32)
            N.check(N.lib().trl_keep_unpack(q.data_ptr(), self.scale.data_ptr(), out.data_ptr(), q.numel() // q.shape[-1], q.shape[-1], N.stream()), "keep_unpack")
        N.count()
        return out


def keep8(x: torch.Tensor) -> Kept8:
    """``x [..., W]`` (fp32) in 8 bits."""
    if x.dtype != torch.float32 or x.dim() < 1:
        raise ValueError(f"keep8 takes fp32 rows, got {tuple(x.shape)} {x.dtype}")
    if not _takes(x):
        return Kept8(*pack(x))
    x = x.contiguous()
    with N.on(x.device):
        kept = Kept8(*_empty(x))
        N.check(N.lib().trl_keep_pack(x.data_ptr(), kept.q.data_ptr(), kept.scale.data_ptr(), x.numel() // x.shape[-1], x.shape[-1], N.stream()), "keep_pack")
    N.count()
    return kept


def swiglu_takes(gu: torch.Tensor) -> bool:
    return _takes(gu) and gu.shape[-1] % 2 == 0


def swiglu(gu: torch.Tensor) -> Tuple[torch.Tensor, Kept8]:
    """SwiGLU of interleaved (gate, up) pairs, and the pairs in 8 bits."""
    gu = gu.contiguous()
    with N.on(gu.device):
        out, kept = torch.empty(*gu.shape[:-1], gu.shape[-1] // 2, dtype=torch.float32, device=gu.device), Kept8(*_empty(gu))
        N.check(N.lib().trl_keep_swiglu(gu.data_ptr(), kept.q.data_ptr(), kept.scale.data_ptr(), out.data_ptr(), gu.numel() // gu.shape[-1], gu.shape[-1],
                                        N.stream()), "keep_swiglu")
    N.count()
    return out, kept


def swiglu_grad(kept: Kept8, g: torch.Tensor) -> torch.Tensor:
    g, q = g.float().contiguous(), kept.q
    with N.on(q.device):
        d = torch.empty_like(q, dtype=torch.float32)
        N.check(N.lib().trl_keep_swiglu_grad(q.data_ptr(), kept.scale.data_ptr(), g.data_ptr(), d.data_ptr(), q.numel() // q.shape[-1], q.shape[-1], N.stream()),
                "keep_swiglu_grad")
    N.count()
    return d

"""Log-probabilities of given tokens from hidden rows and the head, on the kernels of ``csrc/score.cu`` (tcgen05) or in torch."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import native as N
from . import ref

N.register("trl_score_workspace", [N.I] * 5, N.L)
N.register("trl_score", [N.P, N.I, N.P, N.P, N.P] + [N.I] * 3 + [N.P] * 4)

ROWS = 8192               # a call: the tiles' parts of as many rows over 248 320 words are 127 MB
CHUNK = 256               # rows of logits that the torch form has at a time


def takes(h: torch.Tensor, w: torch.Tensor) -> bool:
    """Rows of a multiple of eight values (a copy's rows begin on 16 bytes) and a head in bf16, as the training head is."""
    return (h.is_cuda and h.numel() > 0 and h.shape[-1] % 8 == 0 and h.dtype in (torch.float32, torch.bfloat16) and w.dtype == torch.bfloat16
            and w.shape[0] < 1 << 24 and N.has("trl_score"))


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def score(h, w, targets, mask, entropy: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``h [rows, H]``, ``targets`` int64 and ``mask`` (bool or None) ``[rows]``."""
    lib, (v, hidden) = N.lib(), w.shape
    with N.on(h.device):
        h, w = _aligned(h), _aligned(w)
        n, kind = h.shape[0], int(h.dtype == torch.bfloat16)
        lp = torch.empty(n, dtype=torch.float32, device=h.device)
        ent = torch.empty_like(lp) if entropy else None
        packed = int(mask is not None or not kind)
        for a in range(0, n, ROWS):
            m = min(n - a, ROWS)
            piece = (lambda t: t) if m == n else (lambda t: None if t is None else t[a:a + m])
            work = torch.empty(lib.trl_score_workspace(m, hidden, v, packed, int(entropy)), dtype=torch.uint8, device=h.device)
            N.check(lib.trl_score(piece(h).data_ptr(), kind, w.data_ptr(), piece(targets).data_ptr(), N.ptr(piece(mask)), m, hidden, v, piece(lp).data_ptr(),
                                  N.ptr(piece(ent)), work.data_ptr(), N.stream()), "score")
            N.count(2 + packed)
    return lp, ent


def score_torch(h, w, targets, mask, entropy: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The same in torch, a few rows of logits at a time; on the GPU with bf16 operands and fp32 results, on the CPU in fp32.  (The error word is the
    kernels'.)"""
    cd = torch.bfloat16 if h.is_cuda else torch.float64 if h.dtype == torch.float64 else torch.float32
    wide = torch.float64 if cd == torch.float64 else torch.float32
    wc = w.to(cd)
    lp = torch.zeros(h.shape[0], dtype=wide, device=h.device)
    ent = torch.zeros_like(lp) if entropy else None
    for a in range(0, h.shape[0], CHUNK):
        some = slice(a, a + CHUNK)
        x = h[some].to(cd).to(wide) @ wc.t().to(wide)
        tg, bad = ref.within(targets[some] if mask is None else torch.where(mask[some], targets[some], 0), x.shape[-1])
        m = x.amax(-1, keepdim=True)
        low = x - m
        e = torch.exp(low)
        s = e.sum(-1).double()
        got = low.gather(-1, tg[:, None])[:, 0].double() - torch.log(s)
        if bad is not None:
            got = torch.where(bad, float("nan"), got)
        lp[some] = (got if mask is None else torch.where(mask[some], got, 0.0)).to(wide)
        if entropy:
            got = torch.log(s) - torch.where(e > 0, e * low, 0.0).sum(-1).double() / s
            ent[some] = (got if mask is None else torch.where(mask[some], got, 0.0)).to(wide)
    return lp, ent

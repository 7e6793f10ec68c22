"""Checkpoint merging, streamed tensor by tensor: average, TIES, DARE and iso merges of
fine-tuned checkpoints relative to a base.

Parity: reference ``src/tilerl/merge.py`` (iso / ties / dare / average).
"""
from __future__ import annotations

import math
import os
from typing import Dict, List, Optional, Sequence

import torch

from .formats import INT8Tensor, keep_int8, quantize_int8


def merge_average(deltas: Sequence[torch.Tensor], weights: Optional[Sequence[float]] = None) -> torch.Tensor:
    w = weights or [1.0 / len(deltas)] * len(deltas)
    return sum(d * wi for d, wi in zip(deltas, w))


def merge_ties(deltas: Sequence[torch.Tensor], density: float = 0.2) -> torch.Tensor:
    """Trim each task vector to its top-``density`` magnitudes, elect a sign per element by
    total mass, and average the entries that agree with it."""
    trimmed = []
    for d in deltas:
        k = max(1, int(d.numel() * density))
        thr = d.abs().flatten().kthvalue(d.numel() - k + 1).values
        trimmed.append(torch.where(d.abs() >= thr, d, torch.zeros_like(d)))
    st = torch.stack(trimmed)
    sign = torch.sign(st.sum(0))
    agree = (torch.sign(st) == sign) & (st != 0)
    return (st * agree).sum(0) / agree.sum(0).clamp_min(1)


def merge_dare(deltas: Sequence[torch.Tensor], drop: float = 0.9, seed: int = 0) -> torch.Tensor:
    """Drop each delta entry with probability ``drop`` and rescale the rest by 1/(1-drop)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    out = torch.zeros_like(deltas[0])
    for d in deltas:
        keep = (torch.rand(d.shape, generator=g) >= drop).to(d.dtype).to(d.device)
        out += d * keep / (1.0 - drop)
    return out / len(deltas)


def merge_iso(deltas: Sequence[torch.Tensor]) -> torch.Tensor:
    """Isotropic merge: sum the task vectors, then flatten the spectrum of 2-D tensors to its
    mean singular value so no task dominates a direction."""
    s = sum(deltas)
    if s.dim() != 2 or min(s.shape) < 2:
        return s / len(deltas)
    u, sv, vh = torch.linalg.svd(s.float(), full_matrices=False)
    return (u * sv.mean()) @ vh


METHODS = {"average": merge_average, "ties": merge_ties, "dare": merge_dare, "iso": merge_iso}


def _integers(f) -> Dict[str, str]:
    """Projections in 8-bit integers of a file (own dialect, exports) and the names of their scales."""
    names, out = set(f.keys()), {}
    for name in names:
        for tail, of in ((".w8", ".wscale"), (".weight", ".weight_scale")):
            scale = name[:-len(tail)] + of
            if name.endswith(tail) and scale in names:
                w, n = f.get_slice(name), math.prod(f.get_slice(scale).get_shape())
                if w.get_dtype() == "I8" and len(w.get_shape()) == 2 and n in (1, w.get_shape()[0]):
                    out[name] = scale
    return out


def _int8(f, name: str, scale: str) -> INT8Tensor:
    w = f.get_tensor(name)
    return INT8Tensor(w, f.get_tensor(scale).float().reshape(-1).expand(w.shape[0]).contiguous())


def _dense(f, name: str, integers: Dict[str, str]) -> torch.Tensor:
    return _int8(f, name, integers[name]).dequant() if name in integers else f.get_tensor(name).float()


def merge_checkpoints(base: str, tuned: List[str], out: str, method: str = "average", **kw) -> int:
    """Stream safetensors files: ``out = base + merge(tuned_i - base)`` per tensor; projections in 8-bit integers by what they stand for."""
    from safetensors import safe_open
    from safetensors.torch import save_file
    fn = METHODS[method]
    f_base = safe_open(os.path.join(base, "model.safetensors"), framework="pt")
    f_tuned = [safe_open(os.path.join(t, "model.safetensors"), framework="pt") for t in tuned]
    result: Dict[str, torch.Tensor] = {}
    integers, tuned_integers = _integers(f_base), [_integers(f) for f in f_tuned]
    scales = set(integers.values())
    for name in f_base.keys():
        if name in scales:
            continue
        b = f_base.get_tensor(name)
        if name in integers:              # neither the integers nor the scales have deltas of their own
            scale = integers[name]
            result[name], result[scale] = b, f_base.get_tensor(scale)
            if all(name in i for i in tuned_integers):
                base_q = _int8(f_base, name, scale)
                dense = base_q.dequant()
                merged = dense + fn([_int8(f, name, scale).dequant() - dense for f in f_tuned], **kw)
                q = keep_int8(quantize_int8(merged), base_q, merged)
                result[name], result[scale] = q.w8, q.wscale
            continue
        if not b.dtype.is_floating_point or b.dtype == torch.float8_e4m3fn or any(name not in f.keys() for f in f_tuned):
            result[name] = b
            continue
        deltas = [_dense(f, name, i) - b.float() for f, i in zip(f_tuned, tuned_integers)]
        result[name] = (b.float() + fn(deltas, **kw)).to(b.dtype)
    os.makedirs(out, exist_ok=True)
    save_file(result, os.path.join(out, "model.safetensors"))
    return len(result)

"""Projections over weights in 8-bit integers (``formats.INT8Tensor``): ``csrc/rows_i8.cu``, ``csrc/gemm_i8.cu``.

Served (``linear``, behind the projections of :class:`~tilerl_b200.ops.cuda.CudaOps`): a tick's rows are quantised per token with the
RMSNorm folded in, multiplied in integers, and leave through the same epilogues as the other formats'.  Trained (``forward`` and
``grad``, behind ``tape.linear``): the same product of fp32 rows, not rounded, and its input's gradient from rows in 16 bits.

Sums are of integers, so neither the other rows of a batch nor the kernel that is taken for their number change a row's result: a
token has the same bits in a prompt, in a decode tick and in training.

The reference multiplies in FP8 (``linear_fp8``, packages/tilerl-kernels/src/tilerl_kernels/kernels_linear.py:1442-1813); it has no integer form.
"""
from __future__ import annotations

import threading
from typing import Dict, NamedTuple, Optional, Tuple

import torch

from ..formats import INT8Tensor
from . import native as N

EPI_STORE, EPI_RESIDUAL, EPI_SWIGLU, EPI_STORE_F32 = 0, 1, 2, 3
TYPES = {torch.float32: 0, torch.bfloat16: 1}
MOST = 131072             # values that a sum of 32 bits holds: 127 * 128 times as many is below 2^31 (a gradient's low digits: csrc/gemm_i8.cu)

N.register("trl_rows_i8", [N.P, N.I, N.L, N.P, N.I, N.F, N.P, N.L, N.P, N.L, N.I, N.I, N.P, N.P])
N.register("trl_linear_i8", [N.P, N.I, N.L, N.P, N.F, N.P, N.L, N.P, N.P, N.L, N.P, N.L, N.P, N.I, N.I, N.I, N.I, N.P])
N.register("trl_linear_i8_grad", [N.P, N.I, N.L, N.P, N.L, N.P, N.P, N.L, N.P, N.I, N.I, N.I, N.P])


def there() -> bool:
    """The library has these kernels (one that serves a single architecture has not)."""
    return N.has("trl_linear_i8")


class _Ready(NamedTuple):
    """A weight that the kernels read, looked over once."""
    w8: torch.Tensor
    wscale: torch.Tensor
    n: int
    k: int
    ptr: int
    ld: int
    scales: int
    device: int


def _ready(w: INT8Tensor) -> Optional[_Ready]:
    """Weights that the kernels read: rows of whole 16-byte pieces, on such a boundary, and sums that 32 bits hold."""
    r = w.__dict__.get("_ready")
    if r is not None and r.w8 is w.w8 and r.wscale is w.wscale and r.ptr == r.w8.data_ptr() and r.scales == r.wscale.data_ptr():
        return r
    w8, ws = w.w8, w.wscale
    n, k = w8.shape
    fits = (w8.is_cuda and ws.device == w8.device and ws.is_contiguous() and 0 < k <= MOST and 0 < n <= 1 << 24 and k % 16 == 0
            and w8.stride(1) == 1 and w8.stride(0) % 16 == 0 and w8.stride(0) >= k and w8.data_ptr() % 16 == 0)
    r = w.__dict__["_ready"] = _Ready(w8, ws, n, k, w8.data_ptr(), w8.stride(0), ws.data_ptr(), w8.get_device()) if fits else None
    return r


def takes(w: INT8Tensor) -> bool:
    return _ready(w) is not None


def _refuse_weight(w: INT8Tensor, who: str = "INT8 products take") -> None:
    raise ValueError(f"{who} weights with rows of a multiple of 16 values on 16-byte boundaries, of up to {MOST}, on "
                     f"a GPU with their scales, got {w.shape} with strides {tuple(w.w8.stride())} on {w.w8.device}")


def _refuse_rows(x, r: _Ready, norm_w) -> None:
    shape, k = x.shape, r.k
    if len(shape) != 2 or shape[1] != k or x.dtype not in TYPES or x.get_device() != r.device or x.stride(1) != 1 and k > 1:
        raise ValueError(f"INT8 products take fp32 or bf16 rows [T, {k}] on the weight's device, got {tuple(shape)} {x.dtype} on {x.device}")
    if norm_w is not None and (norm_w.shape != (k,) or norm_w.dtype != torch.float32 or norm_w.get_device() != r.device or not norm_w.is_contiguous()):
        raise ValueError(f"a norm's weight is fp32 [{k}] on the rows' device, got {tuple(norm_w.shape)} {norm_w.dtype} on {norm_w.device}")


def _width(r: _Ready, epi: int) -> int:
    if epi != EPI_SWIGLU:
        return r.n
    if r.n % 2:
        raise ValueError(f"SwiGLU takes rows in (gate, up) pairs, got {r.n}")
    return r.n // 2


def _crosses(y: torch.Tensor, residual: torch.Tensor) -> bool:
    """Whether a result is written over the residual of another one, which another thread may not have read yet.  (Two bf16 tensors of one shape;
    rows apart by different strides count as crossing wherever their ranges do.)"""
    (t, n), apart = y.shape, (residual.data_ptr() - y.data_ptr()) // 2
    ly, lr = (y.stride(0), residual.stride(0)) if t > 1 else (n, n)
    if not t or apart == 0 and ly == lr or apart >= (t - 1) * ly + n or apart + (t - 1) * lr + n <= 0:
        return False
    return ly != lr or apart % ly < n or ly - apart % ly < n


def _refuse_out(y, t: int, r: _Ready, residual, epi: int) -> None:
    width, kind, here = _width(r, epi), torch.float32 if epi == EPI_STORE_F32 else torch.bfloat16, r.device
    if y.shape != (t, width) or y.dtype != kind or y.get_device() != here or t and y.stride(1) != 1 and width > 1 or t > 1 and y.stride(0) < width:
        raise ValueError(f"the output of {t} rows by {r.n} channels is {kind} with channels side by side, got {tuple(y.shape)} {y.dtype} on {y.device}")
    if (epi == EPI_RESIDUAL) != (residual is not None) or residual is not None and residual is not y and (
            residual.shape != y.shape or residual.dtype != torch.bfloat16 or residual.get_device() != here or residual.stride(1) != 1 and r.n > 1):
        raise ValueError("a residual is bf16 rows of the output's shape, given where one is added")
    if residual is not None and residual is not y and _crosses(y, residual):
        raise ValueError("a residual lies where the output does, each value in the place of its own result, or apart from it")


def _scratch(rows: int, width: int, digits: int = 1) -> int:
    """Bytes that the kernels want for rows in 8 bits or in two digits: the integers, a scale a row, and of long rows in digits the largest of every
    2048 values."""
    if digits == 1:
        return rows * (width + 4)
    return rows * (2 * (-(-width // 16) * 16) + 4 + 4 * -(-width // 2048))


def quant_rows(x, q, s, *, norm_w=None, eps: float = 0.0, channels=None) -> None:
    """Rows ``x [T, K]`` into ``q`` (int8 ``[T, >= K]``) and ``s`` (fp32 ``[T]``); with ``channels`` (a gradient's scales) into two rows of digits
    a row of ``x``."""
    scratch = None if channels is None else torch.empty(x.shape[0] * -(-x.shape[1] // 2048), dtype=torch.int32, device=x.device)
    N.check(N.lib().trl_rows_i8(x.data_ptr(), TYPES[x.dtype], x.stride(0), N.ptr(channels if norm_w is None else norm_w), int(norm_w is not None), eps,
                                q.data_ptr(), q.stride(0), s.data_ptr(), x.shape[0], x.shape[1], 1 if channels is None else 2, N.ptr(scratch), N.stream()), "rows_i8")
    N.count()


def _product(x, r: _Ready, out, ldo, scratch, norm_w, eps, residual, epi) -> None:
    if r.device != N._device():
        with torch.cuda.device(r.device):
            return _product(x, r, out, ldo, scratch, norm_w, eps, residual, epi)
    rc = N.lib().trl_linear_i8(x.data_ptr(), TYPES[x.dtype], x.stride(0), None if norm_w is None else norm_w.data_ptr(), eps, r.ptr, r.ld, r.scales,
                               None if residual is None else residual.data_ptr(), 0 if residual is None else residual.stride(0), out.data_ptr(), ldo,
                               scratch.data_ptr(), x.shape[0], r.n, r.k, epi, N.stream())
    if rc >= 0:
        N.check(rc or -1, "linear_i8")
    N.count(-rc)


def _integers(ops, t: int, r: _Ready) -> torch.Tensor:
    """The backend's memory for a product's integers: its kernels run on the weight's device."""
    scratch = ops.ws.get("int8_rows", (_scratch(t, r.k),), torch.int8)
    if scratch.get_device() != r.device:
        raise ValueError(f"the weight is on {r.w8.device}, the backend's buffers on {scratch.device}")
    return scratch


def linear(ops, x, w, y, *, norm_w=None, eps=0.0, residual=None, epi=EPI_STORE) -> None:
    """``y = epi(norm(x) @ W^T)``; ``y`` may be the residual."""
    r = _ready(w)
    if r is None:
        _refuse_weight(w)
    _refuse_rows(x, r, norm_w)
    t = x.shape[0]
    _refuse_out(y, t, r, residual, epi)
    if t:
        _product(x, r, y, y.stride(0), _integers(ops, t, r), norm_w, eps, residual, epi)


def served(ops, name: str, x, w, norm_w, eps: float, epi: int = EPI_STORE) -> torch.Tensor:
    """``linear`` into the backend's own buffer ``name`` (bf16)."""
    r = _ready(w)
    if r is None:
        _refuse_weight(w)
    _refuse_rows(x, r, norm_w)
    t, width = x.shape[0], _width(r, epi)
    y = ops.ws.get(name, (t, width), torch.bfloat16)
    if y.get_device() != r.device:
        raise ValueError(f"the weight is on {w.w8.device}, the backend's buffers on {y.device}")
    if t:
        _product(x, r, y, width, _integers(ops, t, r), norm_w, eps, None, epi)
    return y


# ---- the training tape ------------------------------------------------------------------------------------
def train_takes(x: torch.Tensor, w: INT8Tensor) -> bool:
    """Rows that the kernels take as they are; the torch forms serve the rest (of so many channels that their sums could pass 32 bits, too)."""
    if not x.is_cuda or not there() or x.dtype not in TYPES or x.dim() < 1:
        return False
    r = _ready(w)
    return r is not None and x.get_device() == r.device and x.shape[-1] == r.k and r.n <= MOST


#: memory for the integers of short calls, for each thread and stream: (an allocation takes as long as a launch)
_KEPT = threading.local()
_KEEP = 4 << 20


def _workspace(rows: torch.Tensor, nbytes: int) -> torch.Tensor:
    """Memory that a call's kernels hand to each other.  Up to 4 MB is kept from call to call: calls of one thread on one stream run one
    after the other, while two threads may launch theirs in between each other.  A captured call has its own, as every other of its tensors."""
    if nbytes > _KEEP or _capturing():
        return rows.new_empty(nbytes, dtype=torch.int8)
    kept: Dict[Tuple[int, int], torch.Tensor] = _KEPT.__dict__
    key = (rows.get_device(), _raw_stream(rows.get_device()))
    t = kept.get(key)
    if t is None:
        t = kept[key] = rows.new_empty(_KEEP, dtype=torch.int8)
    return t


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
_raw_stream = N._raw_stream


def _flat(x: torch.Tensor, width: int) -> torch.Tensor:
    if x.requires_grad:
        x = x.detach()
    if x.dim() != 2:
        x = x.reshape(-1, width)
    return x if x.stride(1) == 1 else x.contiguous()


def forward(x: torch.Tensor, w: INT8Tensor) -> torch.Tensor:
    """``x [..., K]`` -> fp32 ``[..., N]``."""
    r = _ready(w)
    rows = _flat(x, r.k)
    t = rows.shape[0]
    out = rows.new_empty((t, r.n), dtype=torch.float32)
    if t:
        _product(rows, r, out, r.n, _workspace(rows, _scratch(t, r.k)), None, 0.0, None, EPI_STORE_F32)
    return out if x.dim() == 2 else out.view(*x.shape[:-1], r.n)


def grad(g: torch.Tensor, w: INT8Tensor) -> torch.Tensor:
    """Gradient of ``forward``'s input, the rounding of ``x`` taken for none: ``g [..., N]`` -> fp32 ``[..., K]``."""
    r = _ready(w)
    rows = _flat(g if g.dtype in TYPES else g.float(), r.n)
    t = rows.shape[0]
    dx = rows.new_empty((t, r.k), dtype=torch.float32)
    if t:
        _gradient(rows, r, dx, _workspace(rows, _scratch(t, r.n, 2)))
    return dx if g.dim() == 2 else dx.view(*g.shape[:-1], r.k)


def _gradient(rows, r: _Ready, dx, scratch) -> None:
    if r.device != N._device():
        with torch.cuda.device(r.device):
            return _gradient(rows, r, dx, scratch)
    N.check(N.lib().trl_linear_i8_grad(rows.data_ptr(), TYPES[rows.dtype], rows.stride(0), r.ptr, r.ld, r.scales, dx.data_ptr(), r.k, scratch.data_ptr(),
                                       rows.shape[0], r.n, r.k, N.stream()), "linear_i8_grad")
    N.count(2)


# ---- weights ---------------------------------------------------------------------------------------------------
def quantize_(src: torch.Tensor, dst: INT8Tensor) -> None:
    """fp32 or bf16 ``[N, K]`` into ``dst`` in place, as ``formats.quantize_int8`` gives it."""
    if not takes(dst):
        _refuse_weight(dst, "quantize_ takes")
    if src.shape != dst.w8.shape or src.dtype not in TYPES or src.device != dst.w8.device:
        raise ValueError(f"quantize_ takes fp32 or bf16 of {dst.shape} on the weight's device, got {tuple(src.shape)} {src.dtype} on {src.device}")
    src = src if src.stride(1) == 1 else src.contiguous()
    with N.on(src.device):
        quant_rows(src, dst.w8, dst.wscale)
    for t in (dst.w8, dst.wscale):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)

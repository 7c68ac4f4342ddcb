"""The global norm over many gradient tensors, and gradients clipped by it (csrc/grad_norm.cu).

    total = grad_norm(grads)                                  # 0-d tensor on the GPU, no host read
    total = clip_grad_norm_(model.parameters(), max_norm=1.0)  # torch.nn.utils.clip_grad_norm_'s call, in place
    clipped, total = clip_grads(grads, 1.0)                    # new tensors, the raw gradients kept

The Adam steps of gs_b200.adam take max_grad_norm and clip as they read the gradients, which saves writing them.

Tensors are float32, bfloat16, float16 or float64 CUDA tensors, mixed in one call, each dense in its own order of
dimensions (contiguous, transposed, channels-last), of any length and at any address. Sums are taken in float64 in an
order that follows from the list's lengths and types, the addresses modulo 16 bytes and the device, so a call on the
same tensors repeats bit for bit; copies at other addresses may differ in the last bits of the float64 sum. None of the
calls waits for the device (error_if_nonfinite apart), and all can be captured into a CUDA graph. Nothing is recorded
for autograd, except that tensors were written: as after torch's own in-place operations, a backward that needs their
old values raises.
"""
from __future__ import annotations

import math
from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib as L

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}  # SPLAT_F32 ... SPLAT_F64
_NORMS = {math.inf: 0, 1.0: 1, 2.0: 2}  # SPLAT_NORM_INF ...
NORM_GIVEN = 3  # SPLAT_NORM_GIVEN


def norm_code(norm_type) -> int:
    try:
        return _NORMS[float(norm_type)]
    except (KeyError, TypeError, ValueError):
        raise ValueError(f"norm_type must be 1, 2 or inf, got {norm_type!r}") from None


def check_max_norm(max_norm) -> float:
    value = float(max_norm)
    if not value >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm!r}")
    return value


def _dense(t: torch.Tensor) -> bool:
    """Every element of the tensor's memory range belongs to it once, in whatever order of dimensions."""
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _refuse(name: str, tensors: list) -> None:
    """Raises for the first tensor that the kernels do not take."""
    first = None
    for i, t in enumerate(tensors):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}[{i}] must be a tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{name}[{i}] must be a CUDA tensor")
        if t.layout != torch.strided or t.dtype not in _CODES:
            raise RuntimeError(f"{name}[{i}] must be a dense float32, bfloat16, float16 or float64 tensor, got "
                               f"{t.dtype} ({t.layout})")
        if t.is_neg():
            raise RuntimeError(f"{name}[{i}] is a view that negates its memory (of a conjugate): call resolve_neg()")
        if t.numel() and not t.is_contiguous() and not _dense(t):
            raise RuntimeError(f"{name}[{i}] must be dense (contiguous, or contiguous with its dimensions in another "
                               f"order), got shape {tuple(t.shape)} with strides {t.stride()}")
        first = t.device if first is None else first
        if t.device != first:
            raise RuntimeError(f"{name} must be on one device, got {first} and {t.device}")


_native = None


def _tensors():
    """The module that reads lists of tensors (csrc/tensor_list.cpp), loaded on first use."""
    global _native
    if _native is None:
        try:
            from . import _tensors as module
        except ImportError as e:
            raise RuntimeError("_tensors.so is not built; run `python 3dgs-project_b200/build.py` "
                               "(or __graft_entry__.build()) first") from e
        _native = module
    return _native


class Described(NamedTuple):
    """A list of tensors as the C ABI takes it."""

    addresses: bytes
    sizes: bytes
    codes: bytes
    device: int
    current: bool  # the device is the current one
    stream: int

    def call(self, function: str, *args) -> None:
        """The library launches on the current device: makes it the tensors'."""
        if self.current:
            L.call(function, *args, self.stream)
        else:
            with torch.cuda.device(self.device):
                L.call(function, *args, self.stream)


def describe(tensors: list) -> Described | None:
    """The list read for the C ABI, or None when the kernels do not take one of its entries."""
    got = _tensors().describe(tensors)
    return None if got is None else Described._make(got)


def _described(name: str, tensors: list) -> Described:
    d = describe(tensors)
    if d is None:
        _refuse(name, tensors)
        raise RuntimeError(f"{name} cannot be read as dense CUDA tensors")
    return d


def _listed(tensors) -> list:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return tensors if isinstance(tensors, (list, tuple)) else list(tensors)


TABLE = 1000  # tensors of one launch: the workspace grows by the launch


@lru_cache(maxsize=None)
def _workspace_bytes(tables: int) -> int:
    return L.query("splat_grad_workspace_size", tables * TABLE)


def scratch(device: int, count: int, f64: bool = False):
    """(norm, its address, workspace, its address, its bytes) for a call over `count` tensors; the workspace is to live
    until the call has returned."""
    size = _workspace_bytes((count + TABLE - 1) // TABLE)
    return (*_tensors().scratch(device, f64, size), size)


def adam_table(groups: list, lean: bool):
    """The groups as a clipped step's C call takes them, (table, device, current, stream), or None when it does not."""
    return _tensors().adam_table(groups, lean)


def written(entries) -> None:
    """Counts a write of the tensors (of a step's groups: of parameters and moments) for autograd."""
    _tensors().written(entries)


def _norm(d: Described, norm: int) -> torch.Tensor:
    f64 = 3 in d.codes
    count = len(d.codes)
    out, out_ptr, ws, ws_ptr, ws_bytes = scratch(d.device, count, f64)
    d.call("splat_grad_norm", count, d.addresses, d.sizes, d.codes, norm, out_ptr, f64, ws_ptr, ws_bytes)
    return out


def _check_finite(norm: torch.Tensor, norm_type) -> None:
    if not bool(torch.isfinite(norm)):
        raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite ({float(norm)}); pass "
                           "error_if_nonfinite=False to go on with it")


def grad_norm(grads, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The norm of all elements of the tensors as one vector: 0-d, float32 (float64 when one of them is float64), on
    their device. norm_type: 1, 2 or inf. NaN when an element is NaN. Squares of float64 elements leave float64's range
    beyond 1e154 (the norm is infinite) and below 1e-162 (they count as 0); those of the other types do not. No tensors:
    0 on the CPU, as torch's clipping gives. error_if_nonfinite raises for an infinite or NaN norm (which waits for the
    device)."""
    norm = norm_code(norm_type)
    tensors = _listed(grads)
    if not tensors:
        return torch.zeros(())
    total = _norm(_described("grads", tensors), norm)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    return total


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None, total_norm: torch.Tensor | None = None):
    """(clipped, total_norm): the gradients times min(1, max_norm / (total_norm + 1e-6)). The factor is taken in float64
    and rounded to float32 for all but float64 gradients; the product of a 16-bit gradient is taken in float32 and rounded
    to its type. A NaN norm makes them all NaN; an infinite one makes them 0, and NaN where they are infinite, unless
    max_norm is infinite too: then they are all NaN (as torch's clipping gives).

    out: the tensors to write, of the gradients' shapes, types and strides; they may not overlap the gradients or one
    another. None makes new ones; `out=grads` (or the same tensors) clips in place, where a norm below max_norm writes
    nothing. total_norm: a norm to clip by in place of the gradients' own (one element, float32 or float64, on their
    device: the norm over all ranks, say); it is returned."""
    norm, limit = norm_code(norm_type), check_max_norm(max_norm)
    tensors = _listed(grads)
    in_place = out is grads
    outs = None if out is None else tensors if in_place else _listed(out)
    if outs is not None and len(outs) != len(tensors):
        raise RuntimeError(f"out has {len(outs)} tensors for {len(tensors)} gradients")
    if not tensors:
        return [], torch.zeros(()) if total_norm is None else total_norm
    d = _described("grads", tensors)
    if outs is None:
        outs = [torch.empty_like(t) for t in tensors]
    to = d if in_place else _described("out", outs)
    if not in_place and (to.device != d.device or not _tensors().same_form(tensors, outs)):
        raise RuntimeError("out must have the gradients' shapes, types, strides and device")
    f64 = 3 in d.codes
    count = len(d.codes)
    if total_norm is None:
        total_norm, norm_ptr, ws, ws_ptr, ws_bytes = scratch(d.device, count, f64)
    else:
        L.check_cuda("total_norm", total_norm)
        if total_norm.dtype not in (torch.float32, torch.float64) or total_norm.numel() != 1 \
                or total_norm.get_device() != d.device:
            raise RuntimeError("total_norm must be one float32 or float64 value on the gradients' device")
        read = total_norm.detach().resolve_neg()
        read = read.double() if f64 else read
        f64 = read.dtype == torch.float64
        norm, norm_ptr, ws_ptr, ws_bytes = NORM_GIVEN, read.data_ptr(), None, 0
    d.call("splat_grad_clip", count, d.addresses, to.addresses, d.sizes, d.codes, norm, limit, norm_ptr, f64, ws_ptr,
           ws_bytes)
    if out is not None:
        written(outs)
    return list(outs), total_norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: bool | None = None) -> torch.Tensor:
    """Scales the parameters' gradients in place so that their norm together is at most max_norm, and returns the norm
    they had (torch.nn.utils.clip_grad_norm_'s call, for dense gradients on one CUDA device; foreach chooses between
    torch's implementations and changes nothing here). Parameters without a gradient are passed over; one gradient may
    not appear twice. error_if_nonfinite raises for an infinite or NaN norm, before anything is scaled (which waits
    for the device)."""
    norm_code(norm_type), check_max_norm(max_norm)
    grads = [p.grad for p in _listed(parameters) if p.grad is not None]
    if not error_if_nonfinite:
        return clip_grads(grads, max_norm, norm_type, out=grads)[1]
    return clip_grads(grads, max_norm, norm_type, out=grads, total_norm=grad_norm(grads, norm_type, True)
                      if grads else None)[1]

"""The global norm over many gradient tensors, and gradients clipped by it (csrc/grad_norm.cu).

    total = grad_norm(grads)                                  # 0-d tensor on the GPU, no host read
    total = clip_grad_norm_(model.parameters(), max_norm=1.0)  # torch.nn.utils.clip_grad_norm_'s call, in place
    clipped, total = clip_grads(grads, 1.0)                    # new tensors, the raw gradients kept

The Adam steps of gs_b200.adam take max_grad_norm and clip as they read the gradients, which saves writing them.

Tensors are float32, bfloat16, float16 or float64 CUDA tensors, mixed in one call, each dense in its own order of
dimensions (contiguous, transposed, channels-last), of any length and at any address. Sums are taken in float64 in an
order that the sizes fix, so a call repeats bit for bit. None of the calls waits for the device (error_if_nonfinite
apart), and all can be captured into a CUDA graph.
"""
from __future__ import annotations

import math
from array import array
from contextlib import nullcontext

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
        if t.numel() and not t.is_contiguous() and not _dense(t):
            raise RuntimeError(f"{name}[{i}] must be dense (contiguous, or contiguous with its dimensions in another "
                               f"order), got shape {tuple(t.shape)} with strides {t.stride()}")
        first = t.device if first is None else first
        if t.device != first:
            raise RuntimeError(f"{name} must be on one device, got {first} and {t.device}")


def _described(name: str, tensors: list) -> tuple[bytes, int]:
    """The tensors' type codes and their device index, or an exception for what the kernels do not take."""
    try:
        codes = bytes([_CODES[t.dtype] for t in tensors])
        devices = {t.get_device() for t in tensors}
        if len(devices) == 1 and min(devices) >= 0 and all([t.is_contiguous() for t in tensors]):
            return codes, devices.pop()
    except (AttributeError, KeyError, RuntimeError):
        pass
    _refuse(name, tensors)
    return codes, tensors[0].get_device()


def _listed(name: str, tensors) -> list:
    if isinstance(tensors, torch.Tensor):
        return [tensors]
    return list(tensors)


def _pointers(tensors: list) -> array:
    return array("Q", [t.data_ptr() for t in tensors])


def _sizes(tensors: list) -> array:
    return array("q", [t.numel() for t in tensors])


def _address(a: array) -> int:
    return a.buffer_info()[0]


def on_device(index: int):
    """The library launches on the current device: makes it the tensors'."""
    return nullcontext() if torch.cuda.current_device() == index else torch.cuda.device(index)


def norm_workspace(count: int, device) -> torch.Tensor:
    return L.workspace(L.query("splat_grad_workspace_size", count), device)


def _norm(tensors: list, codes: bytes, index: int, norm: int) -> torch.Tensor:
    device = tensors[0].device
    f64 = 3 in codes
    out = torch.empty((), dtype=torch.float64 if f64 else torch.float32, device=device)
    ws = norm_workspace(len(tensors), device)
    ptrs, sizes = _pointers(tensors), _sizes(tensors)
    with on_device(index):
        L.call("splat_grad_norm", len(tensors), _address(ptrs), _address(sizes), codes, norm, out.data_ptr(), f64,
               ws.data_ptr(), ws.numel(), L.stream_of(out))
    return out


def _check_finite(norm: torch.Tensor, norm_type) -> None:
    if not bool(torch.isfinite(norm)):
        raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite ({float(norm)}); pass "
                           "error_if_nonfinite=False to go on with it")


@torch.no_grad()
def grad_norm(grads, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """The norm of all elements of the tensors as one vector: 0-d, float32 (float64 when one of them is float64), on
    their device. norm_type: 1, 2 or inf. NaN when an element is NaN. No tensors: 0 on the CPU, as torch's clipping
    gives. error_if_nonfinite raises for an infinite or NaN norm (which waits for the device)."""
    norm = norm_code(norm_type)
    tensors = _listed("grads", grads)
    if not tensors:
        return torch.zeros(())
    total = _norm(tensors, *_described("grads", tensors), norm)
    if error_if_nonfinite:
        _check_finite(total, norm_type)
    return total


@torch.no_grad()
def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None, total_norm: torch.Tensor | None = None):
    """(clipped, total_norm): the gradients times min(1, max_norm / (total_norm + 1e-6)), each rounded once to its own
    type. A NaN norm makes them all NaN; an infinite one makes them 0, and NaN where they are infinite.

    out: the tensors to write, of the gradients' shapes, types and strides; they may not overlap the gradients or one
    another. None makes new ones; `out=grads` (or the same tensors) clips in place, where a norm below max_norm writes
    nothing. total_norm: a norm to clip by in place of the gradients' own (one element, float32 or float64, on their
    device: the norm over all ranks, say); it is returned."""
    norm, limit = norm_code(norm_type), check_max_norm(max_norm)
    tensors = _listed("grads", grads)
    outs = None if out is None else _listed("out", out)
    if outs is not None and len(outs) != len(tensors):
        raise RuntimeError(f"out has {len(outs)} tensors for {len(tensors)} gradients")
    if not tensors:
        return [], torch.zeros(()) if total_norm is None else total_norm
    codes, index = _described("grads", tensors)
    if outs is None:
        outs = [torch.empty_like(t) for t in tensors]
    elif any([o is not t for o, t in zip(outs, tensors)]):
        out_codes, out_index = _described("out", outs)
        if out_codes != codes or out_index != index or [o.shape for o in outs] != [t.shape for t in tensors]:
            raise RuntimeError("out must have the gradients' shapes, types and device")
        if [o.stride() for o in outs if o.numel()] != [t.stride() for t in tensors if t.numel()]:
            raise RuntimeError("out must have the gradients' strides")
    device = tensors[0].device
    f64 = 3 in codes
    given = total_norm is not None
    if given:
        L.check_cuda("total_norm", total_norm)
        if total_norm.dtype not in (torch.float32, torch.float64) or total_norm.numel() != 1 \
                or total_norm.device != device:
            raise RuntimeError("total_norm must be one float32 or float64 value on the gradients' device")
        read = total_norm.double() if f64 else total_norm
        f64 = read.dtype == torch.float64
        ws_ptr, ws_bytes = None, 0
    else:
        read = total_norm = torch.empty((), dtype=torch.float64 if f64 else torch.float32, device=device)
        ws = norm_workspace(len(tensors), device)
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    ptrs, out_ptrs, sizes = _pointers(tensors), _pointers(outs), _sizes(tensors)
    with on_device(index):
        L.call("splat_grad_clip", len(tensors), _address(ptrs), _address(out_ptrs), _address(sizes), codes,
               NORM_GIVEN if given else norm, limit, read.data_ptr(), f64, ws_ptr, ws_bytes, L.stream_of(tensors[0]))
    return outs, total_norm


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the parameters' gradients in place so that their norm together is at most max_norm, and returns the norm
    they had (torch.nn.utils.clip_grad_norm_'s call). Parameters without a gradient are passed over; one gradient may
    not appear twice. error_if_nonfinite raises for an infinite or NaN norm, before anything is scaled (which waits
    for the device)."""
    norm_code(norm_type), check_max_norm(max_norm)
    grads = [p.grad for p in _listed("parameters", parameters) if p.grad is not None]
    if not error_if_nonfinite:
        return clip_grads(grads, max_norm, norm_type, out=grads)[1]
    return clip_grads(grads, max_norm, norm_type, out=grads, total_norm=grad_norm(grads, norm_type, True)
                      if grads else None)[1]

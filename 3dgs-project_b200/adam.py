"""FusedAdam: Faster-GS's optimizer interface (cluster/patches/fastergs_lean_adam.patch:251-307) with every
parameter group updated by ONE launch of adam_step_multi (csrc/adam.cu) instead of one launch per group, and the
lean options of that patch (visibility-sparse update, bfloat16 moments) through adam_step_multi_lean.

State is the torch.optim.Adam layout ('step', 'exp_avg', 'exp_avg_sq' per parameter), so state_dict()
round-trips with torch's Adam and with checkpoints written by the reference's trainer.
"""
from __future__ import annotations

import ctypes
from contextlib import nullcontext

import torch

from . import _lib as L
from . import grad as gs_grad


class _Group(ctypes.Structure):
    """Mirror of adam_group in include/splat_b200.h."""

    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("exp_avg", ctypes.c_void_p),
                ("exp_avg_sq", ctypes.c_void_p), ("n", ctypes.c_longlong), ("lr", ctypes.c_double)]


class _LeanGroup(ctypes.Structure):
    """Mirror of adam_lean_group in include/splat_b200.h."""

    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("exp_avg", ctypes.c_void_p),
                ("exp_avg_sq", ctypes.c_void_p), ("n", ctypes.c_longlong), ("lr", ctypes.c_double),
                ("features", ctypes.c_int), ("lowp_moments", ctypes.c_int)]


MAX_GROUPS = 8


class FusedAdam(torch.optim.Adam):
    """Adam over single-tensor parameter groups, all groups in one kernel launch per step.

    The options of the reference's lean optimizer (cluster/patches/fastergs_lean_adam.patch:251-307), both off by
    default (then this is the original Faster-GS optimizer):
      sparse              only primitives visible in the last differentiable forward (n_touched_tiles > 0, handed
                          over by gs3d._Rasterize.last_visibility) are updated; the others keep their parameters
                          and moments for that step
      lowp_moment_groups  names of parameter groups whose exp_avg / exp_avg_sq are kept in bfloat16 (stochastic
                          rounding on write)
    and one of this build (off by default; with the dense update only):
      fuse_backward       when the six 3DGS tensors of a diff_rasterize call (means, scales, rotations, opacities,
                          sh0, sh_rest) are parameters of this optimizer, each alone in its group, the rasterizer's
                          backward leaves their preprocess backward to step(), which runs it fused with their Adam
                          update (gs3d_backward_preprocess_adam): their gradients are never written, so .grad stays
                          None for them after backward() unless other loss terms contributed (those gradients are
                          added inside the fused step). The parameters, moments and densification statistics are
                          bit-identical to the unfused path for one rendered view per step; with several views per
                          step all but the last are materialised into .grad when the next one arrives.
      max_grad_norm       step() applies the gradients scaled by min(1, max_grad_norm / (norm + 1e-6)), norm the global
                          norm of order grad_norm_type (1, 2 or inf) over every gradient of the step, which it leaves
                          in `grad_norm` (0-d, on the device; no host read). .grad keeps the raw gradients; the
                          update is that of grad.clip_grad_norm_ followed by the plain step, bit for bit. Not with
                          fuse_backward, whose gradients are never written.
    """

    def __init__(self, params, lr, eps, betas=(0.9, 0.999), sparse: bool = False,
                 lowp_moment_groups: tuple = (), fuse_backward: bool = False, max_grad_norm: float | None = None,
                 grad_norm_type: float = 2.0) -> None:
        if max_grad_norm is not None:
            max_grad_norm = gs_grad.check_max_norm(max_grad_norm)
            if fuse_backward:
                raise RuntimeError("max_grad_norm needs the gradients that fuse_backward does not write")
        gs_grad.norm_code(grad_norm_type)
        super().__init__(params=params, lr=lr, eps=eps, betas=betas)
        self.max_grad_norm = max_grad_norm
        self.grad_norm_type = grad_norm_type
        self.grad_norm: torch.Tensor | None = None  # of the last clipped step
        self.sparse = bool(sparse)
        self.lowp_moment_groups = set(lowp_moment_groups)
        self.lean = self.sparse or bool(self.lowp_moment_groups)
        self.n_dense_fallbacks = 0
        self.fuse_backward = bool(fuse_backward)
        self._pending = None  # (PendingBackward, the six parameter tensors)
        if self.fuse_backward and self.lean:
            raise RuntimeError("fuse_backward takes the dense update (no sparse / lowp_moment_groups)")
        from . import gs3d

        gs3d._Rasterize.track_visibility = self.sparse
        if self.fuse_backward:
            gs3d._Rasterize.fused_optimizer = self

    # ---- fused preprocess backward + Adam ----

    def _group_of(self, t: torch.Tensor):
        for group in self.param_groups:
            if len(group["params"]) == 1 and group["params"][0].data_ptr() == t.data_ptr() \
                    and group["params"][0].shape == t.shape:
                return group
        return None

    def _owns(self, six) -> bool:
        """True when the six rasterizer tensors are this optimizer's parameters (one per group, float32 CUDA,
        contiguous), so their preprocess backward can be deferred to step()."""
        if not self.fuse_backward:
            return False
        for t in six:
            if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()) or self._group_of(t) is None:
                return False
        return True

    def _defer(self, pending, six) -> None:
        if self._pending is not None:  # an earlier view of this step: its gradients go to .grad now
            earlier, tensors = self._pending
            grads = earlier.preprocess()
            for p, g in zip(self._params_of(tensors), grads):
                g = g.view(p.shape)
                p.grad = g if p.grad is None else p.grad + g
        self._pending = (pending, six)

    def _params_of(self, tensors):
        return [self._group_of(t)["params"][0] for t in tensors]

    def zero_grad(self, set_to_none: bool = True) -> None:  # noqa: D102
        self._pending = None
        super().zero_grad(set_to_none=set_to_none)

    @torch.no_grad()
    def _fused_step(self) -> set:
        pending, tensors = self._pending
        self._pending = None
        params = self._params_of(tensors)
        groups = [self._group_of(t) for t in tensors]
        exp_avg, exp_avg_sq, steps, lrs, grad_in = [], [], [], [], []
        for p, group in zip(params, groups):
            state = self.state[p]
            if len(state) == 0:
                state["step"] = torch.tensor(0.0)
                state["exp_avg"] = torch.zeros_like(p)
                state["exp_avg_sq"] = torch.zeros_like(p)
            state["step"] += 1
            exp_avg.append(state["exp_avg"])
            exp_avg_sq.append(state["exp_avg_sq"])
            steps.append(int(state["step"].item()))
            lrs.append(float(group["lr"]))
            grad_in.append(p.grad)
        b1, b2 = groups[0]["betas"]
        eps = groups[0]["eps"]
        for group in groups[1:]:
            if tuple(group["betas"]) != (b1, b2) or group["eps"] != eps:
                raise RuntimeError("fuse_backward needs the same betas and eps in the six groups")
        pending.preprocess_adam(params, exp_avg, exp_avg_sq, lrs, steps, (b1, b2), eps, grad_in)
        return {id(p) for p in params}

    @torch.no_grad()
    def step(self, closure=None) -> None:  # noqa: D102
        if closure is not None:
            raise RuntimeError("FusedAdam does not take a closure")
        if self.max_grad_norm is not None:
            self._check_clipped()
        done = self._fused_step() if self._pending is not None else set()
        visibility = None
        if self.sparse:
            from . import gs3d

            visibility = gs3d._Rasterize.last_visibility
        by_key: dict[tuple, list] = {}
        grads: list[torch.Tensor] = []  # in the parameters' order, which the clip's sums follow
        masks: dict[tuple, torch.Tensor | None] = {}
        for group in self.param_groups:
            if len(group["params"]) != 1:
                raise RuntimeError("more than one tensor in group")
            param = group["params"][0]
            if id(param) in done or param.grad is None or param.numel() == 0:
                continue
            L.check_cuda("param", param, torch.float32)
            lowp = group.get("name") in self.lowp_moment_groups
            moment_dtype = torch.bfloat16 if lowp else param.dtype
            state = self.state[param]
            if len(state) == 0:
                state["step"] = torch.tensor(0.0)
                state["exp_avg"] = torch.zeros_like(param, dtype=moment_dtype)
                state["exp_avg_sq"] = torch.zeros_like(param, dtype=moment_dtype)
            elif state["exp_avg"].dtype != moment_dtype:
                # densification concatenates float32 zeros to the moments, which promotes them; convert back
                state["exp_avg"] = state["exp_avg"].to(moment_dtype)
                state["exp_avg_sq"] = state["exp_avg_sq"].to(moment_dtype)
            grad = param.grad if param.grad.is_contiguous() else param.grad.contiguous()
            step = int(state["step"].item()) + 1
            if not self.lean:
                key = ("dense", step, *group["betas"], group["eps"], param.device)
                entry = _Group(param.data_ptr(), grad.data_ptr(), state["exp_avg"].data_ptr(),
                               state["exp_avg_sq"].data_ptr(), param.numel(), float(group["lr"]))
            else:
                vis = visibility
                if vis is not None and vis.numel() != param.shape[0]:
                    vis = None  # stale mask: this group falls back to the dense update
                    self.n_dense_fallbacks += 1
                key = ("lean", step, *group["betas"], group["eps"], param.device, None if vis is None else id(vis))
                masks[key] = vis
                entry = _LeanGroup(param.data_ptr(), grad.data_ptr(), state["exp_avg"].data_ptr(),
                                   state["exp_avg_sq"].data_ptr(), param.numel(), float(group["lr"]),
                                   param.numel() // max(param.shape[0], 1), int(lowp))
            entry._counter = state["step"]
            entry._updated = (param, grad, state["exp_avg"], state["exp_avg_sq"])
            grads.append(grad)
            by_key.setdefault(key, []).append(entry)
        clip = None
        if self.max_grad_norm is not None:
            clip = self._clip(grads, len(by_key) == 1 and len(grads) <= MAX_GROUPS)
        for key, groups in by_key.items():
            kind, step, b1, b2, eps, dev = key[:6]
            for s in range(0, len(groups), MAX_GROUPS):
                chunk = groups[s:s + MAX_GROUPS]
                _launch(kind == "lean", chunk, step, (b1, b2), eps, masks.get(key), dev, clip)
                for entry in chunk:  # a step that ran out of memory, or was refused, has not happened
                    entry._counter += 1
                if clip is not None:
                    gs_grad.written([entry._updated for entry in chunk])

    def _check_clipped(self) -> None:
        """The clipped step's limit, which a caller may set anew between steps, and gradients: one norm is taken over
        them, on one device."""
        gs_grad.check_max_norm(self.max_grad_norm)
        gs_grad.norm_code(self.grad_norm_type)
        devices = set()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    L.check_cuda("param", p, torch.float32)
                    if p.grad.dtype != torch.float32 or not p.grad.is_cuda or p.grad.layout != torch.strided:
                        raise RuntimeError("max_grad_norm needs dense float32 CUDA gradients")
                    if p.grad.is_neg():
                        raise RuntimeError("a gradient is a view that negates its memory: call resolve_neg()")
                    devices.add(p.device)
        if len(devices) > 1:
            raise RuntimeError("max_grad_norm needs the parameters on one device")

    def _clip(self, grads: list, in_step: bool):
        """The clip arguments of the step's launches. A step of one launch takes the norm itself (in_step); for several
        it is taken over all of their gradients first."""
        norm = gs_grad.norm_code(self.grad_norm_type)
        if not grads:
            self.grad_norm = torch.zeros(())
            return None
        if in_step:
            buffers = gs_grad.scratch(grads[0].get_device(), len(grads))
            self.grad_norm = buffers[0]
            return norm, float(self.max_grad_norm), buffers
        self.grad_norm = gs_grad.grad_norm(grads, self.grad_norm_type)
        return gs_grad.NORM_GIVEN, float(self.max_grad_norm), self.grad_norm


def _launch(lean: bool, groups: list, step: int, betas, eps: float, visibility, device, clip) -> None:
    """One launch over at most MAX_GROUPS entries; `clip` = (norm code, max_norm, grad.scratch()'s buffers,
    or with NORM_GIVEN the norm) or None."""
    arr = ((_LeanGroup if lean else _Group) * len(groups))(*groups)
    args = [len(groups), ctypes.addressof(arr), int(step), float(betas[0]), float(betas[1]), float(eps)]
    if lean:
        args += [L.ptr(visibility), 0 if visibility is None else visibility.numel()]
    name = "adam_step_multi_lean" if lean else "adam_step_multi"
    stream = torch.cuda.current_stream(device).cuda_stream
    if clip is None:
        L.call(name, *args, stream)
        return
    code, max_norm, norm = clip
    if code == gs_grad.NORM_GIVEN:
        norm_ptr, ws_ptr, ws_bytes = norm.data_ptr(), None, 0
    else:
        norm_ptr, ws_ptr, ws_bytes = norm[1], norm[3], norm[4]
    with torch.cuda.device(device):
        L.call(name + "_clipped", *args, code, max_norm, norm_ptr, ws_ptr, ws_bytes, stream)


def _refuse_groups(groups: list[tuple], lean: bool) -> None:
    """Raises for the first buffer that a clipped step does not take."""
    for i, (p, g, m, v, _) in enumerate(groups):
        moments = (torch.float32, torch.bfloat16) if lean else (torch.float32,)
        for name, t in (("param", p), ("grad", g), ("exp_avg", m), ("exp_avg_sq", v)):
            L.check_cuda(f"{name} of group {i}", t, torch.float32 if name in ("param", "grad") else None)
            if t.dtype not in moments or (t is v and t.dtype != m.dtype):
                raise RuntimeError(f"moments of group {i} must be float32" + (", or both bfloat16" if lean else
                                   " (adam_step_lean takes bfloat16 ones)"))
            if t.is_neg():
                raise RuntimeError(f"{name} of group {i} is a view that negates its memory: call resolve_neg()")
            if t.numel() != p.numel() or t.device != groups[0][0].device:
                raise RuntimeError(f"{name} of group {i} must have its parameter's size, on the first group's device")
    raise RuntimeError("the groups cannot be read as dense CUDA tensors")


def _clipped_step(groups: list[tuple], lean: bool, step: int, betas, eps: float, visibility, max_grad_norm,
                  norm_type) -> torch.Tensor:
    """adam_step / adam_step_lean with max_grad_norm: the buffers of all groups read and checked in one go."""
    code, limit = gs_grad.norm_code(norm_type), gs_grad.check_max_norm(max_grad_norm)
    read = gs_grad.adam_table(groups, lean)
    if read is None:  # a rate may be another kind of number
        held = [tuple(group) for group in groups]
        groups = [(p, g, m, v, float(lr)) for p, g, m, v, lr in held]
        read = gs_grad.adam_table(groups, lean)
    if read is None:
        _refuse_groups(groups, lean)
    table, device, current, stream = read
    norm, norm_ptr, ws, ws_ptr, ws_bytes = gs_grad.scratch(device, len(groups))
    args = [len(groups), table, int(step), float(betas[0]), float(betas[1]), float(eps)]
    if lean:
        args += [L.ptr(visibility), 0 if visibility is None else visibility.numel()]
    with nullcontext() if current else torch.cuda.device(device):
        L.call("adam_step_multi_lean_clipped" if lean else "adam_step_multi_clipped", *args, code, limit, norm_ptr,
               ws_ptr, ws_bytes, stream)
    gs_grad.written(groups)
    return norm


def adam_step(groups: list[tuple], step: int, betas=(0.9, 0.999), eps: float = 1e-15,
              max_grad_norm: float | None = None, norm_type: float = 2.0) -> torch.Tensor | None:
    """Functional form: groups = [(param, grad, exp_avg, exp_avg_sq, lr), ...] (CUDA float32, contiguous).

    With max_grad_norm the step takes the gradients times min(1, max_grad_norm / (norm + 1e-6)), norm the global norm
    of order norm_type (1, 2 or inf) over the groups' gradients, and returns the norm (0-d, on the device). The
    gradients keep their values, and may share no memory with what is written; nor may the groups, among themselves."""
    if not groups:
        return None if max_grad_norm is None else torch.zeros(())
    if max_grad_norm is not None:
        return _clipped_step(groups, False, step, betas, eps, None, max_grad_norm, norm_type)
    entries = [_Group(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(), float(lr))
               for p, g, m, v, lr in groups]
    _launch(False, entries, step, betas, eps, None, groups[0][0].device, None)
    return None


def adam_step_lean(groups: list[tuple], step: int, visibility: torch.Tensor | None = None, betas=(0.9, 0.999),
                   eps: float = 1e-15, max_grad_norm: float | None = None,
                   norm_type: float = 2.0) -> torch.Tensor | None:
    """Functional lean form (the reference's `_C.adam_step_sparse` for several groups at once): groups =
    [(param, grad, exp_avg, exp_avg_sq, lr), ...]; exp_avg / exp_avg_sq float32 or bfloat16 (stochastic rounding);
    visibility int32 [n_primitives] on the GPU or None. max_grad_norm and norm_type as in adam_step; the norm counts the
    gradients of primitives that are not visible too."""
    if not groups:
        return None if max_grad_norm is None else torch.zeros(())
    if visibility is not None and (visibility.dtype != torch.int32 or not visibility.is_cuda):
        raise RuntimeError("visibility must be int32 [n_primitives] on CUDA")
    if max_grad_norm is not None:
        if visibility is not None:
            L.check_cuda("visibility", visibility)
            if visibility.device != groups[0][0].device:
                raise RuntimeError("visibility must be on the groups' device")
        return _clipped_step(groups, True, step, betas, eps, visibility, max_grad_norm, norm_type)
    entries = []
    for p, g, m, v, lr in groups:
        if m.dtype != v.dtype or m.dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError("moments must share a dtype, float32 or bfloat16")
        entries.append(_LeanGroup(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(), float(lr),
                                  p.numel() // max(p.shape[0], 1), int(m.dtype == torch.bfloat16)))
    _launch(True, entries, step, betas, eps, visibility, groups[0][0].device, None)
    return None

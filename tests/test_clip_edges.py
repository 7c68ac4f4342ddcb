"""Edges of the gradient norm, the clipping and the clipped Adam steps that need no GPU."""
from __future__ import annotations

import ctypes
import importlib.util
import inspect
from array import array
from pathlib import Path

import numpy as np
import pytest
import torch

from gs_b200 import _lib as L
from gs_b200 import adam as A
from gs_b200 import grad as G
from oracle import adam_oracle as O

OK, ERR_ARG = 0, 1
P = 1 << 20  # an address that is never read: the calls below are refused, or have nothing to do


def test_rounding_keeps_what_is_not_finite():
    """The stochastic rounding to bfloat16 of NaN is NaN whatever the noise, of an infinity that infinity."""
    noise = np.arange(1 << 16, dtype=np.uint32)
    for bits in (0x7FFFFFFF, 0x7FC00000, 0x7F800001, 0xFFFFFFFF, 0xFFC00000):
        f = np.full(noise.size, bits, np.uint32).view(np.float32)
        assert np.isnan(O.bf16_bits_to_float(O.float_to_bf16_bits_sr(f, noise))).all()
    for sign in (1.0, -1.0):
        f = np.full(noise.size, sign * np.inf, np.float32)
        assert (O.bf16_bits_to_float(O.float_to_bf16_bits_sr(f, noise)) == sign * np.inf).all()


def _lean_step(groups, visibility=None, n_primitives=0):
    arr = (A._LeanGroup * len(groups))(*groups)
    return L.load().adam_step_multi_lean(len(groups), ctypes.addressof(arr), 1, 0.9, 0.999, 1e-15, visibility,
                                         n_primitives, None)


@pytest.mark.parametrize("features", [0, 1, 45])
def test_lean_groups_without_elements(features):
    """Rows of no elements, or no rows: nothing to do. A group with elements has rows of at least one."""
    empty = A._LeanGroup(None, None, None, None, 0, 1e-3, features, 1)
    assert _lean_step([empty, empty]) == OK
    assert _lean_step([empty], P, 0) == OK
    assert _lean_step([empty, A._LeanGroup(P, P, P, P, 4, 1e-3, 0, 0)]) == ERR_ARG
    assert "bad size" in L.load().splat_last_error().decode()
    assert _lean_step([A._LeanGroup(P, P, P, P, -4, 1e-3, 1, 0)]) == ERR_ARG


@pytest.mark.parametrize("entry", ["norm", "clip"])
@pytest.mark.parametrize("count,gib", [(1000, 70), (999, 70), (481, 70), (2, 20 * 1024), (100_000, 1)])
def test_lists_beyond_the_chunk_index(entry, count, gib):
    """A list may name a large tensor many times: past 32 TiB the index of its chunks no longer fits, nor would its
    launches' partials fit the workspace."""
    ptrs, sizes, codes = array("Q", [P] * count), array("q", [gib << 28] * count), bytes(count)
    args = [count, ptrs.buffer_info()[0]] + ([ptrs.buffer_info()[0]] if entry == "clip" else [])
    args += [sizes.buffer_info()[0], codes, 2] + ([1.0] if entry == "clip" else [])
    size = L.query("splat_grad_workspace_size", count)
    assert getattr(L.load(), f"splat_grad_{entry}")(*args, P, 0, P, size, None) == ERR_ARG
    assert "32 TiB" in L.load().splat_last_error().decode()


@pytest.fixture
def steps(monkeypatch):
    """FusedAdam on the CPU up to its launches, which are listed (step, groups, clip) instead of made."""
    made = []
    monkeypatch.setattr(A.L, "check_cuda", lambda name, t, dtype=None: t)
    monkeypatch.setattr(A.FusedAdam, "_check_clipped", lambda self: None)
    monkeypatch.setattr(A, "_launch", lambda lean, groups, step, betas, eps, visibility, device, clip:
                        made.append((step, len(groups), clip)))
    return made


@pytest.mark.parametrize("count", [2, 11])
def test_a_step_that_runs_out_of_memory_is_not_counted(monkeypatch, steps, count):
    """The buffers of the norm are had before the counters go on (count 11: a norm of its own, for several launches)."""
    params = [torch.nn.Parameter(torch.ones(3)) for _ in range(count)]
    for p in params:
        p.grad = torch.ones(3)
    opt = A.FusedAdam([{"params": [p]} for p in params], lr=1e-3, eps=1e-15, max_grad_norm=1.0)

    def full(*args):
        raise torch.OutOfMemoryError("no memory")

    with monkeypatch.context() as m:
        m.setattr(G, "scratch", full)
        m.setattr(G, "grad_norm", full)
        with pytest.raises(torch.OutOfMemoryError):
            opt.step()
    assert not steps and all(float(opt.state[p]["step"]) == 0 for p in params)
    norm = torch.zeros(())
    monkeypatch.setattr(G, "scratch", lambda *args: (norm, 0, None, 0, 0))
    monkeypatch.setattr(G, "grad_norm", lambda *args: norm)
    for n in (1, 2):
        steps.clear()
        opt.step()
        assert all(float(opt.state[p]["step"]) == n for p in params)
        assert [s[0] for s in steps] == [n] * len(steps) and sum(s[1] for s in steps) == count


@pytest.mark.parametrize("clip", [{}, {"max_grad_norm": 1.0}])
def test_a_launch_that_is_refused_is_not_counted(monkeypatch, steps, clip):
    params = [torch.nn.Parameter(torch.ones(3)) for _ in range(A.MAX_GROUPS + 3)]
    for p in params:
        p.grad = torch.ones(3)
    opt = A.FusedAdam([{"params": [p]} for p in params], lr=1e-3, eps=1e-15, **clip)
    monkeypatch.setattr(G, "grad_norm", lambda *args: torch.zeros(()))

    def second_fails(lean, groups, *args):
        if len(groups) < A.MAX_GROUPS:
            raise RuntimeError("refused")

    monkeypatch.setattr(A, "_launch", second_fails)
    before = [p._version for p in params]
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    written = [p._version - v for p, v in zip(params, before)]  # what was launched has been written all the same
    assert written == [1 if clip else 0] * A.MAX_GROUPS + [0] * 3
    assert [float(opt.state[p]["step"]) for p in params] == [1.0] * A.MAX_GROUPS + [0.0] * 3


def test_a_limit_set_between_steps_is_checked():
    opt = A.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, eps=1e-15, max_grad_norm=1.0)
    for bad in (-1.0, float("nan")):
        opt.max_grad_norm = bad
        with pytest.raises(ValueError):
            opt.step()
    opt.max_grad_norm, opt.grad_norm_type = 2, 3
    with pytest.raises(ValueError):
        opt.step()


def test_writes_are_counted_for_autograd():
    x, y, g = torch.zeros(3), torch.zeros(2, 2)[0], torch.ones(3)
    with torch.inference_mode():
        quiet = torch.zeros(3)
    G.written([x, y, quiet, "x"])
    assert x._version == 1 and y._version == 1
    G.written([(x, g, y, [1], 1e-3), [y, g]])
    assert x._version == 2 and y._version == 3 and g._version == 0
    G.written([])


def _clipped(lean, groups, norm=64 * P, norm_type=2):
    cls = A._LeanGroup if lean else A._Group
    arr = (cls * len(groups))(*[cls(*g, 1e-3, 1, int(lean)) if lean else cls(*g, 1e-3) for g in groups])
    head = (len(groups), ctypes.addressof(arr), 1, 0.9, 0.999, 1e-15)
    tail = (norm_type, 1.0, norm, 128 * P, 1 << 20, None)
    lib = L.load()
    return lib.adam_step_multi_lean_clipped(*head, None, 0, *tail) if lean else lib.adam_step_multi_clipped(*head, *tail)


FIRST, SECOND = (P, 2 * P, 3 * P, 4 * P, 64), (5 * P, 6 * P, 7 * P, 8 * P, 64)


@pytest.mark.parametrize("lean", [False, True])
@pytest.mark.parametrize("groups,kw", [
    ([(P, P, 3 * P, 4 * P, 64)], {}),                              # the gradient is the parameter
    ([(P, 3 * P + 64, 3 * P, 4 * P, 64)], {}),                     # lies in the first moment
    ([(P, 2 * P, 3 * P, 3 * P, 64)], {}),                          # one buffer for both moments
    ([FIRST, (P, *SECOND[1:])], {}),                               # one parameter in two groups
    ([FIRST, (P + 128, *SECOND[1:])], {}),                         # two that share elements
    ([FIRST, (5 * P, P + 240, *SECOND[2:])], {}),                  # a gradient inside the other group's parameter
    ([FIRST, (*SECOND[:2], 4 * P + 96, *SECOND[3:])], {}),
    ([FIRST, SECOND], {"norm": 2 * P + 16}),                       # the norm, written over a gradient
    ([FIRST, SECOND], {"norm": 5 * P, "norm_type": 3}),            # read from a parameter
])
def test_a_clipped_step_on_buffers_that_overlap(lean, groups, kw):
    # a moment's 64 elements have 128 bytes in the lean step here, 256 in the dense one
    assert _clipped(lean, groups, **kw) == ERR_ARG
    assert "overlaps" in L.load().splat_last_error().decode()


def test_the_call_of_torch():
    """clip_grad_norm_ takes what torch's takes, in torch's order."""
    ours, torchs = (list(inspect.signature(f).parameters.values())
                    for f in (G.clip_grad_norm_, torch.nn.utils.clip_grad_norm_))
    assert [(p.name, p.default) for p in ours] == [(p.name, p.default) for p in torchs]
    for foreach in (None, True, False):
        assert float(G.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0, foreach=foreach)) == 0.0


@pytest.fixture
def builder():
    path = Path(L.__file__).with_name("build.py")
    spec = importlib.util.spec_from_file_location("builder_under_test", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("absent", ["torch", "Python.h"])
def test_the_library_builds_without_torch(monkeypatch, tmp_path, capsys, builder, absent):
    """Without torch, or Python's headers, the C ABI library is built and the module that reads tensors is not."""
    monkeypatch.setattr(builder, "TENSORS", tmp_path / "_tensors.so")
    if absent == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name: None if name == "torch" else find(name))
    else:
        monkeypatch.setattr(builder.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert builder.build() == builder.LIB and builder.LIB.exists()
    assert not builder.TENSORS.exists() and f"{absent} is absent" in capsys.readouterr().err


def test_the_library_is_built_first(monkeypatch, builder):
    """A module that does not compile stops the build with an error that names it, after the library."""
    order = []
    monkeypatch.setattr(builder, "build_library", lambda *a: order.append("library"))

    def fails(*args):
        order.append("tensors")
        raise RuntimeError("g++ failed on tensor_list.cpp")

    monkeypatch.setattr(builder, "build_tensors", fails)
    with pytest.raises(RuntimeError, match="tensor_list.cpp"):
        builder.build()
    assert order == ["library", "tensors"]

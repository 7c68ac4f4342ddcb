"""The gradient-norm entry points without a GPU: what the C ABI and the Python layer refuse, before any device work, and
the memory orders that count as dense."""
from __future__ import annotations

import ctypes
import math
from array import array

import pytest
import torch

from gs_b200 import _lib as L
from gs_b200 import adam as A
from gs_b200 import grad as G

ERR_ARG = 1
P = 1 << 20  # an address that is never read: each call below is refused first


def _list(ptrs, sizes, codes):
    p, n = array("Q", ptrs), array("q", sizes)
    return p, n, bytes(codes)


def _norm(ptrs, sizes, codes, norm_type=2, norm=P, f64=0, ws=P, ws_bytes=1 << 20):
    p, n, c = _list(ptrs, sizes, codes)
    return L.load().splat_grad_norm(len(ptrs), p.buffer_info()[0], n.buffer_info()[0], c, norm_type, norm, f64, ws,
                                    ws_bytes, None)


def _clip(ptrs, outs, sizes, codes, norm_type=2, max_norm=1.0, norm=P, f64=0, ws=P, ws_bytes=1 << 20):
    p, n, c = _list(ptrs, sizes, codes)
    o = array("Q", outs)
    return L.load().splat_grad_clip(len(ptrs), p.buffer_info()[0], o.buffer_info()[0], n.buffer_info()[0], c, norm_type,
                                    max_norm, norm, f64, ws, ws_bytes, None)


def _error() -> str:
    return L.load().splat_last_error().decode()


@pytest.mark.parametrize("kw,says", [
    (dict(sizes=[-1]), "negative size"),
    (dict(codes=[4]), "unknown type"),
    (dict(sizes=[1 << 62]), "elements"),
    (dict(sizes=[(1 << 43) + 1]), "elements"),
    (dict(codes=[3]), "float64"),
    (dict(ptrs=[0]), "null buffer"),
    (dict(ptrs=[P + 2]), "not aligned"),
    (dict(ptrs=[P + 1], codes=[1]), "not aligned"),
    (dict(norm_type=3), "unknown norm type"),
    (dict(norm_type=-1), "unknown norm type"),
    (dict(norm=None), "norm's buffer"),
    (dict(norm=P + 2), "norm's buffer"),
    (dict(norm=P + 4, f64=1), "norm's buffer"),
    (dict(ws=None), "workspace"),
    (dict(ws=P + 4), "workspace"),
    (dict(ws_bytes=8), "workspace"),
])
def test_norm_refusals(kw, says):
    args = dict(ptrs=[P], sizes=[4], codes=[0])
    args.update(kw)
    assert _norm(**args) == ERR_ARG
    assert says in _error()


@pytest.mark.parametrize("kw,says", [
    (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=math.nan), "max_norm"),
    (dict(norm_type=4), "unknown norm type"),
    (dict(outs=[0, 8 * P]), "null"),
    (dict(outs=[P + 2, 8 * P]), "not aligned"),
    (dict(outs=[P, 8 * P]), "in place"),                        # one in place, one not
    (dict(outs=[P + 4, 8 * P]), "overlaps"),                     # an output inside its own input
    (dict(outs=[8 * P, 2 * P + 8]), "overlaps"),                 # an output inside an input
    (dict(outs=[8 * P, 8 * P + 60]), "overlaps"),                # two outputs
    (dict(ptrs=[P, P], outs=[P, P]), "overlaps"),                # the same tensor twice, in place
    (dict(ptrs=[P, P + 32], outs=[P, P + 32]), "overlaps"),      # tensors that share elements, in place
    (dict(ws=None), "workspace"),
    (dict(norm=8 * P + 8), "overlaps"),                          # the norm inside an output
    (dict(norm=2 * P + 8), "overlaps"),                          # written over an input
    (dict(norm=8 * P + 8, norm_type=3), "overlaps"),             # read from what is written
])
def test_clip_refusals(kw, says):
    args = dict(ptrs=[P, 2 * P], outs=[8 * P, 16 * P], sizes=[16, 16], codes=[0, 0])
    args.update(kw)
    assert _clip(**args) == ERR_ARG
    assert says in _error()


def test_many_tensors_that_overlap_are_found():
    n = 3000
    ptrs = [P + 64 * i for i in range(n)]
    ptrs[2500] = P + 64 * 17 + 4
    assert _clip(ptrs, ptrs, [16] * n, [0] * n) == ERR_ARG
    assert "overlaps" in _error()


@pytest.mark.parametrize("kw,says", [(dict(norm_type=9), "norm type"), (dict(max_norm=-0.5), "max_norm"),
                                     (dict(norm=None), "norm's buffer"), (dict(norm=P + 1), "norm's buffer"),
                                     (dict(ws=None), "workspace"), (dict(ws=P + 1), "workspace"), (dict(step=0), "step"), (dict(n=-1), "size")])
@pytest.mark.parametrize("lean", [False, True])
def test_clipped_step_refusals(lean, kw, says):
    a = dict(step=1, norm_type=2, max_norm=1.0, norm=P, ws=P, n=4)
    a.update(kw)
    cls = A._LeanGroup if lean else A._Group
    e = cls(P, P, P, P, a["n"], 1e-3, 1, 0) if lean else cls(P, P, P, P, a["n"], 1e-3)
    arr = (cls * 1)(e)
    head = (1, ctypes.addressof(arr), a["step"], 0.9, 0.999, 1e-15)
    tail = (a["norm_type"], a["max_norm"], a["norm"], a["ws"], 1 << 20, None)
    lib = L.load()
    status = lib.adam_step_multi_lean_clipped(*head, None, 0, *tail) if lean else lib.adam_step_multi_clipped(*head, *tail)
    assert status == ERR_ARG
    assert says in _error()


def test_workspace_grows_with_the_list():
    one = L.query("splat_grad_workspace_size", 1)
    assert L.query("splat_grad_workspace_size", 0) == one > 0
    assert L.query("splat_grad_workspace_size", 100_000) >= 100 * one


@pytest.mark.parametrize("bad", [0, 3, 2.5, "two", None, math.nan, -math.inf])
def test_norm_types(bad):
    with pytest.raises(ValueError):
        G.grad_norm([], bad)
    with pytest.raises(ValueError):
        G.clip_grads([], 1.0, bad)
    with pytest.raises(ValueError):
        A.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, eps=1e-15, max_grad_norm=1.0, grad_norm_type=bad)


@pytest.mark.parametrize("bad", [-1.0, math.nan, -math.inf])
def test_limits(bad):
    with pytest.raises(ValueError):
        G.clip_grads([], bad)
    with pytest.raises(ValueError):
        G.clip_grad_norm_([], bad)
    with pytest.raises(ValueError):
        A.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, eps=1e-15, max_grad_norm=bad)


def test_tensors_that_are_refused():
    for bad, kind in ((torch.zeros(3), RuntimeError), ("x", TypeError), (torch.zeros(2, 2).to_sparse(), RuntimeError),
                      (torch.zeros(3, dtype=torch.int32), RuntimeError)):
        with pytest.raises(kind):
            G.grad_norm([bad])
        with pytest.raises(kind):
            G.clip_grads([bad], 1.0)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        G.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="for 1 gradients"):
        G.clip_grads([p.grad], 1.0, out=[])
    with pytest.raises(RuntimeError, match="CUDA"):
        A.adam_step([(p.data, p.grad, p.grad, p.grad, 1e-3)], 1, max_grad_norm=1.0)
    opt = A.FusedAdam([p], lr=1e-3, eps=1e-15, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step()
    assert not opt.state  # refused before any state was made


def test_nothing_to_do():
    assert float(G.grad_norm([])) == 0.0
    assert float(G.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0  # no gradient
    out, total = G.clip_grads([], 1.0)
    assert out == [] and float(total) == 0.0
    assert A.adam_step([], 1) is None
    assert float(A.adam_step([], 1, max_grad_norm=1.0)) == 0.0
    assert float(A.adam_step_lean([], 1, max_grad_norm=1.0)) == 0.0
    opt = A.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, eps=1e-15, max_grad_norm=1.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0


def test_fuse_backward_is_refused():
    with pytest.raises(RuntimeError, match="fuse_backward"):
        A.FusedAdam([torch.nn.Parameter(torch.zeros(3))], lr=1e-3, eps=1e-15, fuse_backward=True, max_grad_norm=1.0)


def test_buffers_that_cannot_be_had():
    with pytest.raises(RuntimeError):
        G._tensors().scratch(0, False, 1 << 62)  # no such memory; without a GPU, no CUDA either
    with pytest.raises(TypeError):
        G._tensors().scratch(0, False)


def test_forms_that_agree():
    same = G._tensors().same_form
    x = torch.zeros(4, 5, 6)
    assert same([x], [torch.zeros(4, 5, 6)]) and same([], [])
    assert not same([x], [torch.zeros(4, 5, 7)]) and not same([x], [x.double()]) and not same([x], [x, x])
    assert not same([x.transpose(0, 1)], [torch.zeros(5, 4, 6)])
    assert same([x.transpose(0, 1)], [torch.ones(4, 5, 6).transpose(0, 1)])
    # the stride of a dimension with one entry says nothing
    a = torch.zeros(9, 1, 2).as_strided((2, 1, 9), (1, 7, 2))
    assert same([a], [torch.zeros(9, 1, 2).as_strided((2, 1, 9), (1, 2, 2))])
    assert not same([x], ["x"])


def test_dense_orders():
    x = torch.zeros(4, 5, 6)
    assert G._dense(x) and G._dense(x.permute(2, 0, 1)) and G._dense(torch.zeros(3, 1, 7).transpose(0, 2))
    assert G._dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))
    assert not G._dense(x[:, :, ::2]) and not G._dense(x[:, 1:]) and not G._dense(torch.zeros(1).expand(4))
    assert G._dense(x[1:]) and G._dense(torch.zeros(1)[0])

"""Edges of the gradient norm, the clipping and the clipped Adam steps on the GPU."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gs_b200 import adam as A
from gs_b200 import grad as G
from gs_b200 import gs3d

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SHAPES_3DGS = [(3,), (3,), (4,), (1,), (1, 3), (15, 3)]


def adam_state(n, device, seed, lowp=(), offset=0):
    """Groups of the six tensors of n 3D Gaussians, each `offset` elements behind the start of its allocation; moments
    of the groups in `lowp` in bfloat16."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def make(shape, scale, dtype=F32):
        flat = torch.empty(math.prod(shape) + offset, device=device, dtype=dtype)
        return flat[offset:].view(shape).copy_(torch.randn(shape, generator=gen, device=device) * scale)

    groups = []
    for k, s in enumerate(SHAPES_3DGS):
        dtype = BF16 if k in lowp else F32
        p, g = make((n, *s), 1.0), make((n, *s), 10.0 ** -k)
        groups.append((p, g, make((n, *s), 1e-2, dtype), make((n, *s), 1e-2, dtype).abs_(), 1e-3 * (k + 1)))
    return groups


def copies(groups):
    return [(p.clone(), g.clone(), m.clone(), v.clone(), lr) for p, g, m, v, lr in groups]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n", [1, 7, 301, 4096, 30_011])
def test_nan_in_bfloat16_moments(cuda, n, masked):
    """One NaN gradient makes the clip factor NaN: every element that is updated gets NaN moments, in bfloat16 as in
    float32, on vectors, their scalar ends and misaligned buffers, in one launch and in several. The elements that the
    mask leaves out keep what they had."""
    vis = None
    if masked:
        vis = (torch.rand(n, device=cuda, generator=torch.Generator(device=cuda).manual_seed(n)) < 0.5).int()
        vis[0] = 1
    for offset in (0, 1):
        a = adam_state(n, cuda, n, lowp=(1, 5), offset=offset)
        a[3][1][n // 2] = math.nan
        b = copies(a)
        assert math.isnan(float(A.adam_step_lean(a, 12, vis, max_grad_norm=1.0)))
        for x, y in zip(a, b):
            on = torch.ones(n, dtype=torch.bool, device=cuda) if vis is None else vis != 0
            for i in (0, 2, 3):
                assert bool(x[i][on].isnan().all()), (offset, x[0].shape, i)
                assert torch.equal(x[i][~on], y[i][~on])


def test_nan_in_bfloat16_moments_without_the_clip(cuda):
    """The same of the step that does not clip: NaN where the gradient is, nowhere else."""
    a = adam_state(5003, cuda, 3, lowp=(0, 1, 2, 3, 4, 5))
    at = torch.randint(0, 5003, (97,), device=cuda)
    for _, g, _, _, _ in a:
        g[at] = math.nan
    A.adam_step_lean(a, 5)
    for p, g, m, v, _ in a:
        for t in (p, m, v):
            assert torch.equal(t.isnan(), g.isnan())


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("clip", [{}, {"max_grad_norm": 0.05}])
def test_lean_groups_without_elements(cuda, clip, masked):
    """A model of SH degree 0 has no higher bases (n, 0, 3): the lean steps pass over that group."""
    n = 501
    vis = (torch.rand(n, device=cuda) < 0.4).int() if masked else None
    a = adam_state(n, cuda, 6, lowp=(4,))
    b = copies(a)
    none = torch.empty(n, 0, 3, device=cuda)
    low = none.bfloat16()
    total = A.adam_step_lean(a[:2] + [(none, none, low, low, 1e-3)] + a[2:], 4, vis, **clip)
    want = A.adam_step_lean(b, 4, vis, **clip)
    assert total is None if want is None else torch.equal(total, want)
    for x, y in zip(a, b):
        assert all(torch.equal(x[i], y[i]) for i in (0, 1, 2, 3))
    for rows in (0, n):  # nothing at all
        t = torch.empty(rows, 0, 3, device=cuda)
        seen = torch.zeros(rows, dtype=torch.int32, device=cuda) if masked else None
        total = A.adam_step_lean([(t, t, t, t, 1e-3)], 4, seen, **clip)
        assert total is None if not clip else float(total) == 0.0
    t = torch.empty(0, 3, device=cuda)  # no Gaussians
    total = A.adam_step_lean([(t, t, t, t, 1e-3)], 4, vis[:0] if masked else None, **clip)
    assert total is None if not clip else float(total) == 0.0


@pytest.mark.parametrize("call", ["clip", "step", "lean step"])
def test_the_cache_is_left_to_others(cuda, call):
    """After a call, passes over a buffer that fits the L2 are as fast as before it: the call holds no lines there. (With
    64 MiB held the passes took 1.17 to 1.19 times as long, for as long as nothing moved gigabytes; without, the times
    differ by 0.4%.)"""
    a = adam_state(300_000, cuda, 1)
    grads = [x[1] for x in a]
    outs = [torch.empty_like(g) for g in grads]
    seen = (torch.rand(300_000, device=cuda) < 0.35).int()
    calls = {"clip": lambda: G.clip_grads(grads, 0.05, out=outs), "step": lambda: A.adam_step(a, 5, max_grad_norm=0.05),
             "lean step": lambda: A.adam_step_lean(a, 5, seen, max_grad_norm=0.05)}
    buffer, total = torch.ones(20 << 20, device=cuda), torch.empty((), device=cuda)  # 80 MiB
    stream = torch.ones(1 << 30, device=cuda)

    def passes(before) -> float:
        times = []
        for _ in range(7):
            stream.add_(1.0)  # 8 GiB through the L2: nothing of an earlier call is left
            before()
            for _ in range(4):
                torch.sum(buffer, dim=0, out=total)
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(40):
                torch.sum(buffer, dim=0, out=total)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    calls[call]()
    assert passes(calls[call]) <= 1.1 * passes(lambda: None)


def test_a_backward_through_what_was_clipped_raises(cuda):
    """As after torch's clipping: a second derivative that needs the raw gradient must not take the clipped one."""
    x = torch.randn(2000, device=cuda, requires_grad=True)
    for call in (lambda: G.clip_grad_norm_([x], 0.1), lambda: G.clip_grads([x.grad.detach()], 0.1, out=[x.grad.detach()]),
                 lambda: G.clip_grad_norm_([x], 0.1, error_if_nonfinite=True)):
        x.grad, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
        again = (x.grad ** 2).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            again.backward()
    x.grad, = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    again = (x.grad ** 2).sum()
    want, = torch.autograd.grad(again, x, retain_graph=True)
    G.clip_grads([x.grad], 0.1)  # into new tensors: nothing is lost
    G.grad_norm([x.grad])
    second, = torch.autograd.grad(again, x)
    assert torch.equal(second, want)
    with torch.inference_mode():
        quiet = torch.randn(2000, device=cuda)
    G.clip_grads([quiet], 0.1, out=[quiet])


@pytest.mark.parametrize("lean", [False, True])
def test_a_backward_through_what_was_stepped_raises(cuda, lean):
    step = A.adam_step_lean if lean else A.adam_step
    groups = adam_state(50, cuda, 1)
    p = groups[0][0].requires_grad_()
    loss = (p ** 2).sum()
    step(groups, 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    p = torch.randn(50, 3, device=cuda, requires_grad=True)
    opt = A.FusedAdam([{"params": [p], "name": "p"}], lr=1e-3, eps=1e-15, max_grad_norm=1.0,
                      lowp_moment_groups=("p",) if lean else ())
    loss = (p ** 2).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("n", [512, 300_000])
def test_groups_side_by_side_in_memory(cuda, n):
    """Buffers that touch do not overlap, and two groups may take one gradient."""
    flat = torch.rand(7 * n, device=cuda) + 0.1
    p0, p1, m0, m1, v0, v1, g = flat.view(7, n)
    groups = [(p0, g, m0, v0, 1e-3), (p1, g, m1, v1, 1e-2)]
    other = copies(groups)
    total = A.adam_step(groups, 3, max_grad_norm=0.5)
    (a, b), want = G.clip_grads([x[1] for x in other], 0.5)
    A.adam_step([(x[0], c, *x[2:]) for x, c in zip(other, (a, b))], 3)
    assert torch.equal(total, want)
    for x, y in zip(groups, other):
        assert all(torch.equal(x[i], y[i]) for i in range(4))
    with pytest.raises(RuntimeError, match="overlaps"):
        A.adam_step([(p0, p0, m0, v0, 1e-3)], 3, max_grad_norm=0.5)


def test_rates_of_other_kinds(cuda):
    """A rate is anything that float() takes; what its conversion does to the caller's list changes nothing."""

    class Rate:
        def __float__(self):
            groups.clear()
            return 2e-3

    want = adam_state(100, cuda, 2)[:3]
    A.adam_step([(*x[:4], lr) for x, lr in zip(want, (1.0, 2e-3, 0.5))], 2, max_grad_norm=0.1)
    for rates in ((1, Rate(), 0.5), (torch.ones((), device=cuda), np.float64(2e-3), np.float32(0.5))):
        kept = adam_state(100, cuda, 2)[:3]
        groups = [[*x[:4], lr] for x, lr in zip(kept, rates)]
        A.adam_step(groups, 2, max_grad_norm=0.1)
        for x, y in zip(kept, want):
            assert all(torch.equal(x[i], y[i]) for i in range(4))
    with pytest.raises((TypeError, ValueError)):
        A.adam_step([(*want[0][:4], "fast")], 2, max_grad_norm=0.1)


def test_views_that_negate_their_memory(cuda):
    """The imaginary part of a lazy conjugate: its memory holds the values of the other sign."""
    z = torch.complex(torch.ones(1, device=cuda), torch.full((1,), 2.0, device=cuda))
    g, plain = z.conj().imag, torch.ones(1, device=cuda)
    assert g.is_neg() and g.is_contiguous() and float(g) == -2.0
    for call in (lambda: G.grad_norm([g]), lambda: G.clip_grads([g], 1.0), lambda: G.clip_grads([plain], 1.0, out=[g]),
                 lambda: A.adam_step([(plain, g, plain.clone(), plain.clone(), 1e-3)], 1, max_grad_norm=1.0)):
        with pytest.raises(RuntimeError, match="negates"):
            call()
    assert float(G.clip_grads([g.resolve_neg()], 1.0)[0][0]) == pytest.approx(-1.0, rel=1e-5)
    p = torch.ones(1, device=cuda, requires_grad=True)
    p.grad = g
    opt = A.FusedAdam([{"params": [p]}], lr=1e-3, eps=1e-15, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="negates"):
        opt.step()
    total = torch.complex(plain, -4.0 * plain).conj().imag  # 4
    assert float(G.clip_grads([plain], 1.0, total_norm=total)[0][0]) == pytest.approx(0.25, rel=1e-5)


@pytest.mark.parametrize("p", [1.0, 2.0])
@pytest.mark.parametrize("n", [900, 60_000, 3_000_017])
def test_every_bit_of_a_float64_norm_repeats(cuda, n, p):
    """One launch, and several: the same tensors give the same float64 sum, through every entry point that takes it."""
    gen = torch.Generator(device=cuda).manual_seed(n)
    grads = [torch.randn(n, generator=gen, device=cuda), torch.randn(n // 3, generator=gen, device=cuda).half()[1:],
             torch.randn(7, generator=gen, device=cuda, dtype=torch.float64)]
    first = G.grad_norm(grads, p)
    assert first.dtype == torch.float64
    outs = [torch.empty_like(g) for g in grads]
    for _ in range(5):
        assert torch.equal(G.grad_norm(grads, p), first)
        assert torch.equal(G.clip_grads(grads, 0.1, p, out=outs)[1], first)


def test_limits_and_norms_at_the_ends_of_the_range(cuda):
    g = torch.tensor([1.0, math.inf, -2.0], device=cuda)
    outs, total = G.clip_grads([g], math.inf)
    assert float(total) == math.inf and bool(outs[0].isnan().all())  # inf / inf, as torch's clipping
    other = torch.nn.Parameter(torch.zeros(3, device=cuda))
    other.grad = g.clone()
    torch.nn.utils.clip_grad_norm_(other, math.inf)
    assert torch.equal(other.grad.isnan(), outs[0].isnan())
    tiny = torch.full((4,), 1e-170, device=cuda, dtype=torch.float64)
    assert float(G.grad_norm([tiny])) == 0.0 and float(G.grad_norm([tiny], 1.0)) > 0.0
    assert float(G.grad_norm([tiny * 1e15])) == pytest.approx(2e-155, rel=1e-12)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("n", [3, 4096, 30_011])
def test_clipped_lean_step_by_every_norm(cuda, n, p, masked):
    """The clipped lean step has the bits of clipping and then stepping, whichever norm and mask choose its kernel."""
    vis = None
    if masked:
        vis = (torch.rand(n, device=cuda, generator=torch.Generator(device=cuda).manual_seed(n)) < 0.4).int()
        vis[0] = 3
    a = adam_state(n, cuda, n, lowp=(2, 5))
    b = copies(a)
    total = A.adam_step_lean(a, 12, vis, max_grad_norm=0.05, norm_type=p)
    grads, want = G.clip_grads([x[1] for x in b], 0.05, p)
    A.adam_step_lean([(x[0], g, *x[2:]) for x, g in zip(b, grads)], 12, vis)
    flat = torch.cat([x[1].double().reshape(-1) for x in a])
    exact = float(flat.abs().max() if p == math.inf else (flat.abs() ** p).sum() ** (1 / p))
    # a float64 sum of fewer than 2^13 additions a path, rounded once to float32
    assert abs(float(total) - exact) <= 2.0 ** -24 * 1.001 * exact and torch.equal(total, want)
    for x, y in zip(a, b):
        assert all(torch.equal(x[i], y[i]) for i in (0, 2, 3))
    if masked:
        start = adam_state(n, cuda, n, lowp=(2, 5))
        assert all(torch.equal(x[i][vis == 0], y[i][vis == 0]) for x, y in zip(a, start) for i in (0, 2, 3))


@pytest.mark.parametrize("stale", [False, True])
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_sparse_optimizer_in_several_launches(cuda, monkeypatch, p, stale):
    """More groups than a launch takes, or groups that a stale mask sends to the dense update: one norm over all of
    them, then masked steps by that norm."""
    n = 2003
    vis = (torch.rand(n, device=cuda) < 0.4).int()
    monkeypatch.setattr(gs3d._Rasterize, "track_visibility", False)  # as it was, when the optimizers have set it
    monkeypatch.setattr(gs3d._Rasterize, "last_visibility", vis, raising=False)
    shapes = [(n, *s) for s in (SHAPES_3DGS * 2)[:4 if stale else 11]] + ([(n + 1, 3)] if stale else [])
    start = [torch.randn(s, device=cuda) for s in shapes]
    a, b = ([t.clone().requires_grad_() for t in start] for _ in range(2))
    kw = {"lr": 1e-3, "eps": 1e-15, "sparse": True, "lowp_moment_groups": ("g1", "g3")}
    oa = A.FusedAdam([{"params": [t], "name": f"g{k}"} for k, t in enumerate(a)], max_grad_norm=0.3, grad_norm_type=p,
                     **kw)
    ob = A.FusedAdam([{"params": [t], "name": f"g{k}"} for k, t in enumerate(b)], **kw)
    for _ in range(3):
        for x, y in zip(a, b):
            x.grad = torch.randn_like(x)
            y.grad = x.grad.clone()
        oa.step()
        want = G.clip_grad_norm_(b, 0.3, p)
        ob.step()
        assert torch.equal(oa.grad_norm, want) and float(want) > 0.3
        for x, y in zip(a, b):
            assert torch.equal(x, y)
            assert all(torch.equal(oa.state[x][k], ob.state[y][k]) for k in ("exp_avg", "exp_avg_sq"))
    assert oa.n_dense_fallbacks == (3 if stale else 0)
    for x, t in zip(a, start):
        if x.shape[0] == n:
            assert torch.equal(x[vis == 0], t[vis == 0]) and not torch.equal(x, t)

"""The global gradient norm, clipping by it and the clipped Adam steps on the GPU, against float64.

Tolerances (u = 2^-24, half a step of float32): a float32 norm is a float64 sum, whose own error (an element passes
through fewer than 2^13 additions of 2^-53 at these sizes) is far below u, rounded once: u. A float64 norm: 2^13 x 2^-53.
The factor is one division in float64 from the rounded norm; rounded to float32 it is off by u (the norm) + u, and the
product by another u: 3 u, plus half a step of the tensor's type (2^-8 bf16, 2^-11 fp16), and half of the smallest
subnormal where the product is that small."""
from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from gs_b200 import _lib as L
from gs_b200 import adam as A
from gs_b200 import grad as G
from gs_b200 import gs3d, scenes

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SLACK = 1.001  # second-order terms
F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
HALF = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def norm64(grads, p):
    flat = torch.cat([g.detach().double().reshape(-1) for g in grads])
    if p == math.inf:
        return flat.abs().max() if flat.numel() else flat.sum()
    return flat.abs().sum() if p == 1.0 else (flat * flat).sum().sqrt()


def close_norm(got, grads, p):
    want = float(norm64(grads, p))
    # below 2^-126 a float32's step is 2^-149 whatever the value, so its rounding is off by up to 2^-150
    tol = 2.0 ** -40 * want if got.dtype == F64 else U * SLACK * want + 2.0 ** -150
    assert abs(float(got.double()) - want) <= tol, (float(got), want)


def close_clip(outs, grads, limit, p):
    norm = float(norm64(grads, p))
    f = min(1.0, limit / (norm + 1e-6))
    for o, g in zip(outs, grads):
        want = g.double() * f
        if g.dtype == F64:
            rel, tiny = 2.0 ** -39, 0.0
        else:
            rel, tiny = (3 * U + HALF[g.dtype]) * SLACK, TINY[g.dtype]
        assert bool(((o.double() - want).abs() <= rel * want.abs() + tiny).all()), (g.dtype, tuple(g.shape))


def scaled_bits(g, total, limit):
    """What the documentation says: the factor in float64 from the norm that the call returns (a Python division:
    torch's `number / tensor` multiplies by a rounded reciprocal), the product in torch."""
    f = limit / (float(total) + 1e-6)
    f = torch.tensor(f if f < 1 or f != f else 1.0, dtype=F64, device=g.device)
    return g * f if g.dtype == F64 else (g.float() * f.float()).to(g.dtype)


def tensors(shapes, types, seed, device, offset=0):
    """Tensors at odd addresses: each lies `offset` elements behind the start of an allocation of its own."""
    gen = torch.Generator(device=device).manual_seed(seed)
    out = []
    for k, (s, t) in enumerate(zip(shapes, types)):
        n = math.prod(s)
        flat = torch.empty(n + offset, dtype=t, device=device)
        v = flat[offset:].view(s)
        v.copy_(torch.randn(s, generator=gen, device=device, dtype=torch.float64) * 10.0 ** (-(k % 3)))
        out.append(v)
    return out


SIZES = [1, 2, 3, 7, 8, 31, 255, 1023, 1024, 4095, 4096, 4097, 8191, 8193, 16385, 100_003]


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F64])
def test_one_tensor_of_every_length_and_alignment(cuda, dtype, p):
    for n in SIZES:
        for offset in (0, 1, 3):
            g, = tensors([(n,)], [dtype], n + offset, cuda, offset)
            total = G.grad_norm([g], p)
            assert total.shape == () and total.dtype == (F64 if dtype == F64 else F32)
            close_norm(total, [g], p)
            limit = 0.37 * float(total)
            outs, got = G.clip_grads([g], limit, p)
            assert torch.equal(got, total)
            close_clip(outs, [g], limit, p)
            assert torch.equal(outs[0], scaled_bits(g, total, limit))


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("count", [2, 6, 16, 17, 128, 129, 400, 1000, 1001, 2503])
def test_many_tensors_of_mixed_types(cuda, count, p):
    gen = torch.Generator().manual_seed(count)
    lens = [int(x) for x in torch.randint(0, 700, (count,), generator=gen)]
    lens[0], lens[-1] = 0, 20_000
    types = [(F32, BF16, F16)[k % 3] for k in range(count)]
    grads = tensors([(n,) for n in lens], types, count, cuda, offset=count % 2)
    total = G.grad_norm(grads, p)
    close_norm(total, grads, p)
    limit = 0.5 * float(total)
    outs, got = G.clip_grads(grads, limit, p)
    assert torch.equal(got, total)
    close_clip(outs, grads, limit, p)
    kept = [g.clone() for g in grads]
    same, _ = G.clip_grads(grads, limit, p, out=grads)
    assert all(a is b for a, b in zip(same, grads))
    assert all(torch.equal(a, b) for a, b in zip(grads, outs))
    assert any(not torch.equal(a, b) for a, b in zip(grads, kept))


def test_float64_among_others(cuda):
    grads = tensors([(1000,), (33, 7), (5,)], [F32, F64, BF16], 3, cuda, offset=1)
    total = G.grad_norm(grads)
    assert total.dtype == F64
    close_norm(total, grads, 2.0)
    outs, _ = G.clip_grads(grads, 0.1, 2.0)
    for o, g in zip(outs, grads):
        assert torch.equal(o, scaled_bits(g, total, 0.1))


def test_outputs_elsewhere_and_their_surroundings(cuda):
    """Outputs at another alignment than their inputs; what lies around them stays as it is."""
    for dtype in (F32, BF16, F16, F64):
        for n in (1, 9, 4099, 50_001):
            for a, b in ((0, 1), (1, 0), (1, 3), (3, 2)):
                src = torch.randn(n + 8, device=cuda).to(dtype)
                dst = torch.full((n + 8,), 7.0, device=cuda, dtype=dtype)
                raw = src.clone()
                g, o = src[a:a + n], dst[b:b + n]
                _, total = G.clip_grads([g], 0.01, out=[o])
                assert torch.equal(o, scaled_bits(g, total, 0.01))
                assert torch.equal(src, raw)
                assert bool((dst[:b] == 7).all()) and bool((dst[b + n:] == 7).all())
                G.clip_grads([g], 0.01, out=[g])
                assert torch.equal(g, o) and torch.equal(src[:a], raw[:a]) and torch.equal(src[a + n:], raw[a + n:])


def test_orders_of_dimensions(cuda):
    x = torch.randn(6, 5, 7, 3, device=cuda)
    grads = [x.permute(3, 1, 0, 2), torch.randn(4, 8, 3, 3, device=cuda).to(memory_format=torch.channels_last),
             torch.randn(9, 1, 2, device=cuda).transpose(0, 2)]
    total = G.grad_norm(grads)
    close_norm(total, grads, 2.0)
    outs, _ = G.clip_grads(grads, 0.5)
    for o, g in zip(outs, grads):
        assert o.shape == g.shape and torch.equal(o, scaled_bits(g, total, 0.5))
    with pytest.raises(RuntimeError, match="strides"):
        G.clip_grads(grads[:1], 0.5, out=[torch.empty(grads[0].shape, device=cuda)])
    for bad in (x[..., ::2], x[:, 1:3], x[:1, :1, :1, :1].expand(2, 2, 2, 2)):
        with pytest.raises(RuntimeError, match="dense"):
            G.grad_norm([bad])


def test_nothing_and_zeros(cuda):
    empty = [torch.empty(0, device=cuda), torch.empty(3, 0, 2, device=cuda, dtype=BF16)]
    for p in (1.0, 2.0, math.inf):
        assert float(G.grad_norm(empty, p)) == 0.0
        outs, total = G.clip_grads(empty, 1.0, p)
        assert float(total) == 0.0 and [o.shape for o in outs] == [e.shape for e in empty]
        z = [torch.zeros(5000, device=cuda), torch.zeros(3, device=cuda)]
        outs, total = G.clip_grads(z, 0.0, p)
        assert float(total) == 0.0 and all(not o.any() for o in outs)
    one = [torch.tensor(3.0, device=cuda)]  # 0-d
    assert float(G.grad_norm(one)) == 3.0
    assert float(G.clip_grads(one, 1.5)[0][0]) == pytest.approx(1.5, rel=1e-5)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, F64])
def test_values_that_are_not_finite(cuda, dtype, p):
    for n, at in ((5, 2), (40_000, 39_999)):
        g = torch.linspace(-1, 1, n, device=cuda).to(dtype)
        for bad, where in ((math.nan, at), (-math.inf, 0), (math.inf, at)):
            x = g.clone()
            x[where] = bad
            total = G.grad_norm([g, x], p)
            assert math.isnan(float(total)) if math.isnan(bad) else float(total) == math.inf
            outs, _ = G.clip_grads([g, x], 1.0, p)
            if math.isnan(bad):
                assert all(bool(o.isnan().all()) for o in outs)
            else:  # the factor is 0
                assert not outs[0].any()
                assert int(outs[1].isnan().sum()) == 1 and bool(outs[1][where].isnan())
            with pytest.raises(RuntimeError, match="not finite"):
                G.grad_norm([x], p, error_if_nonfinite=True)
        x = g.clone()
        x[at], x[0] = math.nan, math.inf  # NaN wins over infinity
        assert math.isnan(float(G.grad_norm([x], p)))


def test_values_far_from_one(cuda):
    """Squares that leave float32's range, and its subnormals."""
    for scale in (1e30, 1e-30, 1e-42):
        g = torch.randn(30_000, device=cuda) * scale
        for p in (1.0, 2.0, math.inf):
            close_norm(G.grad_norm([g], p), [g], p)
    big = torch.full((100,), 3e38, device=cuda)  # the norm itself is no float32
    assert float(G.grad_norm([big])) == math.inf
    assert float(G.grad_norm([big.double()])) == pytest.approx(3e39 * float(big[0]) / 3e38, rel=1e-12)


def test_factor_of_one_changes_nothing(cuda):
    g = torch.randn(10_001, device=cuda)
    g[5] = -0.0
    raw = g.clone()
    for limit in (1e6, math.inf):
        outs, total = G.clip_grads([g], limit)
        assert torch.equal(outs[0].view(torch.int32), raw.view(torch.int32))
        G.clip_grads([g], limit, out=[g])
        assert torch.equal(g.view(torch.int32), raw.view(torch.int32))
    G.clip_grads([g], 0.0, out=[g])
    assert not g.any()


def test_given_norm(cuda):
    grads = tensors([(5000,), (11, 3)], [F32, BF16], 5, cuda)
    for dtype in (F32, F64):
        total = torch.tensor([123.456], device=cuda, dtype=dtype)
        outs, got = G.clip_grads(grads, 2.0, total_norm=total)
        assert got is total
        for o, g in zip(outs, grads):
            assert torch.equal(o, scaled_bits(g, total[0], 2.0))
    outs, _ = G.clip_grads([grads[0].double()], 2.0, total_norm=torch.tensor(123.456, device=cuda))
    assert torch.equal(outs[0], scaled_bits(grads[0].double(), torch.tensor(123.456, device=cuda), 2.0))
    for bad in (torch.tensor([1.0, 2.0], device=cuda), torch.tensor(1, device=cuda), torch.tensor(1.0)):
        with pytest.raises(RuntimeError):
            G.clip_grads(grads, 2.0, total_norm=bad)


def test_clip_grad_norm_against_torch(cuda):
    torch.manual_seed(7)
    params = [torch.nn.Parameter(torch.randn(s, device=cuda)) for s in ((300, 40), (40,), (7, 5, 3), (1,))]
    for p in params[:3]:
        p.grad = torch.randn_like(p)
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for a, b in zip(params, other):
        b.grad = None if a.grad is None else a.grad.clone()
    for p, limit in ((2.0, 1.0), (1.0, 50.0), (math.inf, 0.25), (2.0, 1e4)):
        raw = [a.grad.clone() for a in params[:3]]
        want = torch.nn.utils.clip_grad_norm_(other, limit, p)
        got = G.clip_grad_norm_(params, limit, p)
        # torch sums in float32 (a tree over at most 12,000 elements: 2^5 roundings are more than it makes)
        assert abs(float(got) - float(want)) <= 32 * U * float(want)
        close_clip([a.grad for a in params[:3]], raw, limit, p)
        for a, b in zip(params, other):
            assert (a.grad is None) == (b.grad is None)
            if b.grad is not None:
                b.grad.copy_(a.grad)
    params[0].grad[3, 3] = math.nan
    raw = [a.grad.clone() for a in params[:3]]
    with pytest.raises(RuntimeError, match="not finite"):
        G.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(a.grad.isnan(), b.isnan()) for a, b in zip(params, raw))
    assert torch.equal(params[1].grad, raw[1])
    with pytest.raises(RuntimeError, match="overlaps"):
        G.clip_grad_norm_([params[1], params[1]], 1.0)
    G.clip_grad_norm_(params[1], 0.5, error_if_nonfinite=True)  # one parameter, not a list
    close_clip([params[1].grad], [raw[1]], 0.5, 2.0)


def test_the_same_bits_every_time(cuda):
    grads = tensors([(1_000_003,), (77_777,), (3,)], [F32, BF16, F16], 9, cuda, offset=1)
    first = G.grad_norm(grads)
    for _ in range(5):
        assert torch.equal(G.grad_norm(grads), first)


def test_more_elements_than_32_bits_count(cuda):
    n = (1 << 32) + 12_345
    g = torch.ones(n, dtype=BF16, device=cuda)
    g[-1], g[0], g[1 << 31] = 300.0, -200.0, 100.0
    want = math.sqrt((n - 3) + 300.0 ** 2 + 200.0 ** 2 + 100.0 ** 2)
    total = G.grad_norm([g])
    assert abs(float(total) - want) <= U * SLACK * want
    assert float(G.grad_norm([g], 1.0)) == pytest.approx(n - 3 + 600.0, rel=U)
    assert float(G.grad_norm([g], math.inf)) == 300.0
    G.clip_grads([g], want / 2, out=[g])
    for at in (-1, 0, 1 << 31, 5, (1 << 32) + 3, (1 << 32) - 1):
        raw = {-1: 300.0, 0: -200.0, 1 << 31: 100.0}.get(at, 1.0)
        assert float(g[at]) == raw / 2  # the factor is a half up to 2^-23, and bfloat16 keeps 8 bits
    assert float(G.grad_norm([g], 1.0)) == pytest.approx((n - 3 + 600.0) / 2, rel=U)


# ---- the clipped Adam steps ----

SHAPES_3DGS = [(3,), (3,), (4,), (1,), (1, 3), (15, 3)]


def adam_state(n, device, seed, lowp=False, offset=0, zero=False):
    gen = torch.Generator(device=device).manual_seed(seed)

    def make(shape, scale, dtype=F32):
        flat = torch.empty(math.prod(shape) + offset, device=device, dtype=dtype)
        v = flat[offset:].view(shape)
        return v.copy_(torch.randn(shape, generator=gen, device=device) * scale)

    groups = []
    for k, s in enumerate(SHAPES_3DGS):
        md = BF16 if lowp and k == 5 else F32
        shape = (n, *s)
        m, v = make(shape, 0.0 if zero else 1e-2, md), make(shape, 0.0 if zero else 1e-2, md)
        groups.append((make(shape, 1.0), make(shape, 10.0 ** -k), m, v.abs_(), 1e-3 * (k + 1)))
    return groups


def copies(groups):
    return [(p.clone(), g.clone(), m.clone(), v.clone(), lr) for p, g, m, v, lr in groups]


def same_groups(a, b):
    for k, (x, y) in enumerate(zip(a, b)):
        for i in (0, 2, 3):
            assert torch.equal(x[i], y[i]), (k, i)


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("n", [1, 5, 4096, 30_011, 200_003])
def test_clipped_adam_is_clipping_then_the_step(cuda, n, p):
    for offset in (0, 1):
        for limit in (0.05, 1e9):
            a = adam_state(n, cuda, n, offset=offset)
            b = copies(a)
            raw = [g.clone() for _, g, _, _, _ in a]
            total = A.adam_step(a, 7, max_grad_norm=limit, norm_type=p)
            grads, want = G.clip_grads([x[1] for x in b], limit, p)
            A.adam_step([(x[0], g, *x[2:]) for x, g in zip(b, grads)], 7)
            assert torch.equal(total, want)
            close_norm(total, raw, p)
            same_groups(a, b)
            assert all(torch.equal(x[1], r) for x, r in zip(a, raw))  # the gradients keep their values


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n", [1, 5, 4096, 30_011, 200_003])
def test_clipped_lean_adam_is_clipping_then_the_step(cuda, n, masked):
    vis = None
    if masked:
        vis = (torch.rand(n, device=cuda) < 0.4).int()
        vis[0] = 3
    for offset in (0, 1):
        a = adam_state(n, cuda, n + 1, lowp=True, offset=offset)
        b = copies(a)
        total = A.adam_step_lean(a, 12, vis, max_grad_norm=0.05)
        grads, want = G.clip_grads([x[1] for x in b], 0.05)
        A.adam_step_lean([(x[0], g, *x[2:]) for x, g in zip(b, grads)], 12, vis)
        assert torch.equal(total, want)
        same_groups(a, b)


@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 7, 45, 8191, 32768, 33000])
def test_lean_mask_of_every_width(cuda, width):
    """The lean steps update the rows that are visible as the dense one does, bit for bit, and no others, whatever the
    row's width is to the groups of four and to the tile (with and without the clip)."""
    n = max(3, 50_021 // width)
    torch.manual_seed(width)
    for share in (0.0, 0.3, 1.0):
        vis = (torch.rand(n, device=cuda) < share).int()
        p, g = torch.randn(n, width, device=cuda), torch.randn(n, width, device=cuda)
        m, v = torch.randn(n, width, device=cuda), torch.rand(n, width, device=cuda)
        on = (vis != 0)[:, None]
        for clip in ({}, {"max_grad_norm": 0.5}):
            dense = [(p.clone(), g, m.clone(), v.clone(), 1e-2)]
            lean = copies(dense)
            A.adam_step(dense, 4, **clip)
            A.adam_step_lean(lean, 4, vis, **clip)
            for i, old in ((0, p), (2, m), (3, v)):
                assert torch.equal(lean[0][i], torch.where(on, dense[0][i], old)), (share, clip, i)


def test_clipped_adam_against_the_formula(cuda):
    """One step from zero moments against float64. The factor and the product are off by 3 u together, so m by 4 u and
    v by 8 u; m / sqrt(v) and the other operations add fewer than 16 u, relative to the update."""
    a = adam_state(20_011, cuda, 2, zero=True)
    raw = copies(a)
    limit, step = 0.5, 1
    total = A.adam_step(a, step, max_grad_norm=limit)
    f = min(1.0, limit / (float(norm64([g for _, g, _, _, _ in raw], 2.0)) + 1e-6))
    assert f < 0.1 and float(total) > limit
    b1, b2 = (float(torch.tensor(b, dtype=F32)) for b in (0.9, 0.999))
    for (p, _, m, v, _), (p0, g, m0, v0, lr) in zip(a, raw):
        g = g.double() * f
        m1 = b1 * (m0.double() - g) + g
        v1 = b2 * (v0.double() - g * g) + g * g
        upd = lr / (1 - 0.9) * m1 / (v1.sqrt() / math.sqrt(1 - 0.999) + 1e-15)
        # from zero moments m = fl(b1 (0 - g) + g) and v likewise: one rounding of a fused operation, 1 - b exact
        # in float64; b2 = 0.999 leaves 0.001 g^2 of two terms near g^2, fused, so the product's rounding counts 1000 u
        assert bool(((m.double() - m1).abs() <= 8 * U * m1.abs() + 1e-44).all())
        assert bool(((v.double() - v1).abs() <= 1100 * U * v1.abs() + 1e-44).all())
        assert bool(((p.double() - (p0.double() - upd)).abs() <= U * (p0.abs() + upd.abs()) + 600 * U * upd.abs()).all())


def test_clipped_adam_refusals(cuda):
    a = adam_state(10, cuda, 1)
    with pytest.raises(ValueError):
        A.adam_step(a, 1, max_grad_norm=-1.0)
    with pytest.raises(ValueError):
        A.adam_step(a, 1, max_grad_norm=1.0, norm_type=3)
    with pytest.raises(RuntimeError, match="at most"):
        A.adam_step(a + adam_state(10, cuda, 2), 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="two groups"):
        A.adam_step([a[0], a[0]], 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="size"):
        A.adam_step([(a[0][0], a[0][1][1:], *a[0][2:])], 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="dtype"):
        A.adam_step([(a[0][0], a[0][1].double(), *a[0][2:])], 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="contiguous"):
        A.adam_step([(a[0][0], a[0][1].t().contiguous().t(), *a[0][2:])], 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="float32"):
        A.adam_step([(a[0][0], a[0][1], a[0][2].bfloat16(), a[0][3].bfloat16(), 1e-3)], 1, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="primitives"):
        A.adam_step_lean(a, 1, torch.ones(9, dtype=torch.int32, device=cuda), max_grad_norm=1.0)


def test_a_norm_that_is_not_finite_in_the_step(cuda):
    a = adam_state(100, cuda, 4)
    a[2][1][3, 1] = math.nan
    b = copies(a)
    total = A.adam_step(a, 3, max_grad_norm=1.0)
    grads, _ = G.clip_grads([x[1] for x in b], 1.0)
    A.adam_step([(x[0], g, *x[2:]) for x, g in zip(b, grads)], 3)
    assert math.isnan(float(total))
    for x, y in zip(a, b):
        assert bool(x[0].isnan().all()) and bool(y[0].isnan().all())


# ---- streams, graphs ----

def test_on_streams_of_their_own(cuda):
    """Calls in flight on two streams at once share nothing."""
    lists = [tensors([(400_000,), (9_999,)], [F32, BF16], 1, cuda), tensors([(9_000_001,), (77,)], [F32, F16], 2, cuda)]
    want = [G.clip_grads(g, 1.0) for g in lists]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(G.clip_grads(lists[k], 1.0))
    torch.cuda.synchronize()
    for k in range(2):
        for outs, total in got[k]:
            assert torch.equal(total, want[k][1])
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k][0]))


@pytest.mark.parametrize("n", [4096, 60_000, 200_000])
def test_captured_and_replayed(cuda, n):
    """Norm, clipping and the clipped step in two graphs, replayed side by side with new gradients."""
    states = [adam_state(n, cuda, s) for s in (5, 6)]
    graphs, norms, clips = [], [], []
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # a warm-up outside the capture
        A.adam_step(copies(states[0]), 9, max_grad_norm=0.05)
        G.clip_grads([x[1] for x in states[0]], 0.05)
    torch.cuda.synchronize()
    before = [copies(s) for s in states]
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            total = G.grad_norm([x[1] for x in s])
            outs, clip_total = G.clip_grads([x[1] for x in s], 0.05)
            step_total = A.adam_step(s, 9, max_grad_norm=0.05)
        graphs.append(graph)
        norms.append((total, clip_total, step_total))
        clips.append(outs)
    for s, b in zip(states, before):
        same_groups(s, b)  # a capture runs nothing
        for x, y in zip(s, b):
            x[1].mul_(1.7)  # new gradients in the same place
            y[1].copy_(x[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for s, b, (total, clip_total, step_total), outs in zip(states, before, norms, clips):
        want_outs, want = G.clip_grads([x[1] for x in b], 0.05)
        A.adam_step(b, 9, max_grad_norm=0.05)
        assert torch.equal(total, want) and torch.equal(clip_total, want) and torch.equal(step_total, want)
        assert all(torch.equal(x, y) for x, y in zip(outs, want_outs))
        same_groups(s, b)


# ---- the optimizer, and a run of everything together ----

def make_opt(leaves, **kw):
    return A.FusedAdam([{"params": [t], "lr": 1e-3 * (k + 1), "name": f"g{k}"} for k, t in enumerate(leaves)], lr=0.0,
                       eps=1e-15, **kw)


@pytest.mark.parametrize("count,kw", [(6, {}), (6, {"lowp_moment_groups": ("g5",)}), (11, {}),
                                      (11, {"lowp_moment_groups": ("g5", "g9")})])
def test_optimizer_is_clip_grad_norm_then_its_step(cuda, count, kw):
    """More groups than one launch takes, and groups out of step with one another (several launches, one norm)."""
    shapes = (SHAPES_3DGS * 2)[:count]
    start = [torch.randn(3001, *s, device=cuda) for s in shapes]
    a, b = ([t.clone().requires_grad_() for t in start] for _ in range(2))
    oa, ob = make_opt(a, max_grad_norm=0.3, **kw), make_opt(b, **kw)
    for it in range(4):
        for k, (x, y) in enumerate(zip(a, b)):
            x.grad = None if it == 1 and k == 2 else torch.randn_like(x)  # group 2 misses a step
            y.grad = None if x.grad is None else x.grad.clone()
        if it == 3:
            a[1].grad = a[1].grad.t().contiguous().t() if a[1].dim() == 2 else a[1].grad  # another order in memory
        oa.step()
        want = G.clip_grad_norm_(b, 0.3)
        ob.step()
        # one gradient of the last round lies in another order: its sum is taken in that order
        if it < 3:
            assert torch.equal(oa.grad_norm, want)
            for x, y in zip(a, b):
                assert torch.equal(x, y)
        else:
            close_norm(oa.grad_norm, [x.grad for x in a], 2.0)
    assert set(oa.state_dict()) == set(ob.state_dict())


def test_sparse_optimizer(cuda):
    """FusedAdam(sparse, lowp_moment_groups, max_grad_norm) against clip_grad_norm_ and the same optimizer without it,
    over real forwards (the visibility that the mask comes from)."""
    sc = scenes.gs3d_test_scene("tiny", seed=2)
    cam = sc["cameras"][0]
    names = ("means", "scales", "rotations", "opacities", "sh0", "sh_rest")
    settings = gs3d.RasterizerSettings(*scenes.settings_tuple(cam, sc["active_sh_bases"], cuda))
    a = [sc[k].to(cuda).requires_grad_(True) for k in names]
    b = [t.detach().clone().requires_grad_(True) for t in a]
    kw = {"sparse": True, "lowp_moment_groups": ("g5",)}
    oa, ob = make_opt(a, max_grad_norm=1e-3, **kw), make_opt(b, **kw)
    try:
        for _ in range(3):
            img = gs3d.diff_rasterize(*a, torch.empty(0), settings)
            ((img - 0.5) ** 2).mean().backward()
            for x, y in zip(a, b):
                y.grad = x.grad.clone()
            want = G.clip_grad_norm_(b, 1e-3)
            oa.step()
            ob.step()
            assert torch.equal(oa.grad_norm, want)
            assert all(torch.equal(x, y) for x, y in zip(a, b))
            assert all(torch.equal(oa.state[x]["exp_avg"], ob.state[y]["exp_avg"]) for x, y in zip(a, b))
            oa.zero_grad()
    finally:
        gs3d._Rasterize.track_visibility = False


def test_kernel_timer(cuda):
    """The timer's events between the launches of a clipped step change nothing."""
    for n in (100, 60_000):
        a = adam_state(n, cuda, 8)
        b = copies(a)
        want = A.adam_step(a, 3, max_grad_norm=0.1)
        with L.KernelTimer("k_adam") as timer:
            timer.arm()
            got = A.adam_step(b, 3, max_grad_norm=0.1)
        assert len(timer.times()["k_adam"]) == 1 and timer.times()["k_adam"][0] > 0
        assert torch.equal(got, want)
        same_groups(a, b)


def test_first_call_inside_a_capture(cuda):
    """In a process of its own whose first call of each entry point is captured."""
    code = """
import torch
from __graft_entry__ import load_package
load_package()
from gs_b200 import adam as A, grad as G
g = [torch.ones(70_000, 3, device="cuda"), torch.ones(7, device="cuda")]
one = [torch.ones(5, device="cuda")]
p, m, v = ([torch.ones_like(t) for t in g] for _ in range(3))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    norms = [G.grad_norm(g), G.grad_norm(one)]
    outs = G.clip_grads(g, 1.0)[0] + G.clip_grads(one, 1.0)[0]
    norms.append(A.adam_step(list(zip(p, g, m, v, (1e-3, 1e-3))), 1, max_grad_norm=1.0))
graph.replay()
torch.cuda.synchronize()
n = 210_007 ** 0.5
assert abs(float(norms[0]) - n) < 1e-3 and abs(float(norms[1]) - 5 ** 0.5) < 1e-6 and float(norms[2]) == float(norms[0])
assert abs(float(outs[0][0, 0]) - 1 / n) < 1e-8 and abs(float(outs[2][0]) - 5 ** -0.5) < 1e-6
assert float(p[1][0]) < 1.0
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_for_another_device_than_the_current_one(cuda):
    """The guard that a call takes when its tensors' device is not the current one."""
    g = torch.randn(1000, device=cuda)
    d = G.describe([g])._replace(current=False)
    out, out_ptr, ws, ws_ptr, ws_bytes = G.scratch(0, 1)
    d.call("splat_grad_norm", 1, d.addresses, d.sizes, d.codes, 2, out_ptr, 0, ws_ptr, ws_bytes)
    assert torch.equal(out, G.grad_norm([g]))


def test_training_together(cuda):
    """A 3D scene trained by the rasterizer's backward: the norm read beside the step, gradients clipped in place for
    one model and in the step for the other, both from the same gradients."""
    sc = scenes.gs3d_test_scene("tiny", seed=1)
    cam = sc["cameras"][0]
    names = ("means", "scales", "rotations", "opacities", "sh0", "sh_rest")
    a = [sc[k].to(cuda).requires_grad_(True) for k in names]
    b = [t.detach().clone().requires_grad_(True) for t in a]
    settings = gs3d.RasterizerSettings(*scenes.settings_tuple(cam, sc["active_sh_bases"], cuda))
    oa, ob = make_opt(a, max_grad_norm=1e-3), make_opt(b)
    clipped = 0
    for it in range(6):
        img = gs3d.diff_rasterize(*a, torch.empty(0), settings)
        ((img - 0.5) ** 2).mean().backward()
        for x, y in zip(a, b):
            y.grad = x.grad.clone()
        total = G.grad_norm([x.grad for x in a])
        close_norm(total, [x.grad for x in a], 2.0)
        assert torch.equal(G.clip_grad_norm_(b, 1e-3), total)
        oa.step()
        ob.step()
        assert torch.equal(oa.grad_norm, total)
        clipped += int(float(total) > 1e-3)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        oa.zero_grad()
        ob.zero_grad()
    assert clipped > 0

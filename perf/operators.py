"""The gradient-norm operators' cases: the global norm over many tensors, clipping by it, and the Adam step that clips.

`run` computes a case in plain torch operations, or with `own` through the package's entry points (gs_b200.grad,
gs_b200.adam); `exact` gives the same results in 64 bits.

Layouts of the tensors (they are what a model of this framework has in hand):
    3dgs    the six tensors of n 3D Gaussians: means, scales, rotations, opacities, sh0, sh_rest (`rest` SH bases)
    toy2d   the five parameters of n 2D Gaussians: xy, log_scale, theta, rgb_logit, opacity_logit
    ragged  `count` tensors of very different lengths (1 to `longest` elements), one behind the other in a flat buffer
            per type, so that most start at odd addresses
Types: fp32, bf16, fp16, fp64, or mixed (float32, bfloat16 and float16 in turn).
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "fp64": torch.float64}
LRS_3DGS = (1.6e-4, 5e-3, 1e-3, 5e-2, 2.5e-3, 2.5e-3)
LRS_TOY2D = (1e-1, 1e-2, 1e-2, 1e-2, 1e-2)
BETAS = (0.9, 0.999)
EPS = 1e-15


def listed():
    return [
        # the norm of the toy2d fit's gradients, each step: the smallest call, where latency counts
        {"name": "norm toy2d 4096", "op": "norm", "layout": "toy2d", "n": 4096, "type": "fp32", "p": "2"},
        # the norm of the scene-scale gradients (3M Gaussians, SH degree 3), far beyond the L2
        {"name": "norm 3dgs 3M", "op": "norm", "layout": "3dgs", "n": 3000000, "rest": 15, "type": "fp32", "p": "2"},
        # the norm over a few hundred tensors of half-precision gradients, as a colour network beside the Gaussians has
        {"name": "norm ragged bf16", "op": "norm", "layout": "ragged", "count": 300, "longest": 2000000, "sizes": 11,
         "type": "bf16", "p": "2"},
        # the toy2d fit's gradients clipped each step
        {"name": "clip toy2d 4096", "op": "clip", "layout": "toy2d", "n": 4096, "type": "fp32", "p": "2", "share": 0.3},
        # the single-view scene's gradients (100k Gaussians), limited in their largest element
        {"name": "clip 3dgs 100k inf", "op": "clip", "layout": "3dgs", "n": 100000, "rest": 15, "type": "fp32",
         "p": "inf", "share": 0.3},
        # the batched training step's gradients (1M Gaussians) clipped into buffers of their own, the raw ones kept
        {"name": "clip 3dgs 1M", "op": "clip", "layout": "3dgs", "n": 1000000, "rest": 15, "type": "fp32", "p": "2",
         "share": 0.3},
        # the ragged list in mixed precision
        {"name": "clip ragged mixed", "op": "clip", "layout": "ragged", "count": 200, "longest": 1000000, "sizes": 12,
         "type": "mixed", "p": "2", "share": 0.3},
        # clipped in place in a step whose norm is below the limit, as most steps of a run are: nothing changes
        {"name": "clip in place 3dgs 3M quiet", "op": "clip", "layout": "3dgs", "n": 3000000, "rest": 15,
         "type": "fp32", "p": "2", "share": 4.0},
        # the clipped Adam step of the toy2d fit
        {"name": "adam toy2d 4096", "op": "adam", "layout": "toy2d", "n": 4096, "p": "2", "share": 0.3},
        # of the single-view scene: everything stays in the L2
        {"name": "adam 3dgs 100k", "op": "adam", "layout": "3dgs", "n": 100000, "rest": 15, "p": "2", "share": 0.3},
        # of the scene-scale view
        {"name": "adam 3dgs 3M", "op": "adam", "layout": "3dgs", "n": 3000000, "rest": 15, "p": "2", "share": 0.3},
        # the lean step of the batched scene: a third of the Gaussians visible, bfloat16 SH moments
        {"name": "lean adam 3dgs 1M", "op": "lean", "layout": "3dgs", "n": 1000000, "rest": 15, "p": "2",
         "share": 0.3},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "clip", "adam", "lean"))
    case = {"op": op, "p": rng.choice(("2", "2", "1", "inf"))}
    layout = rng.choice(("3dgs", "3dgs", "toy2d") + (("ragged",) if op in ("norm", "clip") else ()))
    if op == "lean":
        layout = "3dgs"
    case["layout"] = layout
    if layout == "ragged":
        case.update(count=_spread(rng, 1, 400), longest=_spread(rng, 100, 2000000), sizes=rng.randrange(1 << 20))
    elif layout == "3dgs":
        case.update(n=_spread(rng, 1, 3000000), rest=rng.choice((15, 15, 8, 3)))
    else:
        case.update(n=_spread(rng, 1, 200000))
    if op in ("norm", "clip"):
        case["type"] = rng.choice(("fp32", "fp32", "bf16", "fp16", "mixed", "fp64"))
    if op != "norm":
        case["share"] = rng.choice((0.3, 0.01, 4.0))
    return case


def _shapes(case):
    if case["layout"] == "3dgs":
        n, rest = case["n"], case["rest"]
        return [(n, 3), (n, 3), (n, 4), (n, 1), (n, 1, 3), (n, rest, 3)]
    if case["layout"] == "toy2d":
        n = case["n"]
        return [(n, 2), (n, 2), (n,), (n, 3), (n,)]
    rng = random.Random(case["sizes"])
    return [(_spread(rng, 1, case["longest"]),) for _ in range(case["count"])]


def _types(case, count):
    name = case.get("type", "fp32")
    if name == "mixed":
        return [(torch.float32, torch.bfloat16, torch.float16)[i % 3] for i in range(count)]
    return [TYPES[name]] * count


def _scales(case, count):
    """The size of each tensor's gradients: the groups of a Gaussian model differ by orders of magnitude."""
    if case["layout"] == "ragged":
        return [10.0 ** -(i % 4) for i in range(count)]
    return [(1.0, 0.3, 0.03, 0.1, 0.2, 0.02)[i] for i in range(count)]


def _limit(case, shapes, scales):
    """max_norm: `share` of the norm that gradients of these scales have, about."""
    sizes = [math.prod(s) for s in shapes]
    kept = 0.35 if case["layout"] == "3dgs" else 1.0
    if case["p"] == "inf":
        norm = max(s * math.sqrt(2 * math.log(n + 2)) for s, n in zip(scales, sizes))
    elif case["p"] == "1":
        norm = sum(s * n * kept * 0.8 for s, n in zip(scales, sizes))
    else:
        norm = math.sqrt(sum(s * s * n * kept for s, n in zip(scales, sizes)))
    return case["share"] * norm


def _in_place(case):
    """Clipping in place is measured where it changes nothing, so that each pass meets the same gradients."""
    return case["op"] == "clip" and case["share"] > 1.0


def _views(flats, shapes, types):
    at, views = {t: 0 for t in flats}, []
    for s, t in zip(shapes, types):
        n = math.prod(s)
        views.append(flats[t][at[t]:at[t] + n].view(s))
        at[t] += n
    return views


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = _shapes(case)
    types, scales = _types(case, len(shapes)), _scales(case, len(shapes))
    total = {t: sum(math.prod(s) for s, u in zip(shapes, types) if u == t) for t in dict.fromkeys(types)}
    state = {"case": case, "flats": {t: torch.empty(k, dtype=t, device="cuda") for t, k in total.items()}}
    state["grads"] = _views(state["flats"], shapes, types)
    seen = None
    if case["layout"] == "3dgs":  # Gaussians that the view does not show have no gradient
        seen = torch.rand(case["n"], generator=gen, device="cuda") < 0.35
        seen[0] = True
    for g, s in zip(state["grads"], scales):
        x = torch.randn(g.shape, generator=gen, device="cuda").mul_(s)
        if seen is not None:
            x.mul_(seen.view(-1, *[1] * (g.dim() - 1)))
        g.copy_(x)
        del x
    if case["op"] == "norm":
        return state
    state["max_norm"] = _limit(case, shapes, scales)
    if case["op"] == "clip":
        state["out_flats"] = state["flats"] if _in_place(case) else {t: torch.empty_like(f)
                                                                     for t, f in state["flats"].items()}
        state["out"] = state["grads"] if _in_place(case) else _views(state["out_flats"], shapes, types)
        return state
    lrs = LRS_3DGS if case["layout"] == "3dgs" else LRS_TOY2D
    state["groups"], state["step"] = [], 100
    for k, (g, s, lr) in enumerate(zip(state["grads"], scales, lrs)):
        low = torch.bfloat16 if case["op"] == "lean" and k == 5 else torch.float32
        p = torch.randn(g.shape, generator=gen, device="cuda")
        m = torch.randn(g.shape, generator=gen, device="cuda").mul_(0.05 * s)
        v = torch.rand(g.shape, generator=gen, device="cuda").add_(0.1).mul_(0.01 * s * s)
        state["groups"].append((p, g, m.to(low), v.to(low), lr))
    if case["op"] == "lean":
        state["visibility"] = seen.to(torch.int32) * torch.randint(1, 40, seen.shape, generator=gen, device="cuda",
                                                                   dtype=torch.int32)
    return state


# ---- the plain form ----

def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _norm(grads, p):
    kind = torch.float64 if any(g.dtype == torch.float64 for g in grads) else torch.float32
    if p == "inf":
        return torch.stack([_wide(g).abs().max().to(kind) for g in grads if g.numel()]).max()
    if p == "1":
        return torch.stack([_wide(g).abs().sum(dtype=torch.float64) for g in grads]).sum().to(kind)
    return torch.stack([_wide(g).square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().to(kind)


def _factor(norm, max_norm):
    return torch.clamp(max_norm / (norm + 1e-6), max=1.0)


def _mixed_bits(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _to_bf16(f, noise):
    bits = (f.view(torch.int32).to(torch.int64) + (noise & 0xFFFF)) >> 16
    return bits.to(torch.int16).view(torch.bfloat16)


def _adam(p, g, m, v, lr, step, factor, visibility):
    b1, b2 = (torch.tensor(b, dtype=torch.float32).item() for b in BETAS)
    g = g * factor
    m1 = (m.float() - g) * b1 + g
    v1 = (v.float() - g * g) * b2 + g * g
    p1 = p - (lr / (1 - BETAS[0] ** step)) * m1 / (v1.sqrt() * (1 / math.sqrt(1 - BETAS[1] ** step)) + EPS)
    if m.dtype == torch.bfloat16:
        seed = (0x9E3779B9 * step + 0x85EBCA6B) & 0xFFFFFFFF
        r = _mixed_bits(torch.arange(p.numel(), device=p.device).view(p.shape) ^ seed)
        m1, v1 = _to_bf16(m1, r), _to_bf16(v1, _mixed_bits(r))
    if visibility is not None:
        on = (visibility != 0).view(-1, *[1] * (p.dim() - 1))
        p1, m1, v1 = torch.where(on, p1, p), torch.where(on, m1, m), torch.where(on, v1, v)
    return p.copy_(p1), m.copy_(m1), v.copy_(v1)


def _run_plain(state):
    case, grads = state["case"], state["grads"]
    norm = _norm(grads, case["p"])
    if case["op"] == "norm":
        return norm
    factor = _factor(norm, state["max_norm"])
    if case["op"] == "clip":
        _ = [o.copy_(_wide(g) * factor) for g, o in zip(grads, state["out"])]
        return norm, list(state["out_flats"].values())
    state["step"] += 1
    return norm, [_adam(*group, state["step"], factor, state.get("visibility")) for group in state["groups"]]


def _run_own(state):
    from __graft_entry__ import load_package

    load_package()
    from gs_b200 import adam, grad

    case = state["case"]
    p = float(case["p"])
    if case["op"] == "norm":
        return grad.grad_norm(state["grads"], p)
    if case["op"] == "clip":
        _, norm = grad.clip_grads(state["grads"], state["max_norm"], p, out=state["out"])
        return norm, list(state["out_flats"].values())
    state["step"] += 1
    if case["op"] == "adam":
        norm = adam.adam_step(state["groups"], state["step"], BETAS, EPS, max_grad_norm=state["max_norm"],
                              norm_type=p)
    else:
        norm = adam.adam_step_lean(state["groups"], state["step"], state["visibility"], BETAS, EPS,
                                   max_grad_norm=state["max_norm"], norm_type=p)
    return norm, [(p, m, v) for p, _, m, v, _ in state["groups"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ----

def exact(case, seed):
    state = prepare(case, seed)
    flat = torch.cat([f.double() for f in state["flats"].values()])
    if case["p"] == "inf":
        norm = flat.abs().max()
    elif case["p"] == "1":
        norm = flat.abs().sum()
    else:
        norm = torch.dot(flat, flat) ** 0.5
    if case["op"] == "norm":
        return norm
    limit = state["max_norm"] / (float(norm) + 1e-6)
    scale = limit if limit < 1.0 else 1.0
    if case["op"] == "clip":
        return norm, [f.double() * scale for f in state["flats"].values()]
    del flat
    t = state["step"] + 1
    keep = [float(torch.tensor(b, dtype=torch.float32)) for b in BETAS]  # the step holds the betas in float32
    hidden = state["visibility"].eq(0) if case["op"] == "lean" else None
    groups = []
    for param, grad, first, second, lr in state["groups"]:
        was = [x.double() for x in (param, first, second)]
        g = grad.double() * scale
        first_new = keep[0] * was[1] + (1.0 - keep[0]) * g
        second_new = keep[1] * was[2] + (1.0 - keep[1]) * g ** 2
        root = (second_new / (1.0 - BETAS[1] ** t)).sqrt()
        now = [was[0] - lr * (first_new / (1.0 - BETAS[0] ** t)) / (root + EPS), first_new, second_new]
        if hidden is not None:
            now = [x.index_put((hidden,), old[hidden]) for x, old in zip(now, was)]
        groups.append(tuple(now))  # bfloat16 moments: the value before its random rounding
    return norm, groups


def work(case):
    shapes = _shapes(case)
    types = _types(case, len(shapes))
    values = sum(math.prod(s) for s in shapes)
    read = sum(math.prod(s) * torch.empty((), dtype=t).element_size() for s, t in zip(shapes, types))
    if case["op"] == "norm":
        return {"bytes": read + 4, "flops": 2 * values}
    if case["op"] == "clip":  # in place and below the limit nothing has to be written
        return {"bytes": read * (1 if _in_place(case) else 2) + 4, "flops": 3 * values}
    if case["op"] == "adam":
        return {"bytes": 28 * values + 4, "flops": 18 * values}
    # lean: every gradient for the norm; the rest for the visible 35 %, the SH moments in 2 bytes
    n, rest = case["n"], 3 * case["rest"]
    moved = 4 * values + 4 * n + int(0.35 * n * (14 * 24 + rest * 16)) + 4
    return {"bytes": moved, "flops": 2 * values + int(0.35 * 18 * values)}

"""Cases of the gradient operators of nvdiffrecmc_amd.optim, in their plain form and through the framework.

norm   grad_norm(tensors, norm_type, scales): the norm of many gradient tensors as one vector
clip   clip_grad_norm_(parameters, max_norm, norm_type): the same norm, and the gradients scaled by min(1, max_norm / (norm + 1e-6))
step   FusedAdam(max_norm=...).step(): the norm of the gradients as Adam sees them, and the update with the clipped gradients

A set of tensors is named by what it stands for: the trained set of the direct-lighting iteration (kd, ks and normal textures, the light
probe, the vertices), or a network's weights (blocks of square and four-fold matrices with their vectors, an embedding), or a ragged list.
Layouts: `own` = every gradient an allocation of its own; `arena` = views of one buffer at multiples of 512 bytes, with gaps, as a caching
allocator places them; `bucket` = views that follow one another without a gap behind `lead` elements, as in a data-parallel bucket.
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6                               # of the clipping factor
LR, BETA1, BETA2, ADAM_EPS = 0.01, 0.9, 0.999, 1e-8
TILE = 64                                # texels of a tile that receive gradient together


# ---- the cases -----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the probe's gradient alone, 256^2 texels: a monitor's call, where latency counts
        dict(name="norm probe", op="norm", set="probe", probe=256, dtype="fp32", layout="own", p=2.0, size=1.0),
        # everything that the iteration trains with unlocked geometry at 684 k triangles, the probe's gradient times 64
        dict(name="norm scene", op="norm", set="scene", tex=1024, probe=256, verts=342016, touched=0.24, light_scale=64.0, dtype="fp32", layout="own", p=2.0, size=3.0),
        # the largest: the gradients of a network of 24 blocks of width 1600 in fp32, one bucket
        dict(name="norm network", op="norm", set="network", blocks=24, width=1600, rows=32000, dtype="fp32", layout="bucket", lead=0, p=2.0, size=5.0),
        # the largest magnitude of a ragged list of half-precision gradients whose views begin at odd places
        dict(name="norm ragged fp16 max", op="norm", set="ragged", count=120, most=3000000, sizes=7, dtype="fp16", layout="bucket", lead=3, p=math.inf, size=4096.0),
        # probe and vertices of the 10 k triangle mesh, each its own allocation
        dict(name="clip probe and mesh", op="clip", set="light_mesh", probe=256, verts=5344, dtype="fp32", layout="own", p=2.0, size=4.0, max_norm=1.0),
        # the scene's whole set after a view with outliers
        dict(name="clip scene", op="clip", set="scene", tex=1024, probe=256, verts=342016, touched=0.49, dtype="fp32", layout="own", p=2.0, size=4.0, max_norm=1.0),
        # a network's bf16 gradients where an allocator put them
        dict(name="clip network bf16", op="clip", set="network", blocks=24, width=960, rows=32000, dtype="bf16", layout="arena", p=2.0, size=4.0, max_norm=1.0),
        # most steps of a run that has settled: the norm lies below the threshold and the gradients stay as they are
        dict(name="clip network under", op="clip", set="network", blocks=12, width=768, rows=50001, dtype="fp32", layout="arena", p=2.0, size=0.5, max_norm=1.0),
        # many short tensors of odd lengths behind an odd offset, by the sum of magnitudes
        dict(name="clip ragged fp16 sum", op="clip", set="ragged", count=400, most=70000, sizes=11, dtype="fp16", layout="bucket", lead=5, p=1.0, size=60000.0, max_norm=20000.0),
        # the smallest training set: one small probe, the vertices of the 6 k triangle mesh
        dict(name="step probe and mesh", op="step", set="light_mesh", probe=128, verts=2930, size=4.0, max_norm=1.0),
        # the scene's whole set, every texel with a gradient
        dict(name="step scene", op="step", set="scene", tex=1024, probe=256, verts=342016, touched=1.0, sparse=False, size=4.0, max_norm=1.0),
        # the textures by tiles: a quarter of them touched, as by one view
        dict(name="step scene tiles", op="step", set="scene", tex=1024, probe=256, verts=5344, touched=0.24, sparse=True, size=4.0, max_norm=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "step"])
    kind = rng.choice(["probe", "light_mesh", "scene", "network", "ragged"] if op != "step" else ["light_mesh", "scene"])
    c = dict(op=op, set=kind)
    if kind in ("probe", "light_mesh", "scene"):
        c["probe"] = _log(rng, 8, 700)
    if kind in ("light_mesh", "scene"):
        c["verts"] = _log(rng, 3, 342016)
    if kind == "scene":
        c.update(tex=_log(rng, 16, 1500), touched=round(rng.uniform(0.02, 1.0), 3))
    if kind == "network":
        c.update(blocks=_log(rng, 1, 24), width=_log(rng, 16, 960), rows=_log(rng, 100, 32000))
    if kind == "ragged":
        c.update(count=_log(rng, 2, 600), most=_log(rng, 20, 300000), sizes=rng.randrange(1 << 20))
    if op == "step":
        c.update(size=4.0, max_norm=round(math.exp(rng.uniform(-2.5, 2.5)), 3))
        if kind == "scene":
            c["sparse"] = rng.random() < 0.5
        return c
    c["dtype"] = rng.choice(["fp32", "bf16", "fp16"])
    c["p"] = rng.choice([2.0, 2.0, 1.0, math.inf])
    c["layout"] = rng.choice(["arena", "bucket"] if kind in ("network", "ragged") else ["own", "arena", "bucket"])
    if c["layout"] == "bucket":
        c["lead"] = rng.randrange(9)
    c["size"] = round(math.exp(rng.uniform(0.0, 3.0)) * (500.0 if c["dtype"] == "fp16" else 1.0), 3)
    if op == "clip":
        c["max_norm"] = round(c["size"] * rng.choice([0.1, 0.4, 0.8, 2.0]), 4)
    return c


def _shapes(case):
    kind = case["set"]
    light = [(case["probe"], case["probe"], 3)] if "probe" in case else []
    verts = [(case["verts"], 3)] if "verts" in case else []
    if kind == "probe":
        return light
    if kind == "light_mesh":
        return light + verts
    if kind == "scene":
        return [(case["tex"], case["tex"], 3)] * 3 + light + verts
    if kind == "network":
        w = case["width"]
        block = [(w,), (w,), (w, w), (w,), (w, w), (w, w), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
        return [(case["rows"], w)] + block * case["blocks"] + [(w,), (w,)]
    rng = random.Random(case["sizes"])
    sizes = [0 if rng.random() < 0.02 else _log(rng, 1, case["most"]) for _ in range(case["count"])]
    return [(n,) for n in sizes[1:]] + [(case["most"] | 1,)]


def _scales(case):
    """The factor that a gradient of the trained set is seen through: the probe's is larger in a training step."""
    k = case.get("light_scale", 64.0 if case["op"] == "step" else 1.0)
    return [k if len(s) == 3 and s[0] == case.get("probe") and i == (3 if case["set"] == "scene" else 0) else 1.0 for i, s in enumerate(_shapes(case))]


def work(case):
    n = sum(math.prod(s) for s in _shapes(case))
    if case["op"] == "step":
        tex = 9 * case["tex"] ** 2 if case.get("sparse") else 0
        live = n - tex * (1.0 - case.get("touched", 1.0))                 # an untouched texel: its gradient is read, nothing else
        return {"bytes": 28.0 * live + 4.0 * (n - live), "flops": 3.0 * n + 15.0 * live}
    b = DTYPES[case["dtype"]].itemsize
    clipped = case["op"] == "clip" and case["max_norm"] < case["size"]
    return {"bytes": float(n * b * (2 if clipped else 1)), "flops": 2.0 * n + (n if clipped else 0)}


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _values(shape, touched, gen):
    """Gradients of noisy estimates: many small values, a few large ones; in a texture nothing outside the touched tiles."""
    n = math.prod(shape)
    g = torch.randn(n, generator=gen, device="cuda").pow_(3)
    if touched < 1.0 and len(shape) == 3:
        texels = n // 3
        live = torch.rand((texels + TILE - 1) // TILE, generator=gen, device="cuda") < touched
        g = g.view(texels, 3) * live.repeat_interleave(TILE)[:texels, None]
    return g.view(shape)


def _total(grads, p):
    a = [g.abs().max() if p == math.inf else g.abs().pow(p).sum(dtype=torch.float64) for g in grads if g.numel()]
    t = torch.stack([x.double() for x in a])
    return t.max() if p == math.inf else t.sum() ** (1 / p)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes, scales = _shapes(case), _scales(case)
    textures = 3 if case["set"] == "scene" else 0
    values = [_values(s, case.get("touched", 1.0) if i < textures else 1.0, gen) for i, s in enumerate(shapes)]
    # the norm that the case speaks of, to within a few percent from seed to seed
    p = case.get("p", 2.0)
    unit = case["size"] / _total([v * k for v, k in zip(values, scales)], p) * (1 + 0.02 * torch.rand((), generator=gen, device="cuda"))
    values = [v.mul_(unit) for v in values]
    state = {"case": case, "scales": scales, "p": p, "max_norm": case.get("max_norm")}
    if case["op"] == "step":
        state["params"] = [torch.nn.Parameter(torch.rand(s, generator=gen, device="cuda")) for s in shapes]
        for q, v in zip(state["params"], values):
            q.grad = v
        state["bounds"] = _bounds(case)
        state["rates"] = [3.0 if k != 1.0 else 1.0 for k in scales]
        if own:
            from nvdiffrecmc_amd.optim import FusedAdam
            state["opt"] = FusedAdam(state["params"], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, clamps=state["bounds"], grad_scales=scales, lr_scales=state["rates"],
                                     normalize3=[i == 2 and textures > 0 for i in range(len(shapes))],
                                     sparse=[bool(case.get("sparse")) and i < textures for i in range(len(shapes))], max_norm=case["max_norm"])
        else:
            state["m"] = [torch.zeros_like(q) for q in state["params"]]
            state["v"] = [torch.zeros_like(q) for q in state["params"]]
            state["t"] = 0
        return state
    dtype = DTYPES[case["dtype"]]
    if case["layout"] == "own":
        grads = [v.to(dtype) for v in values]
        state["out"] = grads
    else:
        step = 512 // dtype.itemsize if case["layout"] == "arena" else 1
        at, places = case.get("lead", 0), []
        for s in shapes:
            places.append(at)
            at += -(-math.prod(s) // step) * step
        buffer = torch.full((at,), 2.0 ** -14, dtype=dtype, device="cuda")       # (of the gradients' magnitude: a gap that is scaled shows)
        grads = [buffer[o:o + v.numel()].view(v.shape).copy_(v) for o, v in zip(places, values)]
        state["out"] = [buffer]
    state["grads"] = grads
    if case["op"] == "clip":
        state["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
        for q, g in zip(state["params"], grads):
            q.grad = g
    return state


def _bounds(case):
    """The clamps of the training step, tensor by tensor: kd, ks, the normal map, the probe, the vertices."""
    if case["set"] != "scene":
        return [(0.01, None), None]
    lo, hi = torch.tensor([0.0, 0.08, 0.0], device="cuda"), torch.tensor([0.01, 1.0, 1.0], device="cuda")
    return [(0.0, 1.0), (None, None, lo, hi), (-1.0, 1.0), (0.01, None), None]


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "step":
        return _step(state)
    if op == "norm":
        if own:
            from nvdiffrecmc_amd.optim import grad_norm
            return grad_norm(state["grads"], norm_type=state["p"], scales=state["scales"] if "light_scale" in state["case"] else None)
        return _norm(_flat(state["grads"], state["scales"]), state["p"]).float()
    # a threshold that a schedule lowers: every pass over the same gradients has something to scale, as with new gradients
    limit = state["max_norm"]
    if limit < state["case"]["size"]:
        state["max_norm"] *= 0.9999
    if own:
        from nvdiffrecmc_amd.optim import clip_grad_norm_
        norm = clip_grad_norm_(state["params"], limit, norm_type=state["p"])
    else:
        flat = _flat(state["grads"], state["scales"])
        norm = _norm(flat, state["p"])
        scaled = flat * (limit / (norm + EPS)).clamp(max=1.0).float()
        [g.copy_(x.view(g.shape)) for g, x in zip(state["grads"], scaled.split([g.numel() for g in state["grads"]]))]
        norm = norm.float()
    return [norm] + state["out"]


def _flat(grads, scales):
    """All gradients as one vector in 32 bits."""
    if any(k != 1.0 for k in scales):
        grads = [g.float() * k for g, k in zip(grads, scales)]
    return torch.cat([g.reshape(-1) for g in grads]).float()


def _norm(flat, p):
    """Its norm; a sum of many terms in 64 bits."""
    if p == math.inf:
        return flat.abs().max().double()
    if p == 1.0:
        return flat.abs().sum(dtype=torch.float64)
    return flat.square().sum(dtype=torch.float64).sqrt()


@torch.no_grad()
def _step(state):
    params = state["params"]
    if own:
        opt = state["opt"]
        opt.step()
        return {"norm": opt.grad_norm, "params": [q.detach() for q in params], "m": opt.exp_avg, "v": opt.exp_avg_sq}
    norm = _norm(_flat([q.grad for q in params], state["scales"]), 2.0)
    factor = (state["max_norm"] / (norm + EPS)).clamp(max=1.0).float()
    state["t"] += 1
    t = state["t"]
    for i, (q, m, v) in enumerate(zip(params, state["m"], state["v"])):
        g = q.grad * state["scales"][i] * factor
        m.add_((g - m) * (1 - BETA1))
        v.mul_(BETA2).add_(g * g * (1 - BETA2))
        q.sub_(m / (v.sqrt() / math.sqrt(1 - BETA2 ** t) + ADAM_EPS) * (LR * state["rates"][i] / (1 - BETA1 ** t)))
        b = state["bounds"][i]
        if b is not None:
            q.clamp_(b[0], b[1]) if b[0] is not None or b[1] is not None else None
            q.copy_(torch.minimum(torch.maximum(q, b[2]), b[3])) if len(b) > 2 else None
        if i == 2 and state["case"]["set"] == "scene":
            q.div_(q.square().sum(-1, keepdim=True).clamp(min=1e-20).sqrt())
    return {"norm": norm.float(), "params": [q.detach() for q in params], "m": state["m"], "v": state["v"]}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    grads = [q.grad for q in s["params"]] if case["op"] == "step" else s["grads"]
    p, total = s["p"], torch.zeros((), dtype=torch.float64, device="cuda")
    for g, k in zip(grads, s["scales"]):
        if g.numel():
            a = torch.linalg.vector_norm(g.double() * k, ord=p)
            total = torch.maximum(total, a) if p == math.inf else total + a ** p
    norm = total if p == math.inf else total ** (1 / p)
    if case["op"] == "norm":
        return norm
    factor = torch.where(norm + EPS > s["max_norm"], s["max_norm"] / (norm + EPS), torch.ones_like(norm))
    if case["op"] == "clip":
        if case["layout"] == "own":
            return [norm] + [g.double() * factor for g in grads]
        whole = s["out"][0].double()                                     # the gaps stay as they are
        for g in grads:
            whole[g.storage_offset():g.storage_offset() + g.numel()] = g.double().reshape(-1) * factor
        return [norm, whole]
    new, ms, vs = [], [], []
    for i, (q, g) in enumerate(zip(s["params"], grads)):                 # the first step, from moments of zero
        h = g.double() * s["scales"][i] * factor
        ms.append((1 - BETA1) * h)
        vs.append((1 - BETA2) * h * h)
        x = q.detach().double() - LR * s["rates"][i] * h / (h.abs() + ADAM_EPS)
        b = s["bounds"][i]
        if b is not None:
            lo = b[2].double() if len(b) > 2 else torch.tensor(-math.inf if b[0] is None else b[0], dtype=torch.float64, device="cuda")
            hi = b[3].double() if len(b) > 2 else torch.tensor(math.inf if b[1] is None else b[1], dtype=torch.float64, device="cuda")
            x = torch.minimum(torch.maximum(x, lo), hi)
        if i == 2 and case["set"] == "scene":
            x = x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp(min=1e-10)
        new.append(x)
    return {"norm": norm, "params": new, "m": ms, "v": vs}

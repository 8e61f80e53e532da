"""The cases by which the rotary positions and the orthogonalised momentum step are measured.

`own` False: the plain forms, elementary torch operations in 32 bits (the angles in 64). `own` True: the calls a user makes of v1t_amd."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # a, b, c of X <- a X + (b A + c A A) X, A = X X^T
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01
CORE = ((620, 155),) * 3 + ((155, 620), (488, 155), (155, 488))  # q, k, v, projection and the two MLP matrices of a block of the default core


def listed():
    return [
        # the shared core of a training step: 112 images, 29 x 57 patches behind a class token, q and k inside the packed and padded projections
        {"name": "rotary_core_step", "op": "rotary", "batch": 112, "grid": "1x29x57", "lead": 1, "heads": 4, "kv_heads": 4, "dim": 155, "pad": 5,
         "sections": "38,38", "layout": "pairs", "shared": False, "base": 10000.0, "far": 0, "type": "bf16", "backward": False, "packed": True},
        # one mouse's batch in a loop over mice: forward and the gradients of q and k
        {"name": "rotary_mouse_train", "op": "rotary", "batch": 16, "grid": "1x29x57", "lead": 1, "heads": 4, "kv_heads": 4, "dim": 155, "pad": 5,
         "sections": "38,38", "layout": "pairs", "shared": False, "base": 10000.0, "far": 0, "type": "bf16", "backward": True, "packed": True},
        # a clip of 24 such frames as one long prompt, keys shared by four query heads, one ladder of rates over three axes
        {"name": "rotary_clip_prompt", "op": "rotary", "batch": 1, "grid": "24x29x57", "lead": 0, "heads": 16, "kv_heads": 4, "dim": 128, "pad": 0,
         "sections": "16,24,24", "layout": "halves", "shared": True, "base": 10000.0, "far": 0, "type": "bf16", "backward": False, "packed": False},
        # one new token for each of eight streams, far into them: latency
        {"name": "rotary_one_token", "op": "rotary", "batch": 8, "grid": "1x1x1", "lead": 0, "heads": 16, "kv_heads": 4, "dim": 128, "pad": 0,
         "sections": "16,24,24", "layout": "halves", "shared": True, "base": 500000.0, "far": 900000, "type": "bf16", "backward": False, "packed": False},
        # a small odd model in 32 bits, trained: 91 features a head, the last nine without a position
        {"name": "rotary_odd_train", "op": "rotary", "batch": 5, "grid": "3x17x23", "lead": 2, "heads": 6, "kv_heads": 3, "dim": 91, "pad": 0,
         "sections": "11,15,15", "layout": "halves", "shared": False, "base": 100.0, "far": 0, "type": "fp32", "backward": True, "packed": False},
        # one small matrix alone: latency
        {"name": "orthogonal_one_small", "op": "orthogonal", "count": 1, "rows": 155, "cols": 64, "type": "fp32"},
        # a tall matrix of a wide model
        {"name": "orthogonal_tall", "op": "orthogonal", "count": 1, "rows": 8192, "cols": 1024, "type": "fp32"},
        # a large square one, in 16 bits
        {"name": "orthogonal_square", "op": "orthogonal", "count": 1, "rows": 4096, "cols": 4096, "type": "bf16"},
        # a stack of odd ones
        {"name": "orthogonal_odd_stack", "op": "orthogonal", "count": 12, "rows": 777, "cols": 1301, "type": "fp16"},
        # the step over the matrices of the default core: four blocks
        {"name": "muon_core", "op": "muon", "model": "core", "blocks": 4, "width": 0},
        # the step over one block of a model of width 2048
        {"name": "muon_wide", "op": "muon", "model": "wide", "blocks": 1, "width": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "orthogonal", "orthogonal", "muon"))
    if kind == "rotary":
        axes = rng.choice((1, 2, 3))
        sections = [rng.randint(2, 40) for _ in range(axes)]
        dim = 2 * sum(sections) + rng.choice((0, 0, 1, 3, 8))
        heads = rng.choice((1, 2, 4, 6, 12, 16))
        kv = rng.choice([k for k in (1, 2, 3, 4, 16) if heads % k == 0])
        t, h, w = (rng.randint(1, 24), rng.randint(1, 29), _log(rng, 1, 57)) if axes == 3 else (1, rng.randint(1, 29), _log(rng, 1, 57))
        most = max(1, min(112, int(1e8 // (t * h * w * (heads + kv) * dim))))  # no more elements than the largest listed case
        return {"op": "rotary", "batch": _log(rng, 1, most), "grid": "%dx%dx%d" % (t, h, w), "lead": rng.choice((0, 1, 2)), "heads": heads,
                "kv_heads": kv, "dim": dim, "pad": rng.choice((0, 0, 5)), "sections": ",".join(map(str, sections)),
                "layout": rng.choice(("pairs", "halves")), "shared": rng.random() < 0.5, "base": rng.choice((100.0, 10000.0, 500000.0)),
                "far": rng.choice((0, 0, 900000)), "type": rng.choice(("bf16", "bf16", "fp16", "fp32")), "backward": rng.random() < 0.5,
                "packed": heads == kv and rng.random() < 0.5}
    if kind == "orthogonal":
        rows, cols = _log(rng, 24, 4096), _log(rng, 24, 4096)
        most = max(1, min(16, int(1.7e7 // (rows * cols))))
        return {"op": "orthogonal", "count": rng.randint(1, most), "rows": rows, "cols": cols, "type": rng.choice(("fp32", "bf16", "fp16"))}
    if rng.random() < 0.5:
        return {"op": "muon", "model": "core", "blocks": rng.randint(1, 5), "width": 0}
    return {"op": "muon", "model": "wide", "blocks": 1, "width": _log(rng, 100, 2000)}


def _shapes(case):
    if case["model"] == "core":
        return CORE * case["blocks"]
    w = case["width"]
    return ((3 * w, w), (w, w), (4 * w, w), (w, 4 * w)) * case["blocks"]


def _sections(case):
    return tuple(int(s) for s in case["sections"].split(","))


def _gradient(rows, cols, g):
    """What a linear layer's weight receives: the sum over samples of the outer products of two feature vectors whose scales fall off."""
    samples = max(64, max(rows, cols))
    dy = torch.randn(samples, rows, device=DEV, generator=g) * (torch.arange(rows, device=DEV) + 1.0) ** -0.15
    x = torch.randn(samples, cols, device=DEV, generator=g) * (torch.arange(cols, device=DEV) + 1.0) ** -0.15
    return dy.t() @ x / samples


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "orthogonal":
        made = [_gradient(case["rows"], case["cols"], g).to(TYPES[case["type"]]) for _ in range(case["count"])]
        return {"case": case, "updates": made}
    if case["op"] == "muon":
        shapes = _shapes(case)
        return {"case": case, "weights": [torch.randn(r, c, device=DEV, generator=g) * c**-0.5 for r, c in shapes],
                "grads": [_gradient(r, c, g) for r, c in shapes], "moments": [3 * _gradient(r, c, g) for r, c in shapes]}
    sections, dtype = _sections(case), TYPES[case["type"]]
    t, h, w = (int(s) for s in case["grid"].split("x"))
    at = torch.stack(torch.meshgrid(*(torch.arange(s, device=DEV) for s in (t, h, w)), indexing="ij"), -1).reshape(-1, 3)[:, 3 - len(sections):]
    at = torch.cat([at.new_zeros(case["lead"], len(sections)), at + case["far"]])  # the leading tokens have no place: angle zero
    at = at + seed % 7 * (torch.arange(len(at), device=DEV) >= case["lead"])[:, None]  # where the grid begins
    b, n, q, k, d, pad = case["batch"], len(at), case["heads"], case["kv_heads"], case["dim"], case["pad"]

    def values(heads):
        return torch.randn(b, n, heads, d + pad, device=DEV, generator=g).to(dtype)

    if case["packed"]:  # q, k and v of one projection, features padded: the operator gets views
        both = torch.randn(b, n, 3, q, d + pad, device=DEV, generator=g).to(dtype)
        state = {"q": both[:, :, 0, :, :d], "k": both[:, :, 1, :, :d]}
    else:
        state = {"q": values(q)[..., :d], "k": values(k)[..., :d]}
    if case["backward"]:
        state = {"q": state["q"].requires_grad_(), "k": state["k"].requires_grad_(), "dq": values(q)[..., :d], "dk": values(k)[..., :d]}
    return {"case": case, "positions": at.to(torch.int32), **state}


def _cos_sin(at, case):
    """cos and sin of every token's angles in 64 bits, rounded to 32: (tokens, 1, pairs)."""
    sections = _sections(case)
    axis = torch.cat([torch.full((s,), a, device=DEV) for a, s in enumerate(sections)])
    if case["shared"]:
        part = torch.arange(len(axis), device=DEV, dtype=torch.float64) / len(axis)
    else:
        part = torch.cat([torch.arange(s, device=DEV, dtype=torch.float64) / s for s in sections])
    angle = at.to(torch.float64)[:, axis] * torch.pow(torch.tensor(case["base"], dtype=torch.float64, device=DEV), -part)
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotate(x, cos, sin, layout):
    pairs, x32 = cos.shape[-1], x.float()
    if layout == "pairs":
        x0, x1 = x32[..., 0:2 * pairs:2], x32[..., 1:2 * pairs:2]
        turned = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)
    else:
        x0, x1 = x32[..., :pairs], x32[..., pairs:2 * pairs]
        turned = torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1)
    return torch.cat([turned, x32[..., 2 * pairs:]], -1).to(x.dtype)


def _orthogonal(u):
    """Newton-Schulz steps on the update, laid with its shorter side first."""
    x = u.float()
    x = x.t() if u.shape[0] > u.shape[1] else x
    x = x / (x.norm() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def run(state):
    case = state["case"]
    if case["op"] == "orthogonal":
        if own:
            import v1t_amd
            return v1t_amd.orthogonalize(state["updates"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return [_orthogonal(u).to(u.dtype).contiguous() for u in state["updates"]]
    if case["op"] == "muon":
        weights, grads, moments = state["weights"], state["grads"], state["moments"]
        if own:
            import v1t_amd
            v1t_amd.muon_step(weights, grads, moments, lr=LR, momentum=MOMENTUM, weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        else:
            for w, g, m in zip(weights, grads, moments):
                m.mul_(MOMENTUM).add_(g)
                o = _orthogonal(g + MOMENTUM * m)
                w.mul_(1 - LR * DECAY).sub_(o * (LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))))
        return {"weights": weights, "moments": moments}
    q, k, at = state["q"], state["k"], state["positions"]
    if own:
        import v1t_amd
        yq, yk = v1t_amd.rotary(q, at, k=k, sections=_sections(case), base=case["base"], layout=case["layout"], shared=case["shared"])
        if not case["backward"]:
            return yq, yk
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (state["dq"], state["dk"]))
        return yq.detach(), yk.detach(), dq, dk
    with torch.no_grad():
        cos, sin = _cos_sin(at, case)
        out = [_rotate(x, cos, sin, case["layout"]) for x in (q, k)]
        if case["backward"]:  # the gradient turns back
            out += [_rotate(x, cos, -sin, case["layout"]) for x in (state["dq"], state["dk"])]
        return tuple(out)


def work(case):
    if case["op"] == "rotary":
        t, h, w = (int(s) for s in case["grid"].split("x"))
        n = case["batch"] * (t * h * w + case["lead"]) * (case["heads"] + case["kv_heads"]) * case["dim"]
        n *= 2 if case["backward"] else 1
        return {"bytes": 2 * n * (4 if case["type"] == "fp32" else 2), "flops": 3 * n}
    if case["op"] == "orthogonal":
        shapes, size = [(case["rows"], case["cols"])] * case["count"], 2 * (4 if case["type"] == "fp32" else 2)
    else:
        shapes, size = _shapes(case), 5 * 4  # reads weight, gradient and momentum, writes weight and momentum
    flops = 0
    for r, c in shapes:
        m, n = min(r, c), max(r, c)
        # half of each symmetric product; on the short side alone where that is less (two stages: gram, recursion on it, one product back)
        flops += min(STEPS * (3 * m * m * n + m**3), 6 * m * m * n + 13 * m**3)
    return {"bytes": sum(r * c for r, c in shapes) * size, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        sections, at = _sections(case), state["positions"].double()
        pairs = sum(sections)
        turns = torch.empty(len(at), pairs, dtype=torch.complex128, device=DEV)
        j = 0
        for a, s in enumerate(sections):
            for i in range(s):
                rate = math.exp(-math.log(case["base"]) * (j / pairs if case["shared"] else i / s))
                turns[:, j] = torch.polar(torch.ones_like(at[:, a]), at[:, a] * rate)
                j += 1

        def turned(x, t):
            y = x.detach().double().clone()
            if case["layout"] == "pairs":
                first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
            else:
                first, second = slice(0, pairs), slice(pairs, 2 * pairs)
            for i in range(len(y)):  # an image at a time: the complex copies are large
                z = torch.complex(y[i, ..., first].contiguous(), y[i, ..., second].contiguous()) * t[:, None]
                y[i, ..., first], y[i, ..., second] = z.real, z.imag
            return y

        out = [turned(state["q"], turns), turned(state["k"], turns)]
        if case["backward"]:
            out += [turned(state["dq"], turns.conj()), turned(state["dk"], turns.conj())]
        return tuple(out)

    def steps(u):
        """By polynomials of the first Gram matrix, which all commute: O = Q X0."""
        u = u.double()
        flip = u.shape[0] > u.shape[1]
        x = (u.t() if flip else u) / (u.norm() + EPS)
        gram, one = x @ x.t(), torch.eye(min(u.shape), dtype=torch.float64, device=DEV)
        (a, b, c), total = COEFFICIENTS, torch.eye(min(u.shape), dtype=torch.float64, device=DEV)
        for _ in range(STEPS):
            factor = a * one + gram @ (b * one + c * gram)
            total, gram = factor @ total, factor @ gram @ factor
        o = total @ x
        return o.t() if flip else o

    if case["op"] == "orthogonal":
        return [steps(u).contiguous() for u in state["updates"]]
    weights, moments = [], []
    for w, g, m in zip(state["weights"], state["grads"], state["moments"]):
        moments.append(MOMENTUM * m.double() + g.double())
        scale = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        weights.append((1 - LR * DECAY) * w.double() - LR * scale * steps(g.double() + MOMENTUM * moments[-1]))
    return {"weights": weights, "moments": moments}

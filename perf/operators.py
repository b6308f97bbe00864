"""What is measured of the optimizer operators: the norm of many gradient tensors (with its clipping form) and the AdamW
step over many tensors, its states held in 32 bits or in 8.

A case names the operator, the layout of the tensor list and the types; `prepare` makes the tensors, `run` is one pass."""
import math
import random

import torch

own = False

BETAS, EPS, DECAY, LR, FIRST_STEP = (0.9, 0.999), 1e-8, 0.01, 3e-4, 100
QBLOCK = 256             # elements that share a scale of the 8-bit states
E4M3_MAX, TINY = 448.0, 2.0 ** -126
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the tensor lists -----------------------------------------------------------------------------------------------
def _head(K):
    """The seven parameters of the few-shot head: K class rows, two gate layers and the projection, depth 256."""
    return [K * 256] + [256 * 256, 256] * 3


def _denet(K):
    """Everything DENet trains: embedding, the five ASPP branches, their projection, the last convolution and its norm, the head."""
    aspp = [256 * 256, 256] + [256 * 256 * 9, 256] * 3 + [256 * 256, 256]
    return [256 * 1024 * 9, 256] + aspp + [256 * 1280, 256, 256 * 256 * 9, 256, 256] + _head(K)


def _ragged(tensors, elements, salt):
    """`tensors` sizes that differ by up to a factor of a thousand, odd ones and single elements among them."""
    rng = random.Random(salt * 7919 + tensors)
    weight = [math.exp(rng.uniform(0.0, math.log(1000.0))) for _ in range(tensors)]
    total = sum(weight)
    return [1 if tensors > 3 and i % 17 == 5 else max(1, int(elements * x / total)) for i, x in enumerate(weight)]


def _sizes(case):
    if case["layout"] == "head":
        return _head(case["K"])
    if case["layout"] == "denet":
        return _denet(case["K"])
    return _ragged(case["tensors"], case["elements"], case["salt"])


def listed():
    return [
        # the head alone is trained (frozen feature producer): seven tensors, 0.2 M elements, latency counts
        {"name": "norm head", "op": "norm", "layout": "head", "K": 21, "grad": "f32"},
        # what the trainer's clipping does to the gradients of the whole model before any optimizer
        {"name": "clip denet", "op": "clip", "layout": "denet", "K": 21, "grad": "f32"},
        # a long list of odd-sized bf16 gradients (an unfrozen feature producer)
        {"name": "norm ragged bf16", "op": "norm", "layout": "ragged", "tensors": 161, "elements": 25_557_033, "salt": 1, "grad": "bf16"},
        # a few very large gradients, far beyond the caches
        {"name": "norm large", "op": "norm", "layout": "ragged", "tensors": 5, "elements": 536_870_913, "salt": 2, "grad": "f32"},
        # the step of a run that trains the head alone
        {"name": "adamw32 head", "op": "adamw", "bits": 32, "layout": "head", "K": 21, "param": "f32", "grad": "f32", "clip": False},
        # the training step of the framework's own configuration, clipped, with 81 classes
        {"name": "adamw32 denet clip", "op": "adamw", "bits": 32, "layout": "denet", "K": 81, "param": "f32", "grad": "f32", "clip": True},
        # a long list of odd sizes whose gradients a bf16 backward left, fp32 parameters
        {"name": "adamw32 ragged bf16", "op": "adamw", "bits": 32, "layout": "ragged", "tensors": 161, "elements": 25_557_033, "salt": 3, "param": "f32", "grad": "bf16", "clip": False},
        # a model of 0.2 billion parameters: every stream is read and written from memory
        {"name": "adamw32 large", "op": "adamw", "bits": 32, "layout": "ragged", "tensors": 3, "elements": 201_326_611, "salt": 4, "param": "f32", "grad": "f32", "clip": False},
        # the same four with the states in 8 bits: the head with 81 classes
        {"name": "adamw8 head", "op": "adamw", "bits": 8, "layout": "head", "K": 81, "param": "f32", "grad": "f32", "clip": False},
        # the training step of the framework's own configuration, clipped
        {"name": "adamw8 denet clip", "op": "adamw", "bits": 8, "layout": "denet", "K": 21, "param": "f32", "grad": "f32", "clip": True},
        # a model held in bf16 throughout, odd sizes
        {"name": "adamw8 ragged bf16", "op": "adamw", "bits": 8, "layout": "ragged", "tensors": 161, "elements": 25_557_033, "salt": 5, "param": "bf16", "grad": "bf16", "clip": False},
        # where states of a fourth of the size are what makes the model fit
        {"name": "adamw8 large", "op": "adamw", "bits": 8, "layout": "ragged", "tensors": 3, "elements": 201_326_611, "salt": 6, "param": "f32", "grad": "f32", "clip": False},
    ]


def draw(rng):
    case = {"op": rng.choice(("norm", "clip", "adamw", "adamw", "adamw", "adamw"))}
    layout = rng.choice(("head", "denet", "ragged", "ragged", "ragged", "ragged"))
    case["layout"] = layout
    if layout == "ragged":
        case["elements"] = int(math.exp(rng.uniform(math.log(2e3), math.log(1.5e8))))
        case["tensors"] = max(1, min(case["elements"] // 64, int(math.exp(rng.uniform(0.0, math.log(300.0))))))
        case["salt"] = rng.randrange(1 << 20)
    else:
        case["K"] = rng.randrange(2, 129)
    case["grad"] = rng.choice(("f32", "bf16"))
    if case["op"] == "adamw":
        case["bits"] = rng.choice((8, 32))
        case["param"] = rng.choice(("f32", "bf16"))
        case["clip"] = rng.random() < 0.5
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _views(flat, sizes, offsets):
    return [flat[o:o + n] for o, n in zip(offsets, sizes)]


def _quantised(x, positive):
    """e4m3 codes and scales of x [blocks * QBLOCK]."""
    x = x.reshape(-1, QBLOCK)
    scale = (x.abs().amax(dim=1) / E4M3_MAX).clamp(min=TINY)
    y = x * (1.0 / scale)[:, None]
    if positive:
        y = torch.where(y > 0, y.clamp(min=2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).reshape(-1), scale


def prepare(case, seed):
    sizes = _sizes(case)
    eight = case.get("bits") == 8
    # the tensors are views of one buffer: packed without gaps as in a flat gradient bucket, and with each tensor
    # at a multiple of the scale's block where the states have 8 bits (the rest of its last block stays zero)
    offsets, at = [], 0
    for n in sizes:
        offsets.append(at)
        at += -(-n // QBLOCK) * QBLOCK if eight else n
    total = max(at, 1)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    live = torch.zeros(total, device=dev) if eight else None
    # gradients differ by orders of magnitude from tensor to tensor, and rows of 256 without any gradient occur (classes
    # that no episode of the batch shows)
    g = torch.randn(total, device=dev, generator=gen)
    dead = (torch.rand(-(-total // 256), device=dev, generator=gen) < 0.03).repeat_interleave(256)[:total]
    g[dead] = 0.0
    scale = [10.0 ** rng.uniform(-4.0, -1.0) for _ in sizes]
    for o, n, s in zip(offsets, sizes, scale):
        g[o:o + n] *= s
        if eight:
            live[o:o + n] = 1.0
    if eight:
        g *= live
    state = {"case": case, "sizes": sizes, "offsets": offsets, "step": FIRST_STEP}
    state["max_norm"] = 0.5 * float(g.double().square().sum().sqrt()) + 1e-3
    if case["op"] == "adamw":
        p = torch.randn(total, device=dev, generator=gen) * 0.05
        m = torch.randn(total, device=dev, generator=gen)
        r = torch.rand(total, device=dev, generator=gen) + 0.5
        for o, n, s in zip(offsets, sizes, scale):
            m[o:o + n] *= 0.3 * s
            r[o:o + n] *= s
        m[dead] = 0.0
        r[dead] = 0.0
        if eight:
            p, m, r = p * live, m * live, r * live
            state["exp_avg"], state["exp_avg_scale"] = _quantised(m, False)
            state["exp_avg_sqrt"], state["exp_avg_sqrt_scale"] = _quantised(r, True)
        else:
            state["exp_avg"], state["exp_avg_sq"] = m, r.square()
        state["p"] = p.to(TYPES[case["param"]])
    state["g"] = g.to(TYPES[case["grad"]])
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if case["op"] == "norm":
        return _norm_own(state) if own else _norm_plain(state)
    if case["op"] == "clip":
        return _clip_own(state) if own else _clip_plain(state)
    state["step"] += 1
    if own:
        return _adamw_own(state)
    return _adamw8_plain(state) if case["bits"] == 8 else _adamw32_plain(state)


def _outputs(state):
    if state["case"]["bits"] == 8:
        keys = ("p", "exp_avg", "exp_avg_scale", "exp_avg_sqrt", "exp_avg_sqrt_scale")
    else:
        keys = ("p", "exp_avg", "exp_avg_sq")
    return {k: state[k] for k in keys}


def _norm_own(state):
    from denet_amd import ops
    if "plan" not in state:
        state["plan"] = ops.GradNormPlan(_views(state["g"], state["sizes"], state["offsets"]))
    return {"norm": state["plan"].norm()}


def _clip_own(state):
    from denet_amd import ops
    if "plan" not in state:
        state["plan"] = ops.GradNormPlan(_views(state["g"], state["sizes"], state["offsets"]))
    norm = state["plan"].clip_(state["max_norm"])
    return {"norm": norm, "g": state["g"]}


def _adamw_own(state):
    from denet_amd import ops
    if "plan" not in state:
        def views(k):
            return _views(state[k], state["sizes"], state["offsets"])

        if state["case"]["bits"] == 8:
            firsts = [o // QBLOCK for o in state["offsets"]]
            counts = [-(-n // QBLOCK) for n in state["sizes"]]
            scales = [_views(state[k], counts, firsts) for k in ("exp_avg_scale", "exp_avg_sqrt_scale")]
            state["plan"] = ops.AdamWPlan(views("p"), views("g"), views("exp_avg"), views("exp_avg_sqrt"), *scales)
        else:
            state["plan"] = ops.AdamWPlan(views("p"), views("g"), views("exp_avg"), views("exp_avg_sq"))
    norm = state["plan"].step(state["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                              max_norm=state["max_norm"] if state["case"]["clip"] else None)
    out = _outputs(state)
    return dict(out, norm=norm) if state["case"]["clip"] else out


def _norm64(g):
    return g.double().square().sum().sqrt()


def _norm_plain(state):
    return {"norm": _norm64(state["g"]).float()}


def _coef(norm64, max_norm):
    return (max_norm / (norm64 + 1e-6)).clamp(max=1.0).float()


def _clip_plain(state):
    n = _norm64(state["g"])
    state["g"].copy_(state["g"].float() * _coef(n, state["max_norm"]))
    return {"norm": n.float(), "g": state["g"]}


def _update_plain(state, g, m, r):
    """p <- (1 - lr wd) p - lr / (1 - b1^t) m / (r / sqrt(1 - b2^t) + eps), r = sqrt(v)."""
    t = state["step"]
    denom = r * (1.0 / math.sqrt(1.0 - BETAS[1] ** t)) + EPS
    p = state["p"].float() * (1.0 - LR * DECAY) - (m / denom) * (LR / (1.0 - BETAS[0] ** t))
    state["p"].copy_(p)


def _grad_plain(state):
    if not state["case"]["clip"]:
        return state["g"].float(), {}
    n = _norm64(state["g"])
    return state["g"].float() * _coef(n, state["max_norm"]), {"norm": n.float()}


def _adamw32_plain(state):
    g, more = _grad_plain(state)
    m, v = state["exp_avg"], state["exp_avg_sq"]
    m.copy_(m * BETAS[0] + g * (1.0 - BETAS[0]))
    v.copy_(v * BETAS[1] + (g * g) * (1.0 - BETAS[1]))
    _update_plain(state, g, m, v.sqrt())
    return dict(_outputs(state), **more)


def _adamw8_plain(state):
    g, more = _grad_plain(state)
    m = (state["exp_avg"].float().reshape(-1, QBLOCK) * state["exp_avg_scale"][:, None]).reshape(-1)
    r = (state["exp_avg_sqrt"].float().reshape(-1, QBLOCK) * state["exp_avg_sqrt_scale"][:, None]).reshape(-1)
    m = m * BETAS[0] + g * (1.0 - BETAS[0])
    r = ((r * r) * BETAS[1] + (g * g) * (1.0 - BETAS[1])).sqrt()
    _update_plain(state, g, m, r)
    for key, x in (("exp_avg", m), ("exp_avg_sqrt", r)):
        code, scale = _quantised(x, key == "exp_avg_sqrt")
        state[key].copy_(code)
        state[key + "_scale"].copy_(scale)
    return dict(_outputs(state), **more)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    n = sum(_sizes(case))
    G = TYPES[case["grad"]].itemsize
    if case["op"] == "norm":
        return {"bytes": n * G, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * n * G, "flops": 3 * n}
    P = TYPES[case["param"]].itemsize
    flops = (16 if case["bits"] == 8 else 14) + (3 if case["clip"] else 0)
    states = 4 + 16 / QBLOCK if case["bits"] == 8 else 16
    return {"bytes": n * (2 * P + G + states), "flops": n * flops}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------
def _exact_norm(g):
    total = 0.0
    for part in g.split(1 << 26):
        x = part.to(torch.float64)
        total += float(torch.dot(x, x))
    return math.sqrt(total)


def _nearest_e4m3(y):
    """The e4m3 value nearest to each y >= 0 (ties to the even code), y <= 448: a step of 2^(e-3) in [2^e, 2^(e+1)), of 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(y.clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    g = s["g"]
    if case["op"] == "norm":
        return {"norm": torch.tensor(_exact_norm(g), dtype=torch.float64)}
    coef, out = 1.0, {}
    if case["op"] == "clip" or case["clip"]:
        norm = _exact_norm(g)
        coef = min(1.0, s["max_norm"] / (norm + 1e-6))
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
    g = g.to(torch.float64) * coef
    if case["op"] == "clip":
        return dict(out, g=g)
    (b1, b2), t = BETAS, FIRST_STEP + 1

    def held(code, scale):
        return torch.mul(s[code].to(torch.float64), s[scale].to(torch.float64).repeat_interleave(QBLOCK))

    if case["bits"] == 8:
        m, v = held("exp_avg", "exp_avg_scale"), held("exp_avg_sqrt", "exp_avg_sqrt_scale") ** 2
    else:
        m, v = s["exp_avg"].to(torch.float64), s["exp_avg_sq"].to(torch.float64)
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g * g, v, b2)
    m_hat, v_hat = m / (1 - b1 ** t), v / (1 - b2 ** t)
    p = s["p"].to(torch.float64)
    out["p"] = p - LR * (DECAY * p + m_hat / (v_hat.sqrt() + EPS))
    if case["bits"] == 32:
        return dict(out, exp_avg=m, exp_avg_sq=v)
    for key, x in (("exp_avg", m), ("exp_avg_sqrt", v.sqrt())):
        rows = x.reshape(-1, QBLOCK)
        scale = torch.maximum(rows.abs().max(dim=1).values / E4M3_MAX, torch.tensor(TINY, dtype=torch.float64, device=x.device))
        y = rows / scale[:, None]
        code = _nearest_e4m3(y.abs()) * torch.sign(y)
        if key == "exp_avg_sqrt":
            code = torch.where((y > 0) & (code == 0), torch.full_like(code, 2.0 ** -9), code)
        out[key], out[key + "_scale"] = code.reshape(-1), scale
    return out

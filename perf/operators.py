"""The optimizer's operators over many tensors, as cases to time: the AdamW step with its moments in 32 and in 8 bits, and
the clipping of the gradients' global norm, alone and inside a step.

`own = False` computes them in elementary torch operations over one flat buffer, `own = True` calls pde_amd.optim.

Layout of every case: the tensors lie in one flat buffer in order, each at the next multiple of 128 elements (as an
allocator would place them), with zeros between them; moments and master weights lie in float32 or 8-bit buffers of the same layout.

Formulas, t counted from 1 (m, v: the moments; g: the gradient, scaled by the clipping factor where the case clips):
    norm = sqrt(sum of g^2 over all tensors),  factor = min(1, max_norm / (norm + 1e-6))
    m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2
    p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

8-bit moments.  Each block of 128 elements of the layout has one scale 2^(s - 127), s a byte (255: a block with a value that
is not finite), and a byte for each element:
    m: sign, 4 bits of exponent (bias 7), 3 of mantissa, subnormal below 2^-6; the largest magnitude is 1.75 * 2^8
    v: 5 bits of exponent (bias 15), 3 of mantissa, subnormal below 2^-14; the largest is 1.75 * 2^16
The scale is the smallest with which the block's largest magnitude stays below the largest code's (s between 0 and 246 for m,
238 for v; 0 for a block of zeros).  On the scale of the codes (equal steps between neighbours, y real) the code is floor(y + u), u = U / 2^17 with
    U_m = ((0x9E3779B9 i + 0xC13FA9A9 t) mod 2^32) >> 15 | 1,   U_v = ((0x6A09E667 i + 0x91E10DA5 t) mod 2^32) >> 15 | 1
for the element at place i of the layout: over the steps the rounding is even on both sides, so small changes are not lost.
(U is odd, so u averages 1/2 and never lies on the border of a y that is itself on a code, as 0.9 * 1.25 = 1.125 is.)
A v above zero keeps at least the code 1.  The parameters' update takes m and v as they are before they are rounded.
"""
import math
import random

import torch

own = False

BLOCK = 128
LR, B1, B2, EPS, WD, MAX_NORM = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 1.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one 2-50x4-1 net, the size of a training step where only latency counts
        {"name": "adamw one net", "op": "adamw", "layers": "2,50,50,50,50,1", "nets": 1, "dtype": "f32", "master": False, "clip": False, "step": 1000},
        # 24 window models of width 100 stepped together: 240 tensors of 2 to 10 000 elements
        {"name": "adamw 24 nets", "op": "adamw", "layers": "2,100,100,100,100,2", "nets": 24, "dtype": "f32", "master": False, "clip": True, "step": 40},
        # a bf16 model with float32 master weights, odd sizes
        {"name": "adamw bf16 master 67M", "op": "adamw", "tensors": 60, "numel": 67_000_003, "shape_seed": 11, "dtype": "bf16", "master": True, "clip": False, "step": 17},
        # a float32 model far beyond the caches, clipped: the largest
        {"name": "adamw f32 clip 240M", "op": "adamw", "tensors": 120, "numel": 240_000_001, "shape_seed": 12, "dtype": "f32", "master": False, "clip": True, "step": 5000},
        # the same small net with its moments in 8 bits
        {"name": "adamw8 one net", "op": "adamw8", "layers": "2,50,50,50,50,1", "nets": 1, "dtype": "f32", "master": False, "clip": False, "step": 1000},
        # a few million float32 weights in tensors of odd sizes
        {"name": "adamw8 f32 5M", "op": "adamw8", "tensors": 37, "numel": 5_000_011, "shape_seed": 13, "dtype": "f32", "master": False, "clip": False, "step": 3},
        # float32 with clipping inside the step
        {"name": "adamw8 f32 clip 60M", "op": "adamw8", "tensors": 150, "numel": 60_000_007, "shape_seed": 14, "dtype": "f32", "master": False, "clip": True, "step": 200},
        # bf16 weights, where memory is what 8-bit moments are taken for
        {"name": "adamw8 bf16 240M", "op": "adamw8", "tensors": 90, "numel": 240_000_001, "shape_seed": 15, "dtype": "bf16", "master": False, "clip": False, "step": 20000},
        # clipping before somebody else's step: the small net
        {"name": "clip one net", "op": "clip", "layers": "2,50,50,50,50,1", "nets": 1, "dtype": "f32", "master": False, "clip": True, "step": 1},
        # many bf16 gradients of odd sizes
        {"name": "clip bf16 33M", "op": "clip", "tensors": 300, "numel": 33_000_001, "shape_seed": 16, "dtype": "bf16", "master": False, "clip": True, "step": 1},
        # float32 gradients far beyond the caches
        {"name": "clip f32 240M", "op": "clip", "tensors": 48, "numel": 240_000_001, "shape_seed": 17, "dtype": "f32", "master": False, "clip": True, "step": 1},
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "clip"])
    numel = int(math.exp(rng.uniform(math.log(700), math.log(120_000_000))))
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    return {"op": op, "tensors": min(int(math.exp(rng.uniform(0, math.log(400)))), max(1, numel // 20)), "numel": numel,
            "shape_seed": rng.randrange(1 << 20), "dtype": dtype, "master": op != "clip" and dtype != "f32" and rng.random() < 0.5,
            "clip": op == "clip" or rng.random() < 0.4, "step": int(math.exp(rng.uniform(0, math.log(30_000))))}


def shapes_of(case):
    if "layers" in case:
        w = [int(x) for x in case["layers"].split(",")]
        one = [s for i in range(len(w) - 1) for s in ((w[i + 1], w[i]), (w[i + 1],))]
        return one * case["nets"]
    r = random.Random(case["shape_seed"])
    share = [math.exp(r.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    return [(max(1, int(case["numel"] * s / sum(share))),) for s in share]


def layout(case):
    """[(first element, shape)], and the layout's length."""
    at, places = 0, []
    for s in shapes_of(case):
        places.append((at, s))
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return places, at


def inputs(case, seed):
    """Everything a pass reads, in the middle of a training: flat buffers of the layout."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    places, n = layout(case)
    dt = DTYPES[case["dtype"]]
    dist = {k: torch.empty(n, device=dev).normal_(generator=gen) for k in ("p", "g", "m", "v")}
    sizes = torch.tensor([math.prod(s) for _, s in places], device=dev)
    blocks = (sizes + BLOCK - 1) // BLOCK
    tensor = torch.repeat_interleave(torch.arange(len(places), device=dev), blocks * BLOCK, output_size=n)
    first = torch.tensor([a for a, _ in places], device=dev)
    real = torch.arange(n, device=dev) - first[tensor] < sizes[tensor]
    # each tensor has a scale of its own, some elements have no gradient (units that are off)
    size = torch.exp(1.5 * torch.empty(len(places), device=dev).normal_(generator=gen))[tensor] * real
    off = torch.empty(n, device=dev).uniform_(generator=gen) < 0.05
    s = {"p": (0.1 * dist["p"] * real).to(dt), "g": (2e-3 * dist["g"] * size * ~off).to(dt)}
    if case["op"] == "clip":
        s["g"] = (s["g"].float() * (20.0 * MAX_NORM / max(1e-12, float(s["g"].double().square().sum().sqrt())))).to(dt)  # to be clipped by 20
        return s, places, real
    s["t"] = case["step"] - 1
    if case["master"]:
        s["master"] = 0.1 * dist["p"] * real
    m, v = 6e-4 * dist["m"] * size, (2e-3 * size) ** 2 * (0.1 + dist["v"] ** 2)
    if s["t"] == 0:
        m, v = torch.zeros_like(m), torch.zeros_like(v)
    if case["op"] == "adamw":
        s["m"], s["v"] = m, v
    else:
        half = torch.full((n,), 1 << 16, dtype=torch.int64, device=dev)
        s["m"], s["sm"] = encode(m.double(), half, M_FORM)
        s["v"], s["sv"] = encode(v.double(), half, V_FORM)
    return s, places, real


# ---- the 8-bit form, plain: what is exact in float64 stays exact ----
M_FORM = {"bias": 7, "top": 8, "most": 246, "signed": True}
V_FORM = {"bias": 15, "top": 16, "most": 238, "signed": False}


def power(e):
    """2^e for whole e within float64's normal range, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def decode(code, scale, form):
    mag = (code & 127 if form["signed"] else code).to(torch.int64)
    e, f = mag >> 3, mag & 7
    whole = torch.where(e > 0, (8 + f) << (e - 1).clamp(min=0), f).double() * 2.0 ** (-2 - form["bias"])
    if form["signed"]:
        whole = torch.where(code > 127, -whole, whole)
    out = whole.view(-1, BLOCK) * power(scale.to(torch.int64) - 127)[:, None]
    return torch.where((scale == 255)[:, None], math.nan, out).view(-1)


def encode(x, u, form):
    x = x.view(-1, BLOCK)
    most = x.abs().amax(1)
    frac, e = torch.frexp(most)  # most = frac * 2^e, frac in [0.5, 1)
    k = e.to(torch.int64) - 1 + (frac >= 0.875) - form["top"]
    s = torch.where(most > 0, (k + 127).clamp(0, form["most"]), 0)
    a = x.abs() * power(127 - s)[:, None]
    frac, e = torch.frexp(a)
    e = e.to(torch.int64) - 1 + form["bias"]
    y = torch.where(a >= 2.0 ** (1 - form["bias"]), 8.0 * e + 8.0 * (2.0 * frac - 1.0), a * 2.0 ** (2 + form["bias"]))
    code = torch.floor(y + u.view(-1, BLOCK).double() * 2.0 ** -17).clamp(max=126 if form["signed"] else 254).to(torch.int64)
    if form["signed"]:
        code = code + 128 * (x < 0)
    else:
        code = torch.where(x > 0, code.clamp(min=1), code)
    bad = ~torch.isfinite(most)
    return torch.where(bad[:, None], 0, code).to(torch.uint8).view(-1), torch.where(bad, 255, s).to(torch.uint8)


def dither(n, t, place, step, device):
    return ((torch.arange(n, device=device) * place + t * step) & 0xFFFFFFFF) >> 15 | 1


# ---- what a pass runs ----
def prepare(case, seed):
    s, places, _ = inputs(case, seed)
    s["op"], s["clip"] = case["op"], case["clip"]
    s["params"] = []
    for at, shape in places:
        p = torch.nn.Parameter(s["p"][at:at + math.prod(shape)].view(shape))
        p.grad = s["g"][at:at + math.prod(shape)].view(shape)
        s["params"].append(p)
    if own and case["op"] != "clip":
        from pde_amd.optim import GroupedAdamW
        opt = GroupedAdamW(s["params"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=32 if case["op"] == "adamw" else 8,
                           max_norm=MAX_NORM if case["clip"] else None, master_weights=case["master"])
        sd = opt.state_dict()
        held = sd["fused"]
        held["exp_avg"].copy_(s.pop("m"))
        held["exp_avg_sq"].copy_(s.pop("v"))
        if case["op"] == "adamw8":
            held["exp_avg_scale"].copy_(s.pop("sm"))
            held["exp_avg_sq_scale"].copy_(s.pop("sv"))
        if case["master"]:
            held["master"].copy_(s.pop("master"))
        held["device_state"].copy_(torch.tensor([s["t"], B1 ** s["t"], B2 ** s["t"]], dtype=torch.float64).expand(len(places), 3))
        opt.load_state_dict(sd)
        s["opt"] = opt
    return s


def run(s):
    if own:
        return run_own(s)
    if s["op"] == "clip":
        g = s["g"].float()
        norm, factor = norm_and_factor(g)
        s["g"].copy_(g * factor)
        return {"grads": s["g"], "norm": norm.float()}
    out, g = {}, s["g"].float() if s["op"] == "adamw" else s["g"].double()  # 8 bits: a rounding's border asks for 64
    if s["clip"]:
        norm, factor = norm_and_factor(g)
        g = g * factor
        out["norm"] = norm.float()
    s["t"] += 1
    step = plain32 if s["op"] == "adamw" else plain8
    out["exp_avg"], out["exp_avg_sq"] = step(s, g, s["master"] if "master" in s else s["p"])
    if "master" in s:
        s["p"].copy_(s["master"])
        out["master"] = s["master"]
    out["params"] = s["p"]
    return out


def norm_and_factor(g):
    norm = g.square().sum(dtype=torch.float64).sqrt()
    return norm, (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).to(g.dtype)


def plain32(s, g, p):
    m, v, t = s["m"], s["v"], s["t"]
    m.mul_(B1).add_(g, alpha=1 - B1)
    v.mul_(B2).add_(g * g, alpha=1 - B2)
    denom = v.sqrt().mul_(1 / math.sqrt(1 - B2 ** t)).add_(EPS)
    p.copy_(p.float() * (1 - LR * WD) - m / denom * (LR / (1 - B1 ** t)))
    return m, v


def plain8(s, g, p):
    t, n = s["t"], g.numel()
    m = B1 * decode(s["m"], s["sm"], M_FORM) + (1 - B1) * g
    v = B2 * decode(s["v"], s["sv"], V_FORM) + (1 - B2) * g * g
    p.copy_(p.double() * (1 - LR * WD) - m / ((v / (1 - B2 ** t)).sqrt() + EPS) * (LR / (1 - B1 ** t)))
    s["m"], s["sm"] = encode(m, dither(n, t, 0x9E3779B9, 0xC13FA9A9, g.device), M_FORM)
    s["v"], s["sv"] = encode(v, dither(n, t, 0x6A09E667, 0x91E10DA5, g.device), V_FORM)
    return decode(s["m"], s["sm"], M_FORM).float(), decode(s["v"], s["sv"], V_FORM).float()


def run_own(s):
    if s["op"] == "clip":
        from pde_amd.optim import clip_grad_norm_
        norm = clip_grad_norm_(s["params"], MAX_NORM)
        return {"grads": s["g"], "norm": norm}
    opt = s["opt"]
    opt.step()
    m, v = opt.moments()
    out = {"exp_avg": m, "exp_avg_sq": v, "params": s["p"]}
    if s["clip"]:
        out["norm"] = opt.grad_norm
    if opt.master is not None:
        out["master"] = opt.master
    return out


def work(case):
    n = sum(math.prod(s) for s in shapes_of(case))
    w = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":
        return {"bytes": 2 * w * n, "flops": 3 * n}
    weights = 3 * w if not case["master"] else 2 * w + 8  # the gradient read, the weights read and written
    moments = 16 if case["op"] == "adamw" else 4 + 4 / BLOCK + 8  # 8 bits: codes and scales both ways, and the values returned
    return {"bytes": int((weights + moments) * n), "flops": (13 + 3 * case["clip"]) * n}


# ---- the definition in 64 bits, from the formulas and tables of the codes' values ----
def exact(case, seed):
    s, _, _ = inputs(case, seed)
    g = s["g"].double()
    out = {}
    if case["clip"]:
        norm = torch.sqrt(torch.dot(g, g))
        g = g * min(1.0, MAX_NORM / (float(norm) + 1e-6))
        out["norm"] = norm
    if case["op"] == "clip":
        return {"grads": g, "norm": norm}
    t = s["t"] + 1
    if case["op"] == "adamw":
        m, v = s["m"].double(), s["v"].double()
    else:
        m, v = table_values(s["m"], s["sm"], True), table_values(s["v"], s["sv"], False)
    m, v = m + (g - m) * (1 - B1), v + (g ** 2 - v) * (1 - B2)
    p = s["master" if case["master"] else "p"].double()
    hat_m, hat_v = m / (1 - B1 ** t), v / (1 - B2 ** t)
    p = p - LR * WD * p - LR * hat_m / (torch.sqrt(hat_v) + EPS)
    if case["op"] == "adamw8":
        i = torch.arange(m.numel(), device=m.device)
        m = table_round(m, (i * 0x9E3779B9 + t * 0xC13FA9A9) % 2 ** 32 // 2 ** 16 * 2 + 1, True)
        v = table_round(v, (i * 0x6A09E667 + t * 0x91E10DA5) % 2 ** 32 // 2 ** 16 * 2 + 1, False)
    out.update(exp_avg=m, exp_avg_sq=v, params=p)
    if case["master"]:
        out["master"] = p
    return out


def table(signed, device):
    """All magnitudes that a code can mean before its block's scale, in order."""
    bias, count = (7, 127) if signed else (15, 255)
    return torch.tensor([(c % 8) / 8 * 2.0 ** (1 - bias) if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - bias) for c in range(count)],
                        dtype=torch.float64, device=device)


def table_values(code, scale, signed):
    c = code.long()
    tab = table(signed, code.device)
    x = torch.where(c >= 128, -tab[c % 128 % 127], tab[c % 128 % 127]) if signed else tab[c % 255]
    return (x.view(-1, BLOCK) * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), scale.double() - 127)[:, None]).view(-1)


def table_round(x, big_u, signed):
    """The value that x's code stands for: the last entry of the table at or below it, or the next, by the place between them."""
    tab = table(signed, x.device)
    x = x.view(-1, BLOCK)
    a, two = x.abs(), torch.tensor(2.0, dtype=torch.float64, device=x.device)
    scales = torch.pow(two, torch.arange(0, 247 if signed else 239, device=x.device).double() - 127)
    s = torch.searchsorted(scales * tab[-1], a.amax(1)).clamp(max=len(scales) - 1)  # the smallest that holds the largest
    # a largest magnitude of exactly 1.75 * 2^e takes the next scale
    s = torch.where(scales[s] * tab[-1] == a.amax(1), (s + 1).clamp(max=len(scales) - 1), s)
    unit = scales[s][:, None]
    y = a / unit
    c = (torch.searchsorted(tab, y, right=True) - 1).clamp(max=len(tab) - 2)
    up = (y - tab[c]) / (tab[c + 1] - tab[c]) + big_u.view(-1, BLOCK) / 2.0 ** 17 >= 1.0
    c = c + up
    if not signed:
        c = torch.where(a > 0, c.clamp(min=1), c)
    return (torch.where(x < 0, -tab[c], tab[c]) * unit).view(-1)

"""Optimiser operators over many tensors at once: what is measured, and the operators' plain forms.

adamw    AdamW with 32-bit moments (fsgs_amd.optim.FusedAdamW), optionally with fp32 master weights behind 16-bit
         parameters and with the gradients' global norm bounded inside the step
adamw8   the same step on moments held in 8 bits (state_bits=8), and the moments read back as values
clip     the gradients' global 2-norm and their scaling to a bound (fsgs_amd.optim.clip_grad_norm_)

Three layouts of parameters: "cloud" is the six tensors of a cloud of `rows` Gaussians (59 values each, one learning rate
per tensor); "poses" is the two tensors of a track of `rows` frames (quaternions and translations); "layers" is `count` tensors of ragged sizes that sum to about `total`, cut out of one flat buffer on 64-element
boundaries, as programs with one communication bucket hold them.

8-bit moments: blocks of 128 consecutive elements share one power of two per moment.  The first moment is kept as
e4m3 codes of m / 2^E, the second as e4m3 codes of sqrt(v) / 2^E; E is the smallest power that brings the block's largest
value to at most 448.  A value is rounded down or up to a neighbouring code by comparing its remainder with a threshold
in [0, 1) that belongs to the element and the step (a quasi-random sequence), so that the mean over steps is unbiased; a
second moment that is not zero keeps at least the smallest code."""
import math
import random

import torch

own = False

CLOUD = ((3, 8e-4), (3, 2.5e-3), (45, 1.25e-4), (1, 0.05), (3, 5e-3), (4, 1e-3))  # floats per Gaussian, learning rate
POSES = ((4, 0.01), (3, 0.01))
BETAS = (0.9, 0.999)
BLOCK = 128
GOLDEN, ROOT2 = 0x9E3779B9, 0x6A09E667        # 2^32 times the fractions of the golden ratio and of sqrt(2)
R2_X, R2_Y = 0xC13FA9A9, 0x91E10DA5           # 2^32 / plastic number, 2^32 / its square (the R2 sequence)


def listed():
    cloud = dict(layout="cloud", dtype="float32", master=False)
    layers = dict(layout="layers")
    return [
        # the pose optimiser of a tracked frame: two tensors, some thousand floats: nothing but latency
        dict(name="poses of 200 frames", op="adamw", layout="poses", rows=200, dtype="float32", master=False,
             decay=0.0, eps=1e-8, bound=0.0),
        # a mapping step's optimiser at 640x512 / 20 000 Gaussians, 1280x1024 / 300 000 and 1920x1080 / 1 000 000
        dict(name="cloud 20k", op="adamw", rows=20000, decay=0.01, eps=1e-15, bound=0.0, **cloud),
        dict(name="cloud 300k, bounded norm", op="adamw", rows=300000, decay=0.01, eps=1e-15, bound=1.0, **cloud),
        dict(name="cloud 1M", op="adamw", rows=1000000, decay=0.0, eps=1e-15, bound=0.0, **cloud),
        # a network trained in 16 bits: weights and biases, with and without fp32 master weights
        dict(name="160 layers bf16, master", op="adamw", count=160, total=64000000, shape_seed=5, dtype="bfloat16",
             master=True, decay=0.1, eps=1e-8, bound=0.0, **layers),
        dict(name="97 layers fp16", op="adamw", count=97, total=500001, shape_seed=9, dtype="float16", master=False,
             decay=0.01, eps=1e-6, bound=0.5, **layers),
        # the same with the moments in 8 bits, where memory or its bandwidth is what is short
        dict(name="cloud 20k, 8-bit", op="adamw8", rows=20011, decay=0.01, eps=1e-15, bound=0.0, **cloud),
        dict(name="cloud 1M, 8-bit", op="adamw8", rows=1000000, decay=0.01, eps=1e-15, bound=0.0, **cloud),
        dict(name="24 layers bf16, master, 8-bit", op="adamw8", count=24, total=20000000, shape_seed=11,
             dtype="bfloat16", master=True, decay=0.1, eps=1e-8, bound=1.0, **layers),
        # the norm alone (below its bound nothing is scaled) and the norm with the scaling
        dict(name="clip cloud 300k", op="clip", rows=300000, bound=1.0, **cloud),
        dict(name="clip 160 layers bf16", op="clip", count=160, total=64000000, shape_seed=5, dtype="bfloat16",
             master=False, bound=0.5, **layers),
        dict(name="clip 40 layers, below", op="clip", count=40, total=300007, shape_seed=13, dtype="float32",
             master=False, bound=1e9, **layers),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["adamw", "adamw8", "clip"])
    case = dict(op=op, dtype="float32", master=False)
    kind = rng.random()
    if kind < 0.35:
        case.update(layout="cloud", rows=log(3, 900000))
    elif kind < 0.45:
        case.update(layout="poses", rows=log(2, 5000))
    else:
        case.update(layout="layers", count=rng.randint(1, 24 if op == "adamw8" else 200), total=log(300, 40000000),
                    shape_seed=rng.randrange(1 << 20), dtype=rng.choice(["float32", "bfloat16", "float16"]))
        if op != "clip" and case["dtype"] != "float32":
            case["master"] = rng.random() < 0.5
    case["bound"] = rng.choice([0.1, 1.0, 1e9]) if op == "clip" else rng.choice([0.0, 0.0, 0.7])
    if op != "clip":
        case.update(decay=rng.choice([0.0, 0.01, 0.1]), eps=1e-6 if case["dtype"] == "float16" else rng.choice([1e-8, 1e-15]))
    return case


def _shapes(case):
    """[(elements, learning rate)] of the case's tensors."""
    # moments in 8 bits: the decayed rates of a run's later part (a tenth), for all layouts
    late = 0.1 if case["op"] == "adamw8" else 1.0
    if case["layout"] != "layers":
        return [(case["rows"] * k, lr * late) for k, lr in (CLOUD if case["layout"] == "cloud" else POSES)]
    rng = random.Random(case["shape_seed"])
    raw = [math.exp(rng.uniform(0.0, 8.0)) for _ in range(case["count"])]
    return [(max(1, int(case["total"] * r / sum(raw))), late * rng.choice([1e-3, 3e-4])) for r in raw]


def work(case):
    n = sum(k for k, _ in _shapes(case))
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "clip":
        return {"bytes": n * size * (1 if case["bound"] >= 1e9 else 2) + 4, "flops": 3.0 * n}
    moments = 16 if case["op"] == "adamw" else 4 + 4 / BLOCK + 4  # read and written; 8 bits: and given back in 16
    weights = 8 + size if case["master"] else 2 * size
    return {"bytes": n * (weights + size + moments), "flops": (15.0 if case["op"] == "adamw" else 45.0) * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """Parameters, gradients and moments of a run in progress: gradients whose scale differs from row to row by orders
    of magnitude, a part of them exactly zero (what no ray has hit), moments of that scale."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda n: torch.rand(n, device="cuda", generator=gen)  # noqa: E731
    normal = lambda n: torch.randn(n, device="cuda", generator=gen)  # noqa: E731
    shapes = _shapes(case)
    dtype = getattr(torch, case["dtype"])
    starts, end = [], 0
    for n, _ in shapes:
        starts.append(end)
        end += -(-n // 64) * 64
    flat = {k: torch.zeros(end, device="cuda") for k in ("p", "g", "m", "v")}
    cut = {k: [b[a:a + n] for a, (n, _) in zip(starts, shapes)] for k, b in flat.items()}
    for i, (n, _) in enumerate(shapes):
        row = 16 if case["layout"] == "layers" else n // case["rows"]
        scale = torch.exp(2.0 * normal(-(-n // row)) - 4.0)
        scale = scale.repeat_interleave(row)[:n]
        cut["p"][i].copy_(normal(n))
        cut["g"][i].copy_(normal(n) * scale * (rand(n) < 0.8))
        cut["m"][i].copy_(normal(n) * scale * 0.3)
        cut["v"][i].copy_(scale.square() * (0.3 + rand(n)))
    s = {"case": case, "flat": {}, "lr": [lr for _, lr in shapes], "step": int(torch.randint(1, 4000, (1,), device="cuda", generator=gen))}
    if case["layout"] == "layers":
        p, g = flat["p"].to(dtype), flat["g"].to(dtype)
        s["flat"].update(p=p, g=g)
        s["p"], s["g"] = ([b[a:a + n] for a, (n, _) in zip(starts, shapes)] for b in (p, g))
        if case["master"]:
            w = p.float()
            s["flat"]["w"], s["w"] = w, [w[a:a + n] for a, (n, _) in zip(starts, shapes)]
    else:
        s["p"], s["g"] = [t.clone() for t in cut["p"]], [t.clone() for t in cut["g"]]
    if case["op"] == "adamw":
        if case["layout"] == "layers":
            s["flat"].update(m=flat["m"], v=flat["v"])
            s["m"], s["v"] = cut["m"], cut["v"]
        else:
            s["m"], s["v"] = [t.clone() for t in cut["m"]], [t.clone() for t in cut["v"]]
    elif case["op"] == "adamw8":
        enc = [(_encode(m, s["step"], GOLDEN, R2_X, False), _encode(v.sqrt(), s["step"], ROOT2, R2_Y, True))
               for m, v in zip(cut["m"], cut["v"])]
        s["mq"], s["rq"] = [e[0][0] for e in enc], [e[1][0] for e in enc]
        s["scales"] = [torch.stack((e[0][1], e[1][1]), 1).contiguous() for e in enc]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["bound"] = case["bound"]
    s["p"] = [p.detach().requires_grad_(True) for p in s["p"]]
    for p, g in zip(s["p"], s["g"]):
        p.grad = g
    if own:
        s["optim"] = _framework()
        if case["op"] != "clip":
            s["opt"] = s["optim"].FusedAdamW(
                [{"params": [p], "lr": lr} for p, lr in zip(s["p"], s["lr"])], betas=BETAS, eps=case["eps"],
                weight_decay=case["decay"], state_bits=8 if case["op"] == "adamw8" else 32,
                master_weights=case["master"], max_grad_norm=case["bound"] or None)
            for i, p in enumerate(s["p"]):
                st = s["opt"].state[p] = {"step": s["step"]}
                if case["op"] == "adamw":
                    st.update(exp_avg=s["m"][i], exp_avg_sq=s["v"][i])
                else:
                    st.update(exp_avg_q=s["mq"][i], exp_avg_sq_q=s["rq"][i], scales=s["scales"][i])
                if case["master"]:
                    st["master"] = s["w"][i]
    return s


def _framework():
    import os
    import sys

    path = os.path.join(os.getcwd(), "free-surgs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from fsgs_amd import optim

    return optim


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "clip":
        if own:
            norm = s["optim"].clip_grad_norm_(s["p"], s["bound"])
        else:
            norm = _clip_plain(s)
        # the gradients of the next pass are the ones that this pass left, so its bound is a little lower: it clips too
        s["bound"] *= 0.99999
        return {"norm": norm, "g": s["flat"]["g"] if s["flat"] else s["g"]}
    if own:
        s["opt"].step()
        moments = s["opt"].moments(torch.bfloat16) if case["op"] == "adamw8" else None
    else:
        moments = _step8_plain(s) if case["op"] == "adamw8" else _step_plain(s)
    out = {k: s["flat"][k] if k in s["flat"] else s[k] for k in ("p", "w", "m", "v") if k in s}
    if moments is not None:
        out["m"], out["v"] = [m for m, _ in moments], [v for _, v in moments]
    return out


def _coefficient(grads, bound):
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    return norm, (bound / (norm + 1e-6)).clamp(max=1.0)


@torch.no_grad()
def _clip_plain(s):
    norm, coef = _coefficient([s["flat"]["g"]] if s["flat"] else s["g"], s["bound"])
    if s["case"]["dtype"] == "float32":
        torch._foreach_mul_(s["g"], coef)
    else:
        torch._foreach_copy_(s["g"], torch._foreach_mul([g.float() for g in s["g"]], coef))
    return norm


def _grads32(s):
    g = [g.float() for g in s["g"]]
    if s["bound"]:
        _, coef = _coefficient([s["flat"]["g"]] if s["flat"] else s["g"], s["bound"])
        g = torch._foreach_mul(g, coef)
    return g


def _weights32(s):
    """The fp32 weights that the step changes: the masters, the parameters themselves, or a widened copy."""
    p = [p.detach() for p in s["p"]]
    return p, s["w"] if "w" in s else p if s["case"]["dtype"] == "float32" else [x.float() for x in p]


@torch.no_grad()
def _step_plain(s):
    s["step"] += 1
    (b1, b2), t, eps, decay = BETAS, s["step"], s["case"]["eps"], s["case"]["decay"]
    g = _grads32(s)
    p, w = _weights32(s)
    torch._foreach_mul_(s["m"], b1)
    torch._foreach_add_(s["m"], g, alpha=1 - b1)
    torch._foreach_mul_(s["v"], b2)
    torch._foreach_addcmul_(s["v"], g, g, value=1 - b2)
    denom = torch._foreach_sqrt(s["v"])
    torch._foreach_div_(denom, math.sqrt(1 - b2 ** t))
    torch._foreach_add_(denom, eps)
    torch._foreach_mul_(w, [1 - lr * decay for lr in s["lr"]])
    torch._foreach_addcdiv_(w, s["m"], denom, scalars=[-lr / (1 - b1 ** t) for lr in s["lr"]])
    if w is not p:
        torch._foreach_copy_(p, w)


def _threshold(n, step, phase, turn):
    """Twenty bits of the element's threshold at this step."""
    i = torch.arange(n, device="cuda", dtype=torch.int64)
    return ((i * phase + step * turn) & 0xFFFFFFFF) >> 12


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _power(e):
    """2^(e - 127) for biased exponents 1..254."""
    return (e.to(torch.int32) << 23).view(torch.float32)


def _encode(x, step, phase, turn, keep):
    """(e4m3 codes, one biased exponent for each block) of a flat fp32 tensor."""
    f = _blocks(x)
    fine = torch.isfinite(f)
    a = torch.where(fine, f.abs(), torch.zeros_like(f))
    mant, ex = torch.frexp(a.amax(1))
    e = torch.where(mant > 0, (ex - 9 + (mant > 0.875) + 127).clamp(1, 254), torch.ones_like(ex))
    y = a * _power(254 - e)[:, None]
    u = _blocks(_threshold(x.numel(), step, phase, turn))
    code = torch.where(y < 2.0 ** -6, (y.double() * 512 + u.double() / 2 ** 20).floor().to(torch.int64),
                       ((y.view(torch.int32).to(torch.int64) + u) >> 20) - 960)
    if keep:
        code = torch.maximum(code, (a > 0).to(torch.int64))
    code = torch.where(fine, code, torch.full_like(code, 127)) | ((f < 0).to(torch.int64) << 7)
    return code.to(torch.uint8).view(-1)[:x.numel()].view(torch.float8_e4m3fn), e.to(torch.uint8)


def _decode(codes, e):
    return (_blocks(codes.float()) * _power(e)[:, None]).view(-1)[:codes.numel()]


@torch.no_grad()
def _step8_plain(s):
    s["step"] += 1
    p, w = _weights32(s)
    moments = [_one8(s, *a) for a in zip(w, _grads32(s), s["mq"], s["rq"], s["scales"], s["lr"])]
    if w is not p:
        torch._foreach_copy_(p, w)
    return moments


def _one8(s, w, g, mq, rq, scales, lr):
    (b1, b2), t, eps, decay = BETAS, s["step"], s["case"]["eps"], s["case"]["decay"]
    m = _decode(mq, scales[:, 0]) * b1 + g * (1 - b1)
    r = (_decode(rq, scales[:, 1]).square() * b2 + g.square() * (1 - b2)).sqrt()
    w.mul_(1 - lr * decay).sub_((lr / (1 - b1 ** t)) * (m / (r / math.sqrt(1 - b2 ** t) + eps)))
    for codes, column, new in ((mq, 0, _encode(m, t, GOLDEN, R2_X, False)), (rq, 1, _encode(r, t, ROOT2, R2_Y, True))):
        codes.copy_(new[0])
        scales[:, column] = new[1]
    return _decode(mq, scales[:, 0]).bfloat16(), _decode(rq, scales[:, 1]).square().bfloat16()


# ---- in 64 bits, from the definition --------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    grads = [g.double() for g in s["g"]]
    norm = torch.sqrt(sum((g * g).sum() for g in grads))
    factor = min(1.0, case["bound"] / (float(norm) + 1e-6)) if case["bound"] else 1.0
    grads = [g * factor for g in grads]
    if case["op"] == "clip":
        return {"norm": norm, "g": _as_laid_out(s, "g", grads)}
    t = s["step"] + 1
    out = {"p": [], "m": [], "v": []}
    for i, g in enumerate(grads):
        if case["op"] == "adamw":
            m, v = s["m"][i].double(), s["v"][i].double()
        else:
            m, v = _values64(s["mq"][i], s["scales"][i][:, 0]), _values64(s["rq"][i], s["scales"][i][:, 1]) ** 2
        m = BETAS[0] * m + (1 - BETAS[0]) * g
        v = BETAS[1] * v + (1 - BETAS[1]) * g * g
        mhat, vhat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
        w = (s["w"][i] if "w" in s else s["p"][i]).double()
        out["p"].append(w - s["lr"][i] * (mhat / (vhat.sqrt() + case["eps"]) + case["decay"] * w))
        if case["op"] == "adamw8":
            m, v = _rounded64(m, t, GOLDEN, R2_X, False), _rounded64(v.sqrt(), t, ROOT2, R2_Y, True) ** 2
        out["m"].append(m)
        out["v"].append(v)
    if case["op"] == "adamw":
        out["m"], out["v"] = _as_laid_out(s, "m", out["m"]), _as_laid_out(s, "v", out["v"])
    if "w" in s:
        out["w"] = _as_laid_out(s, "w", out["p"])
    out["p"] = _as_laid_out(s, "p", out["p"])
    return out


def _as_laid_out(s, key, values):
    if key not in s["flat"]:
        return values
    flat, at = torch.zeros_like(s["flat"][key], dtype=torch.float64), 0
    for v in values:
        flat[at:at + v.numel()] = v
        at += -(-v.numel() // 64) * 64
    return flat


def _values64(codes, e):
    return codes.double() * torch.exp2(e.double() - 127).repeat_interleave(BLOCK)[:codes.numel()]


def _rounded64(x, step, phase, turn, keep):
    """Every value moved to the code below or above it, by the element's threshold."""
    n = x.numel()
    top = torch.cat((x, x.new_zeros(-n % BLOCK))).view(-1, BLOCK).abs().amax(1)
    power = torch.ceil(torch.log2(top / 448.0)).clamp(min=-126)
    low, high = top <= 448.0 * torch.exp2(power - 1), top > 448.0 * torch.exp2(power)
    power = (power + high.double() - low.double()).clamp(min=-126)
    unit = torch.exp2(power).repeat_interleave(BLOCK)[:n]
    a = x.abs() / unit
    grain = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    grain = torch.where(a / grain >= 16, grain * 2, torch.where((a / grain < 8) & (grain > 2.0 ** -9), grain / 2, grain))
    i = torch.arange(n, device=x.device)
    share = torch.floor(((i * phase + step * turn) % 2 ** 32).double() / 4096) / 2 ** 20
    near = torch.floor(a / grain + share) * grain
    if keep:
        near = torch.where(x > 0, near.clamp(min=2.0 ** -9), near)
    return torch.sign(x) * near * unit

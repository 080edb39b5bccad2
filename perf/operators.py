"""Timed cases of two operators of the training path, each beside its plain form in elementary torch operations:

* AdamW over many tensors at once, moments held in 32 bits or in 8 (``nsr.optim.AdamW``), with or without clipping by the
  norm of all gradients;
* layer norm over the last axis, forward and backward with the reduction of the weight's and the bias' gradients
  (``nsr_hip.ops.layer_norm`` / ``layer_norm_forward`` / ``layer_norm_backward``).

``own = False``: ``run`` computes the plain form.  ``own = True``: ``run`` calls the framework.

The 8-bit moments, as both forms hold them: blocks of 256 consecutive elements with one fp32 scale per block and moment; the
first moment m and the root r = sqrt(v) of the second as e4m3 codes (3 mantissa bits, largest value 448), scale = largest
magnitude of the block / 448.  Codes are rounded stochastically: the lattice point below the value is raised by one when the
fraction between the two plus u reaches 1, with u of 16 random bits from a hash of (seed, step, element).  A root above zero
is never rounded to zero, so a first moment is never divided by nothing but eps.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 256              # elements under one scale; tensors start at multiples of it in the flat state
TOP = 448.0              # largest e4m3 value
LEAST = 2.0 ** -100      # a block's largest magnitude counts as at least this much
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "instant-nsr-pl_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from nsr import optim
    from nsr_hip import ops
    return optim, ops


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _ln(name, direction, rows, width, dtype, affine):
    return {"name": name, "op": "layer_norm", "direction": direction, "rows": rows, "width": width, "dtype": dtype,
            "affine": affine}


def _adamw(name, sizes, dtype, bits, clip, beta2=0.99):
    return {"name": name, "op": "adamw", "sizes": sizes, "dtype": dtype, "bits": bits, "clip": clip, "beta2": beta2}


def _text(sizes):
    return ",".join(str(n) for n in sizes)


def listed():
    # the fp32 heads of a NeuS model: two-layer SDF head, colour head, a variance scalar, with their biases
    heads = [64 * 35, 64, 64, 64 * 13, 13, 13, 64 * 32, 64, 64 * 64, 64, 64 * 3, 3, 1, 32 * 64, 64, 64 * 8, 8, 35, 1]
    # layers of a wider fp32 network (width 257 and the like), weights and biases in turn
    layers = [n for k in range(24) for n in ((131 + 37 * k) * (97 + 11 * k), 131 + 37 * k)]
    return [
        # one query point through one normalised layer of the default width: latency only
        _ln("ln forward, one row", "forward", 1, 64, "fp32", "fp32"),
        # an export chunk of 2097152 points through a layer of 64 neurons
        _ln("ln forward, export chunk", "forward", 2097152, 64, "fp16", "fp16"),
        # a training step's samples (256 rays x 1024) through a layer of 64 neurons
        _ln("ln backward, samples x 64", "backward", 262144, 64, "fp32", "fp32"),
        # a wider network under mixed precision: bf16 activations, fp32 weights
        _ln("ln backward, samples x 256", "backward", 131072, 256, "bf16", "fp32"),
        # rows and width that no vector length divides, both directions
        _ln("ln train, odd sizes", "train", 4099, 777, "fp32", "fp32"),
        # few wide rows: the weight's gradient is as much work as the rows
        _ln("ln train, wide rows", "train", 8192, 4096, "bf16", "bf16"),
        # the small fp32 tensors of a NeuS model, 32-bit moments: latency only
        _adamw("adamw, small heads", _text(heads), "fp32", 32, 0.0),
        # the NeRF model: hash table + density network in one vector, colour network in another
        _adamw("adamw, nerf model", _text([12602992, 7168]), "fp32", 32, 0.0),
        # the same parameters with moments in 8 bits
        _adamw("adamw 8 bit, nerf model", _text([12602992, 7168]), "fp32", 8, 0.0),
        # a NeuS model with its background field: two tables and the heads, clipped by the global norm
        _adamw("adamw 8 bit, neus + background", _text([13949952, 13975553] + heads[:6]), "fp32", 8, 1.0, 0.999),
        # a deeper network in bf16, 48 tensors of odd sizes, clipped
        _adamw("adamw, 48 layers, clipped", _text(layers), "bf16", 32, 1.0, 0.999),
        # a scene table of 2^26 entries with two features: the largest update of one GPU's memory budget for moments
        _adamw("adamw 8 bit, large table", _text([1 << 27]), "fp32", 8, 0.0),
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if rng.random() < 0.5:
        width = spread(8, 16384)  # (two or three values have next to no gradient through their own norm)
        rows = spread(1, min(2097152, max(1, (1 << 25) // width)))
        return {"op": "layer_norm", "direction": rng.choice(["forward", "backward", "train"]), "rows": rows, "width": width,
                "dtype": dtype, "affine": rng.choice([dtype, "fp32"])}
    total, count = spread(1000, 1 << 26), rng.randint(1, 24)
    cuts = sorted(rng.randint(1, total) for _ in range(count - 1))
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [total]) if b > a]
    return {"op": "adamw", "sizes": _text(sizes), "dtype": dtype, "bits": rng.choice([8, 32]), "clip": rng.choice([0.0, 1.0]),
            "beta2": rng.choice([0.99, 0.999])}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _places(sizes):
    """[(start, length)] of tensors laid one behind the other at multiples of BLOCK, and the length of the whole"""
    at, found = 0, []
    for n in sizes:
        found.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return found, at


def _prepare_ln(case, gen):
    rows, width = case["rows"], case["width"]
    dt, wt = DTYPES[case["dtype"]], DTYPES[case["affine"]]
    new = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    s = {"op": "layer_norm", "direction": case["direction"], "eps": 1e-5}
    # activations with a mean of their own per row, weights around one
    s["x"] = (new(rows, width) * 1.5 + 0.5 * new(rows, 1)).to(dt)
    s["weight"], s["bias"] = (1.0 + 0.2 * new(width)).to(wt), (0.1 * new(width)).to(wt)
    if case["direction"] != "forward":
        s["dy"] = new(rows, width).to(dt)
    if case["direction"] == "backward":  # what the forward pass left
        _, s["mean"], s["rstd"] = _plain_ln_forward(s["x"], s["weight"], s["bias"], s["eps"])
    return s


def _prepare_adamw(case, gen):
    sizes = [int(n) for n in case["sizes"].split(",")]
    places, total = _places(sizes)
    dt = DTYPES[case["dtype"]]
    new = lambda: torch.randn(total, generator=gen, device="cuda")  # noqa: E731
    live = torch.zeros(total, device="cuda")
    for at, n in places:
        live[at:at + n] = 1.0
    # gradients over several orders of magnitude, as table entries have them: a factor per run of 64 elements, and entries
    # that no sample touched
    scale = 10.0 ** (-4.0 + 3.0 * torch.rand(-(-total // 64), generator=gen, device="cuda")).repeat_interleave(64)[:total]
    touched = (torch.rand(total, generator=gen, device="cuda") < 0.75).float() * live
    s = {"op": "adamw", "bits": case["bits"], "clip": case["clip"], "t": 1000, "seed": 7, "lr": 0.001, "wd": 0.01,
         "beta1": 0.9, "beta2": case["beta2"], "eps": 1e-15}
    s["params"] = (0.1 * new() * live).to(dt)
    s["grads"] = (new() * scale * touched).to(dt)
    m, r = 0.3 * new() * scale * live, (0.5 + new().abs()) * scale * live
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = m, r * r
    else:
        sm, sr = (x.abs().view(-1, BLOCK).amax(1).clamp_min(LEAST) * (1.0 / TOP) for x in (m, r))
        s["exp_avg"] = (m.view(-1, BLOCK) / sm[:, None]).clamp(-TOP, TOP).view(-1).to(torch.float8_e4m3fn)
        # (codes of roots are at least the smallest one where the root is above zero)
        s["exp_avg_rms"] = ((r.view(-1, BLOCK) / sr[:, None]).clamp(2.0 ** -9, TOP).view(-1) * live).to(torch.float8_e4m3fn)
        s["scales"] = torch.stack([sm, sr])
    if own:
        optim, _ = _framework()
        ps = [torch.nn.Parameter(s["params"][at:at + n]) for at, n in places]
        for p, (at, n) in zip(ps, places):
            p.grad = s["grads"][at:at + n]
        opt = optim.AdamW(ps, lr=s["lr"], betas=(s["beta1"], s["beta2"]), eps=s["eps"], weight_decay=s["wd"],
                          state_bits=s["bits"], min_8bit_size=0, max_grad_norm=s["clip"] or None, rounding_seed=s["seed"])
        opt.set_step(s["t"])
        for key, held in (opt.flat32 if s["bits"] == 32 else opt.flat8).items():
            held.copy_(s[key])
        s["opt"] = opt
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return _prepare_ln(case, gen) if case["op"] == "layer_norm" else _prepare_adamw(case, gen)


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _plain_ln_forward(x, weight, bias, eps):
    xf = x.float()
    n = x.shape[1]
    mean = xf.sum(1, keepdim=True) / n
    c = xf - mean
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / n + eps)
    return (c * rstd * weight.float() + bias.float()).to(x.dtype), mean.view(-1), rstd.view(-1)


def _plain_ln_backward(dy, x, weight, mean, rstd):
    n = x.shape[1]
    rstd = rstd[:, None]
    h = (x.float() - mean[:, None]) * rstd
    d = dy.float()
    g = d * weight.float()
    dx = rstd * (g - g.sum(1, keepdim=True) / n - h * ((g * h).sum(1, keepdim=True) / n))
    return dx.to(x.dtype), (d * h).sum(0).to(weight.dtype), d.sum(0).to(weight.dtype)


def _mix(x):
    """32-bit finaliser (two multiplications and three shifts): int64 tensors that hold 32-bit values"""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(seed, t, total, device):
    """32 random bits for each element of a step"""
    e = torch.arange(total, dtype=torch.int64, device=device)
    key = _mix(_mix(torch.tensor(t, dtype=torch.int64, device=device)) ^ seed)
    return _mix((e & 0xFFFFFFFF) ^ ((key + (e >> 32) * 0x9E3779B9) & 0xFFFFFFFF))


def _plain_codes(x, bits16, least):
    """x[blocks, BLOCK] -> (e4m3 codes, scales): the value scaled by 2^-120 has the bits of the e4m3 lattice in front of 20
    more, to which the random ones are added"""
    top = x.abs().amax(1).clamp_min(LEAST)
    y = x.abs() * (torch.full_like(top, TOP) / top)[:, None]
    code = ((y * 2.0 ** -120).view(torch.int32) + (bits16.view_as(x) * 16 + 8).to(torch.int32)) >> 20
    code = torch.where(x != 0, code.clamp(least, 0x7E), torch.zeros_like(code))
    code = torch.where(x < 0, code + 0x80, code)
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn), top * (1.0 / TOP)


def _plain_adamw(s):
    s["t"] += 1
    t, b1, b2 = s["t"], s["beta1"], s["beta2"]
    out = {"params": s["params"]}
    g = s["grads"].float()
    if s["clip"]:
        norm = torch.sqrt((g.double() * g.double()).sum())
        out["norm"] = norm.float()
        g = g * torch.clamp(s["clip"] / (norm + 1e-6), max=1.0).float()
    if s["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = s["exp_avg"].float().view(-1, BLOCK) * s["scales"][0][:, None]
        r = s["exp_avg_rms"].float().view(-1, BLOCK) * s["scales"][1][:, None]
        g, v = g.view(-1, BLOCK), r * r
    m = b1 * m + (1.0 - b1) * g
    v = b2 * v + (1.0 - b2) * (g * g)
    r = torch.sqrt(v)
    step, root = s["lr"] / (1.0 - b1 ** t), 1.0 / math.sqrt(1.0 - b2 ** t)
    p = s["params"].float() * (1.0 - s["lr"] * s["wd"]) - step * (m / (r * root + s["eps"])).view(-1)
    s["params"].copy_(p)
    if s["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return {**out, "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}
    h = _random_bits(s["seed"], t, p.numel(), p.device)
    s["exp_avg"], sm = _plain_codes(m, h >> 16, 0)
    s["exp_avg_rms"], sr = _plain_codes(r, h & 0xFFFF, 1)
    s["scales"] = torch.stack([sm, sr])
    return {**out, "exp_avg": s["exp_avg"], "exp_avg_rms": s["exp_avg_rms"], "scales": s["scales"]}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    _, ops = _framework()
    if s["op"] == "adamw":
        opt = s["opt"]
        opt.step()
        out = {"params": s["params"], **(opt.flat32 if s["bits"] == 32 else opt.flat8)}
        return {**out, "norm": opt.grad_norm} if s["clip"] else out
    if s["direction"] == "forward":
        return {"y": ops.layer_norm(s["x"], s["weight"], s["bias"], s["eps"])}
    out = {}
    if s["direction"] == "train":
        out["y"], mean, rstd = ops.layer_norm_forward(s["x"], s["weight"], s["bias"], s["eps"])
    else:
        mean, rstd = s["mean"], s["rstd"]
    out["dx"], out["dweight"], out["dbias"] = ops.layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd)
    return out


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "adamw":
        return _plain_adamw(s)
    if s["direction"] == "forward":
        return {"y": _plain_ln_forward(s["x"], s["weight"], s["bias"], s["eps"])[0]}
    out = {}
    if s["direction"] == "train":
        out["y"], mean, rstd = _plain_ln_forward(s["x"], s["weight"], s["bias"], s["eps"])
    else:
        mean, rstd = s["mean"], s["rstd"]
    out["dx"], out["dweight"], out["dbias"] = _plain_ln_backward(s["dy"], s["x"], s["weight"], mean, rstd)
    return out


def work(case):
    size = lambda name: 4 if name == "fp32" else 2  # noqa: E731
    if case["op"] == "adamw":
        n = sum(int(k) for k in case["sizes"].split(","))
        # parameters read and written, gradients read, both moments read and written (and their scales)
        moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * n / BLOCK
        return {"bytes": 3 * size(case["dtype"]) * n + moments, "flops": 14 * n + (2 * n if case["clip"] else 0)}
    n, w = case["rows"] * case["width"], case["width"]
    e, a = size(case["dtype"]), size(case["affine"])
    forward = {"bytes": 2 * e * n + 2 * a * w, "flops": 8 * n}
    backward = {"bytes": 3 * e * n + 8 * case["rows"] + 3 * a * w, "flops": 14 * n}
    if case["direction"] == "forward":
        return forward
    if case["direction"] == "backward":
        return backward
    # x is read once for both passes, the rows' statistics are no input
    return {"bytes": 4 * e * n + 4 * a * w, "flops": forward["flops"] + backward["flops"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_ln(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    out = {}
    if s["direction"] == "backward":
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
    else:
        mean = x.mean(1, keepdim=True)
        rstd = ((x - mean).square().mean(1, keepdim=True) + s["eps"]).rsqrt()
        out["y"] = (x - mean) * rstd * w + b
    if s["direction"] != "forward":
        # the gradient of sum(dy * y) with mean and rstd as functions of x, from the two projections that they take out
        dy = s["dy"].double()
        xhat = (x - mean) * rstd
        along = dy * w
        out["dx"] = rstd * (along - along.mean(1, keepdim=True) - xhat * (along * xhat).mean(1, keepdim=True))
        out["dweight"], out["dbias"] = (dy * xhat).sum(0), dy.sum(0)
    return out


def _exact_round(x, u, keep):
    """nearest lattice points of e4m3 below and above x >= 0 (x <= 448), the upper one where fraction + u reaches 1"""
    _, e = torch.frexp(x)  # x = f 2^e with f in [1/2, 1)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3.0)
    q = (torch.floor(x / step + u) * step).clamp_max(TOP)
    return torch.where(x > 0, q.clamp_min(keep), torch.zeros_like(q))


def _exact_adamw(s):
    t, b1, b2 = s["t"] + 1, s["beta1"], s["beta2"]
    p, g = s["params"].double(), s["grads"].double()
    out = {}
    if s["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, s["clip"] / (float(out["norm"]) + 1e-6))
    if s["bits"] == 32:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    else:
        per = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        m, v = s["exp_avg"].double() * per[0], (s["exp_avg_rms"].double() * per[1]).square()
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + g.square() * (1.0 - b2)
    mhat, vhat = m / (1.0 - b1 ** t), v / (1.0 - b2 ** t)
    out["params"] = p - s["lr"] * s["wd"] * p - s["lr"] * mhat / (vhat.sqrt() + s["eps"])
    if s["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    h = _random_bits(s["seed"], t, p.numel(), p.device)  # the definition's own random numbers
    scales = []
    for key, x, bits, keep in (("exp_avg", m, h >> 16, 0.0), ("exp_avg_rms", v.sqrt(), h & 0xFFFF, 2.0 ** -9)):
        scale = x.abs().view(-1, BLOCK).amax(1).clamp_min(LEAST) / TOP
        y = (x.abs().view(-1, BLOCK) / scale[:, None]).view(-1).clamp_max(TOP)
        out[key] = _exact_round(y, (bits.double() + 0.5) / 65536.0, keep) * x.sign()
        scales.append(scale)
    return {**out, "scales": torch.stack(scales)}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_ln(s) if s["op"] == "layer_norm" else _exact_adamw(s)

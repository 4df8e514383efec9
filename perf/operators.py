"""Cases for the matrix optimizer's operators: orthogonalisation by Newton-Schulz products, the Muon step, the AdamW step.

`run` computes each operator either in its plain form (elementary torch operations) or, with `own` set, through segmi.optim as a
training program calls it; `exact` is the definition once more in 64 bits.  Shapes are the filters of this repository's networks
(a filter [K, C, R, S] is the K x C*R*S matrix of its memory order) or generic odd ones.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # quintic a s + b s^3 + c s^5: every singular value in (0, 1] goes to about 1
EPS = 1e-7

# filters x count, then everything that is no matrix (norm scales and offsets, classifier biases, depthwise filters)
UNET = ("32x3x3x3 64x32x3x3*2 64x64x3x3 128x64x3x3*2 128x128x3x3 256x128x3x3*2 256x256x3x3 512x256x3x3*2 512x512x3x3 "
        "1024x512x3x3*2 512x1024x3x3 1024x512x2x2 256x1024x3x3 512x256x2x2 128x512x3x3 256x128x2x2 64x256x3x3 128x64x2x2 32x128x3x3 2x64x1x1")
UNET_REST = "32*4 64*9 128*9 256*9 512*9 1024*4 2*1"
PSPNET = ("64x3x3x3 64x64x3x3*4 128x64x3x3 64x128x1x1 256x64x1x1*3 256x128x1x1 64x256x1x1*2 128x256x1x1 128x128x3x3*4 512x128x1x1*4 "
          "512x256x1x1 128x512x1x1*3 256x512x1x1 256x256x3x3*6 1024x256x1x1*6 1024x512x1x1 256x1024x1x1*5 512x1024x1x1 512x512x3x3*3 "
          "2048x512x1x1*3 2048x1024x1x1 512x2048x1x1*6 512x4096x3x3 21x512x1x1*2 512x1024x3x3")
PSPNET_REST = "64*16 128*18 256*32 512*34 1024*14 2048*8 21*2"


def listed():
    return [
        # --- orthogonalisation alone: what a program of its own (a shampoo-like or spectral step) asks of a filter's update
        {"name": "ortho_one_stem_filter", "op": "ortho", "shapes": "64x576", "dtype": "float32"},          # latency: one 64-channel 3x3 filter
        {"name": "ortho_ragged", "op": "ortho", "shapes": "21x512 150x257 1x129 333x65 19x2304 7x7 64x27", "dtype": "float32"},   # classifiers, stems, odd sizes
        {"name": "ortho_stage3", "op": "ortho", "shapes": "256x1024*5 256x2304*6 1024x256*6", "dtype": "float32"},  # a residual stage's wide and tall filters
        {"name": "ortho_unet_middle", "op": "ortho", "shapes": "1024x4608", "dtype": "float32"},           # the widest 3x3 filter of the encoder
        {"name": "ortho_bf16_stage4", "op": "ortho", "shapes": "512x2048*3 512x4608*3 2048x512*3", "dtype": "bfloat16"},  # updates held in 16 bits
        {"name": "ortho_pyramid", "op": "ortho", "shapes": "512x36864", "dtype": "float32"},               # the pyramid bottleneck: 72 times as wide as high
        # --- the whole Muon step: momentum, orthogonalisation, decay and update, AdamW for what is no matrix
        {"name": "muon_head", "op": "muon", "filters": "64x64x3x3 21x64x1x1", "rest": "64*2 21", "nesterov": True},   # latency: fine-tuning a small head
        {"name": "muon_unet", "op": "muon", "filters": UNET, "rest": UNET_REST, "nesterov": True},
        {"name": "muon_pspnet", "op": "muon", "filters": PSPNET, "rest": PSPNET_REST, "nesterov": False},
        # --- AdamW
        {"name": "adamw_norms", "op": "adamw", "rest": "64*16 128*18 256*32"},                              # latency: norm layers only
        {"name": "adamw_odd", "op": "adamw", "rest": "1 3 150 4097 65537 1000003 728x1x3x3*4 64x27"},       # ragged sizes, tap-major depthwise filters
        {"name": "adamw_pspnet", "op": "adamw", "rest": PSPNET + " " + PSPNET_REST},                        # every parameter of a network
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ortho", "muon", "adamw"])
    if op == "adamw":
        return {"op": op, "rest": " ".join(str(_log(rng, 1, 4e6)) for _ in range(_log(rng, 1, 120)))}
    mats, cost = [], 0.0
    for _ in range(_log(rng, 1, 24)):
        k, c, taps = _log(rng, 2, 1536), _log(rng, 2, 1536), rng.choice([1, 1, 3])
        m, n = sorted((k, c * taps * taps))
        cost += float(m) * m * n
        if cost > 3e10 and mats:
            break
        mats.append((k, c, taps))
    if op == "ortho":
        return {"op": op, "shapes": " ".join("%dx%d" % (k, c * t * t) for k, c, t in mats), "dtype": rng.choice(["float32", "bfloat16"])}
    return {"op": op, "filters": " ".join("%dx%dx%dx%d" % (k, c, t, t) for k, c, t in mats),
            "rest": " ".join(str(_log(rng, 1, 4096)) for _ in range(_log(rng, 1, 100))), "nesterov": rng.random() < 0.5}


def _shapes(text):
    out = []
    for word in text.split():
        dims, _, times = word.partition("*")
        out += [tuple(int(d) for d in dims.split("x"))] * (int(times) if times else 1)
    return out


def _arena(shapes, dtype=torch.float32):
    """One flat buffer and a view of it per shape, as gradient buckets hold them: 16-byte slots, filters in the memory order this
    repository keeps them in (channels-last, depthwise ones tap-major)."""
    sizes = [(math.prod(s) + 3) & ~3 for s in shapes]
    flat = torch.zeros(sum(sizes), dtype=dtype, device=DEVICE)
    views, at = [], 0
    for s, size in zip(shapes, sizes):
        slot = flat[at:at + math.prod(s)]
        if len(s) == 4 and s[1] == 1:
            slot = slot.view(s[1], s[2], s[3], s[0]).permute(3, 0, 1, 2)
        elif len(s) == 4:
            slot = slot.view(s[0], s[2], s[3], s[1]).permute(0, 3, 1, 2)
        views.append(slot.view(s) if len(s) != 4 else slot)
        at += size
    return flat, views


def _update(shape, gen):
    """A gradient as training sees it: a few strong directions whose strength falls off, under sampling noise, at a layer's own scale."""
    m = shape[0]
    n = int(math.prod(shape[1:]))
    scale = 10.0 ** (-4.0 + 2.5 * torch.rand((), generator=gen, device=DEVICE))
    noise = torch.randn(m, n, generator=gen, device=DEVICE)
    if n > 1 and m > 1:
        r = min(16, m, n)
        fall = 1.0 / (1.0 + torch.arange(r, device=DEVICE, dtype=torch.float32))
        noise = noise + (3.0 * torch.randn(m, r, generator=gen, device=DEVICE) * fall) @ torch.randn(r, n, generator=gen, device=DEVICE)
    return (noise * scale).reshape(shape)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(1 + 7919 * seed)
    if case["op"] == "ortho":
        dt = getattr(torch, case["dtype"])
        return {"op": "ortho", "mats": [_update(s, gen).to(dt) for s in _shapes(case["shapes"])]}
    filters, rest = _shapes(case.get("filters", "")), _shapes(case["rest"])
    st = {"op": case["op"], "nesterov": bool(case.get("nesterov")), "t": 7, "lr": 2e-3, "decay": 0.05, "mu": 0.95, "betas": (0.9, 0.999), "eps": 1e-8}
    flats, views = zip(_arena(filters + rest), _arena(filters + rest), _arena(filters), _arena(rest), _arena(rest))
    st["flats"] = dict(zip(("params", "grads", "momentum", "exp_avg", "exp_avg_sq"), flats))
    ps, gs, bs, ms, vs = views
    k = len(filters)
    st["filters"], st["rest"] = list(zip(ps[:k], gs[:k], bs)), list(zip(ps[k:], gs[k:], ms, vs))
    for p, g, b in st["filters"]:
        p.copy_(torch.randn(p.shape, generator=gen, device=DEVICE) * (2.0 / math.prod(p.shape[1:])) ** 0.5)
        g.copy_(_update(tuple(p.shape), gen))
        b.copy_(6.0 * g + 2.0 * g.square().mean().sqrt() * torch.randn(p.shape, generator=gen, device=DEVICE))    # a running sum of earlier gradients
    for p, g, m, v in st["rest"]:
        p.copy_(1.0 + 0.1 * torch.randn(p.shape, generator=gen, device=DEVICE))
        g.copy_(_update(tuple(p.shape) if p.dim() > 1 else (1, p.numel()), gen).reshape(p.shape))
        m.copy_(0.5 * g + 0.2 * g.abs().mean() * torch.randn(p.shape, generator=gen, device=DEVICE))
        v.copy_((g * g + (0.3 * g.abs().mean()) ** 2) * 0.01)
    if own:
        st["optimizer"] = _optimizer(st)
    return st


def _optimizer(st):
    """The optimizer as a program resumed at step `t` holds it."""
    _package()
    from segmi import optim
    params = []
    for p, g in [q[:2] for q in st["filters"] + st["rest"]]:
        p = torch.nn.Parameter(p)
        p.grad = g
        params.append(p)
    if st["op"] == "muon":
        opt = optim.Muon(params, lr=st["lr"], weight_decay=st["decay"], momentum=st["mu"], nesterov=st["nesterov"], ns_coefficients=COEFFICIENTS,
                         eps=EPS, ns_steps=5, adjust_lr_fn="match_rms_adamw", adamw_betas=st["betas"], adamw_eps=st["eps"])
    else:
        opt = optim.FusedAdamW(params, lr=st["lr"], betas=st["betas"], eps=st["eps"], weight_decay=st["decay"])
    k = len(st["filters"])
    for p, q in zip(params[:k], st["filters"]):
        opt.state[p]["momentum_buffer"] = q[2]
    for p, q in zip(params[k:], st["rest"]):
        opt.state[p].update(step=torch.tensor(float(st["t"])), exp_avg=q[2], exp_avg_sq=q[3])
    return opt


def _package():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pytorch-segmentation_amd")
    if here not in sys.path:
        sys.path.insert(1, here)


def _outputs(st):
    return {k: st["flats"][k] for k in ("params", "momentum", "exp_avg", "exp_avg_sq")}


def run(st):
    if st["op"] == "ortho":
        if own:
            _package()
            from segmi import optim
            return optim.orthogonalize(st["mats"], steps=5, coefficients=COEFFICIENTS, eps=EPS)
        return [_plain_orthogonal(m).to(m.dtype) for m in st["mats"]]
    if own:
        st["optimizer"].step()
        return _outputs(st)
    st["t"] += 1
    for p, g, b in st["filters"]:
        b.mul_(st["mu"]).add_(g)
        u = g + st["mu"] * b if st["nesterov"] else b
        o = _plain_orthogonal(u.reshape(u.shape[0], -1)).reshape(u.shape)
        rows, cols = u.shape[0], u[0].numel()
        p.mul_(1.0 - st["lr"] * st["decay"]).sub_(st["lr"] * 0.2 * math.sqrt(max(rows, cols)) * o)
    b1, b2 = st["betas"]
    c1, c2 = 1.0 - b1 ** st["t"], math.sqrt(1.0 - b2 ** st["t"])
    for p, g, m, v in st["rest"]:
        m.mul_(b1).add_(g * (1.0 - b1))
        v.mul_(b2).add_(g * g * (1.0 - b2))
        p.mul_(1.0 - st["lr"] * st["decay"]).sub_((st["lr"] / c1) * m / (v.sqrt() / c2 + st["eps"]))
    return _outputs(st)


def _plain_orthogonal(u):
    a, b, c = COEFFICIENTS
    x = u.float()
    x = x / x.double().square().sum().sqrt().clamp(min=EPS).float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


def work(case):
    """Bytes: every tensor read and written once.  Operations: of the five quintic steps, whichever way takes fewer — on the matrix
    itself (a Gram product, its square, one product with the matrix a step) or on its Gram matrix (one Gram product, one product with
    the matrix, the rest m x m); a product known to be symmetric counts one triangle."""
    byts = flops = 0.0
    shapes = _shapes(case["shapes"]) if case["op"] == "ortho" else _shapes(case.get("filters", ""))
    for s in shapes:
        k, n = s[0], int(math.prod(s[1:]))
        m, w = min(k, n), max(k, n)
        byts += k * n * (2 * (2 if case["op"] == "ortho" and case["dtype"] == "bfloat16" else 4) if case["op"] == "ortho" else 20)
        flops += min(5.0 * (3.0 * m * m * w + float(m) ** 3), 3.0 * m * m * w + 17.0 * float(m) ** 3) + (0 if case["op"] == "ortho" else 8.0 * k * n)
    for s in _shapes(case.get("rest", "")):
        byts += 28.0 * math.prod(s)
        flops += 14.0 * math.prod(s)
    return {"bytes": byts, "flops": flops}


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "ortho":
        return [_exact_orthogonal(m.to(f64)) for m in st["mats"]]
    lr, wd, mu, t = st["lr"], st["decay"], st["mu"], st["t"] + 1
    b1, b2 = st["betas"]
    filters, rest = _shapes(case.get("filters", "")), _shapes(case["rest"])
    k = len(filters)
    out, views = {}, {}
    for key, shapes in (("params", filters + rest), ("momentum", filters), ("exp_avg", rest), ("exp_avg_sq", rest)):
        out[key], views[key] = _arena(shapes, f64)
    for i, (p, g, b) in enumerate(st["filters"]):
        p, g, b = p.to(f64), g.to(f64), b.to(f64)
        b = b * mu + g
        u = b * mu + g if st["nesterov"] else b
        cols = u.numel() // u.shape[0]
        o = _exact_orthogonal(u.reshape(u.shape[0], cols)).reshape(u.shape)
        views["params"][i].copy_((1 - lr * wd) * p - lr * 0.2 * max(u.shape[0], cols) ** 0.5 * o)
        views["momentum"][i].copy_(b)
    for i, (p, g, m, v) in enumerate(st["rest"]):
        p, g, m, v = p.to(f64), g.to(f64), m.to(f64), v.to(f64)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + st["eps"])
        views["params"][k + i].copy_(p - lr * wd * p - lr * step)
        views["exp_avg"][i].copy_(m)
        views["exp_avg_sq"][i].copy_(v)
    return out


def _exact_orthogonal(u):
    """X <- X (a + b X'X + c (X'X)^2) on the shorter side, from u / max(|u|, eps)."""
    x = u / max(float(torch.linalg.vector_norm(u)), EPS)
    wide = x.shape[1] >= x.shape[0]
    a, b, c = COEFFICIENTS
    for _ in range(5):
        if wide:
            s = torch.mm(x, x.mT)
            x = torch.mm(torch.addmm(b * s, s, s, beta=1.0, alpha=c), x) + a * x
        else:
            s = torch.mm(x.mT, x)
            x = torch.mm(x, torch.addmm(b * s, s, s, beta=1.0, alpha=c)) + a * x
    return x

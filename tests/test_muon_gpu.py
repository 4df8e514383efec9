"""Matrix optimizer on the GPU against its formulas in 64 bits.

Tolerances.  u = 2^-22 bounds the rounding of a value held as an fp16 pair and the term its products leave out; it is also the size
of an fp32 sum's rounding at these lengths.  The iteration's map takes a relative perturbation of X_0 to at most a^5 = 485 times its size
(p'(0) = a a step, |p'| <= a everywhere on [0, 1.2]); per step four products round, so 20 independent roundings of relative
Frobenius size u give sqrt(20) 485 u = 5.2e-4 of |X| in Frobenius norm at the worst spectrum (WORST).  On a full-rank Gaussian matrix
almost every singular value is amplified far less; there the bound is the fp32 iteration's own distance from 64 bits:
at most 4 times it (u is 4 times fp32's 2^-24), or 16 u where that is smaller (SHARP).  That comparison is one of root mean squares: on
sides below 16 a handful of roundings make up either distance and the smallest singular value may be anything (2 x 2: s_min / s_max
is below 1/20 one time in ten), so a single one, amplified by up to a^5, decides, and WORST is the bound."""
import math

import pytest
import torch

from segmi import muon, optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -22
WORST = math.sqrt(20.0) * 3.4445 ** 5 * U
SHARP_FLOOR = 16 * U
E24 = 2.0 ** -24


def iterate(m, steps=5, coef=muon.NS_COEFFICIENTS, eps=1e-7, dtype=torch.float64):
    x = m.to(dtype)
    norm = m.double().square().sum().sqrt().clamp(min=eps)
    x = (x.double() / norm).to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(steps):
        g = x @ x.t().contiguous()
        x = coef[0] * x + (coef[1] * g + coef[2] * (g @ g)) @ x
    return x.t() if tall else x


def matrix(kind, r, c, gen, dev):
    z = torch.randn(r, c, generator=gen, device=dev)
    k = min(r, c)
    if kind == "gauss":
        return z * 3e-3
    if kind == "lowrank":
        q = max(1, k // 8)
        return torch.randn(r, q, generator=gen, device=dev) @ torch.randn(q, c, generator=gen, device=dev) + 1e-2 * z
    if kind == "heavy":
        return z * torch.exp(2.0 * torch.randn(r, c, generator=gen, device=dev))
    if kind == "decay":
        u = torch.linalg.qr(torch.randn(r, k, generator=gen, device=dev, dtype=torch.float64)).Q
        v = torch.linalg.qr(torch.randn(c, k, generator=gen, device=dev, dtype=torch.float64)).Q
        return ((u * torch.logspace(0, -4, k, device=dev, dtype=torch.float64)) @ v.t().contiguous()).float()
    raise ValueError(kind)


def gen_of(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def relative(a, b):
    return float((a.double() - b).norm() / b.norm())


SIZES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 5), (7, 7), (21, 512), (64, 64), (64, 576), (65, 64), (63, 129), (128, 128), (150, 257), (333, 65),
         (192, 1000), (129, 2304), (512, 64), (256, 1024), (320, 320), (1024, 256), (448, 512), (512, 4608)]


@pytest.mark.parametrize("r,c", SIZES, ids=lambda v: str(v))
def test_orthogonalize_gauss(cuda, r, c):
    m = matrix("gauss", r, c, gen_of(cuda, r * 10007 + c), cuda)
    before = m.clone()
    out = optim.orthogonalize(m)
    want = iterate(m)
    assert out.shape == m.shape and out.dtype == m.dtype and torch.equal(m, before)
    here, plain = relative(out, want), relative(iterate(m, dtype=torch.float32), want)
    print("%dx%d: distance %.2e, fp32 iteration %.2e" % (r, c, here, plain))
    assert here <= (max(4 * plain, SHARP_FLOOR) if min(r, c) >= 16 else WORST)


@pytest.mark.parametrize("kind", ["lowrank", "heavy", "decay"])
@pytest.mark.parametrize("r,c", [(64, 64), (96, 700), (500, 130), (512, 512)], ids=lambda v: str(v))
def test_orthogonalize_hard_spectra(cuda, kind, r, c):
    m = matrix(kind, r, c, gen_of(cuda, r + 31 * c), cuda)
    here = relative(optim.orthogonalize(m), iterate(m))
    print("%s %dx%d: distance %.2e" % (kind, r, c, here))
    assert here <= WORST


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
@pytest.mark.parametrize("coef", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5)], ids=str)
def test_orthogonalize_steps_and_coefficients(cuda, steps, coef):
    m = matrix("gauss", 70, 200, gen_of(cuda, steps), cuda)
    here = relative(optim.orthogonalize(m, steps=steps, coefficients=coef), iterate(m, steps, coef))
    # a perturbation grows by at most a a step; `4 steps` roundings
    assert here <= math.sqrt(4.0 * steps) * max(1.0, coef[0]) ** min(steps, 5) * U


def test_orthogonalize_many_sizes_share_their_launches(cuda):
    """More matrices than one launch's descriptors hold, wide and tall, sizes mixed."""
    gen = gen_of(cuda, 5)
    sizes = [(1 + (37 * i) % 190, 1 + (91 * i) % 333) for i in range(101)] + [(300, 900), (64, 64)]
    mats = [matrix("gauss", r, c, gen, cuda) for r, c in sizes]
    outs = optim.orthogonalize(mats)
    assert len(outs) == len(mats)
    for m, o in zip(mats, outs):
        want = iterate(m)
        bound = max(4 * relative(iterate(m, dtype=torch.float32), want), SHARP_FLOOR) if min(m.shape) >= 16 else WORST
        assert relative(o, want) <= bound, tuple(m.shape)
    again = optim.orthogonalize(mats)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))       # no atomics, fixed orders


def test_orthogonalize_bf16(cuda):
    for r, c in ((64, 576), (333, 65), (1, 9), (130, 130)):
        m = matrix("gauss", r, c, gen_of(cuda, r), cuda).bfloat16()
        out = optim.orthogonalize(m)
        want = iterate(m)
        assert out.dtype == torch.bfloat16
        # half a bf16 step (2^-8 relative) on top of the fp32-accurate value
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * want.abs().max()).all())


def test_orthogonalize_strides_and_dimensions(cuda):
    gen = gen_of(cuda, 11)
    base = matrix("gauss", 90, 300, gen, cuda)
    want = iterate(base)
    big = torch.zeros(200, 700, device=cuda)
    cases = {"transposed": base.t().contiguous().t(), "rows apart": torch.as_strided(big, (90, 300), (700, 1), 3), "columns apart": torch.as_strided(big, (90, 300), (700, 2), 5),
             "column-major apart": torch.as_strided(torch.zeros(300, 128, device=cuda), (90, 300), (1, 128), 1)}
    for name, v in cases.items():
        if v.data_ptr() != base.data_ptr() and not torch.equal(v, base):
            v.copy_(base)
        out = optim.orthogonalize(v)
        assert out.shape == v.shape and relative(out, want) <= 1e-5, name
    # a channels-last filter, a contiguous one, and one whose dimensions are not dense
    f = matrix("gauss", 40, 5 * 9, gen, cuda).view(40, 5, 3, 3)
    ref = iterate(f.reshape(40, 45)).reshape(40, 5, 3, 3)
    for v in (f, f.contiguous(memory_format=torch.channels_last), torch.cat([f, f], dim=3)[..., :3], f.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)):
        out = optim.orthogonalize(v)
        assert relative(out, ref) <= 1e-5
    # broadcast rows (stride 0): rank one
    v = torch.randn(1, 33, generator=gen, device=cuda).expand(20, 33)
    assert relative(optim.orthogonalize(v), iterate(v)) <= WORST
    # dense outputs only ever lie in memory of their own
    outs = optim.orthogonalize([base, base])
    assert torch.equal(outs[0], outs[1]) and outs[0].data_ptr() != outs[1].data_ptr()


def test_orthogonalize_empty_zero_and_extreme(cuda):
    e = optim.orthogonalize([torch.zeros(0, 5, device=cuda), torch.zeros(5, 0, device=cuda), torch.zeros(6, 70, device=cuda)])
    assert e[0].shape == (0, 5) and e[1].shape == (5, 0) and torch.equal(e[2], torch.zeros(6, 70, device=cuda))
    assert optim.orthogonalize(torch.zeros(0, 3, device=cuda)).shape == (0, 3)
    m = matrix("gauss", 48, 100, gen_of(cuda, 3), cuda)
    want = iterate(m)
    for scale in (2.0 ** -100, 2.0 ** 60, 2.0 ** 120):                # sums of squares beyond fp32's range
        got = optim.orthogonalize(m * scale, eps=1e-38)
        assert relative(got, want) <= 1e-5, scale
    tiny = m * (1e-9 / float(m.norm()))                               # below eps: divided by eps alone
    assert relative(optim.orthogonalize(tiny, eps=1e-7), iterate(tiny, eps=1e-7)) <= 1e-3


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_orthogonalize_not_finite_stays_in_its_matrix(cuda, bad):
    gen = gen_of(cuda, 17)
    mats = [matrix("gauss", 70, 90, gen, cuda) for _ in range(3)]
    alone = optim.orthogonalize(mats[0])
    mats[1][69, 3] = bad
    outs = optim.orthogonalize(mats)
    assert bool(torch.isnan(outs[1]).all())
    assert torch.equal(outs[0], alone) and bool(torch.isfinite(outs[2]).all())


def test_orthogonalize_on_another_stream_and_in_a_graph(cuda):
    mats = [matrix("gauss", 100, 300, gen_of(cuda, 1), cuda), matrix("gauss", 64, 64, gen_of(cuda, 2), cuda)]
    want = optim.orthogonalize(mats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = optim.orthogonalize(mats)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                   # two graphs of the same work: each has a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = optim.orthogonalize(mats)
        graphs.append((g, outs))
    for k in range(4):
        for m in mats:
            m.mul_(1.0 + 0.25 * k).add_(0.01 * k)
        eager = optim.orthogonalize(mats)
        torch.cuda.synchronize()
        for g, outs in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_result_is_orthogonal(cuda):
    """What the operator is for: singular values near 1 whatever they were."""
    for kind, r, c in (("gauss", 128, 512), ("decay", 100, 100)):
        s = torch.linalg.svdvals(optim.orthogonalize(matrix(kind, r, c, gen_of(cuda, 9), cuda), steps=10, coefficients=(2.0, -1.5, 0.5)).double())
        if kind == "gauss":
            assert float((s - 1).abs().max()) < 1e-3
        assert float(s.max()) < 1.01


# ------------------------------------------------------------------------------------------------ optimizers
def network(dev, seed=0):
    """One parameter of every kind: channels-last, contiguous and transposed filters, depthwise, single row, vectors, scalar."""
    gen = gen_of(dev, seed)
    r = lambda *s: torch.randn(s, generator=gen, device=dev)
    dw = r(3, 3, 24).permute(2, 0, 1).unsqueeze(1)
    raw = [r(64, 16, 3, 3).contiguous(memory_format=torch.channels_last), r(24, 40, 1, 1).contiguous(memory_format=torch.channels_last), r(48, 20, 2, 2), r(130, 33),
           r(20, 65).t(), dw, r(1, 31), r(77), r(1).squeeze(), r(21)]
    ps = [torch.nn.Parameter(t) for t in raw]
    assert ps[5].stride() == dw.stride()
    for p in ps:
        p.grad = torch.empty_like(p).copy_(torch.randn(p.shape, generator=gen, device=dev) * 1e-2)
    return ps


def adamw_reference(p, g, m, v, t, lr, wd, b1, b2, eps):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps), m, v


def close(got, want, scale, what):
    bad = (got.double() - want).abs() > scale
    assert not bool(bad.any()), (what, float(((got.double() - want).abs() / scale.clamp(min=1e-300)).max()))


def test_fused_adamw_matches_the_formula(cuda):
    ps = network(cuda)
    off = torch.zeros(1001, device=cuda)                       # a parameter that does not start on 16 bytes
    odd = torch.nn.Parameter(off[1:].copy_(torch.randn(1000, device=cuda)))
    odd.grad = torch.randn(1003, device=cuda)[3:]
    groups = [{"params": ps[:4]}, {"params": ps[4:] + [odd], "lr": 3e-3, "weight_decay": 0.2, "betas": (0.8, 0.95), "eps": 1e-6}]
    opt = optim.FusedAdamW(groups, lr=1e-2, weight_decay=0.01)
    ref = [[p.detach().double(), torch.zeros_like(p, dtype=torch.float64), torch.zeros_like(p, dtype=torch.float64)] for p in ps + [odd]]
    for t in range(1, 5):
        for p in ps + [odd]:
            p.grad.mul_(1.0 + 0.3 * t).add_(1e-3 * t)
        opt.step()
        for i, p in enumerate(ps + [odd]):
            g = opt.param_groups[0 if i < 4 else 1]
            old = ref[i][0]
            new = adamw_reference(*[ref[i][0], p.grad.double(), ref[i][1], ref[i][2]], t, g["lr"], g["weight_decay"], g["betas"][0], g["betas"][1], g["eps"])
            ref[i] = list(new)
            st = opt.state[p]
            assert float(st["step"]) == t
            # each step adds: m 3, v 4 roundings of size 2^-24; the update (m/., sqrt, the corrections) 8 of its own size, p 2 of p's
            close(st["exp_avg"], ref[i][1], 4 * t * E24 * (ref[i][1].abs() + p.grad.double().abs()) + 1e-30, ("m", i))
            close(st["exp_avg_sq"], ref[i][2], 5 * t * E24 * ref[i][2] + 1e-30, ("v", i))
            close(p, ref[i][0], t * E24 * (3 * old.abs() + 16 * g["lr"] * 10) , ("p", i))


def test_fused_adamw_state_interchanges_with_torch(cuda):
    pa, pb = network(cuda, 3), network(cuda, 3)
    a, b = optim.FusedAdamW(pa, lr=1e-2), torch.optim.AdamW(pb, lr=1e-2)
    for o in (a, b):
        o.step()
    pc = network(cuda, 3)
    for p, q in zip(pc, pb):
        p.data.copy_(q)
    c = optim.FusedAdamW(pc, lr=1e-2)
    c.load_state_dict(b.state_dict())
    d = torch.optim.AdamW(pa, lr=1e-2)
    d.load_state_dict(a.state_dict())
    for o in (b, c, d):
        o.step()
    for x, y, z in zip(pa, pb, pc):
        assert torch.allclose(x, y, rtol=2e-6, atol=2e-7) and torch.allclose(z, y, rtol=2e-6, atol=2e-7)
    assert float(c.state[pc[0]]["step"]) == 2.0


def muon_reference(ps, opt, state, t):
    """One Muon step in 64 bits on copies; returns the new parameters and how large each update was."""
    out = []
    for i, p in enumerate(ps):
        g = next(q for q in opt.param_groups if any(p is x for x in q["params"]))
        old, grad = state[i]["p"], p.grad.double()
        if muon._matrix_of(p) is not None and g.get("algorithm", "auto") == "auto":
            buf = g["momentum"] * state[i].get("b", torch.zeros_like(old)) + grad
            u = grad + g["momentum"] * buf if g["nesterov"] else buf
            k, rest = u.shape[0], u.numel() // u.shape[0]
            f = 0.2 * math.sqrt(max(k, rest)) if g["adjust_lr_fn"] == "match_rms_adamw" else math.sqrt(max(1.0, k / rest))
            o = iterate(u.reshape(k, rest), g["ns_steps"], g["ns_coefficients"], g["eps"]).reshape(u.shape)
            state[i]["b"], state[i]["p"] = buf, old * (1 - g["lr"] * g["weight_decay"]) - g["lr"] * f * o
            # the update's rounding: WORST relative to its own size, plus the momentum buffer's (inside it)
            out.append(("muon", g["lr"] * f * (1e-5 * o.abs().max() + 0 * o)))
        else:
            m, v = state[i].get("m", torch.zeros_like(old)), state[i].get("v", torch.zeros_like(old))
            lr = g["lr"] * g["adamw_lr_ratio"]
            state[i]["p"], state[i]["m"], state[i]["v"] = adamw_reference(old, grad, m, v, t, lr, g["weight_decay"], *g["adamw_betas"], g["adamw_eps"])
            out.append(("adamw", 16 * lr * 10 * E24 * torch.ones_like(old)))
    return out


@pytest.mark.parametrize("nesterov,adjust", [(True, "match_rms_adamw"), (False, None), (True, "original")])
def test_muon_steps_match_the_formula(cuda, nesterov, adjust):
    ps = network(cuda, 7)
    groups = [{"params": ps[:3] + ps[5:8]}, {"params": ps[3:5] + ps[8:9], "lr": 5e-3, "weight_decay": 0.0, "momentum": 0.8},
              {"params": [torch.nn.Parameter(torch.randn(30, 50, device=cuda))] + ps[9:], "algorithm": "adamw", "adamw_lr_ratio": 0.3}]
    plain = groups[2]["params"][0]
    plain.grad = torch.randn(30, 50, device=cuda)
    opt = optim.Muon(groups, lr=2e-2, weight_decay=0.1, nesterov=nesterov, adjust_lr_fn=adjust)
    every = ps[:9] + groups[2]["params"]
    state = [{"p": p.detach().double().clone()} for p in every]
    for t in range(1, 4):
        for p in every:
            p.grad.mul_(0.5).add_(torch.randn_like(p) * 1e-2)
        old = [s["p"] for s in state]
        opt.step()
        slack = muon_reference(every, opt, state, t)
        for i, p in enumerate(every):
            kind, s = slack[i]
            close(p, state[i]["p"], t * (4 * E24 * old[i].abs() + s) + 1e-12, (kind, i, t))
            keys = set(opt.state[p])
            assert keys == ({"momentum_buffer"} if kind == "muon" else {"step", "exp_avg", "exp_avg_sq"})
            if kind == "muon":
                close(opt.state[p]["momentum_buffer"], state[i]["b"], 4 * t * E24 * (state[i]["b"].abs() + 0.1), ("buffer", i))
                assert muon._same_layout(opt.state[p]["momentum_buffer"], p)


def test_muon_resumes_bit_identically(cuda, tmp_path):
    """state_dict -> file -> a new optimizer (state arrives in another memory order) -> the same steps."""
    ps, qs = network(cuda, 1), network(cuda, 1)
    a = optim.Muon(ps, lr=1e-2)
    a.step()
    sd = a.state_dict()
    for k, st in sd["state"].items():
        for key, v in st.items():
            if key != "step":
                st[key] = v.contiguous()                # what a checkpoint written elsewhere holds
    torch.save(sd, tmp_path / "o.pt")
    b = optim.Muon(qs, lr=1e-2)
    for p, q in zip(ps, qs):
        q.data.copy_(p)
        q.grad.copy_(p.grad)
    b.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    for _ in range(2):
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)


def test_muon_moving_gradients_missing_gradients_and_closures(cuda):
    ps, qs = network(cuda, 2), network(cuda, 2)
    a, b = optim.Muon(ps, lr=1e-2), optim.Muon(qs, lr=1e-2)
    held = []
    for k in range(4):
        held.append([p.grad for p in ps])
        for i, (p, q) in enumerate(zip(ps, qs)):
            g = torch.randn_like(p)
            q.grad = torch.empty_like(q)
            q.grad.copy_(g)
            if k == 2 and i in (0, 7):
                p.grad = q.grad = None                   # no gradient: the parameter and its state stay as they are
                continue
            p.grad = torch.empty_like(p).copy_(g)        # another tensor every step
        frozen = [(ps[i].detach().clone(), {k2: torch.as_tensor(v).clone() for k2, v in a.state[ps[i]].items()}) for i in (0, 7)]
        assert a.step(lambda: torch.tensor(3.0)) == 3.0
        b.step()
        if k == 2:
            for i, (p0, st) in zip((0, 7), frozen):
                assert torch.equal(ps[i], p0) and all(torch.equal(torch.as_tensor(a.state[ps[i]][k2]), v) for k2, v in st.items())
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    assert float(a.state[ps[7]]["step"]) == 3.0 and float(a.state[ps[8]]["step"]) == 4.0


def test_optimizers_refuse_what_the_kernels_cannot_read(cuda):
    for cls in (optim.Muon, optim.FusedAdamW):
        for p, g in ((torch.zeros(8, 6, device=cuda), torch.zeros(6, 8, device=cuda).t()),
                     (torch.zeros(8, 6, device=cuda, dtype=torch.bfloat16), torch.zeros(8, 6, device=cuda, dtype=torch.bfloat16)),
                     (torch.zeros(16, 12, device=cuda)[::2, ::2], torch.zeros(16, 12, device=cuda)[::2, ::2])):
            p = torch.nn.Parameter(p)
            p.grad = g
            with pytest.raises(RuntimeError):
                cls([p]).step()
    ps = [torch.nn.Parameter(torch.zeros(4, 4, device=cuda)) for _ in range(2)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = optim.Muon([{"params": ps[:1]}, {"params": ps[1:], "ns_steps": 3}])
    with pytest.raises(ValueError, match="same in all parameter groups"):
        opt.step()


@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_captured_step_follows_schedule_and_step_numbers(cuda, cls):
    make = lambda ps, cap: getattr(optim, cls)(ps, lr=1e-2, weight_decay=0.05, capturable=cap)
    ps, qs = network(cuda, 4), network(cuda, 4)
    a, b = make(ps, True), make(qs, False)
    a.step()
    b.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    with pytest.raises(RuntimeError, match="capturable"):
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2):
            b.step()
    for k in range(5):
        for p, q in zip(ps, qs):
            n = torch.randn_like(p)
            p.grad.copy_(n)
            q.grad.copy_(n)
        for o in (a, b):
            o.param_groups[0]["lr"] = 1e-2 / (k + 1)
        a.push_hyper()
        g.replay()
        b.step()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(ps, qs)):
            # the same kernels; bias corrections and decay are rounded from 64 bits on the device instead of the host
            assert torch.allclose(p, q, rtol=4 * (k + 2) * E24, atol=16 * (k + 2) * E24 * 0.1), (k, i, float((p - q).abs().max()))
    if cls == "FusedAdamW":
        assert float(a.state[ps[0]]["step"]) == 6.0


def test_muon_trains_a_network_and_keeps_replicas_identical(cuda):
    """All operators together as a trainer uses them: UNet forward, loss, backward, Muon step (its AdamW half for the norms), twice
    from the same start: finite, moving, and bit-identical."""
    import models
    from segmi.distributed import DistributedModel
    from utils.losses import CrossEntropyLoss2d
    results = []
    for _ in range(2):
        torch.manual_seed(0)
        m = DistributedModel(models.UNet(3).to(cuda).train())
        opt = optim.Muon(m.parameters(), lr=1e-3, adjust_lr_fn="match_rms_adamw", weight_decay=0.01)
        start = [p.detach().clone() for p in m.parameters()]
        g = torch.Generator().manual_seed(1)
        x, t = torch.randn(2, 3, 64, 64, generator=g).to(cuda), torch.randint(0, 3, (2, 64, 64), generator=g).to(cuda)
        crit = CrossEntropyLoss2d(ignore_index=255)
        for _ in range(2):
            m.zero_grad()
            crit(m(x), t).backward()
            m.finish_gradients()
            opt.step()
        assert all(bool(torch.isfinite(p).all()) for p in m.parameters())
        assert all(not torch.equal(p, s) for p, s in zip(m.parameters(), start) if p.grad is not None)
        kinds = {frozenset(opt.state[p]) for p in m.parameters() if p.grad is not None}
        assert kinds == {frozenset({"momentum_buffer"}), frozenset({"step", "exp_avg", "exp_avg_sq"})}
        results.append([p.detach().clone() for p in m.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ------------------------------------------------------------------------------------------------ borders between the kernels' variants
BORDERS = [(32, 256), (32, 257), (33, 256), (31, 768), (32, 769), (30, 2304), (32, 2305), (33, 768), (64, 768), (64, 769), (65, 256), (64, 257), (127, 254), (128, 255)]


@pytest.mark.parametrize("r,c", BORDERS, ids=lambda v: str(v))
@pytest.mark.parametrize("how", ["plain", "tall", "bf16", "column-major", "expanded source"])
def test_orthogonalize_at_the_variants_borders(cuda, r, c, how):
    m = matrix("gauss", r, c, gen_of(cuda, r * 131 + c), cuda)
    if how == "tall":
        m = m.t().contiguous()
    elif how == "column-major":
        m = m.t().contiguous().t()
    elif how == "bf16":
        m = m.bfloat16()
    elif how == "expanded source":
        m = m[:, :1].expand(r, c)                        # rank one: the rest of the spectrum is exactly zero and stays it
    out, want = optim.orthogonalize(m), iterate(m)
    assert out.shape == m.shape and out.dtype == m.dtype
    if how == "bf16":
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * want.abs().max()).all())
    elif how == "expanded source":
        assert relative(out, want) <= WORST
    else:
        assert relative(out, want) <= max(4 * relative(iterate(m, dtype=torch.float32), want), SHARP_FLOOR)


def test_orthogonalize_mixed_lists(cuda):
    """Small, nearly square and wide matrices in one call: wide ones that go with the square ones, wide ones that are too large to, and
    lists without square ones; the outputs lie where each belongs."""
    gen = gen_of(cuda, 23)
    for sizes in ([(150, 257), (256, 1024), (20, 40)], [(256, 1024), (20, 40)], [(150, 257), (1024, 4608), (33, 64)], [(65, 66)] * 61 + [(130, 500)] * 2):
        mats = [matrix("gauss", r, c, gen, cuda) for r, c in sizes]
        for m, o in zip(mats, optim.orthogonalize(mats)):
            want = iterate(m)
            assert relative(o, want) <= max(4 * relative(iterate(m, dtype=torch.float32), want), SHARP_FLOOR), tuple(m.shape)


def test_orthogonalize_same_matrix_twice_and_on_two_streams_at_once(cuda):
    m = matrix("gauss", 40, 70, gen_of(cuda, 4), cuda)
    big = matrix("gauss", 200, 500, gen_of(cuda, 5), cuda)
    one = optim.orthogonalize([m, big])
    two = optim.orthogonalize([m, big, m, big])
    assert all(torch.equal(two[i], two[i + 2]) for i in range(2))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(optim.orthogonalize([m, big]))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, one))


# ------------------------------------------------------------------------------------------------ optimizers: what a program may do between steps
def test_not_finite_gradient_stays_in_its_parameter(cuda):
    ps, qs = network(cuda, 5), network(cuda, 5)
    a, b = optim.Muon(ps, lr=1e-2), optim.Muon(qs, lr=1e-2)
    a.step()
    b.step()
    for i, bad in ((0, float("nan")), (3, float("inf")), (7, float("nan"))):
        ps[i].grad[(5,) if ps[i].dim() == 1 else (5,) + (1,) * (ps[i].dim() - 1)] = bad
    a.step()
    b.step()
    for i, (p, q) in enumerate(zip(ps, qs)):
        if i in (0, 3):
            assert bool(torch.isnan(p).all())            # a matrix's update mixes all of its entries
        elif i == 7:
            assert int(torch.isnan(p).sum()) == 1
        else:
            assert torch.equal(p, q), i


@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_captured_step_after_load_and_after_a_new_parameter(cuda, cls):
    """A graph keeps pointing at this optimizer's buffers: state that is loaded later, and step numbers that other parameters get later, do
    not leave it behind."""
    make = lambda ps: getattr(optim, cls)(ps, lr=1e-2, capturable=True)
    ps, qs = network(cuda, 6), network(cuda, 6)
    a, b = make(ps), make(qs)
    late = [ps[9].grad, qs[9].grad]
    ps[9].grad = qs[9].grad = None                       # comes later
    a.step()
    b.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    ps[9].grad, qs[9].grad = late
    a.step()                                             # eager, with one parameter more
    b.step()
    churn = [torch.randn(64, device=cuda) for _ in range(64)]       # whatever was freed has other contents now
    saved = None
    for k in range(6):
        for p, q in zip(ps, qs):
            n = torch.randn_like(p)
            p.grad.copy_(n)
            q.grad.copy_(n)
        if k == 2:
            saved = ({i: {n: torch.as_tensor(v).clone() for n, v in s.items()} for i, s in b.state_dict()["state"].items()}, b.state_dict()["param_groups"],
                     [q.detach().clone() for q in qs])
        if k == 4:                                       # back to where step 2 began
            for o in (a, b):
                o.load_state_dict({"state": {i: {n: v.clone() for n, v in s.items()} for i, s in saved[0].items()}, "param_groups": saved[1]})
            for ts in (ps, qs):
                for t, v in zip(ts, saved[2]):
                    t.data.copy_(v)
        a.push_hyper()
        g.replay()
        keep = qs[9].grad
        qs[9].grad = None
        b.step()
        qs[9].grad = keep
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(ps, qs)):
            assert torch.equal(p, q), (k, i)
            for n, v in b.state[q].items():
                assert torch.equal(torch.as_tensor(a.state[p][n]), torch.as_tensor(v)), (k, i, n)
    del churn


@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_copied_and_pickled_optimizers_go_on(cuda, cls, tmp_path):
    import copy
    ps = network(cuda, 8)
    a = getattr(optim, cls)(ps, lr=1e-2)
    a.step()
    qs, b = copy.deepcopy((ps, a))
    for q, p in zip(qs, ps):
        q.grad = torch.empty_like(q).copy_(p.grad)
    assert all(x is y for x, y in zip(b.param_groups[0]["params"], qs))
    for _ in range(2):
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert all(torch.equal(torch.as_tensor(a.state[p][n]), torch.as_tensor(v)) for n, v in b.state[q].items())


def test_changed_strides_at_the_same_address_are_seen(cuda):
    for cls in (optim.Muon, optim.FusedAdamW):
        p = torch.nn.Parameter(torch.zeros(8, device=cuda))
        store = torch.ones(16, device=cuda)
        p.grad = store[:8]
        opt = cls([p])
        opt.step()
        p.grad = store[::2]                              # same address, every other element
        with pytest.raises(RuntimeError, match="dense"):
            opt.step()
        q = torch.nn.Parameter(torch.eye(6, device=cuda))
        q.grad = torch.ones(6, 6, device=cuda)
        opt = cls([q])
        opt.step()
        q.data = q.data.t()
        with pytest.raises(RuntimeError, match="dense"):
            opt.step()


@pytest.mark.parametrize("name", ["Muon", "FusedAdamW"])
def test_train_main_with_the_optimizer_from_config(cuda, tmp_path, name):
    """`python train.py -c config.json` with `"optimizer": {"type": name}`: an epoch, a checkpoint, and the run resumed from it with the
    optimizer's state."""
    import json
    import os
    import train
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    config = json.load(open(os.path.join(root, "pytorch-segmentation_amd", "config.json")))
    config["optimizer"] = {"type": name, "differential_lr": True, "args": {"lr": 1e-3, "weight_decay": 0.01}}
    config["trainer"].update(save_dir=str(tmp_path), log_dir=str(tmp_path), epochs=1, save_period=1)
    tr = train.main(json.loads(json.dumps(config)), None)
    assert type(tr.optimizer) is getattr(optim, name)
    assert all(torch.isfinite(v) for v in tr.iteration_losses)
    config["trainer"]["epochs"] = 2
    again = train.main(config, os.path.join(tr.checkpoint_dir, "checkpoint-epoch1.pth"))
    assert again.start_epoch == 2 and all(torch.isfinite(v) for v in again.iteration_losses)
    steps = {float(st["step"]) for st in again.optimizer.state.values() if "step" in st}
    assert steps == {2.0 * len(tr.iteration_losses)}


def test_small_matrices_beside_large_ones_keep_the_callers_order(cuda):
    """Small matrices run on a stream of their own next to large ones: what the caller queued before a call, and what is queued behind it,
    stay before and behind, on the default stream and on another."""
    gen = gen_of(cuda, 31)
    small, large = matrix("gauss", 30, 200, gen, cuda), matrix("gauss", 200, 900, gen, cuda)
    busy = torch.zeros(1 << 26, device=cuda)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            for k in range(4):
                busy.add_(1.0)                           # keeps the stream occupied while the host goes on
                a, b = small * (k + 1.0), large + 0.01 * k
                x, y = optim.orthogonalize([a, b])
                sums = x.sum() + y.sum()                 # reads what has to be there
                a.zero_()                                # and overwrites what was read
                b.zero_()
                want = optim.orthogonalize([small * (k + 1.0)])[0], optim.orthogonalize([large + 0.01 * k])[0]
                assert torch.equal(x, want[0]) and torch.equal(y, want[1]), k
                assert torch.equal(sums, want[0].sum() + want[1].sum())
        torch.cuda.synchronize()


@pytest.mark.parametrize("r,c", [(2, 112), (5, 41), (162, 5), (7, 1000), (16, 200), (13, 2304)], ids=lambda v: str(v))
def test_few_rows_are_closer_than_fp32(cuda, r, c):
    """With few rows a rounding of A or Q moves all singular values at once, and near 1 the polynomial enlarges it tenfold (the terms of
    0.7 = 3.44 - 4.77 + 2.03 cancel): that is most of the fp32 iteration's distance (2^-24 of each of A, b A, c A^2 and Q a step).  Here these are
    in 64 bits and three fp16 numbers, and what is left are roundings of X, 2^-23 each at most, which are independent over r c entries.
    Compared as root mean squares over 24 matrices, so that one unlucky spectrum decides nothing."""
    gen = gen_of(cuda, 97 * r + c)
    here = plain = 0.0
    for _ in range(24):
        m = matrix("gauss", r, c, gen, cuda)
        want = iterate(m)
        here += relative(optim.orthogonalize(m), want) ** 2
        plain += relative(iterate(m, dtype=torch.float32), want) ** 2
    print("%dx%d: %.2e, fp32 iteration %.2e" % (r, c, math.sqrt(here / 24), math.sqrt(plain / 24)))
    assert here <= plain


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_orthogonalize_views_that_do_not_start_on_a_vector(cuda, dtype):
    """Rows whose addresses are odd, for every class of sizes: the loads of four fall back to single ones."""
    for r, c in ((7, 60), (40, 200), (100, 300), (130, 132)):
        m = matrix("gauss", r, c, gen_of(cuda, r), cuda).to(dtype)
        for v in (torch.zeros(r, c + 5, device=cuda, dtype=dtype)[:, 3:3 + c], torch.zeros(r * c + 1, device=cuda, dtype=dtype)[1:].view(r, c),
                  torch.zeros(c, r + 3, device=cuda, dtype=dtype)[:, 2:2 + r].t()):
            v.copy_(m)
            out, want = optim.orthogonalize(v), iterate(m)
            if dtype is torch.float32:
                assert relative(out, want) <= 1e-5
            else:
                assert bool(((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4 * want.abs().max()).all())


def test_orthogonalize_rows_gigabytes_apart(cuda):
    """Offsets beyond 32 bits, in the source of a matrix that would otherwise be a small one, and of a larger one."""
    store = torch.zeros(1_200_000_000, device=cuda)
    for r, c, stride in ((20, 300, 60_000_000), (100, 300, 12_000_000), (1, 500, 7)):
        m = matrix("gauss", r, c, gen_of(cuda, r), cuda)
        for v in (torch.as_strided(store, (r, c), (stride, 1), 1), torch.as_strided(store, (c, r), (1, stride), 1)):
            v.copy_(m if v.shape == m.shape else m.t())
            assert relative(optim.orthogonalize(v), iterate(v)) <= 1e-5


def test_fused_adamw_large_tensor_and_views(cuda):
    """A tensor of more than 2^31 bytes beside a single number; parameters and gradients as views into one buffer."""
    n = 600_000_000
    flat, grads = torch.zeros(n + 5, device=cuda), torch.full((n + 5,), 1e-3, device=cuda)
    flat[-3:] = 2.0
    big, one = torch.nn.Parameter(flat[:n]), torch.nn.Parameter(flat[n + 4])
    big.grad, one.grad = grads[:n], grads[n + 4]
    opt = optim.FusedAdamW([big, one], lr=1e-2, weight_decay=0.0)
    opt.step()
    # the first step moves by lr g / (|g| + eps)
    step = 1e-2 * 1e-3 / (1e-3 + 1e-8)
    for at in (0, 1, n // 2, n - 1):
        assert abs(float(flat[at]) + step) <= 8 * E24 * 1e-2, at
    assert abs(float(flat[n + 4]) - (2.0 - step)) <= 4 * E24 * 2.0
    assert flat[n:n + 4].tolist() == [0.0, 0.0, 2.0, 2.0]           # what lies between them is left alone

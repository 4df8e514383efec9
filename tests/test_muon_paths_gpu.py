"""Muon steps of matrices beyond the one-workgroup sizes, on the GPU against the formula in 64 bits.

Bound on a parameter's distance, in Frobenius norm, summed over the steps: the update's size lr f |O| times what orthogonalize is held to
(4 times the fp32 iteration's distance from 64 bits, or 16 units of 2^-22), plus t + 1 roundings of the momentum and the Nesterov sum, each like
that of X_0, which the fp32 iteration's distance contains, plus 4 half steps for lr f in fp32 and its product; and 3 half steps of the
parameter itself (decay factor, product, sum)."""
import math

import pytest
import torch

from segmi import muon, optim
from test_muon_gpu import E24, SHARP_FLOOR, gen_of, iterate, relative

pytestmark = pytest.mark.gpu

SETS = {
    # square and wide, even and odd, tall; [K, C, R, S] channels-last and contiguous; "t": the first dimension runs fastest
    "few tiles": ["150x257", "333x90", "128x128x3x3", "t 200x310", "65x64", "129x1000"],
    "wide beside square": ["1024x256x1x1", "128x64x3x3", "70x71", "20x30", "t 64x900", "33x2600"],
    "many tiles": ["512x256x3x3", "256x512x3x3", "256x1024x1x1", "c 512x256x2x2", "t 1024x300", "500x501", "40x50"],
    "large": ["2048x2048", "2048x2048", "t 2048x2048", "1024x512x3x3", "c 1024x512x3x3", "48x48"],
    "large and tall": ["4608x1024", "4608x1024", "t 4608x1024", "2048x1100"],
}


def arena(words, lead, dev):
    """The views of one flat buffer, `lead` numbers before each, and the flat buffer's numbers between them."""
    shapes = [[int(d) for d in w.split()[-1].split("x")] for w in words]
    flat = torch.full((sum(math.prod(s) + lead for s in shapes) + lead,), 7.5, device=dev)
    between = torch.ones_like(flat, dtype=torch.bool)
    views, at = [], 0
    for w, s in zip(words, shapes):
        at += lead
        n = math.prod(s)
        slot = flat[at:at + n]
        between[at:at + n] = False
        at += n
        if w.startswith("t "):
            views.append(slot.view(s[1], s[0]).t())
        elif len(s) == 4 and not w.startswith("c "):
            views.append(slot.view(s[0], s[2], s[3], s[1]).permute(0, 3, 1, 2))
        else:
            views.append(slot.view(s))
    return flat, between, views


@pytest.mark.parametrize("lead", [4, 3], ids=["on 16 bytes", "off 16 bytes"])
@pytest.mark.parametrize("nesterov,capturable", [(True, False), (False, False), (True, True), (False, True)])
@pytest.mark.parametrize("name", list(SETS))
def test_muon_steps_match_the_formula(cuda, name, nesterov, capturable, lead):
    words = SETS[name]
    gen = gen_of(cuda, 1000 + len(name))
    flat, between, views = arena(words, lead, cuda)
    gflat, _, grads = arena(words, lead, cuda)
    ps = []
    for v, g in zip(views, grads):
        v.copy_(0.05 * torch.randn(v.shape, generator=gen, device=cuda))
        p = torch.nn.Parameter(v)
        assert p.data_ptr() == v.data_ptr() and p.stride() == v.stride()
        p.grad = g
        ps.append(p)
    # every group has settings of its own, so that a number taken from another group shows
    groups = [{"params": ps[0::3], "lr": 2e-2, "weight_decay": 0.1, "momentum": 0.95}, {"params": ps[1::3], "lr": 7e-3, "weight_decay": 0.0, "momentum": 0.8},
              {"params": ps[2::3], "lr": 4e-2, "weight_decay": 0.3, "momentum": 0.0, "adjust_lr_fn": "original"}]
    opt = optim.Muon(groups, nesterov=nesterov, adjust_lr_fn="match_rms_adamw", capturable=capturable)
    want = [p.detach().double() for p in ps]
    bufs = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(ps)
    for t in range(1, 4):
        for p in ps:
            p.grad.copy_(1e-2 * torch.randn(p.shape, generator=gen, device=cuda))
        kept = gflat.clone()
        opt.step()
        assert torch.equal(gflat, kept)
        assert bool((flat[between] == 7.5).all())                     # nothing is written beside the parameters
        for i, p in enumerate(ps):
            g = opt.param_groups[i % 3]
            bufs[i] = g["momentum"] * bufs[i] + p.grad.double()
            u = p.grad.double() + g["momentum"] * bufs[i] if nesterov else bufs[i]
            rows, cols = u.shape[0], u[0].numel()
            m = u.reshape(rows, cols)
            o = iterate(m)
            plain = relative(iterate(m.float(), dtype=torch.float32), o)
            f = 0.2 * math.sqrt(max(rows, cols)) if g["adjust_lr_fn"] == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
            move = g["lr"] * f
            old, want[i] = want[i], want[i] * (1 - g["lr"] * g["weight_decay"]) - move * o.reshape(u.shape)
            slack[i] += move * float(o.norm()) * (max(4 * plain, SHARP_FLOOR) + (t + 1) * plain + 4 * E24) + 3 * E24 * float(old.norm())
            off = float((p.detach().double() - want[i]).norm())
            assert off <= slack[i], (words[i], t, off / slack[i])
            assert slack[i] <= 1e-2 * t * move * float(o.norm()) + 1e-6 * float(old.norm())           # the bound is one
            assert relative(opt.state[p]["momentum_buffer"], bufs[i]) <= 2 * t * E24
            assert muon._same_layout(opt.state[p]["momentum_buffer"], p)


@pytest.mark.parametrize("name", list(SETS))
def test_captured_steps_equal_eager_ones(cuda, name):
    words = SETS[name]
    sides = []
    for capturable in (True, False):
        gen = gen_of(cuda, 5)
        ps = []
        for v, g in zip(arena(words, 4, cuda)[2], arena(words, 4, cuda)[2]):
            p = torch.nn.Parameter(v.copy_(0.05 * torch.randn(v.shape, generator=gen, device=cuda)))
            p.grad = g.copy_(torch.randn(v.shape, generator=gen, device=cuda))
            ps.append(p)
        opt = optim.Muon([{"params": ps[0::2], "lr": 2e-2}, {"params": ps[1::2], "lr": 3e-3, "momentum": 0.5}], capturable=capturable)
        opt.step()
        sides.append((ps, opt))
    (ps, a), (qs, b) = sides
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    for k in range(4):
        for p, q in zip(ps, qs):
            n = torch.randn_like(p)
            p.grad.copy_(n)
            q.grad.copy_(n)
        for o in (a, b):
            o.param_groups[0]["lr"] = 1e-2 / (k + 1)
            o.param_groups[1]["weight_decay"] = 0.05 * k
        a.push_hyper()
        g.replay()
        b.step()
        torch.cuda.synchronize()
        for w, p, q in zip(words, ps, qs):
            assert torch.equal(p, q), (w, k)
            assert torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"])


def test_moving_gradients_missing_ones_and_resuming(cuda):
    """The general path through what a program does between steps: gradients elsewhere each step, one that is missing, NaN in one matrix,
    a dictionary loaded into another optimizer."""
    words = SETS["many tiles"]
    make = lambda: [torch.nn.Parameter(v.copy_(0.05 * torch.randn(v.shape, generator=gen, device=cuda))) for v in arena(words, 4, cuda)[2]]
    gen = gen_of(cuda, 9)
    ps = make()
    gen = gen_of(cuda, 9)
    qs = make()
    a, b = optim.Muon(ps, lr=1e-2), optim.Muon(qs, lr=1e-2)
    held = []
    for k in range(4):
        for i, (p, q) in enumerate(zip(ps, qs)):
            n = torch.randn_like(p)
            held.append(p.grad)
            p.grad = None if (k, i) == (2, 1) else torch.empty_like(p).copy_(n)
            if q.grad is None:
                q.grad = torch.empty_like(q)
            q.grad.copy_(n)
            if (k, i) == (3, 4):
                p.grad[3, 5] = float("nan")
        before = qs[1].detach().clone()
        frozen = ps[1].detach().clone()
        a.step()
        b.step()
        if k == 2:
            assert torch.equal(ps[1], frozen)
            with torch.no_grad():
                qs[1].copy_(before)
                b.state[qs[1]]["momentum_buffer"].copy_(a.state[ps[1]]["momentum_buffer"])
        if k == 1:
            c = optim.Muon(ps, lr=1e-2)
            c.load_state_dict(a.state_dict())
            a = c
    for i, (p, q) in enumerate(zip(ps, qs)):
        if i == 4:
            assert bool(torch.isnan(p).all()) and not bool(torch.isnan(q).any())
        else:
            assert torch.equal(p, q), words[i]

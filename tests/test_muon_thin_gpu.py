"""Matrices of few rows and many columns in the matrix optimizer, on the GPU against 64 bits.

Up to 16 rows the Gram matrix, Q and the products with Q are in 64 bits, X is rounded to fp32 once a step: at most 6 roundings of half a
step, 2^-24, each relative to its entry (X_0 and five products).  The fp32 iteration rounds X as often and every product besides, so its
distance, as a root mean square over some matrices, bounds the kernels'."""
import math

import pytest
import torch

from segmi import muon, optim
from test_muon_gpu import E24, WORST, gen_of, iterate, matrix, relative

pytestmark = pytest.mark.gpu


def directions(r, c, gen, dev):
    """Noise under a few strong directions, as gradients are."""
    k = min(r, 4)
    return 0.01 * (torch.randn(r, c, generator=gen, device=dev) + 3.0 * torch.randn(r, k, generator=gen, device=dev) @ torch.randn(k, c, generator=gen, device=dev))


SHAPES = [(2, 5000), (3, 5000), (5, 4096), (8, 10000), (16, 4608), (16, 2305), (1, 2305), (13, 70001), (7, 131073)]


@pytest.mark.parametrize("r,c", SHAPES + [(c, r) for r, c in SHAPES], ids=str)
@pytest.mark.parametrize("kind", ["gauss", "directions"])
def test_few_rows_and_many_columns_are_closer_than_fp32(cuda, r, c, kind):
    gen = gen_of(cuda, 89 * r + c)
    here = plain = 0.0
    for _ in range(16):
        m = matrix("gauss", r, c, gen, cuda) if kind == "gauss" else directions(r, c, gen, cuda)
        want = iterate(m)
        out = optim.orthogonalize(m)
        assert out.shape == m.shape and out.dtype == m.dtype
        here += relative(out, want) ** 2
        plain += relative(iterate(m, dtype=torch.float32), want) ** 2
    print("%dx%d: %.2e, fp32 iteration %.2e" % (r, c, math.sqrt(here / 16), math.sqrt(plain / 16)))
    assert here <= plain


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7])
def test_steps_and_coefficients(cuda, steps):
    """Every rounding of X grows by at most a a step: the sum over `steps` of a^k half steps of an entry of size 1 / sqrt(columns)."""
    for coef in (muon.NS_COEFFICIENTS, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)):
        m = matrix("gauss", 9, 3001, gen_of(cuda, steps), cuda)
        grow = sum(coef[0] ** k for k in range(steps + 1))
        assert relative(optim.orthogonalize(m, steps=steps, coefficients=coef), iterate(m, steps, coef)) <= grow * E24


def test_lists_types_strides_and_limits(cuda):
    gen = gen_of(cuda, 41)
    sizes = [(1 + i % 16, 2305 + 61 * i) for i in range(70)] + [(150, 257), (20, 40), (5, 40), (256, 1024)]      # more than a launch holds, and others
    mats = [matrix("gauss", r, c, gen, cuda) for r, c in sizes]
    outs = optim.orthogonalize(mats)
    again = optim.orthogonalize(mats[::-1])[::-1]
    for i, (m, o, p) in enumerate(zip(mats, outs, again)):
        if 70 > i:
            assert torch.equal(o, p)                                     # no atomics, and nothing else in the list enters
            assert relative(o, iterate(m)) <= (WORST if m.shape[0] > 1 else 2 * E24 * 485)
    m = matrix("gauss", 12, 4001, gen, cuda)
    want = optim.orthogonalize(m)
    store = torch.zeros(12, 8017, device=cuda)
    views = [m.t().contiguous().t(), torch.as_strided(store, (12, 4001), (8017, 2), 3), torch.zeros(12, 4010, device=cuda)[:, 5:4006],
             torch.zeros(4001, 20, device=cuda)[:, 3:15].t(), m.view(12, 4001, 1, 1)]
    for v in views:
        if v.shape != m.shape:
            assert torch.equal(optim.orthogonalize(v), want.view(v.shape))
            continue
        v.copy_(m)
        # sums of squares in another order: the norm differs in its last bits of 64, X_0 in one rounding at most
        assert relative(optim.orthogonalize(v), want.double()) <= 1e-6
    wide = m.bfloat16()
    out, ref = optim.orthogonalize(wide), iterate(wide)
    assert out.dtype == torch.bfloat16 and bool(((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-6 * ref.abs().max()).all())
    rank1 = torch.randn(1, 3000, generator=gen, device=cuda).expand(6, 3000)
    assert relative(optim.orthogonalize(rank1), iterate(rank1)) <= WORST
    assert not optim.orthogonalize(torch.zeros(4, 2500, device=cuda)).any()
    for bad in (float("nan"), float("inf")):
        spoilt = m.clone()
        spoilt[11, 4000] = bad
        outs = optim.orthogonalize([spoilt, m])
        assert bool(torch.isnan(outs[0]).all()) and torch.equal(outs[1], want)
    for scale in (2.0 ** -100, 2.0 ** 100):
        assert torch.equal(optim.orthogonalize(m * scale, eps=1e-38), want)


def test_few_rows_gigabytes_apart(cuda):
    """Few columns too, but offsets beyond 32 bits."""
    store = torch.zeros(1_200_000_000, device=cuda)
    for r, c, stride in ((5, 7, 240_000_000), (16, 300, 70_000_000), (2, 2, 1_000_000_000)):
        m = matrix("gauss", r, c, gen_of(cuda, r), cuda)
        for v in (torch.as_strided(store, (r, c), (stride, 1), 1), torch.as_strided(store, (c, r), (1, stride), 1)):
            v.copy_(m if v.shape == m.shape else m.t())
            assert relative(optim.orthogonalize(v), iterate(v)) <= WORST


def test_graph_replays_and_streams(cuda):
    mats = [matrix("gauss", 3, 5000, gen_of(cuda, 1), cuda), matrix("gauss", 16, 90000, gen_of(cuda, 2), cuda), matrix("gauss", 20, 30, gen_of(cuda, 3), cuda)]
    graphs = []
    optim.orthogonalize(mats)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = optim.orthogonalize(mats)
        graphs.append((g, outs))
    for k in range(3):
        for m in mats:
            m.mul_(1.0 + 0.25 * k).add_(0.001 * k)
        eager = optim.orthogonalize(mats)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = optim.orthogonalize(mats)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(eager, outs, other))


@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
def test_muon_on_few_rows(cuda, nesterov, capturable):
    """[classes, channels * taps] heads and their transposes, in two groups, against the formula in 64 bits."""
    gen = gen_of(cuda, 77)
    shapes = [(5, 4096), (2, 300, 3, 3), (4000, 7), (12, 333, 3, 3)]
    ps = []
    for s in shapes:
        t = torch.randn(s, generator=gen, device=cuda) * 0.05
        ps.append(torch.nn.Parameter(t.contiguous(memory_format=torch.channels_last) if len(s) == 4 else t))
    groups = [{"params": ps[:2]}, {"params": ps[2:], "lr": 5e-3, "weight_decay": 0.2, "momentum": 0.8}]
    opt = optim.Muon(groups, lr=2e-2, weight_decay=0.1, nesterov=nesterov, adjust_lr_fn="match_rms_adamw", capturable=capturable)
    want = [p.detach().double() for p in ps]
    bufs = [torch.zeros_like(w) for w in want]
    slack = [0.0] * len(ps)
    for t in range(1, 4):
        for p in ps:
            p.grad = torch.empty_like(p).copy_(1e-2 * torch.randn(p.shape, generator=gen, device=cuda))
        opt.step()
        for i, p in enumerate(ps):
            g = opt.param_groups[0 if i < 2 else 1]
            bufs[i] = g["momentum"] * bufs[i] + p.grad.double()
            u = p.grad.double() + g["momentum"] * bufs[i] if nesterov else bufs[i]
            flat = u.reshape(u.shape[0], -1)
            o = iterate(flat).reshape(u.shape)
            plain = relative(iterate(flat.float(), dtype=torch.float32).reshape(u.shape), o)
            move = g["lr"] * 0.2 * math.sqrt(max(flat.shape))
            old, want[i] = want[i], want[i] * (1 - g["lr"] * g["weight_decay"]) - move * o
            # the iteration as far off as in fp32, t + 1 roundings of the update on top, enlarged like that of X_0 (which `plain` has); the fp32
            # factor of the update and its product: 4 roundings; the parameter: 3 of its own
            slack[i] += move * float(o.norm()) * ((2 + t) * plain + 4 * E24) + 3 * E24 * float(old.norm())
            assert float((p.double() - want[i]).norm()) <= slack[i], (i, t)
            assert relative(opt.state[p]["momentum_buffer"], bufs[i]) <= 2 * t * E24 * 2

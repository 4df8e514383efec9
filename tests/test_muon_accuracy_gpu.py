"""How far orthogonalize is from 64-bit results where it is hardest, on the GPU: spectra that fall off, ranks that are not full, rows and
columns of very different sizes.

Whole matrices.  A rounding here is at most 4 times an fp32 one (2^-22 against 2^-24, an fp16 pair), so the distance, as a root mean
square over some matrices, is at most 4 times the fp32 iteration's, or 16 units of 2^-22 where that is smaller.

Single rows.  Beside these relative roundings a pair has an absolute one: fp16's smallest step is 2^-24, and the scale puts a matrix's bound s
between 2^14 and 2^15, so a value is off by up to 2^-25 / 2^14 = 2^-39 s.  Of a row of norm rho (the matrix's being 1), n wide, that is
sqrt(n) 2^-39 in X_0, and less by the factor a = 3.44 by which such a row grows in each step behind it: 1.5 sqrt(n) 2^-39 together (s <= 1.22).
A and Q = b A + c A^2 (bounds 1 and 5 in the first step, |b| = 4.8) have it too, in m entries of the row, which the product spreads over X, of
norm at most 1.22: (4.8 + 5) 1.22 sqrt(m) 2^-39, with the steps behind it 17 sqrt(m) 2^-39.  So a row is off by at most

    4 times the worst row of the fp32 iteration, or 16 units of 2^-22, and (1.5 sqrt(n) + 17 sqrt(m)) 2^-39 / rho      of its norm.

One row for all.  Then all entries are alike, their roundings too, and those do not average out: a sum of K / 16 instructions' results is off by up to
K / 16 half steps, 2^-24, times kappa, the sum of its terms' sizes over its result, and the two parts of a product with the identity's share
nearly cancel.  The one singular value goes 1, 0.70, 1.11, 0.72, 1.09, 0.70, where |p'| <= 1.31, so behind any error come factors of at most 3.  Two steps at
once: A^2 twice, c s^4 / 0.7 = 4.6 each; W = Q A and A' = W Q, kappa = (3.44 + 2.74) / 0.70 = 8.8 each; P = Q Q', (3.44 + 2.74) (3.44 + 1.86) / 1.11 = 29;
P X, (11.9 + 10.8) / 1.11 = 20: 76.  One step: 4.6, and (b A + c A^2) X, at most 10: 15.  Each Gram sum, K = n, 1.4 times.  Together
3 (2 76 + 15) = 500 times m / 16 and 3 3 1.4 = 13 times n / 16 half steps."""
import math

import pytest
import torch

from segmi import optim
from test_muon_gpu import SHARP_FLOOR, gen_of, iterate, matrix, relative

pytestmark = pytest.mark.gpu

DRAWS = 8


@pytest.mark.parametrize("kind", ["lowrank", "heavy", "decay", "one row for all"])
@pytest.mark.parametrize("r,c", [(32, 200), (64, 64), (64, 500), (96, 700), (500, 130), (512, 512), (300, 2000), (20, 3000), (1024, 1100)], ids=str)
def test_hard_spectra_relative_to_the_fp32_iteration(cuda, kind, r, c):
    gen = gen_of(cuda, r + 37 * c)
    here = plain = 0.0
    for _ in range(DRAWS):
        m = torch.randn(1, c, generator=gen, device=cuda).expand(r, c) if kind == "one row for all" else matrix(kind, r, c, gen, cuda)
        want = iterate(m)
        here += relative(optim.orthogonalize(m), want) ** 2
        plain += relative(iterate(m, dtype=torch.float32), want) ** 2
    here, plain = math.sqrt(here / DRAWS), math.sqrt(plain / DRAWS)
    print("%s %dx%d: %.2e, fp32 iteration %.2e, ratio %.2f" % (kind, r, c, here, plain, here / plain))
    if kind == "one row for all":
        m, n = min(r, c), max(r, c)
        assert here <= (500 * math.ceil(m / 16) + 13 * math.ceil(n / 16)) * 2.0 ** -24
    else:
        assert here <= max(4 * plain, SHARP_FLOOR)


def by_row(a, b):
    return (a.double() - b).norm(dim=1) / b.norm(dim=1)


@pytest.mark.parametrize("which", ["rows", "columns"])
@pytest.mark.parametrize("decades", [2, 4, 6, 8])
@pytest.mark.parametrize("r,c", [(12, 400), (16, 4608), (64, 576), (200, 200), (256, 1024), (300, 5000)], ids=str)
def test_rows_of_different_sizes(cuda, r, c, decades, which):
    """Rows (or columns) from 1 down to 10^-decades, each against 64 bits, relative to its own size."""
    gen = gen_of(cuda, r + 41 * c + decades)
    m = torch.randn(r, c, generator=gen, device=cuda) * torch.logspace(0, -decades, r, device=cuda)[:, None]
    if which == "columns":
        m = m.t().contiguous()
    want, rho = iterate(m), m.double().norm(dim=0 if which == "columns" else 1) / m.double().norm()
    turn = (lambda x: x.t()) if which == "columns" else (lambda x: x)
    here, plain = by_row(turn(optim.orthogonalize(m)), turn(want)), by_row(turn(iterate(m, dtype=torch.float32)), turn(want))
    floor = (1.5 * math.sqrt(c) + 17 * math.sqrt(r)) * 2.0 ** -39 / rho
    print("%s %dx%d, 1e-%d: worst row %.2e, fp32 iteration %.2e" % (which, r, c, decades, float(here.max()), float(plain.max())))
    assert bool((here <= max(4 * float(plain.max()), SHARP_FLOOR) + floor).all())

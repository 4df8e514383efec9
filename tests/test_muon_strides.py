"""The C entry of the orthogonalisation with strides that torch has no views for: negative ones (the first element is not the lowest)."""
import ctypes as C

import numpy as np
import pytest
import torch

from segmi import muon
from segmi._lib import check, lib

COEF = (C.c_double * 3)(*muon.NS_COEFFICIENTS)


def descriptor(rows, cols, src=256, dst=512, src_strides=None, dst_strides=None):
    d = np.zeros(1, dtype=muon._NS_DTYPE)
    d["src"], d["dst"], d["rows"], d["cols"] = src, dst, rows, cols
    d["src_rs"], d["src_cs"] = src_strides or (cols, 1)
    d["dst_rs"], d["dst_cs"] = dst_strides or (cols, 1)
    return d


def test_negative_strides_are_not_addressed_with_32_bits():
    """One-workgroup sizes need no workspace (256 bytes stand for none); with a negative stride their 32-bit offsets do not reach."""
    need = lambda d: lib.segmi_ns_workspace(d.ctypes.data, 1)
    assert need(descriptor(20, 30)) == 256
    for strides in ((-1, 20), (30, -1), (-30, 1), (1, -20), (-30, -1), (1 << 62, 1)):
        assert need(descriptor(20, 30, src_strides=strides)) > 256, strides
        assert need(descriptor(20, 30, dst_strides=strides)) > 256, strides
        assert need(descriptor(5, 30, src_strides=strides)) > 256, strides


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(20, 30), (5, 40), (40, 5), (64, 700), (100, 130), (3, 3000), (130, 700)], ids=str)
@pytest.mark.parametrize("flip_rows,flip_cols,order", [(True, False, "rows"), (False, True, "rows"), (True, True, "rows"), (True, False, "columns"), (False, True, "columns")])
def test_matrices_read_and_written_backwards(cuda, rows, cols, flip_rows, flip_cols, order):
    """The orthogonal factor of a matrix with its rows or columns in the other order is the factor in that order."""
    gen = torch.Generator(device=cuda)
    gen.manual_seed(rows * 1009 + cols)
    m = torch.randn(rows, cols, generator=gen, device=cuda) * 0.01
    flips = [k for k, f in ((0, flip_rows), (1, flip_cols)) if f]
    rs, cs = (cols, 1) if order == "rows" else (1, rows)
    lay = lambda t: t.contiguous() if order == "rows" else t.t().contiguous()
    src = lay(m)                                          # read backwards: m.flip(flips)
    guard = 64
    dst = torch.full((rows * cols + 2 * guard,), 7.5, device=cuda)
    first = (rows - 1) * rs * flip_rows + (cols - 1) * cs * flip_cols
    strides = (-rs if flip_rows else rs, -cs if flip_cols else cs)
    d = descriptor(rows, cols, src.data_ptr() + 4 * first, dst.data_ptr() + 4 * (guard + first), strides, strides)
    nbytes = lib.segmi_ns_workspace(d.ctypes.data, 1)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
    check(lib.segmi_ns_orthogonalize(d.ctypes.data, 1, COEF, 5, 1e-7, ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream), "ns_orthogonalize")
    torch.cuda.synchronize()
    assert bool((dst[:guard] == 7.5).all()) and bool((dst[-guard:] == 7.5).all())
    body = dst[guard:-guard]
    got = (body.view(rows, cols) if order == "rows" else body.view(cols, rows).t()).flip(flips)      # in the order it was read in
    x = m.flip(flips).double()
    x = x / x.norm()
    tall = rows > cols
    x = x.t() if tall else x
    for _ in range(5):
        g = x @ x.t().contiguous()
        x = COEF[0] * x + (COEF[1] * g + COEF[2] * (g @ g)) @ x
    x = x.t() if tall else x
    # as in the tests of orthogonalize on strides: results of a full-rank Gaussian matrix lie within 1e-5
    assert float((got.double() - x).norm() / x.norm()) <= 1e-5

"""State, checkpoints and captured steps of the matrix optimizer on the GPU, beyond test_muon_gpu.py (whose helpers it uses)."""
import pytest
import torch

from segmi import optim
from test_muon_gpu import network

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_reset_state_steps_like_a_new_optimizer(cuda, cls, capturable):
    ps, qs = network(cuda, 12), network(cuda, 12)
    a = getattr(optim, cls)(ps, lr=1e-2, capturable=capturable)
    for _ in range(2):
        a.step()
    for p, q in zip(ps, qs):
        q.data.copy_(p)
    a.state.clear()
    b = getattr(optim, cls)(qs, lr=1e-2, capturable=capturable)
    for k in range(2):
        a.step()
        b.step()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q)
            assert a.state[p].keys() == b.state[q].keys()
            assert all(torch.equal(torch.as_tensor(a.state[p][n]), torch.as_tensor(v)) for n, v in b.state[q].items())


@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_captured_step_after_a_load_without_state(cuda, cls):
    """A new optimizer's dictionary starts a captured step anew, in the buffers the graph points at."""
    ps, qs = network(cuda, 14), network(cuda, 14)
    make = lambda ts: getattr(optim, cls)(ts, lr=1e-2, capturable=True)
    a = make(ps)
    a.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.step()
    g.replay()
    a.load_state_dict(make(qs).state_dict())
    churn = [torch.randn(4096, device=cuda) for _ in range(64)]          # whatever was freed has other contents now
    for p, q in zip(ps, qs):
        q.data.copy_(p)
    b = make(qs)
    for k in range(3):
        for p, q in zip(ps, qs):
            n = torch.randn_like(p)
            p.grad.copy_(n)
            q.grad.copy_(n)
        a.push_hyper()
        g.replay()
        b.step()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(ps, qs)):
            assert torch.equal(p, q), (k, i)
            assert all(torch.equal(a.state[p][n], v) for n, v in b.state[q].items()), (k, i)
    del churn


def test_negated_views_are_what_they_stand_for(cuda):
    """The imaginary part of a conjugate is a view whose memory holds the opposite sign."""
    z = torch.randn(40, 70, dtype=torch.complex64, device=cuda)
    view = z.conj().imag
    assert view.is_neg()
    assert torch.equal(optim.orthogonalize(view), optim.orthogonalize((-z.imag).contiguous()))
    p = torch.nn.Parameter(torch.zeros(40, 70, device=cuda))
    p.grad = torch._neg_view(torch.ones(40, 70, device=cuda))
    for cls in (optim.Muon, optim.FusedAdamW):
        with pytest.raises(RuntimeError, match="negated"):
            cls([p]).step()


@pytest.mark.parametrize("cls", ["Muon", "FusedAdamW"])
def test_gradients_of_another_shape_are_refused(cuda, cls):
    """`p.data = ...` lets a parameter outgrow its gradient."""
    for shape, larger in (((8,), (16,)), ((6, 5), (12, 5))):
        p = torch.nn.Parameter(torch.zeros(shape, device=cuda))
        p.grad = torch.ones(shape, device=cuda)
        opt = getattr(optim, cls)([p])
        opt.step()
        p.data = torch.zeros(larger, device=cuda)
        with pytest.raises(RuntimeError):
            opt.step()

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

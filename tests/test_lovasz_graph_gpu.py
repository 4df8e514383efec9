"""The Lovasz loss inside a captured graph: every replay against the eager result, with eager work and synchronisations between."""
import pytest
import torch

from utils.losses import LovaszSoftmax

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("classes,size", [(5, 40), (21, 97), (150, 64)], ids=str)
def test_captured_loss_and_gradient_equal_eager_ones(cuda, classes, size):
    gen = torch.Generator(device=cuda)
    gen.manual_seed(classes)
    crit = LovaszSoftmax(ignore_index=255)
    x = torch.randn(2, classes, size, size, generator=gen, device=cuda).contiguous(memory_format=torch.channels_last)
    t = torch.randint(0, classes, (2, size, size), generator=gen, device=cuda)
    t[:, :3] = 255

    def both():
        leaf = x.detach().requires_grad_(True)
        loss = crit(leaf, t)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss, grad = both()
    for k in range(4):
        x.mul_(1.0 + 0.5 * k).add_(0.1 * torch.randn(x.shape, generator=gen, device=cuda))
        t.copy_(torch.randint(0, max(2, classes - k), t.shape, generator=gen, device=cuda))
        t[:, :k + 1] = 255
        want = both()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]), k
        assert torch.equal(grad, want[1]), k

"""Muon on calls whose matrices follow different phases in shared launches, and on more shapes than a launch takes."""
import pytest
import torch

from tests.test_gpu_orthogonal_accuracy import error, newton_schulz, noise, times

pytestmark = pytest.mark.gpu

WIDE = ((256, 1024),) * 20 + ((1024, 300),) * 8  # work enough that narrow ones beside them keep phases of their own
MANY = tuple((70 + 3 * k, 130 + 7 * k) for k in range(30)) + WIDE


@pytest.mark.parametrize("shapes", [WIDE + ((64, 128),) * 8 + ((600, 64),) * 4 + ((128, 128),) * 4 + ((16, 700),) * 8, MANY], ids=["kinds", "shapes"])
def test_an_update_from_zero_of_each_kind(device, shapes):
    """Errors of the matrices up to 95 rows and near square (single steps), and of the others, each beside f32 products'."""
    from protoseg_amd import optim
    ps = [torch.nn.Parameter(torch.zeros(s, device=device)) for s in shapes]
    for k, p in enumerate(ps):
        p.grad = noise(device, p.shape, 200 + k)
    opt = optim.Muon(ps, lr=1.0, momentum=0.5, nesterov=False)
    opt.step()
    sums = {}
    for p in ps:
        m, n = sorted(p.shape)
        kind = (m < 64, m < 96 or 2 * n < 3 * m)
        scale = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        exact = -scale * newton_schulz(p.grad[None], torch.float64)[0]
        s = sums.setdefault(kind, [0.0, 0.0, p.shape])
        s[0] += error(p.detach(), exact) ** 2
        s[1] += error(-scale * newton_schulz(p.grad[None], torch.float32)[0], exact) ** 2
        assert torch.equal(opt.state[p]["momentum_buffer"], p.grad)
    assert len(sums) >= 2
    for got, plain, shape in sums.values():
        assert got <= times(shape) ** 2 * plain, shape

"""Matrices of zeros and of values at the end of the float range, through both kernels (one workgroup a matrix, tiles)."""
import pytest
import torch

from tests.test_gpu_muon import check

pytestmark = pytest.mark.gpu

SHAPES = [(40, 60), (60, 40), (130, 200), (600, 70)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_zeros_without_eps(device, shape, dtype):
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(1)
    g = torch.randn(3, *shape, generator=gen).to(dtype).to(device)
    g[1] = 0
    out = optim.orthogonalize(g, eps=0.0)
    assert not bool(out[1].any())  # and no NaN
    for i in (0, 2):
        check(out[i], g[i], eps=0.0)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_a_zero_gradient_without_eps(device, shape):
    """What zero_grad leaves in a parameter that a step has not used."""
    from protoseg_amd import optim
    p = torch.nn.Parameter(torch.ones(shape, device=device))
    p.grad = torch.zeros_like(p)
    optim.Muon([p], lr=0.1, eps=0.0, weight_decay=0.5).step()
    assert torch.equal(p, torch.full_like(p, 1 - 0.1 * 0.5))


@pytest.mark.parametrize("eps", [1e-7, 0.0, 2.0 ** -140])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_subnormal_values(device, shape, eps):
    """Multiples of 2^-149 up to 8 of them, which f32 holds exactly. Where eps is far larger than the matrix, the
    result is as small against 1 as X0 is, and the bound with it."""
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(2)
    g = (torch.randint(-8, 9, shape, generator=gen).double() * 2.0 ** -149).float()
    assert bool((g != 0).any()) and g.abs().max().item() < 2.0 ** -126
    g = g.to(device)
    check(optim.orthogonalize(g, eps=eps), g, eps=eps)

"""Group norm and the orthogonalisation refuse dual tensors (forward-mode differentiation), whose tangent they would drop."""
import pytest
import torch
from torch.autograd import forward_ad

from protoseg_amd import _lib, norm, optim


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("leaf", [False, True])
def test_group_norm(device, which, leaf):
    args = {"x": torch.ones(1, 8, 4, 4, device=device), "weight": torch.ones(8, device=device), "bias": torch.zeros(8, device=device)}
    if leaf:
        args["x"].requires_grad_(True)
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(_lib.ProtosegError, match="forward-mode"):
            norm.group_norm(args["x"], 2, args["weight"], args["bias"])
        with torch.no_grad(), pytest.raises(_lib.ProtosegError, match="forward-mode"):  # tangents live on there
            norm.group_norm(args["x"], 2, args["weight"], args["bias"])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_orthogonalize(device):
    g = torch.ones(4, 6, device=device)
    with forward_ad.dual_level():
        with pytest.raises(_lib.ProtosegError, match="forward-mode"):
            optim.orthogonalize(forward_ad.make_dual(g, g))


@pytest.mark.gpu
def test_tensors_without_a_tangent_pass_an_open_level(device):
    x, g = torch.randn(1, 8, 4, 4, device=device), torch.randn(4, 6, device=device)
    want = norm.group_norm(x, 2), optim.orthogonalize(g)
    with forward_ad.dual_level():
        assert torch.equal(norm.group_norm(x, 2), want[0]) and torch.equal(optim.orthogonalize(g), want[1])

"""Muon on a momentum that was saved in another layout than the parameters have now."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def made(device, seed):
    """A channels-last parameter, its optimizer with a contiguous model's state, and a twin that never changed layout."""
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(32, 16, 3, 3, generator=gen).to(device)
    grads = [torch.randn(32, 16, 3, 3, generator=gen).to(device) for _ in range(6)]
    old = torch.nn.Parameter(w.clone())
    saved = optim.Muon([old], lr=0.05)
    old.grad = grads[0]
    saved.step()
    state = copy.deepcopy(saved.state_dict())
    p = torch.nn.Parameter(old.detach().contiguous(memory_format=torch.channels_last))
    opt = optim.Muon([p], lr=0.05)
    opt.load_state_dict(copy.deepcopy(state))
    twin = torch.nn.Parameter(old.detach().contiguous(memory_format=torch.channels_last))
    opt_t = optim.Muon([twin], lr=0.05)
    opt_t.state[twin]["momentum_buffer"] = state["state"][0]["momentum_buffer"].contiguous(memory_format=torch.channels_last)
    p.grad, twin.grad = (torch.empty_like(p).copy_(grads[1]) for _ in range(2))
    return p, opt, twin, opt_t, grads


def test_a_captured_step_needs_the_layout_first(device):
    from protoseg_amd import _lib
    p, opt, twin, opt_t, grads = made(device, 3)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.ProtosegError, match="one step before"):
        with torch.cuda.graph(graph):
            p.grad.add_(0)
            opt.step()
    opt.step()
    opt_t.step()
    assert torch.equal(p, twin)


def test_replays_after_one_step_are_successive_steps(device):
    p, opt, twin, opt_t, grads = made(device, 4)
    opt.step()
    opt_t.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for g in grads[2:]:
        p.grad.copy_(g)
        twin.grad.copy_(g)
        graph.replay()
        opt_t.step()
        torch.cuda.synchronize()
        assert torch.equal(p, twin) and torch.equal(opt.state[p]["momentum_buffer"], opt_t.state[twin]["momentum_buffer"])

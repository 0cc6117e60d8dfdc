"""Traced and compiled calls of group norm and the orthogonalisation give the eager ones' bits."""
import pytest
import torch

from tests.test_gpu_norm import make

pytestmark = pytest.mark.gpu


def test_traced_backbone(device):
    from protoseg_amd.deeplab import deeplabv2_resnet101_features
    torch.manual_seed(0)
    net = deeplabv2_resnet101_features(n_blocks=(1, 1, 1, 1), scales=[], norm="group").to(device).to(memory_format=torch.channels_last)
    gen = torch.Generator().manual_seed(1)
    image = torch.randn(1, 3, 65, 65, generator=gen).to(device).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        traced = torch.jit.trace(net.base.layer1, (image,))
        assert "protoseg::group_norm" in str(traced.inlined_graph)
        other = torch.randn(1, 3, 65, 65, generator=gen).to(device).contiguous(memory_format=torch.channels_last)
        for x in (image, other):
            got, want = traced(x), net.base.layer1(x)
            assert torch.equal(got, want)


@pytest.mark.parametrize("act", ["identity", "relu", "silu"])
def test_traced_and_compiled_gradients(device, act):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 24, 9, 7, torch.bfloat16, 81)

    def f(x, w, b):
        return norm.group_norm(x, 6, w, b, 1e-5, act)

    def grads(g):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = g(*leaves)
        return (y, *torch.autograd.grad(y, leaves, gy))

    want = grads(f)
    traced = torch.jit.trace(f, (x, w, b))
    compiled = torch.compile(f, backend="aot_eager", fullgraph=True)
    for g in (traced, compiled):
        got = grads(g)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        frozen = w.clone()  # a gradient of x alone
        xl = x.detach().requires_grad_(True)
        gx, = torch.autograd.grad(g(xl, frozen, b), xl, gy)
        assert torch.equal(gx, want[1])


def test_under_a_dispatch_mode(device):
    from protoseg_amd import norm, optim

    class Names(torch.utils._python_dispatch.TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    x, w, b, gy = make(device, 2, 24, 9, 7, torch.float32, 82)
    leaf = x.detach().requires_grad_(True)
    with Names() as mode:
        y = norm.group_norm(leaf, 6, w, b, activation="silu")
        gx, = torch.autograd.grad(y, leaf, gy)
        out = optim.orthogonalize(w.view(6, 4))
    assert {"protoseg.group_norm.default", "protoseg.group_norm_backward.default", "protoseg.orthogonalize.default"} <= set(mode.names)
    leaf2 = x.detach().requires_grad_(True)
    y2 = norm.group_norm(leaf2, 6, w, b, activation="silu")
    assert torch.equal(y, y2) and torch.equal(gx, torch.autograd.grad(y2, leaf2, gy)[0])
    assert torch.equal(out, optim.orthogonalize(w.view(6, 4)))


def test_traced_orthogonalize(device):
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(83)
    g, other = torch.randn(2, 40, 70, generator=gen).to(device), torch.randn(2, 40, 70, generator=gen).to(device)
    traced = torch.jit.trace(lambda g: optim.orthogonalize(g) * 2, (g,))
    assert "protoseg::orthogonalize" in str(traced.graph)
    assert torch.equal(traced(other), optim.orthogonalize(other) * 2)
    leaf = g.clone().requires_grad_(True)
    assert not optim.orthogonalize(leaf).requires_grad


def test_traced_calls_without_autograd(device):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 24, 9, 7, torch.float32, 84)

    def both(x, gy):
        y, stats = norm.group_norm_forward(x, w, b, 6, 1e-5, 3)
        return (y, *norm.group_norm_backward(x, gy, w, b, stats, 6, 3))

    x2, _, _, gy2 = make(device, 2, 24, 9, 7, torch.float32, 85)
    traced = torch.jit.trace(both, (x, gy))
    assert all(torch.equal(a, c) for a, c in zip(traced(x2, gy2), both(x2, gy2)))

"""CPU: tracers and dispatch modes see group norm and the orthogonalisation as operators (fake tensors: nothing runs)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from protoseg_amd import _lib, norm, optim


def targets(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]


def test_group_norm_is_an_operator_to_a_tracer():
    with FakeTensorMode():
        x = torch.empty(2, 8, 5, 4, device="cuda:0").contiguous(memory_format=torch.channels_last)
        w, b = torch.empty(8, device="cuda:0"), torch.empty(8, device="cuda:0")
        y = norm.group_norm(x[:, :4], 2, w[:4], b[:4], activation="silu")
        assert y.shape == (2, 4, 5, 4) and y.is_contiguous(memory_format=torch.channels_last)
        graph = make_fx(lambda x, w, b: norm.group_norm(x, 2, w, b, activation="relu"))(x, w, b)
        assert "protoseg.group_norm.default" in targets(graph)
        with pytest.raises(_lib.ProtosegError, match="no HIP kernel"):
            norm.group_norm(x, 2, activation="gelu")


def test_the_calls_without_autograd_are_operators_too():
    with FakeTensorMode():
        x = torch.empty(2, 8, 5, 4, device="cuda:0").contiguous(memory_format=torch.channels_last)
        w = torch.empty(8, device="cuda:0")

        def both(x, w):
            y, stats = norm.group_norm_forward(x, w, None, 2, 1e-5, 1)
            gx, gw, gb = norm.group_norm_backward(x, y, w, None, stats, 2, 1, need_x=False)
            assert gx is None and gw.shape == gb.shape == (8,)
            return gw

        names = targets(make_fx(both)(x, w))
        assert "protoseg.group_norm.default" in names and "protoseg.group_norm_backward.default" in names


def test_orthogonalize_is_an_operator_to_a_tracer():
    with FakeTensorMode():
        g = torch.empty(3, 40, 20, device="cuda:0", dtype=torch.bfloat16)
        out = optim.orthogonalize(g.mT)
        assert out.shape == (3, 20, 40) and out.dtype == g.dtype and out.is_contiguous()
        assert targets(make_fx(lambda g: optim.orthogonalize(g))(g)) == ["protoseg.orthogonalize.default"]


def test_which_calls_go_to_memory_at_once():
    t = torch.zeros(2)
    assert _lib.direct(t, None, torch.nn.Parameter(t))
    seen = []
    torch.jit.trace(lambda t: (seen.append(_lib.direct(t)), t + 1)[1], (t,), check_trace=False)
    assert seen == [False]

    class Mode(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Mode():
        assert not _lib.direct(t)

    class Sub(torch.Tensor):
        pass

    assert not _lib.direct(t.as_subclass(Sub))


def test_cpu_tensors_are_refused_under_a_tracer_too():
    with pytest.raises(_lib.ProtosegError, match="CPU|cpu"):
        torch.jit.trace(lambda x: norm.group_norm(x, 2), (torch.zeros(1, 8, 4, 4),))
    with pytest.raises(_lib.ProtosegError, match="CPU|cpu"):
        torch.jit.trace(lambda g: optim.orthogonalize(g), (torch.zeros(4, 4),))

"""Group norm, the prototype layer, Muon and Adam together, as a training step uses them. Each operator is
held to its own bound (tests/test_gpu_norm.py, tests/test_gpu_muon.py) on the values that it meets there."""
import pytest
import torch

from tests.test_gpu_muon import reference_step
from tests.test_gpu_norm import close, reference

pytestmark = pytest.mark.gpu


def test_training_step_with_group_norm_and_muon(device):
    from protoseg_amd import norm
    from protoseg_amd.deeplab import deeplabv2_resnet101_features
    from protoseg_amd.model import construct_PPNet
    from protoseg_amd.optim import Adam, Muon
    from protoseg_amd.train import PatchClassificationStep, muon_param_groups
    torch.manual_seed(0)
    feats = deeplabv2_resnet101_features(n_blocks=(1, 1, 1, 1), scales=[], norm="group")
    net = construct_PPNet(img_size=65, prototype_shape=(38, 64, 1, 1), num_classes=19, add_on_layers_type="deeplab_simple",
                          patch_classification=True, features=feats).to(device).to(memory_format=torch.channels_last)
    matrices, vectors = muon_param_groups(net)
    muon, adam = Muon(matrices, lr=2e-3), Adam(vectors, lr=2.5e-4)
    step = PatchClassificationStep(net, [muon, adam])
    gen = torch.Generator().manual_seed(1)
    image = torch.randn(2, 3, 65, 65, generator=gen).to(device).contiguous(memory_format=torch.channels_last)
    target = torch.randint(0, 20, (2, 65, 65), generator=gen).to(device)

    seen = {}

    def watch(module, args, out):
        rec = seen.setdefault(module, {"x": args[0].detach(), "y": out.detach()})
        args[0].register_hook(lambda g: rec.__setitem__("gx", g))
        out.register_hook(lambda g: rec.__setitem__("gy", g))

    gns = [m for m in net.modules() if isinstance(m, norm.GroupNorm)]
    hooks = [m.register_forward_hook(watch) for m in gns]
    affine = {m: (m.weight.detach().clone(), m.bias.detach().clone()) for m in gns}
    before = {p: p.detach().clone() for g in muon.param_groups for p in g["params"]}
    step(image, target)
    for h in hooks:
        h.remove()
    assert len(seen) == len(gns) == 17
    for m, rec in seen.items():
        w, b = affine[m]
        ref = reference(rec["x"], m.num_groups, w, b, m.eps, m.activation, rec["gy"])
        close(rec["y"], ref, "y")
        close(rec["gx"], ref, "gx")
        close(m.weight.grad, ref, "gw")
        close(m.bias.grad, ref, "gb")
    checked = 0
    for g in muon.param_groups:
        for p in g["params"]:
            if p.numel() > 300_000:
                continue
            # columns in the parameter's own order: a permutation of the matrix's, for p, g and B alike
            new, tol, _, _ = reference_step(before[p], p.grad, torch.zeros_like(p), 2e-3, 0.95, True, g["weight_decay"], "original")
            got = p.detach().cpu().double().reshape(new.shape)
            assert torch.linalg.norm(got - new).item() <= tol, tuple(p.shape)
            checked += 1
    assert checked >= 8
    for _ in range(2):
        step(image, target)
    assert all(bool(torch.isfinite(p).all()) for p in net.parameters())


def test_captured_step_of_all_operators_replays(device):
    """group norm -> prototype layer -> their backward -> Muon and Adam in one graph: every replay equals
    the eager twin's step bit for bit, with eager work in between."""
    from protoseg_amd import norm, ops
    from protoseg_amd.optim import Adam, Muon
    gen = torch.Generator().manual_seed(2)
    start = [torch.rand(38, 64, generator=gen), torch.randn(19, 38, generator=gen) * 0.1, 1 + 0.1 * torch.randn(64, generator=gen),
             0.1 * torch.randn(64, generator=gen)]

    class Program:
        def __init__(self):
            self.params = [torch.nn.Parameter(t.to(device)) for t in start]
            for p in self.params:
                p.grad = torch.zeros_like(p)
            self.x = torch.zeros(2, 17, 15, 64, device=device).permute(0, 3, 1, 2)
            self.gl = torch.zeros(2, 17, 15, 19, device=device)
            self.muon, self.adam = Muon(self.params[:2], lr=1e-2), Adam(self.params[2:], lr=1e-3)

        def step(self):
            protos, w_last, w, b = self.params
            y = norm.group_norm(self.x, 32, w, b, activation="sigmoid")
            _, logits, _ = ops.prototype_layer(y, protos, w_last)
            for p, g in zip(self.params, torch.autograd.grad(logits, self.params, self.gl)):
                p.grad.copy_(g)
            self.muon.step()
            self.adam.step()

        def feed(self, seed):
            g = torch.Generator().manual_seed(seed)
            self.x.copy_(torch.randn(2, 17, 15, 64, generator=g).permute(0, 3, 1, 2))
            self.gl.copy_(torch.randn(2, 17, 15, 19, generator=g))

    a, twin = Program(), Program()
    for prog in (a, twin):
        prog.feed(10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a.step()  # eager once: optimizer state, scratch
    torch.cuda.current_stream().wait_stream(stream)
    twin.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a.step()
    for k in range(4):
        for prog in (a, twin):
            prog.feed(20 + k)
        graph.replay()
        twin.step()
        torch.cuda.synchronize()
        for p, t in zip(a.params, twin.params):
            assert torch.equal(p, t), k

"""CPU: a training step follows its ``optimizer`` attribute, as a program that changes phases sets it."""
import torch

from protoseg_amd.train import PatchClassificationStep
from tests.test_train_dp import TinyPPNet, _data, _kld, _resize


def test_an_optimizer_set_later_is_the_one_that_steps():
    model = TinyPPNet()
    ps = list(model.parameters())
    step = PatchClassificationStep(model, torch.optim.SGD(ps[:1], lr=0.5), kld_fn=_kld, resize_fn=_resize)
    step(*_data(0, 0))
    for new in (torch.optim.SGD(ps[1:], lr=0.5), [torch.optim.SGD(ps[1:], lr=0.5)]):
        before = [p.detach().clone() for p in ps]
        step.optimizer = new
        step(*_data(1, 0))
        assert torch.equal(ps[0], before[0])
        assert any(not torch.equal(p, b) for p, b in zip(ps[1:], before[1:]))

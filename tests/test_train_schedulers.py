"""CPU: a training step of several optimizers steps a scheduler of each."""
import pytest
import torch

from protoseg_amd.train import PatchClassificationStep
from tests.test_train_dp import TinyPPNet, _data, _kld, _resize


def _run(optimizers, schedulers, steps=4):
    model = TinyPPNet()
    ps = list(model.parameters())
    opts = optimizers(ps)
    step = PatchClassificationStep(model, opts, iter_size=2, kld_fn=_kld, resize_fn=_resize, lr_scheduler=schedulers(opts))
    for s in range(steps):
        step(*_data(s, 0))
    assert step.iter_steps == 0
    return opts


@pytest.mark.parametrize("kind", [list, tuple])
def test_a_scheduler_for_each_optimizer(kind):
    opts = _run(lambda ps: [torch.optim.SGD(ps[:1], lr=0.5), torch.optim.SGD(ps[1:], lr=0.25)],
                lambda opts: kind(torch.optim.lr_scheduler.ExponentialLR(o, g) for o, g in zip(opts, (0.5, 0.1))))
    assert opts[0].param_groups[0]["lr"] == pytest.approx(0.5 * 0.5 ** 2)  # two boundaries in four micro-steps
    assert opts[1].param_groups[0]["lr"] == pytest.approx(0.25 * 0.1 ** 2)


def test_one_scheduler_or_none():
    opt = _run(lambda ps: torch.optim.SGD(ps, lr=0.5), lambda o: torch.optim.lr_scheduler.ExponentialLR(o, 0.5))
    assert opt.param_groups[0]["lr"] == pytest.approx(0.125)
    opts = _run(lambda ps: [torch.optim.SGD(ps[:1], lr=0.5), torch.optim.SGD(ps[1:], lr=0.25)],
                lambda opts: [None, torch.optim.lr_scheduler.ExponentialLR(opts[1], 0.5)])
    assert [o.param_groups[0]["lr"] for o in opts] == [0.5, pytest.approx(0.0625)]


def test_a_scheduler_given_later():
    model = TinyPPNet()
    opt = torch.optim.SGD(model.parameters(), lr=0.5)
    step = PatchClassificationStep(model, opt, kld_fn=_kld, resize_fn=_resize)
    step(*_data(0, 0))
    step.lr_scheduler = torch.optim.lr_scheduler.ExponentialLR(opt, 0.5)
    step(*_data(1, 0))
    assert opt.param_groups[0]["lr"] == pytest.approx(0.25)

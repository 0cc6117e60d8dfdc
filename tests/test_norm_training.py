"""CPU: a backbone with group norm, its parameter groups, and a training step of several optimizers."""
import pytest
import torch

from protoseg_amd import norm
from protoseg_amd.deeplab import deeplabv2_resnet101_features
from protoseg_amd.model import construct_PPNet
from protoseg_amd.train import PatchClassificationStep, group_norm_params, joint_param_groups, muon_param_groups
from tests.test_train_dp import TinyPPNet, _data, _kld, _resize


def _net(kind):
    feats = deeplabv2_resnet101_features(n_blocks=(1, 1, 1, 1), scales=[], norm=kind)
    return construct_PPNet(img_size=65, prototype_shape=(38, 64, 1, 1), num_classes=19, add_on_layers_type="deeplab_simple",
                           patch_classification=True, features=feats)


def test_group_norm_takes_the_place_of_batch_norm():
    batch, group = _net("batch"), _net("group")
    assert not any(isinstance(m, torch.nn.BatchNorm2d) for m in group.modules())
    assert not any(isinstance(m, norm.GroupNorm) for m in batch.modules())
    assert sum(isinstance(m, norm.GroupNorm) for m in group.modules()) == sum(
        isinstance(m, torch.nn.BatchNorm2d) for m in batch.modules())
    names = {k for k in batch.state_dict() if ".bn." not in k}
    assert names == {k for k in group.state_dict() if ".gn." not in k}
    block = group.features.base.layer2.block1
    assert block.reduce.gn.activation == "relu" and block.increase.gn.activation == "identity"
    group.features.base.freeze_bn()  # nothing to freeze
    with pytest.raises(ValueError, match="norm"):
        deeplabv2_resnet101_features(n_blocks=(1, 1, 1, 1), norm="layer")


def test_parameter_groups():
    batch, group = _net("batch"), _net("group")
    assert len(joint_param_groups(batch)) == 5  # the reference's groups
    groups = joint_param_groups(group)
    assert len(groups) == 6 and groups[-1]["weight_decay"] == 0.0
    assert [id(p) for p in groups[-1]["params"]] == [id(p) for p in group_norm_params(group.features)]
    for net in (batch, group):
        matrices, vectors = muon_param_groups(net)
        flat = [p for g in matrices + vectors for p in g["params"]]
        assert sorted(map(id, flat)) == sorted(id(p) for g in joint_param_groups(net) for p in g["params"])
        assert all(p.dim() >= 2 for g in matrices for p in g["params"]) and all(p.dim() < 2 for g in vectors for p in g["params"])
        decay = {id(p): g["weight_decay"] for g in matrices + vectors for p in g["params"]}
        assert decay[id(net.prototype_vectors)] == 0.0
        assert decay[id(net.features.base.aspp.c0.weight)] == 5e-4


def test_a_list_of_optimizers_steps_like_one():
    def run(split):
        torch.manual_seed(0)
        model = TinyPPNet()
        ps = list(model.parameters())
        opt = [torch.optim.SGD(ps[:1], lr=0.5), torch.optim.SGD(ps[1:], lr=0.5)] if split else torch.optim.SGD(ps, lr=0.5)
        step = PatchClassificationStep(model, opt, loss_weight_kld=0.25, iter_size=2, kld_fn=_kld, resize_fn=_resize)
        for s in range(4):
            step(*_data(s, 0))
        return [p.detach().clone() for p in ps]

    assert all(torch.equal(a, b) for a, b in zip(run(False), run(True)))

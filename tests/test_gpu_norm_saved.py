"""Group norm's backward on saved tensors that hooks brought back in another layout."""
import pytest
import torch

from tests.test_gpu_norm import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["cl", "slice", "nchw"])
@pytest.mark.parametrize("how", ["pinned host memory", "nchw", "wider"])
def test_saved_map_of_another_layout(device, layout, how):
    x, w, b, gy = make(device, 2, 48, 17, 9, torch.bfloat16, 91, layout=layout)
    want = run(x, 12, w, b, 1e-5, "silu", gy)

    def wider(t):
        if t.dim() != 4:
            return t
        big = torch.full((t.shape[0], t.shape[1], t.shape[2], t.shape[3] + 5), float("nan"), dtype=t.dtype, device=t.device)
        big[..., :t.shape[3]] = t
        return big[..., :t.shape[3]]

    hooks = {"pinned host memory": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
             "nchw": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
             "wider": lambda: torch.autograd.graph.saved_tensors_hooks(wider, lambda t: t)}[how]
    with hooks():
        got = run(x, 12, w, b, 1e-5, "silu", gy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_map_changed_in_place_is_refused(device):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 48, 17, 9, torch.float32, 92)
    wl = w.clone().requires_grad_(True)
    x = x.clone(memory_format=torch.preserve_format)
    y = norm.group_norm(x, 12, wl, b)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(gy)

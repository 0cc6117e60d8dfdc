"""Group norm's gradient sums of mixed sign are held in 64 bits: where gz is the incoming gradient itself (identity, relu),
g_bias is off by the rounding of each workgroup's partial sum to f32, u = 2^-24 of it, and by its own. Maps of at most
4096 elements are one workgroup a sample."""
import pytest
import torch

from tests.test_gpu_norm import U, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,groups", [((19, 2, 16, 11), 1), ((2, 1, 61, 67), 1), ((3, 4, 32, 31), 2), ((5, 16, 15, 17), 4), ((4, 3, 33, 40), 3)],
                         ids=str)
@pytest.mark.parametrize("act", ["identity", "relu"])
def test_bias_gradient(device, shape, groups, dtype, act):
    B, C, H, W = shape
    assert C * H * W <= 4096
    x, w, b, gy = make(device, *shape, dtype, 101)
    gb = run(x, groups, w, b, 1e-5, act, gy)[3].cpu().double()
    ref = reference(x, groups, w, b, 1e-5, act, gy)
    z64 = ref["y"] if act == "relu" else None
    gz = gy.cpu().double() * (1.0 if z64 is None else (z64 > 0).double())
    parts = gz.sum((2, 3))
    want = parts.sum(0)
    assert torch.allclose(want, ref["gb"], rtol=1e-12, atol=1e-12)
    tol = U * parts.abs().sum(0) + U * want.abs() + 2.0 ** -60 * gz.abs().sum((0, 2, 3)) + 2.0 ** -126
    assert bool(((gb - want).abs() <= tol).all())

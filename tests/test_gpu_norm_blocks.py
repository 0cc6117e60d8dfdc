"""Group norm where a group's channels lie in two workgroups (more channels than a workgroup's 256 vectors): one set
of statistics, the same bits on every run."""
import pytest
import torch

from tests.test_gpu_norm import close, make, reference, run

pytestmark = pytest.mark.gpu

# channels per workgroup: 512 (C = 750, 2 bf16 a vector), 1024 (4 f32), 2048 (8 bf16), 256 (odd C, one element)
STRADDLING = [((2, 750, 65, 65), 6, torch.bfloat16), ((8, 1536, 65, 65), 32, torch.float32), ((2, 2400, 17, 19), 5, torch.bfloat16),
              ((3, 645, 21, 13), 15, torch.float16), ((2, 1536, 33, 31), 3, torch.float32)]


@pytest.mark.parametrize("shape,groups,dtype", STRADDLING, ids=str)
def test_same_bits_every_run(device, shape, groups, dtype):
    from protoseg_amd import norm
    x, w, b, gy = make(device, *shape, dtype, 61)
    first = None
    for _ in range(6):
        y, stats = norm.group_norm_forward(x, w, b, groups, 1e-5, 1)
        grads = norm.group_norm_backward(x, gy, w, b, stats, groups, 1)
        first = first or (y, stats, *grads)
        assert all(torch.equal(a, c) for a, c in zip(first, (y, stats, *grads)))


@pytest.mark.parametrize("shape,groups,dtype", [s for s in STRADDLING if s[0][0] < 8], ids=str)
def test_against_the_definition(device, shape, groups, dtype):
    x, w, b, gy = make(device, *shape, dtype, 62)
    ref = reference(x, groups, w, b, 1e-5, "silu", gy)
    for v, key in zip(run(x, groups, w, b, 1e-5, "silu", gy), ("y", "gx", "gw", "gb")):
        close(v, ref, key)

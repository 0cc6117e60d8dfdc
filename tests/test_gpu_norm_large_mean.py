"""Group norm of maps whose mean is far larger than their spread.

tests/test_gpu_norm.py's bounds, and the mean's own rounding: the kernels hold it as an f32 pair, whose second part
(at most half a step of the first, 2^-24 |mean|) is rounded by at most 2^-24 of itself, so x - mean is off by
2^-48 |mean| more, xh by that times rstd. The statistics' sums start from a value of the group: nothing of the
mean's size is in them, and they err by far less (2^-53 of the spread's square times the terms of a chain)."""
import pytest
import torch

from tests.test_gpu_norm import close, reference, run

pytestmark = pytest.mark.gpu


def far(device, B, C, H, W, groups, spreads, seed, dtype=torch.float32):
    """Groups of unit spread around +-spreads, not the same in every group; exact in f32 up to 2^20."""
    gen = torch.Generator().manual_seed(seed)
    centre = spreads * torch.where(torch.rand(groups, generator=gen) < 0.5, -1.0, 1.0) * (0.75 + 0.25 * torch.rand(groups, generator=gen))
    x = torch.randn(B, H, W, groups, C // groups, generator=gen) + centre[:, None]
    w, b = 1 + 0.3 * torch.randn(C, generator=gen), 0.3 * torch.randn(C, generator=gen)
    gy = torch.randn(B, H, W, C, generator=gen)
    return (x.reshape(B, H, W, C).to(dtype).to(device).permute(0, 3, 1, 2), w.to(device), b.to(device),
            gy.to(dtype).to(device).permute(0, 3, 1, 2))


@pytest.mark.parametrize("log2", [12, 14, 16, 18, 20])
@pytest.mark.parametrize("shape,groups", [((1, 64, 65, 65), 32), ((2, 24, 65, 65), 2), ((1, 7, 129, 131), 1), ((2, 700, 33, 35), 10)], ids=str)
def test_far_means(device, shape, groups, log2):
    x, w, b, gy = far(device, *shape, groups, 2.0 ** log2, 71)
    ref = reference(x, groups, w, b, 1e-5, "identity", gy)
    parts = x.detach().cpu().double().reshape(shape[0], groups, -1)
    mean, rstd = parts.mean(2), 1 / (parts.var(2, unbiased=False) + 1e-5).sqrt()
    off = (2.0 ** -48 * mean.abs() * rstd).repeat_interleave(shape[1] // groups, 1)[:, :, None, None]  # of xh
    wc = w.cpu().double().abs().view(1, -1, 1, 1)
    g64 = gy.cpu().double()
    ref["y_tol"] = ref["y_tol"] + off * wc
    ref["gw_tol"] = ref["gw_tol"] + (off * g64.abs()).sum((0, 2, 3))
    c2 = (wc * g64.abs()).mean() * 4  # |mean of w gz xh| is below that of |w gz| by far; 4 covers |xh|'s mean square root
    rs = rstd.repeat_interleave(shape[1] // groups, 1)[:, :, None, None]
    ref["gx_tol"] = ref["gx_tol"] + 2 * rs * off * c2 * 4
    for v, key in zip(run(x, groups, w, b, 1e-5, "identity", gy), ("y", "gx", "gw", "gb")):
        close(v, ref, key)


def test_statistics_themselves(device):
    """mean and rstd within a few roundings of f64 of 64 bits' two-pass ones (chains of 2^12 terms at most)."""
    from protoseg_amd import norm
    x, w, b, _ = far(device, 2, 64, 65, 65, 8, 2.0 ** 20, 73)
    _, stats = norm.group_norm_forward(x, w, b, 8, 1e-5, 0)
    parts = x.detach().cpu().double().reshape(2, 8, -1)
    centred = parts - parts[:, :, :1]  # exact
    mean = parts[:, :, 0] + centred.mean(2)
    rstd = 1 / (centred.var(2, unbiased=False) + 1e-5).sqrt()
    got = stats.cpu()
    assert bool(((got[..., 0] - mean).abs() <= 2.0 ** -52 * mean.abs() + 2.0 ** -41).all())
    assert bool(((got[..., 1] - rstd).abs() <= 2.0 ** -41 * rstd * 32).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_first_value_far_out(device, dtype):
    """The pivot lies 2^10 spreads from all others: the variance is its doing."""
    x, w, b, gy = far(device, 2, 32, 21, 19, 4, 0.0, 74, dtype)
    x = x.clone(memory_format=torch.preserve_format)
    x[0, ::8, 0, 0] = 1024.0
    ref = reference(x, 4, w, b, 1e-5, "identity", gy)
    for v, key in zip(run(x, 4, w, b, 1e-5, "identity", gy), ("y", "gx", "gw", "gb")):
        close(v, ref, key)

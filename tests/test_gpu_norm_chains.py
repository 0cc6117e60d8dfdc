"""Group norm's backward where a workgroup's sums are longest: 2^18 elements, whose threads add up 1024 / V values each (V
channels a vector) and whose 256 rows are joined one after the other. float64 on the GPU; the bound is that of f32 chains
of n values, n u sum |value| with u = 2^-24, which sums in 64 bits keep far below."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("shape,dtype,vector", [((512, 1, 512, 512), torch.bfloat16, 1), ((128, 4, 512, 512), torch.float32, 4),
                                                ((171, 3, 512, 512), torch.float32, 1)], ids=str)
def test_longest_chains(device, shape, dtype, vector):
    from protoseg_amd import norm
    B, C, H, W = shape
    gen = torch.Generator(device=device).manual_seed(5)
    x = torch.randn(B, H, W, C, generator=gen, device=device).to(dtype).permute(0, 3, 1, 2)
    gy = (torch.randn(B, H, W, C, generator=gen, device=device) + 0.25).to(dtype).permute(0, 3, 1, 2)
    w = 1 + 0.3 * torch.randn(C, generator=gen, device=device)
    y, stats = norm.group_norm_forward(x, w, None, C, 1e-5, 0)
    gx, gw, gb = norm.group_norm_backward(x, gy, w, None, stats, C, 0)

    chain = 1024 // vector + 256 + 8  # and the value's own roundings
    mean = torch.stack([p.double().mean((2, 3)) for p in x.split(32)]).reshape(-1, C) if B % 32 == 0 else x.double().mean((2, 3))
    want_w, want_b, tol_w, tol_b = (torch.zeros(C, dtype=torch.float64, device=device) for _ in range(4))
    for k in range(0, B, 16):
        xk, gk = x[k:k + 16].double(), gy[k:k + 16].double()
        d = xk - mean[k:k + 16, :, None, None]
        rstd = 1 / (d.square().mean((2, 3), keepdim=True) + 1e-5).sqrt()
        xh = d * rstd
        want_w += (gk * xh).sum((0, 2, 3))
        want_b += gk.sum((0, 2, 3))
        tol_w += chain * U * (gk * xh).abs().sum((0, 2, 3))
        tol_b += chain * U * gk.abs().sum((0, 2, 3))
        # a channel is a group: g_x = rstd w (gy - mean(gy) - xh mean(gy xh))
        wk = w.double().view(1, C, 1, 1)
        c1, c2 = gk.mean((2, 3), keepdim=True), (gk * xh).mean((2, 3), keepdim=True)
        ref = rstd * wk * (gk - c1 - xh * c2)
        e1, e2 = (chain * U * v.abs().mean((2, 3), keepdim=True) for v in (gk, gk * xh))
        tol = torch.finfo(dtype).eps / 2 * ref.abs() + rstd * wk.abs() * (
            4 * U * gk.abs() + e1 + xh.abs() * e2 + 6 * U * (gk.abs() + c1.abs() + xh.abs() * c2.abs())) + 2.0 ** -126
        assert bool(((gx[k:k + 16].double() - ref).abs() <= tol).all())
        fwd = wk * xh
        assert bool(((y[k:k + 16].double() - fwd).abs() <= torch.finfo(dtype).eps / 2 * fwd.abs() + 5.5 * U * fwd.abs() + 2.0 ** -126).all())
    assert bool(((gw.double() - want_w).abs() <= tol_w + U * want_w.abs()).all())
    assert bool(((gb.double() - want_b).abs() <= tol_b + U * want_b.abs()).all())

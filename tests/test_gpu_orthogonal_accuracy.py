"""The orthogonalisation and the Muon step against 64 bits, beside the error of the same formula in f32 products.

How many times that error a result may have: an operand held as a pair of f16 values (hi, lo of 11 bits each) is
off by 1.5 times an f32's rounding in the root mean square (lo lies in its top binade half of the time, with a step
of 2^-22, in the next one a quarter, ...; 2 times at most), and the dropped lo lo products are as large again:
sqrt(1.5^2 + 1.5^2) = 2.1 where nothing else errs, below 64 rows. The MFMA rounds twice in 16 products
where an f32 chain rounds 16 times, so from sums of 64 terms on a result has no more than the formula's own error.
1.25 times each for the sampling: errors are sums of some thousand roundings of the same size.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
PAIRS, SAMPLING = 2.1, 1.25


def newton_schulz(g, dtype, steps=5, eps=1e-7):
    """The formula in ``dtype`` products on the GPU, matrices [count, rows, cols]."""
    a, b, c = NS
    x = g.to(dtype)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + eps)
    for _ in range(steps):
        s = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    return x.transpose(1, 2) if tall else x


def noise(device, shape, seed):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, generator=gen, device=device)


def times(shape):
    return (PAIRS if min(shape[-2:]) < 64 else 1.0) * SAMPLING


def error(got, want):
    return torch.linalg.vector_norm(got.double() - want).item()


SHAPES = [(24, 8, 8), (24, 8, 2000), (24, 16, 512), (24, 32, 32), (12, 32, 2000), (24, 48, 60), (24, 64, 64), (24, 64, 128), (24, 361, 64),
          (12, 96, 96), (12, 96, 160), (12, 128, 128), (8, 300, 257), (8, 256, 1024), (1, 2000, 512), (2, 512, 512), (1, 64, 18432)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_f32_results(device, shape):
    from protoseg_amd import optim
    g = noise(device, shape, 3)
    got, want, plain = optim.orthogonalize(g), newton_schulz(g, torch.float64), newton_schulz(g, torch.float32)
    assert error(got, want) <= times(shape) * error(plain, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(64, 64, 64), (64, 64, 128), (64, 361, 64), (24, 96, 96), (24, 256, 1024), (8, 512, 513)], ids=str)
def test_16_bit_results_round_as_often_to_the_other_side(device, dtype, shape):
    """A result is off from the rounding of the 64-bit one where its error crosses a rounding border, which is
    as rare as the error is small. Some 10^3 crossings at least: their number varies by 3 %."""
    from protoseg_amd import optim
    g = noise(device, shape, 4).to(dtype)
    want, plain = newton_schulz(g, torch.float64).to(dtype), newton_schulz(g, torch.float32).to(dtype)
    crossed, plain_crossed = int((optim.orthogonalize(g) != want).sum()), int((plain != want).sum())
    assert crossed <= times(shape) * plain_crossed


@pytest.mark.parametrize("shapes", [((64, 64),) * 24, ((64, 128),) * 24, ((361, 64),) * 12, ((96, 200),) * 8, ((256, 1024),) * 4,
                                    ((64, 128),) * 8 + ((300, 257),) * 2 + ((64, 600),) * 4, ((16, 300),) * 24], ids=str)
def test_an_update_from_zero(device, shapes):
    """Parameters and momentum that start at zero: the step is the update alone."""
    from protoseg_amd import optim
    ps = [torch.nn.Parameter(torch.zeros(s, device=device)) for s in shapes]
    for k, p in enumerate(ps):
        p.grad = noise(device, p.shape, 50 + k)
    optim.Muon(ps, lr=1.0, momentum=0.5, nesterov=False).step()
    got = want = plain = 0.0
    for p in ps:
        scale = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        exact = -scale * newton_schulz(p.grad[None], torch.float64)[0]
        got += error(p.detach(), exact) ** 2
        plain += error(-scale * newton_schulz(p.grad[None], torch.float32)[0], exact) ** 2
    limit = max(times(s) for s in shapes)
    assert got <= limit ** 2 * plain


@pytest.mark.parametrize("shape", [(2, 65, 129), (3, 129, 65), (2, 100, 257), (1, 1, 900), (2, 63, 385), (2, 257, 130), (1, 700, 900),
                                   (1, 40, 3001), (30, 130, 201), (100, 257, 130)], ids=str)
def test_every_element_and_the_last_row_and_column(device, shape):
    """No element is off by more than the largest errors of the formula: errors are about normal, so the largest of
    n lies near sqrt(2 ln n) <= 6 deviations for both; the last row and column hold the sizes' remainders. A wrong or
    unwritten element is off by 10^4 times as much."""
    from protoseg_amd import optim
    g = noise(device, shape, 5)
    want = newton_schulz(g, torch.float64)
    off, plain = (optim.orthogonalize(g).double() - want).abs(), (newton_schulz(g, torch.float32).double() - want).abs()
    deviation = plain.square().mean().sqrt().item()
    assert off.max().item() <= 6 * times(shape) * deviation
    for part in (off[:, -1], off[:, :, -1]):
        assert part.max().item() <= 6 * times(shape) * deviation

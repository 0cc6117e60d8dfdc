"""Group norm with an activation (protoseg_group_norm_fwd / _bwd, norm.py) against the definition in
float64 on the CPU.

Tolerances, per element (u = 2^-24, one f32 rounding). Statistics are f64 sums of exact inputs: no
error of their own. Forward: t = (x - mean) rstd w takes 4 roundings and z = t + b one more, so
|dz| <= 5 u (|t| + |b|); every activation's slope is at most 1.1; sigmoid adds a relative
2 u (|z| + 3) (exponent's argument, v_exp, v_rcp, sum), silu one rounding more; the result is rounded
by at most half a step of its type. Backward: gz carries |gy| (the activation's error above, doubled
for s (1 - s) and s (1 + z (1 - s))); a sum of gz over n values in f32 chains of at most CHAIN errs by
CHAIN u sum |gz|; g_x adds up three such terms."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CHAIN = 400  # pixels a thread adds up, plus the rows joined in a workgroup (at most 256), plus the formula's own
ACTS = ("identity", "relu", "sigmoid", "silu")
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def act64(z, act):
    return {"identity": lambda t: t, "relu": torch.relu, "sigmoid": torch.sigmoid, "silu": lambda t: t * torch.sigmoid(t)}[act](z)


def reference(x, groups, w, b, eps, act, gy=None):
    """Everything of the definition in float64 on the CPU, and the error bounds of y, gx, gw, gb."""
    dt = x.dtype
    half, tiny = torch.finfo(dt).eps / 2, SMALLEST[dt]
    x = x.detach().cpu().double().contiguous()
    B, C, H, W = x.shape
    w64 = torch.ones(C, dtype=torch.float64) if w is None else w.detach().cpu().double()
    b64 = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().cpu().double()
    xs = x.clone().requires_grad_(True)
    ws, bs = w64.clone().requires_grad_(True), b64.clone().requires_grad_(True)
    parts = xs.reshape(B, groups, -1)
    mean, var = parts.mean(2, keepdim=True), parts.var(2, unbiased=False, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    xh = ((parts - mean) * rstd).reshape(x.shape)
    t = xh * ws.view(1, -1, 1, 1)
    z = t + bs.view(1, -1, 1, 1)
    y = act64(z, act)
    size = (t.abs() + b64.abs().view(1, -1, 1, 1)).detach()
    zd, yd, xh = z.detach(), y.detach(), xh.detach()
    extra = 2 * U * (zd.abs() + 4) if act in ("sigmoid", "silu") else 0.0
    out = {"y": yd, "y_tol": half * yd.abs() + tiny + 1.1 * 5 * U * size + extra * yd.abs()}
    if gy is None:
        return out
    gy = gy.detach().cpu().double().contiguous()
    gx, gw, gb = torch.autograd.grad(y, (xs, ws, bs), gy)
    zr = zd.clone().requires_grad_(True)
    gz, = torch.autograd.grad(act64(zr, act), zr, gy)
    gz_err = gy.abs() * (2 * U * (zd.abs() + 4) * 2 + 5 * U * size * (0.5 if act in ("sigmoid", "silu") else 0.0))
    if act == "identity":
        gz_err = gz_err * 0
    rs = rstd.detach().expand(-1, -1, C // groups).reshape(B, C, 1, 1)
    wc = w64.abs().view(1, -1, 1, 1)
    M = H * W * (C // groups)

    def over_group(v):
        return v.reshape(B, groups, -1).sum(2, keepdim=True).expand(-1, -1, C // groups).reshape(B, C, 1, 1) / M

    e1 = over_group(wc * (gz_err + CHAIN * U * gz.abs()))
    e2 = over_group(wc * xh.abs() * (gz_err + CHAIN * U * gz.abs()))
    c1 = over_group(w64.view(1, -1, 1, 1) * gz).abs()
    c2 = over_group(w64.view(1, -1, 1, 1) * gz * xh).abs()
    gx_tol = half * gx.abs() + tiny + rs * (wc * (gz_err + 4 * U * gz.abs()) + e1 + xh.abs() * e2
                                            + 6 * U * (wc * gz.abs() + c1 + xh.abs() * c2))
    out.update(gx=gx, gw=gw, gb=gb, gx_tol=gx_tol,
               gw_tol=((gz_err + CHAIN * U * gz.abs()) * xh.abs()).sum((0, 2, 3)) + U * gw.abs() + 1e-30,
               gb_tol=(gz_err + CHAIN * U * gz.abs()).sum((0, 2, 3)) + U * gb.abs() + 1e-30)
    return out


def close(got, ref, key):
    err = (got.detach().cpu().double() - ref[key]).abs()
    bad = ~(err <= ref[key + "_tol"])
    assert not bool(bad.any()), f"{key}: {int(bad.sum())} of {bad.numel()} off, worst {err[bad].max():.3e}"


def make(device, B, C, H, W, dtype, seed, mean=1.0, layout="cl"):
    gen = torch.Generator().manual_seed(seed)
    spread = torch.rand(C, generator=gen) + 0.5
    centre = mean * torch.randn(C, generator=gen)
    x = (torch.randn(B, H, W, C, generator=gen) * spread + centre).to(dtype)
    w, b = 1 + 0.3 * torch.randn(C, generator=gen), 0.3 * torch.randn(C, generator=gen)
    gy = torch.randn(B, H, W, C, generator=gen).to(dtype)
    x, gy = x.to(device), gy.to(device)

    def lay(t):
        if layout == "cl":
            return t.permute(0, 3, 1, 2)
        if layout == "nchw":
            return t.permute(0, 3, 1, 2).contiguous()
        pad = {"slice": 8, "odd": 1}[layout]  # channels `pad` to `pad` + C of a wider map
        wide = torch.full((B, H, W, C + 2 * pad), float("nan"), dtype=t.dtype, device=device)
        wide[..., pad:pad + C] = t
        return wide.permute(0, 3, 1, 2)[:, pad:pad + C]

    return lay(x), w.to(device), b.to(device), lay(gy)


def run(x, groups, w, b, eps, act, gy):
    from protoseg_amd import norm
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = norm.group_norm(args[0], groups, args[1], args[2], eps, act)
    return (y, *torch.autograd.grad(y, leaves, gy))


SHAPES = [  # B, C, H, W, groups
    (2, 64, 13, 11, 32), (1, 64, 1, 1, 32), (1, 64, 1, 1, 64), (3, 150, 7, 5, 6), (1, 1, 5, 3, 1), (2, 7, 9, 4, 7), (1, 2048, 9, 11, 32),
    (2, 2056, 3, 3, 8), (4, 320, 12, 10, 1), (1, 190, 33, 31, 19), (1, 4099, 2, 2, 1), (5, 24, 1, 40, 6), (2, 64, 65, 65, 32), (2, 8, 129, 127, 2),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(device, shape, dtype):
    B, C, H, W, groups = shape
    act = ACTS[(C + H + (dtype == torch.float32)) % 4]
    x, w, b, gy = make(device, B, C, H, W, dtype, 7)
    y, gx, gw, gb = run(x, groups, w, b, 1e-5, act, gy)
    assert y.dtype == dtype and gx.dtype == dtype and y.shape == x.shape
    assert y.is_contiguous(memory_format=torch.channels_last) and gw.dtype == gb.dtype == torch.float32
    ref = reference(x, groups, w, b, 1e-5, act, gy)
    for got, key in ((y, "y"), (gx, "gx"), (gw, "gw"), (gb, "gb")):
        close(got, ref, key)


@pytest.mark.parametrize("shape,dtype,act", [((2, 64, 271, 263), torch.float32, "silu"), ((1, 512, 181, 189), torch.bfloat16, "relu"),
                                             ((1, 516, 181, 189), torch.float16, "identity")], ids=str)
def test_maps_beyond_the_caches(device, shape, dtype, act):
    """Results of more than 32 MiB, in 16-B vectors and (516 halves) in 4-B ones."""
    x, w, b, gy = make(device, *shape, dtype, 19)
    assert x.numel() * x.element_size() > 32 << 20
    got = run(x, 4, w, b, 1e-5, act, gy)
    ref = reference(x, 4, w, b, 1e-5, act, gy)
    for v, key in zip(got, ("y", "gx", "gw", "gb")):
        close(v, ref, key)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("layout", ["cl", "nchw", "slice", "odd"])
def test_layouts_and_activations(device, layout, act):
    x, w, b, gy = make(device, 3, 48, 17, 9, torch.bfloat16, 11, layout=layout)
    got = run(x, 12, w, b, 1e-5, act, gy)
    ref = reference(x, 12, w, b, 1e-5, act, gy)
    for v, key in zip(got, ("y", "gx", "gw", "gb")):
        close(v, ref, key)


def test_every_second_sample_and_broadcast_gradient(device):
    x, w, b, _ = make(device, 6, 32, 8, 8, torch.float32, 13)
    gy = torch.ones((), device=device).expand(3, 32, 8, 8)
    got = run(x[::2], 8, w, b, 1e-5, "silu", gy)
    ref = reference(x[::2], 8, w, b, 1e-5, "silu", gy)
    for v, key in zip(got, ("y", "gx", "gw", "gb")):
        close(v, ref, key)


def test_strided_pixels_are_copied(device):
    """Every second column: no single pixel stride, so the map is copied first."""
    x, w, b, gy = make(device, 2, 16, 6, 10, torch.float32, 17)
    xs, gs = x[..., ::2], gy[..., ::2]
    ref = reference(xs, 4, w, b, 1e-5, "relu", gs)
    for v, key in zip(run(xs, 4, w, b, 1e-5, "relu", gs), ("y", "gx", "gw", "gb")):
        close(v, ref, key)


@pytest.mark.parametrize("which", ["weight", "bias", "none"])
def test_without_weight_or_bias(device, which):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 40, 9, 9, torch.float32, 19)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    ref = reference(x, 5, w, b, 1e-5, "sigmoid", gy)
    got = run(x, 5, w, b, 1e-5, "sigmoid", gy)
    close(got[0], ref, "y")
    close(got[1], ref, "gx")
    if which != "none":
        close(got[2], ref, "gw" if which == "weight" else "gb")
    # a gradient of the weight alone: no g_x is written
    if which == "weight":
        wl = w.clone().requires_grad_(True)
        gw, = torch.autograd.grad(norm.group_norm(x, 5, wl, None, 1e-5, "sigmoid"), wl, gy)
        close(gw, ref, "gw")


def test_map_beyond_32_bit_offsets(device):
    """2.2e9 elements (bf16): statistics from f64 sums of slabs, y and the gradients at the far end."""
    from protoseg_amd import norm
    C, H, W, groups = 64, 5860, 5860, 8
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.empty((1, H, W, C), dtype=torch.bfloat16, device=device)
    for part in x[0].chunk(20):
        part.copy_(torch.randn(part.shape, generator=gen, device=device) + 0.5)
    x = x.permute(0, 3, 1, 2)
    assert x.numel() > 2 ** 31
    y, stats = norm.group_norm_forward(x, None, None, groups, 1e-5, 2)
    total = sum(p.double().reshape(-1, groups, C // groups).sum((0, 2)) for p in x[0].permute(1, 2, 0).chunk(20))
    square = sum(p.double().square().reshape(-1, groups, C // groups).sum((0, 2)) for p in x[0].permute(1, 2, 0).chunk(20))
    M = H * W * (C // groups)
    mean, var = total / M, square / M - (total / M) ** 2
    rstd = 1 / (var + 1e-5).sqrt()
    assert torch.allclose(stats[0, :, 0], mean, rtol=1e-12, atol=0) and torch.allclose(stats[0, :, 1], rstd, rtol=1e-12, atol=0)
    m, r = (v.repeat_interleave(C // groups) for v in (mean, rstd))
    last = (x[0, :, -3:].double().permute(1, 2, 0) - m) * r
    ref = torch.sigmoid(last)
    err = (y[0, :, -3:].double().permute(1, 2, 0) - ref).abs()
    # half a step of bf16: finfo.eps = 2^-7 between 1 and 2, so 2^-8 of the value
    assert bool((err <= (2.0 ** -8 + 4 * U * (last.abs() + 4)) * ref).all())
    gx, gw, gb = norm.group_norm_backward(x, y, None, None, stats, groups, 2)
    # gb of y itself: sum of y * y (1 - y) with the f64 sigmoid of z; every term is positive
    want = torch.zeros(C, dtype=torch.float64, device=device)
    for px, py in zip(x[0].permute(1, 2, 0).chunk(40), y[0].permute(1, 2, 0).chunk(40)):
        s = torch.sigmoid((px.double() - m) * r)
        want += (py.double() * s * (1 - s)).sum((0, 1))
    assert bool(((gb.double() - want).abs() <= 3 * CHAIN * U * want).all())
    assert bool(torch.isfinite(gx[0, :, -1]).all()) and bool((gx[0, :, -1] != 0).any())


def test_mean_far_larger_than_the_spread(device):
    """|mean| about 3000 spreads in f32: the statistics and x - mean keep full precision."""
    x, w, b, gy = make(device, 2, 32, 21, 19, torch.float32, 23, mean=3000.0)
    ref = reference(x, 32, w, b, 1e-5, "identity", gy)  # groups of one channel: the mean is the channel's
    for v, key in zip(run(x, 32, w, b, 1e-5, "identity", gy), ("y", "gx", "gw", "gb")):
        close(v, ref, key)


def test_constant_group_and_zero_eps(device):
    x = torch.full((1, 8, 4, 4), 3.0, device=device).contiguous(memory_format=torch.channels_last)
    from protoseg_amd import norm
    assert torch.equal(norm.group_norm(x, 2), torch.zeros_like(x))
    assert bool(torch.isnan(norm.group_norm(x, 2, eps=0.0)).all())  # 0 / 0, as the formula says


def test_not_finite_values_stay_in_their_group(device):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 32, 6, 6, torch.float32, 29)
    x = x.clone()
    x[0, 3, 2, 2] = float("nan")
    x[1, 30, 0, 0] = float("inf")
    y = norm.group_norm(x, 8, w, b)
    bad = torch.zeros(2, 8, dtype=torch.bool, device=device)
    bad[0, 0] = bad[1, 7] = True
    nan = torch.isnan(y).reshape(2, 8, -1)
    assert bool(nan[bad].all()) and not bool(nan[~bad].any())


def test_empty_maps(device):
    from protoseg_amd import norm
    for shape in ((0, 16, 4, 4), (2, 16, 0, 4), (2, 16, 4, 0)):
        x = torch.empty(shape, device=device, requires_grad=True)
        w = torch.ones(16, device=device, requires_grad=True)
        b = torch.zeros(16, device=device, requires_grad=True)
        y = norm.group_norm(x, 4, w, b, activation="silu")
        assert y.shape == x.shape
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any())


def test_same_bits_every_run(device):
    x, w, b, gy = make(device, 2, 64, 65, 65, torch.bfloat16, 31)
    first = run(x, 32, w, b, 1e-5, "relu", gy)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, run(x, 32, w, b, 1e-5, "relu", gy)))


def test_gradient_against_differences(device):
    """<g, v> against (L(x + h v) - L(x - h v)) / 2h in f32, L = <gy, y> summed in f64: the quotient's
    rounding is at most 2 * 6 u sum|gy| (|z| + 1) / 2h, its cut-off h^2 / 6 times a third derivative
    of order sum |gy| / n^(3/2)-directions (v has unit entries): h = 2^-6 keeps both below the bound."""
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 12, 8, 8, torch.float32, 37)
    _, gx, gw, gb = run(x, 3, w, b, 1e-5, "silu", gy)
    gen = torch.Generator().manual_seed(5)
    h = 2.0 ** -6
    for k, (t, g) in enumerate(((x, gx), (w, gw), (b, gb))):
        v = torch.randint(0, 2, t.shape, generator=gen).float().mul(2).sub(1).to(device)

        def loss(sign):
            a = [x, w, b]
            a[k] = t + sign * h * v
            return (gy.double() * norm.group_norm(a[0], 3, a[1], a[2], 1e-5, "silu").double()).sum()

        quotient = ((loss(1) - loss(-1)) / (2 * h)).item()
        exact = (g.double() * v.double()).sum().item()
        z = 4.0  # |z| of these inputs stays below 4 spreads but for a few
        bound = 6 * U * gy.abs().sum().item() * (z + 1) / h + h * h * gy.abs().double().sum().item()
        assert abs(quotient - exact) <= bound, (k, quotient, exact, bound)


def test_graph_replays_follow_the_inputs(device):
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 64, 33, 31, torch.bfloat16, 41)
    static = [x.clone(), gy.clone()]

    def step():
        y, stats = norm.group_norm_forward(static[0], w, b, 32, 1e-5, 1)
        return (y, *norm.group_norm_backward(static[0], static[1], w, b, stats, 32, 1, True, True, True))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x2, _, _, gy2 = make(device, 2, 64, 33, 31, torch.bfloat16, 50 + k)
        static[0].copy_(x2)
        static[1].copy_(gy2)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(x2, 32, w, b, 1e-5, "relu", gy2)
        assert all(torch.equal(a, c) for a, c in zip(out, eager))


def test_two_streams_at_once(device):
    x, w, b, gy = make(device, 2, 96, 40, 41, torch.bfloat16, 43)
    x2, _, _, gy2 = make(device, 2, 96, 40, 41, torch.bfloat16, 44)
    want = [run(x, 12, w, b, 1e-5, "silu", gy), run(x2, 12, w, b, 1e-5, "silu", gy2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, args in zip(streams, ((x, gy), (x2, gy2))):
            with torch.cuda.stream(s):
                got.append(run(args[0], 12, w, b, 1e-5, "silu", args[1]))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, c) for a, c in zip(g, want[k % 2]))


def test_module_and_autocast_weights(device):
    """norm.GroupNorm trains; bf16 parameters are widened and get bf16 gradients."""
    from protoseg_amd import norm
    x, w, b, gy = make(device, 2, 24, 10, 10, torch.bfloat16, 47)
    m = norm.GroupNorm(6, 24, activation="relu").to(device).to(torch.bfloat16)
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xl = x.detach().requires_grad_(True)
    m(xl).backward(gy)
    ref = reference(x, 6, m.weight, m.bias, 1e-5, "relu", gy)
    close(xl.grad, ref, "gx")
    assert m.weight.grad.dtype == torch.bfloat16
    ref["gw_tol"] = ref["gw_tol"] + 2.0 ** -8 * ref["gw"].abs()  # narrowed once more
    close(m.weight.grad, ref, "gw")


def test_refusals_on_the_device(device):
    from protoseg_amd import _lib, norm
    leaf = torch.zeros(2, 12, 4, 4, device=device, requires_grad=True)
    with pytest.raises(_lib.ProtosegError, match="second derivative"):
        torch.autograd.grad(norm.group_norm(leaf, 4).sum(), leaf, create_graph=True)
    x = torch.zeros(2, 12, 4, 4, device=device)
    with pytest.raises(_lib.ProtosegError, match="groups"):
        norm.group_norm(x, 5)
    with pytest.raises(_lib.ProtosegError, match="B, C, H, W"):
        norm.group_norm(x[0], 4)
    with pytest.raises(_lib.ProtosegError, match="weight"):
        norm.group_norm(x, 4, torch.ones(11, device=device))
    with pytest.raises(_lib.ProtosegError, match="dtype"):
        norm.group_norm(x.double(), 4)
    with pytest.raises(_lib.ProtosegError, match="no HIP kernel"):
        norm.group_norm(x, 4, activation="tanh")
    with pytest.raises(_lib.ProtosegError, match="eps"):
        norm.group_norm(x, 4, eps=-1.0)
    with pytest.raises(_lib.ProtosegError):
        norm.group_norm(x, 4, torch.ones(12))  # a CPU weight
    lib = _lib.load()
    p, null = ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(None)
    st = lib.protoseg_group_norm_fwd(p, _lib.F32, 2, 16, 12, 192, 12, 4, null, null, 1e-5, 0, p, p, null, 0, null)
    assert st == _lib.ERR_INVALID and b"workspace" in lib.protoseg_last_error()

"""Newton-Schulz orthogonalisation and the Muon step (muon.hip, optim.py) against the definition in float64.

Error bound, in the Frobenius norm. One step X -> f(X) (odd polynomial of the singular values) has the
Lipschitz constant LIP = max |f'| over the values met (below 4 for the coefficients here), and a step rounds
at most ROUNDINGS operands to pairs of f16 (2^-22 of their norm each: X, A, P, T, Q, and the f32 sums, whose
chains of 16-wide products keep below one such unit for the sizes here). An error of relative size e put in
before step k is at most e LIP^(steps - k) |X_k| in the result:
    |X - exact| <= ROUNDINGS 2^-22 sum_k LIP^(steps - k) |X_k|.
A 16-bit result is rounded once more, by at most half a step of its own values."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NS = (3.4445, -4.7750, 2.0315)
ROUNDINGS, LIP = 6, 4.0
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def exact(g, steps=5, coefficients=NS, eps=1e-7):
    """(result, error bound in the Frobenius norm) of one matrix, float64 on the CPU."""
    a, b, c = coefficients
    x = g.detach().cpu().double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (torch.linalg.norm(x) + eps)
    bound = 0.0
    for _ in range(steps):
        bound = LIP * (bound + ROUNDINGS * 2.0 ** -22 * torch.linalg.norm(x).item())
        s = x @ x.T
        x = a * x + (b * s + c * s @ s) @ x
    bound += ROUNDINGS * 2.0 ** -22 * torch.linalg.norm(x).item()
    return (x.T if tall else x), bound


def check(got, g, **kw):
    ref, bound = exact(g, **kw)
    err = torch.linalg.norm(got.detach().cpu().double() - ref).item()
    tiny = 2.0 ** -25 * math.sqrt(got.numel()) if got.dtype == torch.float16 else 0.0
    assert err <= bound + HALF[got.dtype] * torch.linalg.norm(ref).item() + tiny, (tuple(g.shape), err, bound)


def matrix(shape, seed, kind="noise"):
    gen = torch.Generator().manual_seed(seed)
    g = torch.randn(shape, generator=gen)
    r, c = shape[-2:]
    if kind == "spiked":
        g = g + 3 * torch.randn(*shape[:-1], 2, generator=gen) @ torch.randn(*shape[:-2], 2, c, generator=gen)
    if kind == "rank1":
        g = torch.randn(*shape[:-1], 1, generator=gen) @ torch.randn(*shape[:-2], 1, c, generator=gen)
    if kind == "graded":
        k = min(r, c)
        q1, q2 = torch.linalg.qr(torch.randn(r, k, generator=gen))[0], torch.linalg.qr(torch.randn(c, k, generator=gen))[0]
        g = q1 @ torch.diag(torch.logspace(0, -6, k)) @ q2.T
    return g


SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5), (64, 64), (65, 63), (19, 361), (361, 64), (130, 257), (64, 4608), (300, 513), (1152, 128), (256, 1024)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(device, shape, dtype):
    from protoseg_amd import optim
    g = matrix(shape, 1).to(dtype).to(device)
    out = optim.orthogonalize(g)
    assert out.shape == g.shape and out.dtype == dtype and out.is_contiguous()
    check(out, g)


def check_batch(out, g):
    """check() of every matrix of a batch, float64 on the GPU."""
    a, b, c = NS
    x = g.double()
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if tall else x
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + 1e-7)
    norms = lambda t: torch.linalg.vector_norm(t, dim=(1, 2))  # noqa: E731
    bound = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(5):
        bound = LIP * (bound + ROUNDINGS * 2.0 ** -22 * norms(x))
        s = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * s + c * torch.bmm(s, s), x)
    bound += (ROUNDINGS * 2.0 ** -22 + HALF[out.dtype]) * norms(x)
    x = x.transpose(1, 2) if tall else x
    assert bool((norms(out.double() - x) <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    (300, 30, 61),      # one workgroup a matrix
    (1, 64, 384), (1, 385, 64),  # the largest of those, and the first beyond
    (2, 512, 700),      # 32 x 32 tiles, the contraction over the waves
    (1, 64, 18432), (1, 20001, 70),  # the same with a split contraction
    (30, 130, 200),     # 64 x 64 tiles
    (12, 200, 2100), (12, 2100, 200),  # with a split contraction
    (100, 64, 500), (90, 64, 570), (90, 570, 60), (5, 700, 800),  # two halves of a contraction beside each other
    (100, 257, 130), (100, 130, 257),  # 128 x 128 tiles of Q X
], ids=str)
def test_every_kernel_path(device, shape, dtype):
    from protoseg_amd import optim
    gen = torch.Generator(device=device).manual_seed(21)
    g = torch.randn(shape, generator=gen, device=device).to(dtype)
    check_batch(optim.orthogonalize(g), g)


def test_a_matrix_beyond_32_bit_offsets_of_its_neighbours(device):
    """Two matrices 2^31 elements apart in memory, and one of 1.2e8 elements."""
    from protoseg_amd import optim
    far = torch.zeros(2 ** 31 + 70 * 90, dtype=torch.bfloat16, device=device)
    g = far.as_strided((2, 70, 90), (2 ** 31, 90, 1))
    g.copy_(matrix((2, 70, 90), 22).to(torch.bfloat16))
    check_batch(optim.orthogonalize(g), g)
    del far, g
    gen = torch.Generator(device=device).manual_seed(23)
    g = torch.randn((1, 40, 3_000_001), generator=gen, device=device)
    check_batch(optim.orthogonalize(g), g)


@pytest.mark.parametrize("kind", ["spiked", "rank1", "graded"])
@pytest.mark.parametrize("shape", [(96, 200), (200, 96), (128, 128)], ids=str)
def test_conditioning(device, shape, kind):
    from protoseg_amd import optim
    g = matrix(shape, 2, kind).to(device)
    check(optim.orthogonalize(g), g)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 12])
def test_steps(device, steps):
    from protoseg_amd import optim
    g = matrix((70, 150), 3, "spiked").to(device)
    check(optim.orthogonalize(g, steps=steps), g, steps=steps)


@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (3.0, -3.2, 1.2)])
def test_coefficients(device, coefficients):
    from protoseg_amd import optim
    g = matrix((100, 140), 4).to(device)
    check(optim.orthogonalize(g, 6, coefficients), g, steps=6, coefficients=coefficients)


def test_batches_and_strides(device):
    from protoseg_amd import optim
    g = matrix((2, 3, 40, 90), 5).to(device)
    out = optim.orthogonalize(g)
    for i in range(2):
        for k in range(3):
            check(out[i, k], g[i, k])
    flat = g.reshape(6, 40, 90)
    for view in (flat[::2], flat.mT, flat[:, :, :50], flat[:, 3:30], flat[1:2].expand(3, -1, -1), g[0].permute(1, 0, 2)):
        out = optim.orthogonalize(view)
        assert out.shape == view.shape
        for i in range(view.shape[0]):
            check(out[i], view[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("start,apart", [(0, 40 * 64), (0, 40 * 64 + 8), (0, 40 * 64 + 4), (1, 40 * 64 + 3)])
def test_rows_of_any_alignment(device, dtype, start, apart):
    from protoseg_amd import optim
    flat = torch.zeros(start + 2 * apart + 40 * 64, dtype=dtype, device=device)
    g = flat.as_strided((3, 40, 64), (apart, 64, 1), start)
    g.copy_(matrix((3, 40, 64), 25).to(dtype))
    check_batch(optim.orthogonalize(g), g)


def test_matrices_do_not_touch_each_other(device):
    from protoseg_amd import optim
    g = matrix((5, 48, 80), 6).to(device)
    clean = optim.orthogonalize(g)
    g[1] = 0
    g[2, 5, 7] = float("nan")
    g[3, 0, 0] = float("inf")
    out = optim.orthogonalize(g)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[4], clean[4])
    assert not bool(out[1].any()) and bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[3]).all())


@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e25, 1e36])
def test_scale_of_the_input(device, scale):
    from protoseg_amd import optim
    g = (matrix((40, 60), 7) * scale).to(device)
    check(optim.orthogonalize(g), g)


def test_empty(device):
    from protoseg_amd import optim
    for shape in ((0, 4, 5), (3, 0, 5), (0, 5), (4, 0)):
        assert optim.orthogonalize(torch.empty(shape, device=device)).shape == shape


def test_refusals(device):
    from protoseg_amd import _lib, optim
    g = torch.ones(4, 4, device=device)
    for bad, text in ((dict(steps=0), "steps"), (dict(steps=33), "steps"), (dict(coefficients=(9.0, 0.0, 0.0)), "grow"),
                      (dict(coefficients=(float("nan"), 0.0, 0.0)), "coefficients"), (dict(eps=-1.0), "eps")):
        with pytest.raises(_lib.ProtosegError, match=text):
            optim.orthogonalize(g, **bad)
    with pytest.raises(_lib.ProtosegError, match="dtype"):
        optim.orthogonalize(g.double())
    with pytest.raises(_lib.ProtosegError, match="rows, cols"):
        optim.orthogonalize(g[0])
    p = torch.nn.Parameter(torch.zeros(4, 4, device=device, dtype=torch.bfloat16))
    p.grad = torch.ones_like(p)
    with pytest.raises(_lib.ProtosegError, match="float32"):
        optim.Muon([p]).step()
    q = torch.nn.Parameter(torch.zeros(4, 8, device=device)[:, ::2])
    q.grad = torch.ones(4, 4, device=device)
    with pytest.raises(_lib.ProtosegError, match="dense"):
        optim.Muon([q]).step()


def reference_step(p, g, buf, lr, mu, nesterov, wd, scale):
    p64, g64, b64 = (t.detach().cpu().double().reshape(t.shape[0], -1) for t in (p, g, buf))
    nb = mu * b64 + g64
    u = g64 + mu * nb if nesterov else nb
    o, bound = exact(u)
    r, c = u.shape
    s = math.sqrt(max(1.0, r / c)) if scale == "original" else 0.2 * math.sqrt(max(r, c))
    # the update's own roundings (3 u of its norm) pass through five steps; the last line rounds three times
    norm_u = torch.linalg.norm(u).item()
    bound += 3 * U * LIP ** 5 * (1.0 if norm_u else 0.0)
    new = (1 - lr * wd) * p64 - lr * s * o
    tol = lr * s * bound + 4 * U * (torch.linalg.norm(p64).item() + lr * s * torch.linalg.norm(o).item())
    btol = 2 * U * ((mu * b64).abs() + g64.abs())
    return new, tol, nb, btol


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["original", "rms"])
def test_muon_step(device, nesterov, scale):
    from protoseg_amd import optim
    shapes = [(361, 64, 1, 1), (19, 361), (32, 16, 3, 3), (5, 3), (64, 64), (19, 361), (200, 80)]
    gen = torch.Generator().manual_seed(8)
    ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device) * 0.1) for s in shapes]
    ps[2] = torch.nn.Parameter(ps[2].detach().contiguous(memory_format=torch.channels_last))
    opt = optim.Muon(ps, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
    bufs = [torch.zeros_like(p) for p in ps]
    for _ in range(3):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(device)  # contiguous, also where p is channels last
        before = [p.detach().clone() for p in ps]
        opt.step()
        for k, p in enumerate(ps):
            new, tol, nb, btol = reference_step(before[k], p.grad, bufs[k], 0.02, 0.9, nesterov, 0.1, scale)
            got = p.detach().cpu().double().reshape(new.shape)
            assert torch.linalg.norm(got - new).item() <= tol, (k, shapes[k])
            buf = opt.state[p]["momentum_buffer"]
            assert bool(((buf.cpu().double().reshape(nb.shape) - nb).abs() <= btol).all())
            bufs[k] = buf.clone()


def test_muon_more_shapes_than_one_run_and_missing_gradients(device):
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(9)
    ps = [torch.nn.Parameter(torch.randn(4 + k, 6 + 2 * k, generator=gen).to(device)) for k in range(50)]
    ps.append(torch.nn.Parameter(torch.zeros(0, 5, device=device)))
    ps[-1].grad = torch.zeros(0, 5, device=device)
    opt = optim.Muon(ps, lr=0.1)
    for k, p in enumerate(ps[:-1]):
        if k % 7:
            p.grad = torch.randn(p.shape, generator=gen).to(device)
    before = [p.detach().clone() for p in ps]
    opt.step()
    for k, p in enumerate(ps[:-1]):
        if k % 7 == 0:
            assert torch.equal(p, before[k])
            continue
        new, tol, _, _ = reference_step(before[k], p.grad, torch.zeros_like(p), 0.1, 0.95, True, 0.0, "original")
        assert torch.linalg.norm(p.detach().cpu().double() - new).item() <= tol


def test_muon_neighbours_in_a_flat_buffer_stay(device):
    from protoseg_amd import optim
    flat = torch.full((64 * 70 + 128,), 7.0, device=device)
    p = torch.nn.Parameter(flat[64:64 + 64 * 70].view(64, 70))
    p.grad = matrix((64, 70), 10).to(device)
    optim.Muon([p], lr=0.5).step()
    assert bool((flat[:64] == 7).all()) and bool((flat[-64:] == 7).all()) and not bool((p == 7).any())


def test_muon_state_round_trip(device):
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(11)
    grads = [torch.randn(30, 50, generator=gen).to(device) for _ in range(4)]
    a = torch.nn.Parameter(torch.randn(30, 50, generator=gen).to(device))
    b = torch.nn.Parameter(a.detach().clone())
    opt_a = optim.Muon([a])
    opt_b = optim.Muon([b])
    for g in grads[:2]:
        a.grad = g
        opt_a.step()
    opt_b.load_state_dict(copy.deepcopy(opt_a.state_dict()))
    with torch.no_grad():
        b.copy_(a)
    for g in grads[2:]:
        a.grad = b.grad = g
        opt_a.step()
        opt_b.step()
    assert torch.equal(a, b)


def test_graph_replays_are_successive_steps(device):
    """Two captured steps with workspaces of their own, replayed in turn with eager work between."""
    from protoseg_amd import optim
    gen = torch.Generator().manual_seed(12)
    made = []
    for k in range(2):
        ps = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device)) for s in ((96, 130), (361, 64), (19, 361))]
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(device)
        opt = optim.Muon(ps, lr=0.01)
        opt.step()
        twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        opt_t = optim.Muon(twin, lr=0.01)
        for p, t in zip(ps, twin):
            t.grad = p.grad.clone()
            opt_t.state[t]["momentum_buffer"] = opt.state[p]["momentum_buffer"].clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            opt.step()
        made.append((graph, ps, opt_t, twin, opt))  # opt: its momentum buffers have to outlive the graph
    for _ in range(3):
        for graph, ps, opt_t, twin, _ in made:
            for p, t in zip(ps, twin):
                g = torch.randn(p.shape, generator=gen).to(device)
                p.grad.copy_(g)
                t.grad.copy_(g)
            graph.replay()
            opt_t.step()
        torch.cuda.synchronize()
        for _, ps, _, twin, _ in made:
            assert all(torch.equal(p, t) for p, t in zip(ps, twin))


def test_two_streams_at_once_and_same_bits(device):
    from protoseg_amd import optim
    gs = [matrix((3, 128, 300), 13).to(device), matrix((3, 300, 128), 14).to(device)]
    want = [optim.orthogonalize(g) for g in gs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(3):
        for s, g in zip(streams, gs):
            with torch.cuda.stream(s):
                got.append(optim.orthogonalize(g))
    torch.cuda.synchronize()
    for k, o in enumerate(got):
        assert torch.equal(o, want[k % 2])


def test_a_step_is_seen_by_autograd(device):
    """Parameters are changed in place: a graph that saved their old values refuses its backward."""
    from protoseg_amd import optim
    p = torch.nn.Parameter(matrix((20, 30), 41).to(device))
    x = torch.ones(30, device=device, requires_grad=True)
    opt = optim.Muon([p])
    y = (p * p) @ x
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_first_step_is_not_captured(device):
    from protoseg_amd import _lib, optim
    p = torch.nn.Parameter(matrix((20, 30), 42).to(device))
    p.grad = torch.ones_like(p)
    opt = optim.Muon([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(_lib.ProtosegError, match="one step before"):
        with torch.cuda.graph(graph):
            p.grad.add_(0)
            opt.step()
    opt.step()

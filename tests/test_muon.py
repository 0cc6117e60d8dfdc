"""CPU: refusals and host logic of the orthogonalisation and of Muon (no GPU call is made)."""
import ctypes

import pytest
import torch

from protoseg_amd import _lib, optim

NULL, SOME = ctypes.c_void_p(None), ctypes.c_void_p(4096)
NS = optim.NS_COEFFICIENTS


def orth(g=SOME, dtype=0, count=1, rows=100, cols=200, stride=20000, steps=5, abc=NS, eps=1e-7, out=SOME, ws=NULL, nbytes=0):
    return _lib.load().protoseg_orthogonalize(g, dtype, count, rows, cols, stride, steps, *abc, eps, out, ws, nbytes, NULL)


@pytest.mark.parametrize("bad, status, text", [
    (dict(dtype=2), _lib.ERR_UNSUPPORTED, b"dtype"),
    (dict(count=-1), _lib.ERR_INVALID, b"-1 matrices"),
    (dict(rows=-2), _lib.ERR_INVALID, b"-2 x 200"),
    (dict(rows=40000, cols=40000), _lib.ERR_UNSUPPORTED, b"at most"),
    (dict(rows=17000, cols=17000), _lib.ERR_UNSUPPORTED, b"at most"),
    (dict(steps=0), _lib.ERR_INVALID, b"steps"),
    (dict(steps=33), _lib.ERR_INVALID, b"steps"),
    (dict(abc=(4.5, 0.0, 0.0)), _lib.ERR_UNSUPPORTED, b"grow"),
    (dict(abc=(2.0, 0.5, 0.0)), _lib.ERR_UNSUPPORTED, b"grow"),
    (dict(abc=(float("inf"), 0.0, 0.0)), _lib.ERR_INVALID, b"coefficients"),
    (dict(eps=float("nan")), _lib.ERR_INVALID, b"eps"),
    (dict(g=NULL), _lib.ERR_INVALID, b"non-null"),
    (dict(out=NULL), _lib.ERR_INVALID, b"non-null"),
    (dict(count=2, stride=19999), _lib.ERR_INVALID, b"overlap"),
    (dict(), _lib.ERR_INVALID, b"workspace"),
])
def test_orthogonalize_refusals(bad, status, text):
    assert orth(**bad) == status
    assert text in _lib.load().protoseg_last_error()


def test_empty_calls_need_nothing():
    for empty in (dict(count=0), dict(rows=0), dict(cols=0)):
        assert orth(g=NULL, out=NULL, **empty) == _lib.OK
    lib = _lib.load()
    assert lib.protoseg_orthogonalize_workspace_size(0, 4, 4) == 0
    assert lib.protoseg_muon_step(0, None, None, None, None, None, 0.9, 1, 0.1, 0.0, 0, 5, *NS, 1e-7, NULL, 0, NULL) == _lib.OK


def test_muon_refusals():
    lib = _lib.load()

    def step(n=1, mu=0.9, eps=1e-7, kind=0, steps=5, rows=100, null=False):
        ptrs = (ctypes.c_void_p * 1)(None if null else 4096)
        r, c = (ctypes.c_int32 * 1)(rows), (ctypes.c_int32 * 1)(200)
        return lib.protoseg_muon_step(n, ptrs, ptrs, ptrs, r, c, mu, 1, 0.1, 0.0, kind, steps, *NS, eps, NULL, 0, NULL)

    for bad, text in ((dict(n=-1), b"-1 tensors"), (dict(mu=1.0), b"momentum"), (dict(eps=-1.0), b"eps"), (dict(kind=2), b"scale"),
                      (dict(steps=0), b"steps"), (dict(rows=-1), b"-1 x 200"), (dict(null=True), b"null pointer"), (dict(), b"workspace")):
        assert step(**bad) == _lib.ERR_INVALID and text in lib.protoseg_last_error(), bad


def test_workspace_covers_every_run_of_shapes():
    lib = _lib.load()
    n = 60
    rows, cols = (ctypes.c_int32 * n)(*range(80, 80 + n)), (ctypes.c_int32 * n)(*range(90, 90 + n))
    whole = lib.protoseg_muon_workspace_size(n, rows, cols)
    first = lib.protoseg_muon_workspace_size(24, rows, cols)
    assert 0 < first <= whole and whole % 256 == 0
    # matrices that one workgroup takes whole need none
    assert lib.protoseg_orthogonalize_workspace_size(7, 361, 64) == 0 < lib.protoseg_orthogonalize_workspace_size(7, 385, 64)
    small_r, small_c = (ctypes.c_int32 * 2)(361, 19), (ctypes.c_int32 * 2)(64, 361)
    assert lib.protoseg_muon_workspace_size(2, small_r, small_c) == 0


def test_python_refusals():
    with pytest.raises(_lib.ProtosegError, match="CPU|cpu"):
        optim.orthogonalize(torch.ones(3, 4))
    with pytest.raises(ValueError, match="matrices"):
        optim.Muon([torch.nn.Parameter(torch.zeros(4))])
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(scale="adam")):
        with pytest.raises(ValueError, match="hyper-parameters"):
            optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))], **bad)
    p = torch.nn.Parameter(torch.zeros(4, 4))
    p.grad = torch.ones(4, 4)
    with pytest.raises(_lib.ProtosegError, match="CPU|cpu"):
        optim.Muon([p]).step()


def test_which_layouts_are_rows():
    assert optim._dense_rows(torch.zeros(4, 6))
    assert optim._dense_rows(torch.zeros(4, 3, 2, 2).contiguous(memory_format=torch.channels_last))
    assert optim._dense_rows(torch.zeros(1, 3, 2, 2))
    assert not optim._dense_rows(torch.zeros(6, 4).t())
    assert not optim._dense_rows(torch.zeros(4, 8)[:, ::2])
    assert not optim._dense_rows(torch.zeros(8, 4)[::2])


def test_a_group_is_checked_as_it_is_added():
    from protoseg_amd import optim
    p, q = torch.nn.Parameter(torch.zeros(4, 3)), torch.nn.Parameter(torch.zeros(2, 5))
    opt = optim.Muon([p])
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        opt.add_param_group({"params": [q, q]})
    with pytest.raises(ValueError, match=r"\(7,\)"):
        opt.add_param_group({"params": [q, torch.nn.Parameter(torch.zeros(7))]})
    with pytest.raises(ValueError):
        opt.add_param_group({"params": p})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": q, "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [2e-2, 0.5]


def test_a_tensor_twice_in_a_call_is_refused():
    lib = _lib.load()
    size, other = (ctypes.c_int32 * 2)(100, 100), (ctypes.c_int32 * 2)(200, 200)
    once, twice = (ctypes.c_void_p * 2)(4096, 8192), (ctypes.c_void_p * 2)(4096, 4096)
    for params, bufs in ((twice, once), (once, twice)):
        assert lib.protoseg_muon_step(2, params, once, bufs, size, other, 0.9, 1, 0.1, 0.0, 0, 5, *NS, 1e-7, NULL, 0,
                                      NULL) == _lib.ERR_INVALID
        assert b"twice" in lib.protoseg_last_error()

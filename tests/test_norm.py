"""CPU: refusals and host logic of the group norm (no GPU call is made)."""
import ctypes

import pytest
import torch

from protoseg_amd import _lib, norm

NULL, SOME = ctypes.c_void_p(None), ctypes.c_void_p(4096)


def fwd(dtype=0, B=1, HW=4, C=8, sb=32, sp=8, groups=2, eps=1e-5, act=0, x=SOME, y=SOME, stats=SOME, ws=NULL, nbytes=0):
    return _lib.load().protoseg_group_norm_fwd(x, dtype, B, HW, C, sb, sp, groups, NULL, NULL, eps, act, y, stats, ws, nbytes, NULL)


@pytest.mark.parametrize("bad, status, text", [
    (dict(dtype=2), _lib.ERR_UNSUPPORTED, b"dtype"),
    (dict(groups=3), _lib.ERR_INVALID, b"groups"),
    (dict(groups=0), _lib.ERR_INVALID, b"groups"),
    (dict(C=0), _lib.ERR_INVALID, b"groups"),
    (dict(B=-1), _lib.ERR_INVALID, b"B -1"),
    (dict(B=70000), _lib.ERR_UNSUPPORTED, b"at most"),
    (dict(eps=-1.0), _lib.ERR_INVALID, b"eps"),
    (dict(eps=float("nan")), _lib.ERR_INVALID, b"eps"),
    (dict(act=4), _lib.ERR_INVALID, b"activation"),
    (dict(x=NULL), _lib.ERR_INVALID, b"x must"),
    (dict(sp=7), _lib.ERR_INVALID, b"overlap"),
    (dict(B=2, sb=31), _lib.ERR_INVALID, b"overlap"),
    (dict(y=NULL), _lib.ERR_INVALID, b"non-null"),
    (dict(stats=NULL), _lib.ERR_INVALID, b"non-null"),
    (dict(), _lib.ERR_INVALID, b"workspace"),
])
def test_forward_refusals(bad, status, text):
    assert fwd(**bad) == status
    assert text in _lib.load().protoseg_last_error()


def test_backward_refusals():
    lib = _lib.load()

    def bwd(gy=SOME, gsp=8, stats=SOME, gx=SOME, nbytes=0):
        return lib.protoseg_group_norm_bwd(SOME, gy, 0, 1, 4, 8, 32, 8, 32, gsp, 2, NULL, NULL, 0, stats, gx, NULL, NULL, NULL, nbytes, NULL)

    for bad, text in ((dict(gy=NULL), b"g_y"), (dict(gsp=4), b"overlap"), (dict(stats=NULL), b"stats"), (dict(), b"workspace")):
        assert bwd(**bad) == _lib.ERR_INVALID and text in lib.protoseg_last_error()
    assert bwd(gx=NULL) == _lib.OK  # nothing is asked for: nothing runs


def test_empty_calls_need_nothing():
    assert fwd(B=0, x=NULL, y=NULL) == _lib.OK
    assert fwd(HW=0, x=NULL, y=NULL) == _lib.OK
    assert _lib.load().protoseg_group_norm_workspace_size(0, 0, 4, 8, 2, 1) == 0


def test_workspace_grows_with_the_map():
    lib = _lib.load()
    for back in (0, 1):
        a, b = (lib.protoseg_group_norm_workspace_size(_lib.BF16, 2, hw, 256, 32, back) for hw in (64, 4225))
        assert 0 < a <= b and a % 256 == b % 256 == 0


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.ProtosegError, match="CPU|cpu"):
        norm.group_norm(torch.zeros(1, 8, 4, 4), 2)


def test_what_is_read_in_place():
    cl = torch.zeros(2, 24, 6, 5).contiguous(memory_format=torch.channels_last)
    for view in (cl, cl[:, 8:16], cl[1:], cl[::2], cl[:, :, :, :1][:, :, :1], cl[:, :, :, :1]):
        assert norm._rows(view)[0].data_ptr() == view.data_ptr()
    assert norm._rows(cl[:, 8:16])[1:] == (24 * 30, 24)
    assert norm._rows(cl[:, :, :, :1])[1:] == (24 * 30, 24 * 5)  # one column: the pixel stride is the rows'
    for view in (cl[..., ::2], cl[:, :, ::2], torch.zeros(2, 24, 6, 5), cl[:1].expand(3, -1, -1, -1), cl[:, :1].expand(-1, 8, -1, -1)):
        rows, sb, sp = norm._rows(view)
        assert rows.data_ptr() != view.data_ptr() and rows.is_contiguous(memory_format=torch.channels_last)
        assert (sb, sp) == (view.shape[2] * view.shape[3] * view.shape[1], view.shape[1])
    one = torch.zeros(1, 1, 4, 3)  # a single channel is both layouts at once
    assert norm._rows(one)[1:] == (12, 1)


def test_module_refusals():
    with pytest.raises(ValueError, match="groups"):
        norm.GroupNorm(5, 12)
    with pytest.raises(ValueError, match="activation"):
        norm.GroupNorm(4, 12, activation="gelu")
    assert norm.GroupNorm(4, 12, affine=False).weight is None

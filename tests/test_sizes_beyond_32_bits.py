"""CPU: sizes whose low 32 bits alone would reach the library, or whose padded size leaves an int, are refused."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from protoseg_amd import _lib, norm, optim

NULL, SOME = ctypes.c_void_p(None), ctypes.c_void_p(4096)


@pytest.mark.parametrize("shape", [(1, 1, 65536, 65537), (1, 2, 1 << 16, 1 << 15), ((1 << 32) + 1, 2, 1, 1), (65536, 1, 1, 1), (1, (1 << 20) + 2, 1, 1)])
def test_group_norm_maps(shape):
    with pytest.raises(_lib.ProtosegError, match="at most"):
        norm._sizes(torch.bfloat16, torch.Size(shape), 1)


def test_orthogonalize():
    with FakeTensorMode():
        for shape in ((1, 1, (1 << 32) + 64), ((1 << 32) + 2, 8, 8), (1 << 16, (1 << 16) + 1, 4, 4), ((1 << 31), 3)):
            with pytest.raises(_lib.ProtosegError, match="at most 2147483647"):
                optim.orthogonalize(torch.empty(shape, dtype=torch.bfloat16, device="cuda:0"))


@pytest.mark.parametrize("rows, cols", [(1, 0x7FFFFFFF), (0x7FFFFFFF, 1), (1, 0x7FFFFFC1), (0x7FFFFFFF, 0x7FFFFFFF), (1, (1 << 23) + 1)])
def test_padded_sizes_beyond_an_int(rows, cols):
    lib = _lib.load()
    status = lib.protoseg_orthogonalize(SOME, 1, 1, rows, cols, rows * cols, 5, *optim.NS_COEFFICIENTS, 1e-7, SOME, NULL, 0, NULL)
    assert status == _lib.ERR_UNSUPPORTED and b"at most" in lib.protoseg_last_error()
    ptr, r, c = (ctypes.c_void_p * 1)(4096), (ctypes.c_int32 * 1)(rows), (ctypes.c_int32 * 1)(cols)
    status = lib.protoseg_muon_step(1, ptr, ptr, ptr, r, c, 0.9, 1, 0.1, 0.0, 0, 5, *optim.NS_COEFFICIENTS, 1e-7, NULL, 0, NULL)
    assert status == _lib.ERR_UNSUPPORTED


def test_muon():
    class Large:  # stands for a parameter of 2^32 + 8 columns
        pass

    p = torch.nn.Parameter(torch.zeros(4, 4))
    p.grad = torch.ones(4, 4)
    opt = optim.Muon([p])
    fake = Large()
    fake.grad, fake.shape, fake.dtype = p.grad, (1, (1 << 32) + 8), torch.float32
    fake.numel, fake.dim = (lambda: (1 << 32) + 8), (lambda: 2)
    opt.param_groups[0]["params"] = [fake]
    with pytest.raises(_lib.ProtosegError, match="at most 2147483647"):
        opt.step()

"""CPU: the flags that the kernels' results rest on reach every compile line, and a change of them rebuilds (dry runs of make)."""
import subprocess

from protoseg_amd import _lib

MAKE = ["make", "-n", "-C", str(_lib.CSRC_DIR)]


def lines(*args):
    out = subprocess.run([*MAKE, *args], check=True, capture_output=True, text=True).stdout
    return [line for line in out.splitlines() if " -c " in line]


def test_flags_of_every_object():
    for given in ((), ("HIPFLAGS=-O1 -std=c++17 -fPIC",)):
        compiled = lines("-B", *given)
        assert len(compiled) >= 14
        assert all("-Xclang -target-feature -Xclang -packed-fp32-ops" in line for line in compiled)
        contract = [line for line in compiled if "-ffp-contract=off" in line]
        assert len(contract) == 1 and "bbox.hip" in contract[0]


def test_other_flags_rebuild():
    assert any("norm.hip" in line for line in lines("-W", "Makefile", "norm.o"))


def test_diagnostic_targets_too():
    for target in ("stamps", "resource-usage"):
        out = subprocess.run([*MAKE, target], check=True, capture_output=True, text=True).stdout
        compiled = [line for line in out.splitlines() if "hipcc" in line and "-shared" not in line]
        assert compiled and all("-packed-fp32-ops" in line for line in compiled)

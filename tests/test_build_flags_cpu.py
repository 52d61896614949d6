"""What the Makefile compiles with, read from `make -n`: every device compilation leaves packed fp32 instructions out."""
import os
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "humanoid-vision-system_amd")


def compilations(*args):
    """The hipcc command lines that compile a HIP source, by source."""
    out = subprocess.run(["make", "-C", PKG, "-n", "-B", *args], check=True, capture_output=True, text=True).stdout
    return {w: line for line in out.splitlines() if " -c " in line for w in line.split() if w.startswith("csrc/") and w.endswith(".hip")}


@pytest.mark.parametrize("target", ["all", "debug"])
def test_no_packed_fp32(target):
    """v_pk_add / mul / fma_f32 come from ordinary float code; hipcc makes none with this feature off."""
    got = compilations(target)
    assert set(got) == {"csrc/" + f for f in os.listdir(os.path.join(PKG, "csrc")) if f.endswith(".hip")}
    for source, line in got.items():
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, source


@pytest.mark.parametrize("target", ["all", "debug"])
def test_flags_of_the_caller_do_not_lose_it(target):
    for source, line in compilations(target, "CXXFLAGS=-O2 -fPIC --offload-arch=gfx950", "DBGFLAGS=-O0 -fPIC --offload-arch=gfx950").items():
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, source


@pytest.mark.parametrize("target", ["all", "debug"])
def test_a_changed_makefile_compiles_everything(target):
    """Its flags are part of what an object is made of (the library's provenance hash covers them too)."""
    out = subprocess.run(["make", "-C", PKG, "-n", "-W", "Makefile", target], check=True, capture_output=True, text=True).stdout
    got = {w for line in out.splitlines() if " -c " in line for w in line.split() if w.startswith("csrc/") and w.endswith(".hip")}
    assert got == {"csrc/" + f for f in os.listdir(os.path.join(PKG, "csrc")) if f.endswith(".hip")}

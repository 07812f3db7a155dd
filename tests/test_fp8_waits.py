"""The waits of the kernels that multiply 8-bit codes, in the code that was built for gfx950.

A wait lets as many vector loads stay outstanding as were issued behind those that have to have landed.  The
scales of x are loaded by each lane for itself, those of w for a whole wave: a compiler may make the latter a
scalar load, which the vector loads' counter does not count, and a wait that counts it then ends too early.  So
either that load is a vector load, which is seen here, or the waits do not count it."""

import re
import shutil
import subprocess

import pytest

from ttlhip import _lib as L

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{name: (its code, the vmcnt values that it waits for)}"""
    if not shutil.which(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    d = tmp_path_factory.mktemp("fp8")
    shutil.copy(L.LIB_PATH, d / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=d, check=True, capture_output=True)
    found = {}
    for obj in sorted(d.glob("lib.so.*gfx950")):
        if b"fp8_block_kernel" not in obj.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", str(obj)], check=True, capture_output=True,
                              text=True).stdout
        for part in re.split(r"^[0-9a-f]+ <", text, flags=re.M)[1:]:
            name = part.split(">:", 1)[0]
            found[name] = part, set(map(int, re.findall(r"s_waitcnt vmcnt\((\d+)\)", part)))
    assert found
    return found


def _count(code, load):
    return len(re.findall(rf"\b{load}\b", code))


@pytest.mark.parametrize("tx,tw", [(1, 1), (1, 2), (2, 2), (2, 4)])
def test_blocks_that_share_loads(kernels, tx, tw):
    names = [n for n in kernels if f"fp8_block_kernelILi{tx}ELi{tw}E" in n]
    assert len(names) == 2
    loads = 2 * (tx + tw)  # of a group, which may be outstanding
    for name in names:
        code, waits = kernels[name]
        if "Lb1E" in name:  # into f32: x's scales alone are counted
            assert loads + tx in waits and loads + tx + 1 not in waits, (name, waits)
        else:  # before the loop and three times in it: x's scales and w's
            assert loads + tx + 1 in waits, (name, waits)
            assert _count(code, "global_load_dword") == 4 * (tx + 1), name


def test_the_largest_blocks(kernels):
    names = [n for n in kernels if "fp8_large_kernel" in n]
    assert len(names) == 2
    for name in names:
        code, waits = kernels[name]
        assert 16 + 5 in waits, (name, waits)
        assert _count(code, "global_load_dword") == 2 * 5, name


@pytest.mark.parametrize("mt,nt,waves", [(1, 1, 8), (2, 1, 8), (2, 2, 4), (2, 2, 8), (2, 4, 4), (4, 4, 4)])
def test_waves_that_divide_k(kernels, mt, nt, waves):
    names = [n for n in kernels if f"fp8_direct_kernelILi{mt}ELi{nt}ELi{waves}E" in n]
    assert len(names) == 2
    for name in names:  # two groups before the loop and two in it: x's scales and w's
        code, waits = kernels[name]
        assert 2 * (mt + nt) + mt + 1 in waits, (name, waits)
        assert _count(code, "global_load_ubyte") == 4 * (mt + 1), name

"""The waits of the kernels that multiply 8-bit codes, in the code that was built for gfx950.

The scales of x are loaded by each lane for itself, those of w for a whole wave: a compiler may make the
latter a scalar load, which the vector loads' counter does not count.  A wait that lets the scales' loads
stay outstanding must therefore count x's alone, or it may end before the codes in front of them have landed."""

import re
import shutil
import subprocess

import pytest

from ttlhip import _lib as L

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    """{kernel: the vmcnt values it waits for} of the kernels whose waits count the scales' loads."""
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
            if "fp8_block_kernel" in name or "fp8_large_kernel" in name:
                found[name] = set(map(int, re.findall(r"s_waitcnt vmcnt\((\d+)\)", part)))
    assert found
    return found


def _check(values, loads, x_scales, name):
    assert loads + x_scales in values, (name, values)
    if "Lb1E" not in name:  # (into f32 there may be other code with other waits)
        assert loads + x_scales + 1 not in values, (name, values)


@pytest.mark.parametrize("tx,tw", [(1, 1), (1, 2), (2, 2), (2, 4)])
def test_blocks_that_share_loads(waits, tx, tw):
    names = [n for n in waits if f"fp8_block_kernelILi{tx}ELi{tw}E" in n]
    assert len(names) == 2
    for name in names:  # a group's loads may be outstanding
        _check(waits[name], 2 * (tx + tw), tx, name)


def test_the_largest_blocks(waits):
    names = [n for n in waits if "fp8_large_kernel" in n]
    assert len(names) == 2
    for name in names:
        _check(waits[name], 16, 4, name.replace("Lb1E", ""))

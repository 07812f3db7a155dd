"""How the exponents of two scales are divided between operands in bf16 (csrc/ttlh_fp8.h), for every pair
of scales, compiled for the host."""

import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LEAST, MOST = 2.0 ** -9, 448.0  # magnitudes of codes


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp8")
    src = d / "r.cpp"
    src.write_text('#include "ttlh_fp8.h"\nusing namespace ttlh;\nextern "C" {\n'
                   'int w(int ew) { return wide_w(ew); }\n'
                   'int rest(int ex, int ew) { return wide_rest(ex, ew); }\n'
                   'int x(int ex, int ew) { return wide_x(wide_rest(ex, ew)); }\n'
                   'int far_(int ex, int ew) { return wide_far(wide_rest(ex, ew)); }\n}\n')
    so = d / "r.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "tt-lang_amd", "csrc"),
                    str(src), "-o", str(so)], check=True)
    return ctypes.CDLL(str(so))


def _held(scale):
    """bf16 holds every code times 2^(scale - 127) as a normal number (or zero)."""
    s = 2.0 ** (scale - 127)
    return LEAST * s >= 2.0 ** -126 and MOST * s < 2.0 ** 128 * (1 - 2.0 ** -8)


def test_every_pair_of_scales(rules):
    exact = lost = far = 0
    for ew in range(255):
        w = rules.w(ew)
        assert _held(w)
        for ex in range(255):
            x, e = rules.x(ex, ew), ex + ew - 254
            if rules.far_(ex, ew):
                far += 1
                # rest = ex + ceil(ew / 2) - 42 > 246 and ex <= 254: ew >= 69, e >= 35 + floor(ew / 2)
                assert e >= 69
            elif x + w - 254 == e and _held(x):
                exact += 1
            else:
                # x's operand may be anything up to its largest magnitude here: the product that is
                # meant, and any that comes of it, less than 2^-149; or it is off by 2^-126 at most
                assert 1 <= x < 10
                largest = MOST * 2.0 ** (x - 127) * MOST * 2.0 ** (w - 127)
                if x + w - 254 != e:
                    assert largest < 2.0 ** -149 and MOST * MOST * 2.0 ** e < 2.0 ** -149
                assert 2.0 ** -126 * MOST * 2.0 ** (w - 127) < 2.0 ** -149
                lost += 1
    assert exact > 40000 and far and lost

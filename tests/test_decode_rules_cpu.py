"""Rules and limits of the decode-step operators that are plain C++ (tests/decode_rules_unit.cc)."""
import math
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules_and_limits(tmp_path):
    exe = str(tmp_path / "decode_rules_unit")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                           os.path.join(ROOT, "tests", "decode_rules_unit.cc")])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


@pytest.mark.parametrize("dim,base,original,low,high", [
    (64, 2.0, 8192.0, 1.0, 32.0),          # the slowest pair still turns 660 times
    (128, 1.5, 1e6, 1.0, 32.0), (64, 1.0000001, 8192.0, 1.0, 32.0),
    (64, 10000.0, 0.5, 1.0, 32.0),         # the fastest pair does not turn once
    (32, 100.0, 3.0, 4.0, 8.0), (64, 1.0000001, 0.5, 1.0, 32.0), (64, 10000.0, 1e-300, 1.0, 32.0)])
def test_a_ramp_that_lies_outside_the_pairs(dim, base, original, low, high):
    """Pairs of at least `high` turns stay, of at most `low` are slowed, also where that is all of them."""
    from mace_b200 import capi
    plain = base ** (-2.0 * np.arange(dim // 2) / dim)
    turns = original * plain / (2 * math.pi)
    assert (turns >= high).all() or (turns <= low).all()
    f, _ = capi.rope_frequencies(dim, base=base, scaling=capi.ROPE_RAMP, factor=4.0, original_length=original, low=low, high=high)
    assert np.allclose(f, plain if turns[0] > high else plain / 4.0, rtol=1e-14)


@pytest.mark.parametrize("dim", [4, 32, 64, 80, 128])
@pytest.mark.parametrize("base", [1.2, 10.0, 1e4, 1e6])
@pytest.mark.parametrize("original", [0.01, 1.0, 50.0, 4096.0, 1e7])
def test_a_ramp_slows_slower_pairs_more(dim, base, original):
    """No pair is slowed less than a faster one."""
    from mace_b200 import capi
    plain = base ** (-2.0 * np.arange(dim // 2) / dim)
    for low, high in ((1.0, 2.0), (1.0, 32.0), (0.001, 1e5)):
        f, _ = capi.rope_frequencies(dim, base=base, scaling=capi.ROPE_RAMP, factor=8.0, original_length=original, low=low, high=high)
        share = f / plain
        assert (np.diff(share) <= 1e-14).all() and (share <= 1 + 1e-14).all() and (share >= 1 / 8.0 - 1e-14).all()

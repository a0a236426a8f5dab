"""What the decode-step operators do on the host: page arithmetic, refusals, rotary frequencies."""
import math
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_pages_and_refusals(tmp_path):
    """tests/kv_cache_unit.cc: bad pages and lengths, every refusal of every call."""
    exe = str(tmp_path / "kv_cache_unit")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                           os.path.join(ROOT, "tests", "kv_cache_unit.cc")])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_calls_without_a_context_are_refused():
    import mace_b200
    lib = mace_b200.lib()
    z = None
    assert lib.mb_rope(z, z, z, z, z, 1, 1, 2, 2, 2, 2, 2, 2, 0, 0, 1.0, 0) == 1
    assert lib.mb_rope_kv_append(*[z] * 10, *[1] * 11, 0, 1.0, 0) == 1
    assert lib.mb_paged_attention(*[z] * 10, *[1] * 12, 1.0, 0) == 1
    assert lib.mb_kv_evict(*[z] * 12, *[1] * 13, 0) == 1
    assert lib.mb_quantize_mxfp4(z, z, z, z, 1, 1, 1, 0) == 1
    assert lib.mb_dequantize_mxfp4(z, z, z, z, 1, 1, 1, 0) == 1
    assert lib.mb_gemm_mxfp4(*[z] * 7, 1, 1, 1, 1, 0) == 1


def test_scale_bytes():
    from mace_b200 import capi
    assert capi.mxfp4_scale_bytes(1, 1) == 512
    assert capi.mxfp4_scale_bytes(129, 129) == 4 * 512
    assert capi.mxfp4_scale_bytes(0, 5) == 0
    assert capi.mxfp4_scale_bytes(1 << 20, 1 << 20) == (1 << 13) * (1 << 13) * 512


@pytest.mark.parametrize("dim", [0, 2, 32, 64, 128, 80])
def test_rope_frequencies(dim):
    from mace_b200 import capi
    i = np.arange(dim // 2)
    plain = 10000.0 ** (-2.0 * i / max(dim, 1))
    f, m = capi.rope_frequencies(dim)
    assert m == 1.0 and np.allclose(f, plain, rtol=1e-14)
    f, m = capi.rope_frequencies(dim, scaling=capi.ROPE_LINEAR, factor=4.0)
    assert m == 1.0 and np.allclose(f, plain / 4.0, rtol=1e-14)
    if dim >= 4:
        f, _ = capi.rope_frequencies(dim, scaling=capi.ROPE_BASE, factor=4.0)
        assert f[0] == 1.0 and math.isclose(f[-1], plain[-1] / 4.0, rel_tol=1e-12)
    # bands: pairs of many turns stay, those of few are slowed, turns in between mix linearly
    kw = dict(factor=8.0, original_length=8192.0, low=1.0, high=4.0)
    f, m = capi.rope_frequencies(dim, scaling=capi.ROPE_BANDS, **kw)
    turns = 8192.0 * plain / (2 * math.pi)
    kept = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
    assert m == 1.0 and np.allclose(f, plain * (kept + (1 - kept) / 8.0), rtol=1e-13)
    # ramp: the same ends, linear in the pair's number
    f, m = capi.rope_frequencies(dim, scaling=capi.ROPE_RAMP, **kw)
    assert math.isclose(m, 0.1 * math.log(8.0) + 1.0, rel_tol=1e-6)
    assert np.allclose(f[turns >= 4.0 * 1.5], plain[turns >= 4.0 * 1.5], rtol=0.3)
    assert (f <= plain * (1 + 1e-14)).all() and (f >= plain / 8.0 * (1 - 1e-14)).all()
    share = (f / plain - 1 / 8.0) / (7 / 8.0)
    inner = share[(share > 1e-9) & (share < 1 - 1e-9)]
    assert np.allclose(np.diff(inner, 2), 0.0, atol=1e-9)


def test_rope_frequencies_refuse():
    from mace_b200 import capi
    for kw in (dict(rotary_dim=3), dict(rotary_dim=-2), dict(base=0.0), dict(base=float("nan")), dict(scaling=5), dict(scaling=-1),
               dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("inf")), dict(scaling=2, rotary_dim=2),
               dict(scaling=3, factor=2.0), dict(scaling=3, factor=2.0, original_length=100.0, low=4.0, high=4.0),
               dict(scaling=4, factor=2.0, original_length=100.0, low=0.0), dict(scaling=4, factor=2.0, original_length=100.0, base=1.0)):
        with pytest.raises(capi.MaceB200Error) as e:
            capi.rope_frequencies(**{"rotary_dim": 64, **kw})
        assert e.value.code == 1, kw


def test_eviction_with_strided_weights_wants_a_context():
    import mace_b200
    assert mace_b200.lib().mb_kv_evict_strided(*[None] * 12, *[1] * 14, 0) == 1

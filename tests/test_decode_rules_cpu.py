"""Rules and limits of the decode-step operators that are plain C++ (tests/decode_rules_unit.cc)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules_and_limits(tmp_path):
    exe = str(tmp_path / "decode_rules_unit")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", exe,
                           os.path.join(ROOT, "tests", "decode_rules_unit.cc")])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr

"""What the 4-bit product of few rows reads of its operands, on the host: no byte in front of
a weight's first row or behind its last one, whatever the row's length and address."""
import os
import subprocess


def test_loads_stay_in_the_matrix(tmp_path):
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "fp4_load.cpp")
    exe = str(tmp_path / "fp4_load")
    r = subprocess.run(["g++", "-std=c++17", "-O1", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "fine\n", r.stdout

"""Refusals, launch plans and the 4-bit layout of the layer operators, on the host (no device)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_layer_args(tmp_path):
    exe = str(tmp_path / "layer_args_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra",
                    "-o", exe, os.path.join(HERE, "layer_args_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr

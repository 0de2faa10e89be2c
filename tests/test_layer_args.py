"""Refusals, launch plans and the 4-bit layout of the layer operators, on the host (no device)."""
import os
import struct
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_layer_args(tmp_path):
    exe = str(tmp_path / "layer_args_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra",
                    "-o", exe, os.path.join(HERE, "layer_args_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


class Calls:
    """In the library's place: keeps each call's arguments."""

    def __getattr__(self, name):
        def call(*args):
            self.name, self.args = name, args
            return 0
        return call


@pytest.fixture
def eng():
    from matmulfreellmcpu_amd import Engine
    e = Engine.__new__(Engine)
    e.h, e.lib = None, Calls()
    return e


def test_row_types_are_the_tensors(eng):
    """Without a type the first input's own is taken; addresses alone are fp32; bytes are storage of any type."""
    import torch
    from matmulfreellmcpu_amd import BF16, F16, F32, I8
    f, h, b, c, raw = (torch.zeros(8, dtype=t) for t in (torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.uint8))
    for x, t in ((f, F32), (b, BF16), (h, F16), (64, F32), (raw, F32)):
        eng.add_rmsnorm_q8(c, f, x, f, 1, 8, res=x, h=x)
        assert eng.lib.args[1] == t and eng.lib.args[2:5] == (c.data_ptr(), f.data_ptr(), x if isinstance(x, int) else x.data_ptr())
        eng.w4_linear(0, x, x, 1)
        assert eng.lib.args[2] == t and eng.lib.args[5] == t
        eng.short_conv(x, x, f, 1, 8, 4)
        assert eng.lib.args[1] == t
        eng.selective_scan(x, x, x, f, x, x, 1, 8, 8, z=x)
        assert struct.unpack_from("@2i", eng.lib.args[1])[0] == t
    eng.w4_linear(0, c, h, 1, scales=f)
    assert (eng.lib.args[2], eng.lib.args[5]) == (I8, F16)
    eng.w4_linear(0, raw, raw, 1, dtype=BF16, out_dtype=F16)
    assert (eng.lib.args[2], eng.lib.args[5]) == (BF16, F16)


def test_rows_of_another_type_are_refused(eng):
    """A tensor whose type is not the call's would be read, or written, past its end."""
    import torch
    from matmulfreellmcpu_amd import BF16, F32, I8
    f, b, c, d = (torch.zeros(8, dtype=t) for t in (torch.float32, torch.bfloat16, torch.int8, torch.float64))
    calls = [lambda: eng.add_rmsnorm_q8(c, f, b, f, 1, 8, dtype=F32), lambda: eng.add_rmsnorm_q8(f, f, f, f, 1, 8),
             lambda: eng.add_rmsnorm_q8(c, f, f, f, 1, 8, res=b), lambda: eng.add_rmsnorm_q8(c, f, b, f, 1, 8, h=f),
             lambda: eng.add_rmsnorm_q8(c, f, f, f, 1, 8, y=b), lambda: eng.add_rmsnorm_q8(c, f, 64, f, 1, 8, res=b),
             lambda: eng.w4_linear(0, b, f, 1, dtype=F32), lambda: eng.w4_linear(0, f, b, 1, out_dtype=F32),
             lambda: eng.w4_linear(0, f, f, 1, dtype=I8), lambda: eng.w4_linear(0, d, f, 1),
             lambda: eng.short_conv(f, b, f, 1, 8, 4), lambda: eng.short_conv(b, f, f, 1, 8, 4, dtype=F32)]
    for k in ("out", "u", "dt", "B", "C", "z"):
        kw = dict(out=f, u=f, dt=f, B=f, C=f, z=f)
        kw[k] = b
        calls.append(lambda kw=kw: eng.selective_scan(A=f, rows=1, D=8, N=8, dtype=F32, **kw))
    for call in calls:
        eng.lib.name = None
        with pytest.raises(ValueError, match="type"):
            call()
        assert eng.lib.name is None

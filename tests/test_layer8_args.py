"""Refusals, launch plans and the 8-bit layout of the linear attention layer's operators, on the host (no device)."""
import os
import struct
import subprocess

import pytest

from test_layer_args import HERE, eng  # noqa: F401  (an engine whose library only keeps each call's arguments)


def test_layer8_args(tmp_path):
    exe = str(tmp_path / "layer8_args_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra",
                    "-o", exe, os.path.join(HERE, "layer8_args_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_structs_are_the_headers(tmp_path):
    """The packed arguments lie as the C structs do."""
    from matmulfreellmcpu_amd import _BLOCK_ARGS, _DECAY_ARGS, _LOGP_ARGS
    src = tmp_path / "sizes.c"
    src.write_text("""#include <stdio.h>
#include <stddef.h>
#include "mmfree_hip.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(mmf_decay_args), sizeof(mmf_block_args), sizeof(mmf_logp_args),
         offsetof(mmf_decay_args, seqs), offsetof(mmf_decay_args, ldg), offsetof(mmf_block_args, rows), offsetof(mmf_block_args, scale),
         offsetof(mmf_logp_args, rows));
  return 0;
}
""")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(HERE, "..", "include"), "-o", exe, str(src)], check=True)
    got = [int(n) for n in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [_DECAY_ARGS.size, _BLOCK_ARGS.size, _LOGP_ARGS.size, 8 + 8 * 8, _DECAY_ARGS.size - 8, 8 + 8 * 10, _BLOCK_ARGS.size - 8, 8 + 8 * 6]


def test_types_of_tensors(eng):  # noqa: F811
    """Row types are the tensors' own; tensors of another type are refused wherever they stand."""
    import torch
    from matmulfreellmcpu_amd import BF16, F16, F32
    f, h, b, c, i = (torch.zeros(8, dtype=t) for t in (torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.int64))
    for x, t in ((f, F32), (b, BF16), (h, F16), (64, F32)):
        eng.decay_attention(x, x, x, x, 1, 1, 8, 8, decay=f, gates=f, state=f)
        assert struct.unpack_from("@if", eng.lib.args[1]) == (t, struct.unpack("f", struct.pack("f", 8 ** -0.5))[0])
        eng.block_norm_q8(c, f, x, 1, 8, x=x, gate=x, act=1, w_post=f, h=x, y=x)
        assert struct.unpack_from("@2i", eng.lib.args[1]) == (t, 1)
        eng.token_logprobs(x, 1, 8, ids=i, logprobs=f, top=1, top_ids=i, top_logprobs=f)
        assert struct.unpack_from("@if", eng.lib.args[1]) == (t, 1.0)
        eng.w8_linear(0, c, f, x, 1, bias=f)
        assert eng.lib.args[5] == t
    for call in (lambda: eng.decay_attention(b, b, b, h, 1, 1, 8, 8), lambda: eng.decay_attention(b, b, b, b, 1, 1, 8, 8, gates=b),
                 lambda: eng.decay_attention(b, b, b, b, 1, 1, 8, 8, state=b), lambda: eng.block_norm_q8(c, f, b, 1, 8, x=f),
                 lambda: eng.block_norm_q8(c, f, b, 1, 8, w_pre=b), lambda: eng.block_norm_q8(b, f, b, 1, 8),
                 lambda: eng.token_logprobs(b, 1, 8, ids=f, logprobs=f), lambda: eng.token_logprobs(b, 1, 8, ids=i, logprobs=b),
                 lambda: eng.w8_linear(0, f, f, f, 1), lambda: eng.w8_linear(0, c, b, f, 1), lambda: eng.w8_linear(0, c, f, f, 1, bias=b)):
        with pytest.raises(ValueError, match="place of"):
            call()


def test_w8_codes_are_int8(eng):  # noqa: F811
    """Weights of another type are taken where they are int8 numbers, and never wrapped or cut."""
    import numpy as np
    for codes in ([[128]], [[-129]], [[1.5]], [[float("nan")]], np.array([[200]], np.uint8), np.array([[1 << 40]])):
        with pytest.raises(ValueError, match="no int8 numbers"):
            eng.register_w8(codes, [1.0])
    for codes in ([[127, -128]], np.array([[3.0, -4.0]]), np.array([[7, 100]], np.uint8), np.array([[1, -1]], np.int8)):
        eng.register_w8(codes, [1.0])


def test_heads_of_no_size_are_refused_by_the_library(eng):  # noqa: F811
    """The default scale of a head of 0 is no division by 0: the call reaches the library, which says what is wrong."""
    eng.decay_attention(64, 64, 64, 64, 1, 1, 0, 8)
    assert eng.lib.args

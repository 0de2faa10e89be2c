"""Numbers near the ends of their types in the norms around a block and in log probabilities, against plain numpy in 64 bits.

U = 2^-24 is fp32's half step.
"""
import numpy as np
import pytest

from test_gpu_layer import F16, F32, BF16, FLOATS, I8, U, Rows, close, coded, out_rows, value
from test_gpu_layer8 import block_ref
from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu


# ---- norms around a block -----------------------------------------------------------------------


def block(eng, t, b, w_pre=None, x=None, eps=1e-6):  # noqa: F811
    """(h, y, codes, scales) of rows b (and x)."""
    rows, cols = b.shape
    B, X = Rows(eng, coded(b, t), t), Rows(eng, coded(x, t), t) if x is not None else None
    W = Dev(eng, w_pre) if w_pre is not None else None
    H, Y, Q, S = out_rows(eng, b.shape, t), out_rows(eng, b.shape, t), out_rows(eng, b.shape, I8), out_rows(eng, (rows, 1), F32)
    eng.block_norm_q8(Q.ptr, S.ptr, B.ptr, rows, cols, x=X.ptr if X else None, w_pre=W.ptr if W else None, h=H.ptr, y=Y.ptr, eps=eps,
                      dtype=t)
    eng.sync()
    return value(H.get(), t), value(Y.get(), t), Q.get(), S.get()[:, 0]


@pytest.mark.parametrize("t,cols", [(BF16, 16384), (F16, 16384), (F32, 20000), (BF16, 20000), (F16, 20000)])
def test_block_scales_past_fp32(eng, t, cols):  # noqa: F811
    """A row with one element has a norm of sqrt(cols) there; by the largest weight its scale passes fp32: such a row has no codes.
    Just below, the codes and the scale are numbers. (Rows in registers, and longer ones.)"""
    print(f"block scales t={t} cols={cols}", flush=True)
    b, w = np.zeros((3, cols)), np.ones(cols, np.float32)
    b[0, 7], b[1, 5], b[2, 9], b[2, 11] = 2.0, 2.0, 1.0, -0.5
    w[7], w[5] = 3.4e38, 3.4e38 * 126.9 / np.sqrt(cols)
    h, y, q, s = block(eng, t, b, w, eps=0.0)
    assert (h == b).all()
    assert np.isnan(s[0]) and not q[0].any(), (s[0], np.unique(q[0]))
    _, _, real, scales = block_ref(b[1:], None, None, 0, None, w, None, 1.0, 0.0)
    assert (q[1:] == np.round(real)).all() and (np.abs(s[1:] - scales) <= 1.001 * U * scales).all()
    assert np.isinf(y[0, 7]) and np.isinf(y[1, 5]) and not np.delete(y[:2], (5, 7), 1).any()


@pytest.mark.parametrize("cols", [100, 20000])
def test_block_codes_of_rows_past_fp16(eng, cols):  # noqa: F811
    """h and y past fp16's range are stored as infinities; codes and scales are those of the fp32 h."""
    print(f"block past fp16 cols={cols}", flush=True)
    rng = np.random.default_rng(cols)
    b, x = value(coded(rng.uniform(3e4, 6e4, (2, cols)), F16), F16), value(coded(rng.uniform(3e4, 6e4, (2, cols)), F16), F16)
    x[1] *= 0.25
    b[1] *= 0.25
    h, y, q, s = block(eng, F16, b, None, x)
    want, _, real, scales = block_ref(b, x, None, 0, None, None, None, 1.0, 1e-6)
    ref = value(coded(want, F16), F16)
    assert (h == ref).all() and (y == ref).all() and np.isinf(h[0]).any() and np.isfinite(h[1]).all()
    assert (np.abs(q - real) <= 0.5 + 127 * 2.0 ** -40).all() and (np.abs(s - scales) <= 1.001 * U * scales).all()

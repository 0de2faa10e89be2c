"""Numbers near the ends of their types in the norms around a block and in log probabilities, against plain numpy in 64 bits.

U = 2^-24 is fp32's half step.
"""
import numpy as np
import pytest

from test_gpu_layer import BF16, F16, F32, I8, U, Rows, close, coded, out_rows, value
from test_gpu_layer8 import block_ref, logp_ref
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


# ---- log probabilities --------------------------------------------------------------------------


def logprobs(eng, t, x, ids, T, top):  # noqa: F811
    rows, V = x.shape
    f = np.float32
    X, I, lp, ent = Rows(eng, coded(x, t), t), Dev(eng, ids), Dev(eng, shape=(rows,)), Dev(eng, shape=(rows,))
    ti, tl = Dev(eng, np.zeros((rows, top), np.int64)), Dev(eng, np.zeros((rows, top), f))
    eng.token_logprobs(X.ptr, rows, V, ids=I.ptr, logprobs=lp.ptr, entropy=ent.ptr, top=top, top_ids=ti.ptr, top_logprobs=tl.ptr,
                       temperature=T, dtype=t)
    eng.sync()
    return lp.get(), ent.get(), ti.get(), tl.get()


@pytest.mark.parametrize("V", [2, 300, 9000, 70000])
@pytest.mark.parametrize("T", [1e37, 5e37, 3e38])
@pytest.mark.parametrize("t", [F32, BF16])
def test_logprobs_of_large_logits(eng, t, T, V):  # noqa: F811
    """Logits to the ends of fp32 at temperatures as large: differences of two pass fp32 where their quotients by the temperature
    do not; some tokens cannot come.

    The bound is that of other logits, which counts 1 U for 1 / T and 2 U for an exponent's product with log2 e. Of T = 3e38 both
    are subnormal: 2 / T = 6.7e-39 and 9.6e-39 in steps of 1.4e-45 round by 1.8 U and 1.2 U, 1 U more in all of the 3 U or 5 U that
    it counts of z: within twice the bound."""
    print(f"large logits t={t} T={T} V={V}", flush=True)
    rng, top = np.random.default_rng(V), 2
    x = rng.uniform(-3.3e38, 3.3e38, (5, V))
    x[0, 0], x[1, V // 2:] = 3.3e38, -np.inf
    x[2], x[2, 1] = -3.3e38, 3.3e38
    x[3] = -3.3e38
    x[4], x[4, 0] = -3e38, 0.0
    x = value(coded(x, t), t)
    ids = np.array([1, 0, 0, 1, 1])
    lp, ent, ti, tl = logprobs(eng, t, x, ids, T, top)
    want, H, all_lp, err, ent_err = logp_ref(x, ids, T)
    more, order, at = 2 if T > 1e38 else 1, np.argsort(-x, axis=1, kind="stable")[:, :top], np.arange(5)
    err = np.where(np.isfinite(all_lp), more * err, 0)
    close(lp, want, err[at, ids], F32, "logprobs")
    close(ent, H, more * ent_err, F32, "entropy")
    assert (ti == order).all()
    close(tl, np.take_along_axis(all_lp, order, 1), np.take_along_axis(err, order, 1), F32, "top")

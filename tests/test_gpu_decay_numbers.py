"""What attention with decays keeps of its numbers: matrix products of rows cut into bf16 parts have the digits of fp32 products,
and states that grow or shrink far between the tiles of a long sequence are those of the recurrence.

U = 2^-24 is fp32's half step.
"""
import numpy as np
import pytest

from test_gpu_layer import BF16, F16, F32, FLOATS, U, Rows, close, coded, out_rows, value
from test_gpu_layer8 import decay_ref
from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu


def attention(eng, t, q, k, v, lens, state=None, decay=None, gates=None, scale=1.0):  # noqa: F811
    """(out, state after) of q, k, v [rows, heads, D]."""
    rows, H, Dk = q.shape
    Dv, f = v.shape[2], np.float32
    Q, K, V = (Rows(eng, coded(x.reshape(rows, -1), t), t) for x in (q, k, v))
    for x, r in ((q, Q), (k, K), (v, V)):
        assert (value(r._in(r.host), t) == x.reshape(rows, -1)).all(), "inputs that the type does not hold"
    O = out_rows(eng, (rows, H * Dv), t)
    S = Dev(eng, (np.zeros((len(lens), H, Dk, Dv)) if state is None else state).astype(f))
    D, G = (Dev(eng, x.astype(f)) if x is not None else None for x in (decay, gates))
    eng.decay_attention(O.ptr, Q.ptr, K.ptr, V.ptr, rows, H, Dk, Dv, decay=D.ptr if D else None, gates=G.ptr if G else None,
                        state=S.ptr, lens=lens, scale=scale, dtype=t)
    eng.sync()
    return value(O.get(), t).reshape(rows, H, Dv), S.get()


# ---- digits ---------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [2, 40, 300])
@pytest.mark.parametrize("t", [BF16, F16])
def test_weights_that_cancel(eng, t, rows):  # noqa: F811
    """Two rows whose weights are large and cancel. All numbers are integers and every partial sum stays below 2^24, so that fp32
    sums of any order are exact: outputs have to be the exact ones, rounded once."""
    bits, H, rng = {BF16: 8, F16: 11}[t], 16, np.random.default_rng(rows + t)
    print(f"weights that cancel t={t} rows={rows}", flush=True)
    q = rng.integers(2 ** (bits - 1), 2 ** bits, (rows, H, 2)) | 1
    k, v = np.zeros((rows, H, 2), int), np.zeros((rows, H, 1), int)
    k[0] = rng.integers(2 ** (bits - 1) + 2, 2 ** bits - 2, (H, 2)) | 1
    k[1] = k[0] + rng.integers(-1, 2, (H, 2))
    v[0], v[1] = 1, -1
    out, state = attention(eng, t, q, k, v, [rows])
    want = (q * (k[0] - k[1])).sum(2)
    want[0] = (q[0] * k[0]).sum(1)
    want = value(coded(want.astype(np.float64), t), t)
    assert (out[:, :, 0] == want).all(), (np.abs(out[:, :, 0] - want).max(), np.argwhere(out[:, :, 0] != want)[:3])
    assert (state[0, :, :, 0] == k[0] - k[1]).all()


@pytest.mark.parametrize("rows", [2, 40, 300])
@pytest.mark.parametrize("t", [BF16, F16])
def test_states_that_cancel(eng, t, rows):  # noqa: F811
    """Two rows of the state that are large and cancel, integers of 22 bits whose sums fp32 holds: outputs are exact."""
    H, Dv, rng = 8, 24, np.random.default_rng(rows + t + 50)
    print(f"states that cancel t={t} rows={rows}", flush=True)
    state = rng.integers(2 ** 21, 2 ** 22, (1, H, 2, Dv)) | 1
    state[:, :, 1] = state[:, :, 0] + rng.integers(-100, 101, (1, H, Dv))
    q = np.ones((rows, H, 2), int)
    q[:, :, 1] = -1
    out, after = attention(eng, t, q, np.zeros((rows, H, 2)), np.zeros((rows, H, Dv)), [rows], state=state)
    assert (out == state[:, :, 0] - state[:, :, 1]).all(), np.abs(out - (state[:, :, 0] - state[:, :, 1])).max()
    assert (after == state).all()


def digits(rng, shape):
    """fp32 numbers from 1 to 2 whose lower bits are set, where a part that is cut off leaves the most."""
    return (1 + (rng.integers(0, 2 ** 23, shape) | 0xFE7F) / 2 ** 23).astype(np.float32)


def test_products_have_the_digits_of_fp32(eng):  # noqa: F811
    """Single products: of a query and a key (out = q_i k_0), of a key and a value (the state), of a query and the state. All have
    three parts; the sums of the products of parts are below 1/8 of the product but for the last step, and what is left out (the
    last part by the last) is below 2^-28. So with additions that are off by a step (2 U) at most, and the cut of what is no
    number of 24 bits, a product is within 2.3 U. A further product or sum (out of weight and value 1, of the state) is exact."""
    rng, H, rows = np.random.default_rng(3), 64, 64
    print("digits", flush=True)
    q, k, v = np.zeros((rows, H, 1)), np.zeros((rows, H, 1)), np.zeros((rows, H, 2))
    q[:], k[0], v[0] = digits(rng, (rows, H, 1)), digits(rng, (H, 1)), digits(rng, (H, 2))
    v[0, :, 0] = 1
    out, state = attention(eng, F32, q, k, v, [rows])
    qk = q[:32, :, 0] * k[0, :, 0]
    assert (np.abs(out[:32, :, 0] - qk) <= 2.3 * U * qk).all(), (np.abs(out[:32, :, 0] - qk) / qk).max() / U
    kv = k[0] * v[0]
    assert (np.abs(state[0, :, 0] - kv) <= 2.3 * U * kv).all(), (np.abs(state[0, :, 0] - kv) / kv).max() / U
    s = state[0, :, 0].astype(np.float64)  # the second chunk reads the state that the first left
    qs = q[32:] * s
    assert (np.abs(out[32:] - qs) <= 2.3 * U * qs).all(), (np.abs(out[32:] - qs) / qs).max() / U


@pytest.mark.parametrize("t", FLOATS)
def test_long_prompts_repeat_themselves(eng, t):  # noqa: F811
    """The same call gives the same bits: several tiles, blocks of eight waves, of many heads at once."""
    rng, rows, H, D = np.random.default_rng(5 + t), 2048, 16, 128
    f = np.float32
    q, k, v = (Rows(eng, coded(rng.standard_normal((rows, H * D)), t), t) for _ in range(3))
    g, st = Dev(eng, (-0.1 * rng.random((rows, H))).astype(f)), rng.standard_normal((1, H, D, D)).astype(f)
    first = None
    for i in range(12):
        print(f"repeats t={t} {i}", flush=True)
        O, S = out_rows(eng, (rows, H * D), t), Dev(eng, st)
        eng.decay_attention(O.ptr, q.ptr, k.ptr, v.ptr, rows, H, D, D, gates=g.ptr, state=S.ptr, dtype=t)
        eng.sync()
        got = O.get().view(np.uint8), S.get().view(np.uint8)
        first = first or got
        assert (got[0] == first[0]).all() and (got[1] == first[1]).all()


# ---- range ----------------------------------------------------------------------------------


def far_states(eng, t, H, lens, log_decay, state, scale, keys=5, q_from=0):  # noqa: F811
    """Rows whose keys are 0 but for the last `keys` of each sequence, and whose queries are 0 before row q_from of it, at
    log decays [rows]; against the recurrence.

    An exponent of a chunk of 32 rows rounds to fp32, half a step (U) relative of at most 32 * 2 / ln 2, which is 64 U of its
    exponential (a factor between tiles: 2 U), and the recurrence's own bound counts 3 U a row, 96 U a chunk."""
    rng, D, rows, f = np.random.default_rng(t + H + len(lens)), 8, sum(lens), np.float32
    print(f"far states t={t} H={H} lens={lens} scale={scale}", flush=True)
    q, k, v = (value(coded(rng.standard_normal((rows, H, D)), t), t) for _ in range(3))
    at = np.concatenate([np.arange(n) for n in lens])
    k[at < np.repeat(lens, lens) - keys] = 0
    q[at < q_from] = 0
    gates = np.broadcast_to(np.asarray(log_decay, f)[:, None], (rows, H))
    st = (state * (1 + rng.random((len(lens), H, D, D)))).astype(f)
    out, got = attention(eng, t, q, k, v, lens, state=st, gates=np.ascontiguousarray(gates), scale=scale)
    want, bound, new, err = decay_ref(q, k, v, gates, st, lens, float(f(scale)))
    most = np.abs(new).max(), np.abs(want).max()
    assert most[0] < 3e38 and most[1] < 60000
    close(out, want, bound, t, "out")
    close(got, new, err, F32, "state")


# one tile, tiles of 64 rows, both in a call, tiles of 128 rows
FAR = [(1, [128]), (1, [256]), (1, [128, 300]), (16, [2048])]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("H,lens", FAR)
def test_states_that_grow_past_a_tile(eng, H, lens, t):  # noqa: F811
    """A small state grows by e^126 over a tile's rows, more than fp32 holds, and stays finite; it is e^126 smaller in the end."""
    a = np.concatenate([np.where(np.arange(n) < 63, 2.0, np.where(np.arange(n) < 126, -2.0, 0.0)) for n in lens])
    far_states(eng, t, H, lens, a, 1e-30, 1e-25)
    a = np.concatenate([np.where(np.arange(n) < 63, 2.0, 0.0) for n in lens])
    far_states(eng, t, H, lens, a, 1e-30, 1e-25)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("H,lens", FAR)
def test_states_that_shrink_past_a_tile(eng, H, lens, t):  # noqa: F811
    """A large state shrinks by e^-96 over a tile's rows, less than fp32 holds, and is still a number."""
    a = np.concatenate([np.where(np.arange(n) < 64, -1.5, 0.0) for n in lens])
    far_states(eng, t, H, lens, a, 1e30, 1e12, keys=0, q_from=64)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("H,lens", FAR)
def test_forgotten_states_do_not_grow_back(eng, H, lens, t):  # noqa: F811
    """A log decay of -infinity before rows that grow."""
    a = np.concatenate([np.where(np.arange(n) < 1, -np.inf, np.where(np.arange(n) < 128, 2.0, 0.0)) for n in lens])
    far_states(eng, t, H, lens, a, 1e35, 1.0)

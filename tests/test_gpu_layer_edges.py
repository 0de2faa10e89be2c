"""The layer operators at the edges of their launch plans, against plain numpy in 64 bits."""
import numpy as np
import pytest

from test_gpu_layer import BF16, F16, F32, FLOATS, I8, U, W4, Rows, coded, out_rows, run_norm, run_w4, value
from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu


# ---- norm -----------------------------------------------------------------------------------


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n", range(1, 9))
def test_norm_vectors_of_a_thread(eng, n, t):  # noqa: F811
    """Rows that a block's 256 threads, and from 2048 rows on a wave's 64, hold in n vectors of 16 bytes each."""
    rng = np.random.default_rng(100 * n + t)
    V = 4 if t == F32 else 8
    full = n * 256 * V
    for cols in (full - V, full - 1, full + 1):
        run_norm(eng, rng, t, 3, cols)
    full = n * 64 * V
    for cols in (full - 1, full + 1):
        run_norm(eng, rng, t, 2048, cols, y=False)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("cols", [1600, 1792, 2816, 3500, 3584, 5632, 6145, 6912, 7168, 8192, 12289,
                                  13824, 14336, 16384, 16385, 32768, 32769])
def test_norm_widths(eng, cols, t):  # noqa: F811
    rng = np.random.default_rng(cols + t)
    run_norm(eng, rng, t, 2, cols, pads=(1, 0, 2, 0, 3), offs=(1, 0, 1, 0, 1))
    if cols < 7000:
        run_norm(eng, rng, t, 2050, cols, h=False, y=False)


# ---- 4-bit products ---------------------------------------------------------------------------


def test_w4_groups_beyond_the_row(eng):  # noqa: F811
    """A group of any size that holds the row is one group a row, and is the shape that is given back."""
    rng = np.random.default_rng(30)
    for group in (96, 2 ** 20, 2 ** 31 - 32, 2 ** 31, 2 ** 32, 2 ** 32 + 32, 2 ** 62):
        for t in (F32, I8):
            run_w4(eng, rng, t, 3, 77, 21, group, zeros=True)
    with pytest.raises(ValueError, match="negative"):
        eng.register_w4(np.zeros((4, 10), np.uint8), np.zeros((4, 0), np.float16), K=20, group=-32)


def way(t, rows, K, N):
    """The kernel of a product (w4_way): of few rows, of few rows laid out, by tiles of many."""
    work = rows * K * N
    if rows > 16 and work > (1.6e9 if t == F32 else 2.5e9):
        return "tiles"
    return "laid" if t == F32 and rows > 5 and work > 0.102e9 else "few"


WAYS = [(F32, "few", 1, 2048, 700), (F32, "few", 12, 1031, 700), (F32, "laid", 16, 2048, 8192), (F32, "laid", 20, 2048, 8192),
        (F32, "tiles", 90, 4100, 8001), (BF16, "few", 3, 2048, 700), (BF16, "few", 40, 1031, 700), (BF16, "tiles", 90, 4100, 8001),
        (F16, "few", 3, 2048, 700), (F16, "few", 40, 1031, 700), (F16, "tiles", 130, 1600, 13000)]


def product(eng, w, t, x):  # noqa: F811
    """(fp32 outputs of the rows x, which are in t's storage, the exact ones, sums of the terms' magnitudes)."""
    rows, K = x.shape
    X, O = Rows(eng, x, t), out_rows(eng, (rows, w.w.shape[0]), F32)
    eng.w4_linear(w.id, X.ptr, O.ptr, rows, dtype=t, out_dtype=F32)
    eng.sync()
    xv = value(x, t).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return O.get(), xv @ w.w.T, np.abs(xv) @ np.abs(w.w).T


@pytest.mark.parametrize("t,how,rows,K,N", WAYS)
@pytest.mark.parametrize("group", [32, 64, 128, 0])
def test_w4_large_input_at_weights_of_zero(eng, t, how, rows, K, N, group):  # noqa: F811
    """An input 1e4 times the others that meets weights of 0 leaves the others' sum alone: an output is off by the
    roundings of its own terms. These are U of partial sums below the sum of magnitudes: at most 4 * 6 inside a
    chunk's matrix instructions, of a chunk's share, and one for each scale. Independent, for 4100 inputs with a scale
    for 32: sqrt(129 + 24 / 33) / sqrt(3) = 7 U at one standard deviation if each partial sum were the whole sum.
    fp32 rows in two parts add U for each input, and 2^-40 * 1e4 / 0.8 < 0.2 U of the others."""
    assert way(t, rows, K, N) == how
    print(f"zero weights t={t} {how} rows={rows} K={K} N={N} group={group}", flush=True)
    rng = np.random.default_rng(rows + K + group)
    w = W4(eng, rng, N, K, group, True)
    eng.w4_release(w.id)
    size = group or K
    for k in (5, K - 1):
        w.q[:, k] = w.z[:, k // size]
        w.w[:, k] = 0
    q = np.concatenate([w.q, np.zeros((N, K % 2), np.uint8)], 1)
    w.id = eng.register_w4(q[:, 0::2] | (q[:, 1::2] << 4), w.s, w.z, K=K, group=group)
    x = rng.standard_normal((rows, K))
    x[:, 5], x[:, K - 1] = 1e4, -2e4
    got, want, mag = product(eng, w, t, coded(x, t))
    assert (np.abs(got - want) <= 17 * U * mag).all(), (np.abs(got - want) / (U * mag)).max()
    eng.w4_release(w.id)


@pytest.mark.parametrize("t,how,rows,K,N", [c for c in WAYS if c[0] != F16])
@pytest.mark.parametrize("group", [32, 128])
def test_w4_ranges_by_kernel(eng, t, how, rows, K, N, group):  # noqa: F811
    """Rows from 1e-30 to 1e30 keep their digits, and so do inputs of one row that lie far apart, down to 2^-40 of the
    largest of their run's group; rows of 1e35 throughout stay finite. Bounds as above."""
    assert way(t, rows, K, N) == how
    print(f"ranges t={t} {how} rows={rows} K={K} N={N} group={group}", flush=True)
    rng = np.random.default_rng(rows + group)
    w = W4(eng, rng, N, K, group, True)
    x = rng.standard_normal((rows, K)) * 10.0 ** np.linspace(-28, 30, rows)[:, None]
    got, want, mag = product(eng, w, t, coded(x, t))
    assert (np.abs(got - want) <= 17 * U * mag).all(), (np.abs(got - want) / (U * mag)).max(1)
    x = rng.standard_normal((rows, K)) * 2.0 ** rng.integers(-45, 1, (rows, K))
    got, want, mag = product(eng, w, t, coded(x, t))
    # (the largest input of any run is below 2^3)
    assert (np.abs(got - want) <= 17 * U * mag + 2.0 ** -37 * np.abs(w.w).sum(1)).all()
    x = np.full((rows, K), 1e35) * rng.choice([-1, 1], (rows, 1))
    got, want, mag = product(eng, w, t, coded(x, t))
    over = np.abs(want) > 3e38  # an output beyond fp32
    assert (np.abs(got - want)[~over] <= (17 * U * mag)[~over]).all()
    eng.w4_release(w.id)


@pytest.mark.parametrize("t,how,rows,K,N", WAYS)
def test_w4_rows_without_a_number(eng, t, how, rows, K, N):  # noqa: F811
    """A row with an infinity or NaN has no finite output, wherever it stands, and the other rows keep their bits."""
    assert way(t, rows, K, N) == how
    print(f"infinities t={t} {how} rows={rows} K={K} N={N}", flush=True)
    rng = np.random.default_rng(rows)
    w = W4(eng, rng, N, K, 64, True)
    x = rng.standard_normal((rows, K))
    got, _, _ = product(eng, w, t, coded(x, t))
    hurt = sorted({0, rows // 2, rows - 1})
    for r, v in zip(hurt, (np.inf, np.nan, -np.inf)):
        x[r, (7 * r + 3) % K if r else K - 1] = v
    again, _, _ = product(eng, w, t, coded(x, t))
    assert not np.isfinite(again[hurt]).any()
    keep = np.setdiff1d(np.arange(rows), hurt)
    assert (again[keep] == got[keep]).all()
    eng.w4_release(w.id)


@pytest.mark.parametrize("how,rows,K,N", [c[1:] for c in WAYS if c[0] == F16])
def test_w4_fp16_range(eng, how, rows, K, N):  # noqa: F811
    """fp16 rows below fp16's normal range and at its largest values."""
    assert way(F16, rows, K, N) == how
    rng = np.random.default_rng(rows)
    w = W4(eng, rng, N, K, 64, True)
    for x in (rng.integers(-8, 9, (rows, K)) * 2.0 ** -24, rng.choice([-65504.0, 65504.0], (rows, K)), np.full((rows, K), 65504.0)):
        got, want, mag = product(eng, w, F16, coded(x, F16))
        assert (np.abs(got - want) <= 17 * U * mag).all()
    eng.w4_release(w.id)


# ---- selective scan ---------------------------------------------------------------------------


def test_scan_growth_beyond_fp32(eng):  # noqa: F811
    """A rate of +infinity, or one that grows past fp32, leaves its state infinite at every length, also where the last
    group of steps is ragged; a NaN rate stays NaN, and other channels keep their numbers."""
    rng = np.random.default_rng(17)
    D, N = 70, 16
    for T in (1, 2, 3, 4, 5, 31, 33, 69):
        print(f"growth T={T}", flush=True)
        u, dt = rng.standard_normal((T, D)).astype(np.float32), np.full((T, D), 0.5, np.float32)
        B, Cm = (rng.standard_normal((T, N)).astype(np.float32) for _ in range(2))
        A = -np.ones((D, N), np.float32)
        A[3], A[9], A[20] = np.inf, 3e38, np.nan
        d = {k: Dev(eng, v) for k, v in dict(u=u, dt=dt, B=B, C=Cm, A=A).items()}
        S, O = Dev(eng, np.ones((1, N, D), np.float32)), Dev(eng, shape=(T, D))
        eng.selective_scan(O.ptr, d["u"].ptr, d["dt"].ptr, d["A"].ptr, d["B"].ptr, d["C"].ptr, T, D, N, state=S.ptr,
                           softplus=False)
        eng.sync()
        o, s = O.get(), S.get()[0]
        assert (s[:, [3, 9]] == np.inf).all() and not np.isfinite(o[:, [3, 9]]).any()
        assert np.isnan(s[:, 20]).all() and np.isnan(o[:, 20]).all()
        others = np.setdiff1d(np.arange(D), [3, 9, 20])
        assert np.isfinite(s[:, others]).all() and np.isfinite(o[:, others]).all()

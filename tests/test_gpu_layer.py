"""The layer operators (norm with int8 codes, 4-bit products, short convolution, selective scan)
against plain numpy in 64 bits: sizes on both sides of every tile, odd strides and addresses, all
types, empty and one-row sequences, carried states, captured graphs.

u = 2^-24 is fp32's half step; an output of type t is off by half a step of its type more.
"""
import ctypes as C

import numpy as np
import pytest

from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu

F32, BF16, F16, I8 = 0, 1, 2, 3
FLOATS = [F32, BF16, F16]
U = 2.0 ** -24
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}  # half a step, relative
TINY = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -25}  # below the normal range: half a step, absolute
STORE = {F32: np.float32, BF16: np.uint16, F16: np.float16, I8: np.int8}
SENTINEL = 0x5A


def coded(a, t):
    """float array -> the type's storage (to nearest, ties to even)."""
    a = np.asarray(a)
    if t != BF16:
        with np.errstate(over="ignore"):  # fp16 beyond 65504: infinity
            return a.astype(STORE[t])
    b = np.ascontiguousarray(a, np.float32).view(np.uint32)
    up = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), up)


def value(a, t):
    """Storage -> float32 values."""
    if t != BF16:
        return a.astype(np.float32)
    return (a.astype(np.uint32) << 16).view(np.float32)


class Rows:
    """A [rows, cols] tensor on the device, `pad` elements longer from row to row, `off` elements past an
    aligned address, in memory filled with a pattern that has to stay around it."""

    def __init__(self, eng, a, t, pad=0, off=0):  # noqa: F811
        self.t, (self.rows, self.cols) = t, a.shape
        self.ld, self.off = self.cols + pad, off
        host = np.full((off + self.rows * self.ld + 64) * np.dtype(STORE[t]).itemsize, SENTINEL, np.uint8)
        self.host = host.view(STORE[t])
        self._in(self.host)[:] = a
        self.dev = Dev(eng, self.host)
        self.ptr = self.dev.ptr + off * self.host.itemsize

    def _in(self, flat):
        return flat[self.off:self.off + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def get(self):
        got = self.dev.get()
        around = got.copy()
        self._in(around)[:] = self._in(self.host)
        assert (around.view(np.uint8) == self.host.view(np.uint8)).all(), "memory around the tensor was written"
        return self._in(got).copy()


def out_rows(eng, shape, t, pad=0, off=0):  # noqa: F811
    a = np.empty(shape, STORE[t])
    a.view(np.uint8)[...] = SENTINEL
    return Rows(eng, a, t, pad, off)


def close(got, want, bound, t, what):
    """|got - want| <= bound + half a step of the type, element by element; NaN and infinities alike."""
    got = np.asarray(got, np.float64)
    tol = bound + HALF[t] * 1.001 * (np.abs(want) + bound) + TINY[t]
    off = np.abs(got - want)
    with np.errstate(invalid="ignore"):
        bad = ~((off <= tol) | (np.isnan(want) & np.isnan(got)) | (got == want))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.size} off; first {i}: {got[i]!r} for {want[i]!r}, "
                             f"allowed {tol[i]!r}")


# ---- norm -----------------------------------------------------------------------------------


def norm_ref(x, res, w, eps):
    """h (fp32), y, codes' real values and scales in 64 bits, from fp32 inputs."""
    with np.errstate(all="ignore"):
        h = x + res if res is not None else x.copy()  # one fp32 rounding
        d = h.astype(np.float64)
        rstd = 1.0 / np.sqrt((d * d).mean(1, keepdims=True) + np.float64(np.float32(eps)))
        y = d * w.astype(np.float64) * rstd
        m = np.maximum(np.abs(y).max(1, keepdims=True), 1e-5)
    return h, y, y * 127.0 / m, (m / 127.0)[:, 0]


def run_norm(eng, rng, t, rows, cols, res=True, h=True, y=True, pads=(0, 0, 0, 0, 0), offs=(0, 0, 0, 0, 0), in_place=None,  # noqa: F811
             x=None, w=None, eps=1e-6):
    print(f"norm t={t} rows={rows} cols={cols} res={res} h={h} y={y} pads={pads} offs={offs} {in_place}", flush=True)
    x = (rng.standard_normal((rows, cols)) * 0.5).astype(np.float32) if x is None else x
    r = (rng.standard_normal((rows, cols)) * np.where(rng.random(cols) < 0.02, 30, 2)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32) if w is None else w
    X, R = Rows(eng, coded(x, t), t, pads[0], offs[0]), Rows(eng, coded(r, t), t, pads[1], offs[1]) if res else None
    H, Y = out_rows(eng, (rows, cols), t, pads[2], offs[2]), out_rows(eng, (rows, cols), t, pads[3], offs[3])
    Q, S = out_rows(eng, (rows, cols), I8, pads[4], offs[4]), out_rows(eng, (rows, 1), F32)
    W = Rows(eng, w[None], F32, 0, offs[0])
    if in_place:
        H = {"x": X, "res": R}[in_place]
    eng.add_rmsnorm_q8(Q.ptr, S.ptr, X.ptr, W.ptr, rows, cols, res=R.ptr if res else None, h=H.ptr if h else None,
                       y=Y.ptr if y else None, eps=eps, dtype=t, ldx=X.ld, ldres=R.ld if res else 0, ldh=H.ld, ldy=Y.ld,
                       ldcodes=Q.ld)
    eng.sync()
    hw, yw, real, scale = norm_ref(value(coded(x, t), t), value(coded(r, t), t) if res else None, w, eps)
    q, s = Q.get().astype(np.float64), S.get()[:, 0]
    if h:
        assert (H._in(H.dev.get()) == coded(hw, t)).all() if in_place else (H.get() == coded(hw, t)).all(), "h"
    # the code is the nearest integer in 64 bits: 2^-40 for the sums' own rounding
    assert (np.abs(q - real) <= 0.5 + 2.0 ** -40 * 127).all(), np.abs(q - real).max()
    assert (np.abs(s - scale) <= U * 1.001 * scale).all()
    if y:
        close(value(Y.get(), t), yw, U * np.abs(yw), t, "y")


# around the lengths that one thread, one wave and one block hold, and beyond all registers
NORM_COLS = [1, 3, 7, 64, 100, 255, 256, 257, 511, 1024, 1031, 2048, 2050, 4095, 4097, 8192, 8200, 16391, 40000]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("cols", NORM_COLS)
def test_norm_lengths(eng, cols, t):  # noqa: F811
    rng = np.random.default_rng(cols)
    run_norm(eng, rng, t, 5, cols)
    run_norm(eng, rng, t, 3, cols, pads=(1, 2, 3, 5, 1), offs=(1, 3, 5, 2, 1))
    run_norm(eng, rng, t, 1, cols, res=False, h=False, y=False)
    run_norm(eng, rng, t, 2, cols, in_place="res")
    run_norm(eng, rng, t, 2, cols, in_place="x", y=False)


@pytest.mark.parametrize("t", FLOATS)
def test_norm_many_rows(eng, t):  # noqa: F811
    rng = np.random.default_rng(4)
    for rows, cols in ((1000, 70), (700, 1030), (2100, 256), (600, 2560)):
        run_norm(eng, rng, t, rows, cols, pads=(2, 0, 4, 0, 3))


def test_norm_special_rows(eng):  # noqa: F811
    """Zero rows keep the smallest scale; rows with an infinity or NaN have NaN for a scale and codes 0;
    huge and tiny rows do not overflow or vanish in their squares."""
    rng = np.random.default_rng(9)
    rows, cols = 7, 300
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= np.float32(1e-30)
    x[3, 7], x[4, 299], x[5, 0] = np.inf, np.nan, -np.inf
    w = np.ones(cols, np.float32)
    X, W = Rows(eng, x, F32), Rows(eng, w[None], F32)
    Q, S, Y = out_rows(eng, (rows, cols), I8), out_rows(eng, (rows, 1), F32), out_rows(eng, (rows, cols), F32)
    eng.add_rmsnorm_q8(Q.ptr, S.ptr, X.ptr, W.ptr, rows, cols, y=Y.ptr)
    eng.sync()
    q, s = Q.get(), S.get()[:, 0]
    _, yw, real, scale = norm_ref(x, None, w, 1e-6)
    fine = [0, 1, 2, 6]
    assert np.isnan(s[[3, 4, 5]]).all() and (q[[3, 4, 5]] == 0).all()
    assert (q[0] == 0).all() and s[0] == np.float32(1e-5 / 127.0)
    assert (np.abs(s[fine] - scale[fine]) <= U * 1.001 * scale[fine]).all()
    assert (np.abs(q[fine] - real[fine]) <= 0.5 + 1e-9).all()
    close(Y.get()[fine], yw[fine], U * np.abs(yw[fine]), F32, "y")


def test_norm_codes_are_the_products_input(eng):  # noqa: F811
    """The codes equal the Int8Absmax ones of the engine's own rule wherever fp32 rounding leaves no
    choice: both round y * 127 / max|y|, and differ only where that is within 1e-3 of a half."""
    rng = np.random.default_rng(12)
    rows, cols = 16, 1000
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float32)
    X, W, Y = Rows(eng, x, F32), Rows(eng, w[None], F32), out_rows(eng, (rows, cols), F32)
    Q, S = out_rows(eng, (rows, cols), I8), out_rows(eng, (rows, 1), F32)
    eng.rmsnorm(Y.ptr, X.ptr, W.ptr, rows, cols)
    eng.add_rmsnorm_q8(Q.ptr, S.ptr, X.ptr, W.ptr, rows, cols)
    eng.sync()
    y = Y.get()
    sa = np.float32(127) / np.maximum(np.abs(y).max(1, keepdims=True), np.float32(1e-5))
    scaled = (y * sa).astype(np.float32)
    sure = np.abs(np.abs(scaled - np.rint(scaled)) - 0.5) > 1e-3
    assert (Q.get()[sure] == np.rint(scaled)[sure]).all()


# ---- 4-bit products ---------------------------------------------------------------------------


class W4:
    def __init__(self, eng, rng, N, K, group, zeros, exact=False):  # noqa: F811
        G = -(-K // group) if group else 1
        self.q = rng.integers(0, 16, (N, K)).astype(np.uint8)
        self.z = rng.integers(0, 16, (N, G)).astype(np.uint8) if zeros else None
        # exact: powers of two, so that products and sums of small integers have no rounding at all
        self.s = (2.0 ** rng.integers(-3, 3, (N, G)) if exact else 0.01 * (0.5 + rng.random((N, G)))).astype(np.float16)
        q = np.concatenate([self.q, np.zeros((N, K % 2), np.uint8)], 1)
        self.id = eng.register_w4(q[:, 0::2] | (q[:, 1::2] << 4), self.s, self.z, K=K, group=group)
        at = np.arange(K) // (group or K)
        self.v = self.q.astype(np.float64) - (self.z[:, at].astype(np.float64) if zeros else 8.0)  # integers
        self.w = self.v * self.s.astype(np.float64)[:, at]
        assert eng.w4_shape(self.id) == (N, K, group or K)


def run_w4(eng, rng, t, rows, K, N, group, zeros, out_t=F32, exact=True, padx=0, offx=0, pado=0, offo=0):  # noqa: F811
    print(f"w4 t={t} rows={rows} K={K} N={N} group={group} zeros={zeros} out={out_t} exact={exact} "
          f"{padx, offx, pado, offo}", flush=True)
    w = W4(eng, rng, N, K, group, zeros, exact)
    if t == I8:
        x = rng.integers(-128, 128, (rows, K)).astype(np.int8)
        xs = (2.0 ** rng.integers(-4, 2, (rows, 1)) if exact else 0.02 + 0.03 * rng.random((rows, 1))).astype(np.float32)
    else:
        x = coded(rng.integers(-4, 5, (rows, K)) if exact else rng.standard_normal((rows, K)), t)
        xs = None
    X, O = Rows(eng, x, t, padx, offx), out_rows(eng, (rows, N), out_t, pado, offo)
    S = Rows(eng, xs, F32) if t == I8 else None
    eng.w4_linear(w.id, X.ptr, O.ptr, rows, dtype=t, out_dtype=out_t, scales=S.ptr if S else None, ldx=X.ld, ldo=O.ld)
    eng.sync()
    xv = value(x, t).astype(np.float64)
    want = xv @ w.w.T
    if t == I8:
        want = want * xs
    got = value(O.get(), out_t)
    if exact:
        # all terms are integers times 2^-3 (int8: 2^-7), and their sums stay below 2^24 of that unit:
        # every order of summation gives the sum itself
        assert np.abs(xv).sum(1).max() * 15 * 4 * (128 if t == I8 else 8) < 2 ** 24 or t == I8
        ref = value(coded(want.astype(np.float32), out_t), out_t) if t != I8 else None
        if t != I8:
            assert (got == ref).all(), (np.argwhere(got != ref)[:3], got[got != ref][:3], ref[got != ref][:3])
        else:  # exact integers per group, then an fp32 sum over the groups: G + 2 roundings
            G = -(-K // group) if group else 1
            mag = np.abs(xv) @ np.abs(w.w.T) * xs
            rounded = value(coded(want.astype(np.float32), out_t), out_t)
            want = np.where(np.isinf(rounded), rounded, want)  # beyond fp16's largest value, 65504
            close(got, want, U * (-(-K // 32) + 3) * mag, out_t, "w4 int8")
    else:
        # each of the sums' roundings is half a step of a partial sum, and these stay below the sums of
        # magnitudes: 128 / 4 additions inside a group at most, and one per group and split, all of
        # |x| (|q - z| + 32) s. Independent, so their squares add: 4 standard deviations, as a norm.
        assert np.linalg.norm(got - want) <= (4e-6 + HALF[out_t]) * np.linalg.norm(want)
        at = np.arange(K) // (group or K)
        mag = np.abs(xv) @ ((np.abs(w.v) + 32) * w.s.astype(np.float64)[:, at]).T * (xs if t == I8 else 1)
        close(got, want, U * 16 * mag, out_t, "w4")
    eng.w4_release(w.id)


W4_SHAPES = [(1, 1, 1), (1, 64, 16), (1, 2048, 64), (2, 77, 33), (3, 128, 17), (5, 129, 40), (6, 300, 100), (8, 96, 31),
             (16, 1031, 70), (17, 256, 48), (21, 160, 129), (33, 500, 65), (64, 384, 200), (65, 130, 16), (100, 1031, 133),
             (130, 640, 257)]


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
@pytest.mark.parametrize("group", [32, 64, 128, 0, 96, 256])
def test_w4_layouts(eng, t, group):  # noqa: F811
    """Sums without rounding: any misplaced code, scale, zero point or row shows."""
    rng = np.random.default_rng(group + t)
    for i, (rows, K, N) in enumerate(W4_SHAPES):
        run_w4(eng, rng, t, rows, K, N, group, zeros=i % 2 == 0, padx=i % 3, offx=i % 5, pado=i % 4, offo=i % 2)


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
def test_w4_many_rows(eng, t):  # noqa: F811
    rng = np.random.default_rng(t)
    for rows, K, N, group in ((300, 256, 144, 128), (257, 1000, 300, 32), (513, 192, 1100, 64), (1030, 70, 40, 0)):
        run_w4(eng, rng, t, rows, K, N, group, zeros=True, padx=3, pado=1)


@pytest.mark.parametrize("group", [32, 64, 128, 0])
def test_w4_laid_rows(eng, group):  # noqa: F811
    """fp32 rows that are laid out for the kernel of few rows: one and two column tiles, one and two output tiles."""
    rng = np.random.default_rng(60 + group)
    for i, (rows, K, N) in enumerate(((7, 5000, 4400), (16, 9001, 1200), (17, 2049, 4500), (50, 1031, 3000))):
        run_w4(eng, rng, F32, rows, K, N, group, zeros=i % 2 == 0, padx=i, offx=1, pado=3, out_t=FLOATS[i % 3])


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
@pytest.mark.parametrize("i", [0, 1, 2])
def test_w4_tiles(eng, t, i):  # noqa: F811
    """Products of many rows: inputs split over blocks, over a block's waves, and not at all."""
    rng = np.random.default_rng(70 + t)
    rows, K, N = ((80, 4100, 8001), (131, 1301, 16300), (701, 600, 6500))[i]
    for k in (0, 1):
        group = (32, 64, 128, 0)[(t + i + 2 * k) % 4]
        run_w4(eng, rng, t, rows, K, N, group, zeros=k == 0, padx=k, pado=1 - k, out_t=F32 if k else FLOATS[(t + i) % 3])


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_tiles_of_every_step(eng, t, group):  # noqa: F811
    """Many rows with scales for 32, 64 and 128 inputs: few outputs and many, inputs in one run and in several."""
    rng = np.random.default_rng(90 + group + t)
    for i, (rows, K, N) in enumerate(((3100, 6900, 120), (90, 4100, 8001), (701, 600, 6500), (700, 2000, 2100),
                                      (1515, 737, 2809))):
        run_w4(eng, rng, t, rows, K, N, group, zeros=i % 2 == 0, padx=i, pado=i % 3)


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
@pytest.mark.parametrize("out_t", FLOATS)
def test_w4_rounding(eng, t, out_t):  # noqa: F811
    """Real inputs: the fp32 rows keep all their digits."""
    rng = np.random.default_rng(17 + t + out_t)
    for rows, K, N in ((1, 2048, 130), (4, 6912, 48), (24, 1031, 70), (70, 512, 100), (300, 640, 160), (90, 2048, 1100),
                       (130, 1600, 13000)):
        run_w4(eng, rng, t, rows, K, N, group=[32, 64, 128][rows % 3], zeros=rows != 4, out_t=out_t, exact=False)


def test_w4_wide_range(eng):  # noqa: F811
    """fp32 rows from 1e-30 to 1e30 keep their digits, and rows do not touch each other."""
    rng = np.random.default_rng(3)
    w = W4(eng, rng, 50, 200, 32, True)
    x = (rng.standard_normal((9, 200)) * 10.0 ** np.linspace(-30, 30, 9)[:, None]).astype(np.float32)
    X, O = Rows(eng, x, F32), out_rows(eng, (9, 50), F32)
    eng.w4_linear(w.id, X.ptr, O.ptr, 9)
    eng.sync()
    want, got = x.astype(np.float64) @ w.w.T, O.get()
    for r in range(9):
        assert np.linalg.norm(got[r] - want[r]) <= 4e-6 * np.linalg.norm(want[r]), r
    x[2, 3], x[5, 199] = np.nan, np.inf
    X = Rows(eng, x, F32)
    eng.w4_linear(w.id, X.ptr, O.ptr, 9)
    eng.sync()
    again = O.get()
    assert not np.isfinite(again[[2, 5]]).any()
    keep = [0, 1, 3, 4, 6, 7, 8]
    assert (again[keep] == got[keep]).all()


@pytest.mark.parametrize("t", [F32, BF16, F16, I8])
def test_w4_long_rows_and_many(eng, t):  # noqa: F811
    """One row of many inputs; more rows than one launch or pass takes."""
    rng = np.random.default_rng(40 + t)
    run_w4(eng, rng, t, 1, 12000, 40, 128, zeros=True)
    run_w4(eng, rng, t, 3, 9999, 17, 32, zeros=False, padx=5)
    run_w4(eng, rng, t, 66000, 640 if t != F32 else 160, 64, 64, zeros=True, padx=1)


def test_w4_small_values(eng):  # noqa: F811
    """fp16 rows below fp16's normal range, and fp32 rows whose largest input is 1e6 times the others, by both kernels."""
    rng = np.random.default_rng(41)
    for rows, K, N in ((3, 256, 48), (40, 2048, 8192)):
        w = W4(eng, rng, N, K, 64, True)
        x = (rng.integers(-8, 9, (rows, K)) * 2.0 ** -24).astype(np.float16)
        X, O = Rows(eng, x, F16), out_rows(eng, (rows, N), F32)
        eng.w4_linear(w.id, X.ptr, O.ptr, rows, dtype=F16)
        eng.sync()
        want = x.astype(np.float64) @ w.w.T
        assert np.linalg.norm(O.get() - want) <= 4e-6 * np.linalg.norm(want)
        x = rng.standard_normal((rows, K)).astype(np.float32)
        x[:, 5] *= 1e6
        X = Rows(eng, x, F32)
        eng.w4_linear(w.id, X.ptr, O.ptr, rows)
        eng.sync()
        # less the large input's own share, which is exact in fp32 to half a step of it: what is left of the
        # others is off by a few steps of the sum's size at most
        want = x.astype(np.float64) @ w.w.T
        assert (np.abs(O.get() - want) <= 16 * U * (np.abs(x[:, 5:6] * w.w[:, 5]) + np.linalg.norm(want) / np.sqrt(want.size))).all()


def test_offsets_beyond_32_bits(eng):  # noqa: F811
    """Rows 2.4 GB apart: the same outputs as of neighbouring rows."""
    rng = np.random.default_rng(42)
    cols, ld = 100, 1_200_000_000
    x = coded(rng.standard_normal((3, cols)), BF16)
    near = Rows(eng, x, BF16)
    p = C.c_void_p()
    eng._chk(eng.lib.mmf_malloc(eng.h, C.byref(p), (2 * ld + cols) * 2))
    try:
        for r in range(3):
            row = np.ascontiguousarray(x[r])
            eng._chk(eng.lib.mmf_upload(eng.h, p.value + 2 * r * ld, row.ctypes.data_as(C.c_void_p), row.nbytes))
        w, f = W4(eng, rng, 30, cols, 32, True), np.float32
        nw, cw = Dev(eng, np.ones(cols, f)), Dev(eng, rng.standard_normal((cols, 4)).astype(f))
        A = Dev(eng, -np.ones((cols, 16), f))
        B = Rows(eng, coded(rng.standard_normal((3, 16)), BF16), BF16)
        for what in ("norm", "w4", "conv", "scan"):
            got = []
            for ptr, step in ((near.ptr, cols), (p.value, ld)):
                O, S = out_rows(eng, (3, cols if what != "w4" else 30), I8 if what == "norm" else BF16), out_rows(eng, (3, 1), F32)
                if what == "norm":
                    eng.add_rmsnorm_q8(O.ptr, S.ptr, ptr, nw.ptr, 3, cols, dtype=BF16, ldx=step)
                elif what == "w4":
                    eng.w4_linear(w.id, ptr, O.ptr, 3, dtype=BF16, out_dtype=BF16, ldx=step)
                elif what == "conv":
                    eng.short_conv(O.ptr, ptr, cw.ptr, 3, cols, 4, dtype=BF16, ldx=step)
                else:
                    eng.selective_scan(O.ptr, ptr, ptr, A.ptr, B.ptr, B.ptr, 3, cols, 16, dtype=BF16, ldu=step, lddt=step)
                eng.sync()
                got.append(O.get())
            assert (got[0].view(np.uint8) == got[1].view(np.uint8)).all(), what
    finally:
        eng.lib.mmf_free(eng.h, p)


def test_w4_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    rng = np.random.default_rng(1)
    q, s = rng.integers(0, 255, (4, 32)).astype(np.uint8), np.ones((4, 2), np.float16)
    wid = eng.register_w4(q, s, group=32)
    x, o = Dev(eng, np.zeros((2, 64), np.float32)), Dev(eng, shape=(2, 4))
    for kw, why in ((dict(dtype=5), "dtype"), (dict(out_dtype=I8), "out_dtype"), (dict(ldx=63), "stride"),
                    (dict(dtype=I8), "scales")):
        with pytest.raises(MmfError, match=why):
            eng.w4_linear(wid, x.ptr, o.ptr, 2, **kw)
    with pytest.raises(MmfError, match="group"):
        eng.register_w4(q, np.ones((4, 2), np.float16), group=48)
    with pytest.raises(MmfError, match="zero points"):
        eng.register_w4(q, s, np.full((4, 2), 16, np.uint8), group=32)
    with pytest.raises(ValueError):
        eng.register_w4(q, s, group=64)
    eng.w4_release(wid)
    with pytest.raises(MmfError, match="released"):
        eng.w4_linear(wid, x.ptr, o.ptr, 2)
    with pytest.raises(MmfError, match="invalid w4_id"):
        eng.w4_shape(10 ** 6)


# ---- short convolution ------------------------------------------------------------------------


def silu(x):
    return x / (1.0 + np.exp(-x))


def conv_ref(x, w, bias, state, lens, act):
    """(out, error bound, new state) in 64 bits."""
    W = w.shape[1]
    outs, bounds, states, r = [], [], [], 0
    w = w.astype(np.float64)
    for s, n in enumerate(lens):
        ext = np.concatenate([state[s] if state is not None else np.zeros((W - 1, x.shape[1])), x[r:r + n]]).astype(np.float64)
        y = np.zeros((n, x.shape[1])) + (bias if bias is not None else 0)
        mag = np.abs(y)
        for j in range(W):
            y = y + ext[j:j + n] * w[:, j]
            mag = mag + np.abs(ext[j:j + n] * w[:, j])
        o = silu(y) if act else y
        # W roundings of sums below mag, through a slope of at most 1.1; silu's own 6 (exp, +, rcp, product)
        # and the exponent's product |y| log2(e) rounded twice
        outs.append(o)
        bounds.append(U * (1.1 * W * mag + (6 + 2 * np.abs(y)) * np.abs(o)) if act else U * W * mag)
        states.append(ext[n:])
        r += n
    return np.concatenate(outs), np.concatenate(bounds), np.stack(states)


def run_conv(eng, rng, t, lens, D, W, bias=True, state=True, act=True, pads=(0, 0), offs=(0, 0), seqs=None):  # noqa: F811
    print(f"conv t={t} lens={lens if len(lens) < 20 else len(lens)} D={D} W={W} {bias, state, act} {pads, offs}", flush=True)
    rows, n = sum(lens), len(lens)
    x = coded(rng.standard_normal((rows, D)) * 2, t)
    w = rng.standard_normal((D, W)).astype(np.float32)
    b = rng.standard_normal(D).astype(np.float32) if bias else None
    st = rng.standard_normal((n, W - 1, D)).astype(np.float32) if state else None
    X, O = Rows(eng, x, t, pads[0], offs[0]), out_rows(eng, (rows, D), t, pads[1], offs[1])
    WD, B = Rows(eng, w, F32, 0, offs[0]), Rows(eng, b[None], F32, 0, offs[1]) if bias else None
    S = Rows(eng, st.reshape(1, -1), F32, 0, offs[0]) if state and W > 1 else None
    want, bound, new = conv_ref(value(x, t), w, b, st, lens, act)
    eng.short_conv(O.ptr, X.ptr, WD.ptr, rows, D, W, bias=B.ptr if bias else None, state=S.ptr if S else None,
                   lens=None if seqs else lens, seqs=seqs or 1, silu=act, dtype=t, ldx=X.ld, ldo=O.ld)
    eng.sync()
    close(value(O.get(), t), want, bound, t, "conv")
    if S:
        assert (S.get().reshape(new.shape) == new).all(), "conv state"


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("W", [1, 2, 3, 4, 7, 8])
def test_conv_sequences(eng, t, W):  # noqa: F811
    rng = np.random.default_rng(W * 3 + t)
    run_conv(eng, rng, t, [1], 5, W)
    run_conv(eng, rng, t, [3, 0, 1, 2, 17, 0, 64, 9, 0], 100, W, pads=(3, 1), offs=(1, 3))
    run_conv(eng, rng, t, [8, 16, 7, 15, 33], 257, W, bias=False, pads=(5, 2), offs=(3, 1))
    run_conv(eng, rng, t, [40], 130, W, state=False, act=False)
    run_conv(eng, rng, t, [2, 0, 5], 64, W, state=False)


@pytest.mark.parametrize("t", FLOATS)
def test_conv_steps_and_many_sequences(eng, t):  # noqa: F811
    rng = np.random.default_rng(t)
    run_conv(eng, rng, t, [1] * 64, 512, 4, seqs=64)
    run_conv(eng, rng, t, [5] * 7, 1030, 4, seqs=7)
    run_conv(eng, rng, t, [int(n) for n in rng.integers(0, 6, 700)], 33, 4)  # several tables of sequences
    run_conv(eng, rng, t, [1] * 500, 40, 3)
    run_conv(eng, rng, t, [700, 300], 1111, 4, pads=(1, 0))


def test_conv_carries_its_state(eng):  # noqa: F811
    """A sequence in pieces gives what it gives at once."""
    rng = np.random.default_rng(8)
    D, W, T = 200, 4, 50
    x, w = rng.standard_normal((T, D)).astype(np.float32), rng.standard_normal((D, W)).astype(np.float32)
    X, WD, S = Dev(eng, x), Dev(eng, w), Dev(eng, np.zeros((W - 1, D), np.float32))
    whole, parts = Dev(eng, shape=(T, D)), Dev(eng, shape=(T, D))
    eng.short_conv(whole.ptr, X.ptr, WD.ptr, T, D, W)
    r = 0
    for n in (1, 1, 2, 9, 1, 30, 6):
        eng.short_conv(parts.ptr + 4 * r * D, X.ptr + 4 * r * D, WD.ptr, n, D, W, state=S.ptr)
        r += n
    eng.sync()
    assert r == T and (whole.get() == parts.get()).all()
    assert (S.get() == x[T - 3:]).all()


# ---- selective scan ---------------------------------------------------------------------------


def scan_ref(u, dt, A, B, C, skip, z, bias, state, lens, softplus):
    """(out, bound, state, its bound) in 64 bits; the bounds follow the roundings through the recurrence."""
    f = np.float64
    u, dt, A, B, C = (a.astype(f) for a in (u, dt, A.T, B, C))
    N, D = A.shape
    if bias is not None:
        dt = dt + bias
    # dt: the sum's rounding reaches softplus with its size, softplus itself has 6 of its own
    dmag = U * (np.abs(dt) + (np.abs(bias) if bias is not None else 0))
    if softplus:
        dt = np.maximum(dt, 0) + np.log1p(np.exp(-np.abs(dt)))
        dmag = np.minimum(dmag, dmag) + 8 * U * dt
    out, bound = np.zeros_like(u), np.zeros_like(u)
    new = np.zeros((len(lens), N, D))
    err = np.zeros_like(new)
    r = 0
    for s, n in enumerate(lens):
        h = state[s].astype(f) if state is not None else np.zeros((N, D))
        e = np.zeros_like(h)
        for p in range(r, r + n):
            a, b = np.exp(dt[p] * A), dt[p] * u[p] * B[p][:, None]
            # the exponent's relative roundings (3: A log2 e, its product, dt's sum over a chunk), exp's own 2,
            # the product with h; dt's error in both terms
            e = a * e + np.abs(a * h) * (U * (4 + 6 * np.abs(dt[p] * A)) + dmag[p] * np.abs(A)) \
                + np.abs(b) * U * 4 + dmag[p] * np.abs(u[p] * B[p][:, None])
            h = a * h + b
            e = e + U * np.abs(h)
            y = (C[p][:, None] * h).sum(0)
            ye = (np.abs(C[p])[:, None] * (e + U * N * np.abs(h))).sum(0)
            if skip is not None:
                y, ye = y + skip * u[p], ye + 2 * U * np.abs(skip * u[p]) + U * np.abs(y)
            if z is not None:
                g = silu(z[p].astype(f))
                y, ye = y * g, ye * np.abs(g) + U * (8 + 2 * np.abs(z[p])) * np.abs(y * g)
            out[p], bound[p] = y, ye
        new[s], err[s] = h, e
        r += n
    return out, bound, new, err


def run_scan(eng, rng, t, lens, D, N, skip=True, z=True, bias=True, state=True, softplus=True, pads=(0,) * 6,  # noqa: F811
             offs=(0,) * 6, seqs=None):
    print(f"scan t={t} lens={lens if len(lens) < 20 else len(lens)} D={D} N={N} {skip, z, bias, state, softplus} "
          f"{pads, offs}", flush=True)
    rows, n = sum(lens), len(lens)
    f = np.float32
    data = {"u": rng.standard_normal((rows, D)), "dt": rng.standard_normal((rows, D)) * 0.7 - (0 if bias else 2),
            "B": rng.standard_normal((rows, N)), "C": rng.standard_normal((rows, N)), "z": rng.standard_normal((rows, D)) * 2}
    if not softplus:
        data["dt"] = np.abs(data["dt"]) * 0.1
    data = {k: coded(v, t) for k, v in data.items()}
    A = (-np.arange(1, N + 1) * np.exp(0.1 * rng.standard_normal((D, N)))).astype(f)
    sk = rng.standard_normal(D).astype(f) if skip else None
    bi = (rng.standard_normal(D) * 0.5 - 3).astype(f) if bias and softplus else None
    st = rng.standard_normal((n, N, D)).astype(f) if state else None
    dev = {k: Rows(eng, v, t, pads[i], offs[i]) for i, (k, v) in enumerate(data.items())}
    O = out_rows(eng, (rows, D), t, pads[5], offs[5])
    AD = Rows(eng, A, F32, 0, offs[0])
    SK, BI = (Rows(eng, v[None], F32, 0, offs[1]) if v is not None else None for v in (sk, bi))
    S = Rows(eng, st.reshape(1, -1), F32, 0, offs[2]) if state else None
    v = {k: value(a, t) for k, a in data.items()}
    want, bound, new, err = scan_ref(v["u"], v["dt"], A, v["B"], v["C"], sk, v["z"] if z else None, bi, st, lens, softplus)
    eng.selective_scan(O.ptr, dev["u"].ptr, dev["dt"].ptr, AD.ptr, dev["B"].ptr, dev["C"].ptr, rows, D, N,
                       skip=SK.ptr if SK else None, z=dev["z"].ptr if z else None, dt_bias=BI.ptr if BI else None,
                       state=S.ptr if S else None, lens=None if seqs else lens, seqs=seqs or 1, softplus=softplus, dtype=t,
                       ldo=O.ld, ldu=dev["u"].ld, lddt=dev["dt"].ld, ldb=dev["B"].ld, ldc=dev["C"].ld, ldz=dev["z"].ld)
    eng.sync()
    close(value(O.get(), t), want, bound, t, "scan")
    if state:
        got = S.get().reshape(new.shape)
        for s, k in enumerate(lens):
            if not k:
                assert (got[s] == st[s]).all(), "state of an empty sequence"
        off = np.abs(got - new)
        assert (off <= err + U * np.abs(new) + 1e-37).all(), (off - err).max()


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("N", [1, 2, 4, 5, 8, 15, 16, 17, 24, 33, 64, 128])
def test_scan_states(eng, t, N):  # noqa: F811
    rng = np.random.default_rng(N * 3 + t)
    run_scan(eng, rng, t, [1], 3, N)
    run_scan(eng, rng, t, [1] * 9, 70, N, seqs=9, pads=(1, 2, 0, 3, 1, 2), offs=(1, 0, 3, 1, 2, 3))
    run_scan(eng, rng, t, [3, 0, 1, 20, 0, 40, 9], 100, N, pads=(3, 1, 2, 0, 5, 1), offs=(1, 3, 1, 5, 2, 1))
    run_scan(eng, rng, t, [33], 65, N, skip=False, z=False, bias=False, state=False)
    run_scan(eng, rng, t, [17, 5], 64, N, softplus=False)


@pytest.mark.parametrize("t", FLOATS)
def test_scan_long(eng, t):  # noqa: F811
    """Sequences that are cut into chunks, with ragged ends."""
    rng = np.random.default_rng(t)
    run_scan(eng, rng, t, [700], 130, 16)
    run_scan(eng, rng, t, [1000, 1, 0, 333, 64, 65], 64, 16, pads=(1,) * 6)
    run_scan(eng, rng, t, [1025], 33, 64, state=False)
    run_scan(eng, rng, t, [300, 511], 192, 5, z=False)
    run_scan(eng, rng, t, [513], 20, 128)


def test_scan_many_sequences(eng):  # noqa: F811
    rng = np.random.default_rng(5)
    run_scan(eng, rng, F32, [int(n) for n in rng.integers(0, 5, 600)], 40, 16)  # several tables of sequences
    run_scan(eng, rng, F32, [1] * 500, 70, 16)
    run_scan(eng, rng, F32, [12] * 300, 24, 4, seqs=300)
    run_scan(eng, rng, F32, [700] + [1, 0, 2] * 90 + [900, 400], 64, 16)  # chunks in two of the tables


def test_scan_strong_decay_and_large_steps(eng):  # noqa: F811
    """Decays that underflow to 0 forget the state; steps of exactly 0 keep it bit for bit."""
    rng = np.random.default_rng(6)
    T, D, N = 200, 64, 16
    u, dt = rng.standard_normal((T, D)).astype(np.float32), np.zeros((T, D), np.float32)
    B, Cm = (rng.standard_normal((T, N)).astype(np.float32) for _ in range(2))
    A = -np.ones((D, N), np.float32) * 50
    st = rng.standard_normal((1, N, D)).astype(np.float32)
    d = {k: Dev(eng, v) for k, v in dict(u=u, dt=dt, B=B, C=Cm, A=A).items()}
    S, O = Dev(eng, st), Dev(eng, shape=(T, D))
    eng.selective_scan(O.ptr, d["u"].ptr, d["dt"].ptr, d["A"].ptr, d["B"].ptr, d["C"].ptr, T, D, N, state=S.ptr,
                       softplus=False)
    eng.sync()
    assert (S.get() == st).all()
    d["dt"] = Dev(eng, np.full((T, D), 100, np.float32))
    eng.selective_scan(O.ptr, d["u"].ptr, d["dt"].ptr, d["A"].ptr, d["B"].ptr, d["C"].ptr, T, D, N, state=S.ptr,
                       softplus=False)
    eng.sync()
    want = 100.0 * u[-1].astype(np.float64) * B[-1].astype(np.float64)[:, None]
    assert (np.abs(S.get()[0] - want) <= 2 * U * np.abs(want)).all()


def test_scan_infinite_decay_and_nan(eng):  # noqa: F811
    """A decay rate of -infinity keeps nothing of the state, at a sequence's ragged end too; a NaN stays in its channel."""
    rng = np.random.default_rng(16)
    T, D, N = 69, 70, 16  # a ragged group of steps
    u, dt = rng.standard_normal((T, D)).astype(np.float32), np.full((T, D), 0.5, np.float32)
    B, Cm = (rng.standard_normal((T, N)).astype(np.float32) for _ in range(2))
    A = -np.ones((D, N), np.float32)
    A[3], u[5, 40] = -np.inf, np.nan
    d = {k: Dev(eng, v) for k, v in dict(u=u, dt=dt, B=B, C=Cm, A=A).items()}
    S, O = Dev(eng, np.ones((1, N, D), np.float32)), Dev(eng, shape=(T, D))
    eng.selective_scan(O.ptr, d["u"].ptr, d["dt"].ptr, d["A"].ptr, d["B"].ptr, d["C"].ptr, T, D, N, state=S.ptr,
                       softplus=False)
    eng.sync()
    o, s = O.get(), S.get()[0]
    want = 0.5 * u[:, 3].astype(np.float64)[:, None] * B
    assert (np.abs(s[:, 3] - want[-1]) <= 2 * U * np.abs(want[-1])).all()
    assert (np.abs(o[:, 3] - (want * Cm).sum(1)) <= 20 * U * np.abs(want * Cm).sum(1)).all()
    others = np.arange(D) != 40
    assert np.isfinite(o[:, others]).all() and np.isfinite(s[:, others]).all()
    assert np.isfinite(o[:5, 40]).all() and np.isnan(o[5:, 40]).all() and np.isnan(s[:, 40]).all()


def test_scan_carries_its_state(eng):  # noqa: F811
    """A prompt and then single tokens give what the whole sequence gives, to rounding."""
    rng = np.random.default_rng(7)
    T, D, N = 150, 96, 16
    x = {k: rng.standard_normal((T, D if k in "u dt z".split() else N)).astype(np.float32) * 0.5 for k in ("u", "dt", "z", "B", "C")}
    A = (-np.arange(1, N + 1) * np.ones((D, 1))).astype(np.float32)
    want, bound, new, err = scan_ref(x["u"], x["dt"], A, x["B"], x["C"], None, x["z"], None, None, [T], True)
    d, AD = {k: Dev(eng, v) for k, v in x.items()}, Dev(eng, A)
    S, O = Dev(eng, np.zeros((1, N, D), np.float32)), Dev(eng, shape=(T, D))
    r = 0
    for n in (100, 1, 1, 30, 1, 17):
        eng.selective_scan(O.ptr + 4 * r * D, d["u"].ptr + 4 * r * D, d["dt"].ptr + 4 * r * D, AD.ptr,
                           d["B"].ptr + 4 * r * N, d["C"].ptr + 4 * r * N, n, D, N, z=d["z"].ptr + 4 * r * D, state=S.ptr)
        r += n
    eng.sync()
    close(O.get(), want, bound, F32, "pieces")
    assert (np.abs(S.get() - new) <= err + U * np.abs(new)).all()


def test_layer_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    b = [Dev(eng, np.zeros((4, 64), np.float32)) for _ in range(8)]
    p = [x.ptr for x in b]
    with pytest.raises(MmfError, match="width"):
        eng.short_conv(p[0], p[1], p[2], 4, 64, 9)
    with pytest.raises(MmfError, match="sum to the rows"):
        eng.short_conv(p[0], p[1], p[2], 4, 64, 4, lens=[1, 2])
    with pytest.raises(MmfError, match="overlaps"):
        eng.short_conv(p[0], p[0], p[2], 4, 64, 4)
    with pytest.raises(MmfError, match="states"):
        eng.selective_scan(p[0], p[1], p[2], p[3], p[4], p[5], 4, 64, 200)
    with pytest.raises(MmfError, match="divide"):
        eng.selective_scan(p[0], p[1], p[2], p[3], p[4], p[5], 4, 64, 16, seqs=3)
    with pytest.raises(MmfError, match="overlaps"):
        eng.selective_scan(p[1], p[1], p[2], p[3], p[4], p[5], 4, 64, 16)
    with pytest.raises(MmfError, match="null"):
        eng.add_rmsnorm_q8(p[0], p[1], None, p[2], 4, 64)
    with pytest.raises(MmfError, match="overlaps"):
        eng.add_rmsnorm_q8(p[0], p[1], p[2], p[3], 4, 64, y=p[2])
    # no rows: nothing to do, whatever the pointers
    eng.add_rmsnorm_q8(None, None, None, None, 0, 64)
    eng.short_conv(None, None, None, 0, 64, 4, lens=[0, 0])
    eng.selective_scan(None, None, None, None, None, None, 0, 64, 16, seqs=3)
    eng.sync()


# ---- together -----------------------------------------------------------------------------------


class Layer:
    """One layer of a recurrent low-bit model on device buffers: norm and codes, input projection,
    convolution, projections of dt, B and C, scan, output projection, and the next norm."""

    def __init__(self, eng, rng, H, D, N, W, seqs, rows):  # noqa: F811
        self.eng, self.H, self.D, self.N, self.W, self.seqs, self.rows, self.R = eng, H, D, N, W, seqs, rows, 16
        self.w = {"in": W4(eng, rng, 2 * D, H, 64, True), "proj": W4(eng, rng, self.R + 2 * N, D, 32, False),
                  "dt": W4(eng, rng, D, self.R, 0, False), "out": W4(eng, rng, H, D, 128, True)}
        f = np.float32
        self.host = {"norm": (1 + 0.1 * rng.standard_normal(H)).astype(f), "conv": rng.standard_normal((D, W)).astype(f) / 2,
                     "bias": rng.standard_normal(D).astype(f) * f(0.1), "A": -np.exp(rng.standard_normal((D, N))).astype(f),
                     "skip": np.ones(D, f), "dt_bias": (rng.standard_normal(D) - 3).astype(f)}
        self.p = {k: Dev(eng, v) for k, v in self.host.items()}
        self.conv_state = np.zeros((seqs, W - 1, D), f)
        self.state = np.zeros((seqs, N, D), f)
        self.d_conv, self.d_state = Dev(eng, self.conv_state), Dev(eng, self.state)
        s = dict(res=H, x=H, codes=None, scales=1, xz=2 * D, u=D, proj=self.R + 2 * N, dt=D, y=D, out=H)
        self.b = {k: Dev(eng, np.zeros((rows, n), f)) for k, n in s.items() if n}
        self.b["codes"] = Dev(eng, np.zeros((rows, H), np.int8))

    def run(self, rows, lens=None):
        e, b, p, H, D, N, R = self.eng, self.b, self.p, self.H, self.D, self.N, self.R
        kw = dict(lens=lens, seqs=self.seqs)
        e.add_rmsnorm_q8(b["codes"].ptr, b["scales"].ptr, b["x"].ptr, p["norm"].ptr, rows, H, res=b["res"].ptr, h=b["res"].ptr)
        e.w4_linear(self.w["in"].id, b["codes"].ptr, b["xz"].ptr, rows, dtype=I8, scales=b["scales"].ptr)
        e.short_conv(b["u"].ptr, b["xz"].ptr, p["conv"].ptr, rows, D, self.W, bias=p["bias"].ptr, state=self.d_conv.ptr,
                     ldx=2 * D, **kw)
        e.w4_linear(self.w["proj"].id, b["u"].ptr, b["proj"].ptr, rows)
        e.w4_linear(self.w["dt"].id, b["proj"].ptr, b["dt"].ptr, rows, ldx=R + 2 * N)
        e.selective_scan(b["y"].ptr, b["u"].ptr, b["dt"].ptr, p["A"].ptr, b["proj"].ptr + 4 * R, b["proj"].ptr + 4 * (R + N),
                         rows, D, N, skip=p["skip"].ptr, z=b["xz"].ptr + 4 * D, dt_bias=p["dt_bias"].ptr,
                         state=self.d_state.ptr, ldb=R + 2 * N, ldc=R + 2 * N, ldz=2 * D, **kw)
        e.w4_linear(self.w["out"].id, b["y"].ptr, b["x"].ptr, rows)

    def ref(self, x, res, lens):
        """The same in 64 bits: (x, res) for the next layer."""
        h = self.host
        r, _, real, scale = norm_ref(x.astype(np.float32), res.astype(np.float32), h["norm"], 1e-6)
        xz = (np.rint(real) * scale[:, None]) @ self.w["in"].w.T
        u, _, self.conv_state = conv_ref(xz[:, :self.D], h["conv"], h["bias"], self.conv_state, lens, True)
        proj = u @ self.w["proj"].w.T
        dt = proj[:, :self.R] @ self.w["dt"].w.T
        y, _, self.state, _ = scan_ref(u, dt, h["A"], proj[:, self.R:self.R + self.N], proj[:, self.R + self.N:], h["skip"],
                                       xz[:, self.D:], h["dt_bias"], self.state, lens, True)
        return y @ self.w["out"].w.T, r


def near(got, want, tol, what):
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= tol, f"{what}: {off:.2e}"


def test_layer_prompt_then_tokens(eng):  # noqa: F811
    """Ragged prompts and then single tokens through the whole layer. Each operator keeps a relative
    error of some 1e-6 in norm; the products carry it on, six of them, with a factor of order one."""
    rng = np.random.default_rng(21)
    lens = [37, 1, 90, 5]
    L = Layer(eng, rng, 200, 320, 16, 4, len(lens), sum(lens))
    for rows, ls in ((sum(lens), lens), (4, None), (4, None)):
        x, res = (rng.standard_normal((rows, 200)).astype(np.float32) for _ in range(2))
        for k, v in (("x", x), ("res", res)):
            eng._chk(eng.lib.mmf_upload(eng.h, L.b[k].ptr, v.ctypes.data_as(C.c_void_p), v.nbytes))
        L.run(rows, ls)
        eng.sync()
        wx, wres = L.ref(x, res, ls or [1] * 4)
        near(L.b["res"].get()[:rows], wres, 1e-7, "residual")
        near(L.b["x"].get()[:rows], wx, 5e-5, "output")
        near(L.d_state.get(), L.state, 5e-5, "state")
        near(L.d_conv.get(), L.conv_state, 5e-5, "carried inputs")


def hip_graphs():
    hip = C.CDLL("libamdhip64.so.7")
    for n in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch",
              "hipGraphExecDestroy", "hipGraphDestroy"):
        getattr(hip, n).restype = C.c_int
    return hip


def captured(hip, stream, work):
    """(graph, executable graph) of work() on the stream."""
    graph, ge = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    work()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ge), graph, None, None, C.c_size_t(0)) == 0
    return graph, ge


def test_workspace_in_graphs():
    """The workspace's first use is refused under capture, and leaves the capture alone; two graphs that share
    it, a long scan and a product of many rows, replay in turn with eager calls between them."""
    from matmulfreellmcpu_amd import Engine, MmfError
    e, hip = Engine(0), hip_graphs()
    try:
        rng, f = np.random.default_rng(50), np.float32
        T, D, N, R, K, M = 700, 128, 16, 80, 1024, 8192
        u, B, A = rng.standard_normal((T, D)).astype(f), rng.standard_normal((T, N)).astype(f), -np.ones((D, N), f)
        d = {k: Dev(e, v) for k, v in dict(u=u, B=B, A=A, x=rng.standard_normal((R, K)).astype(f)).items()}
        w = W4(e, rng, M, K, 128, True)
        y, o = Dev(e, np.zeros((T, D), f)), Dev(e, np.zeros((R, M), f))
        scan = lambda: e.selective_scan(y.ptr, d["u"].ptr, d["u"].ptr, d["A"].ptr, d["B"].ptr, d["B"].ptr, T, D, N)  # noqa: E731
        product = lambda: e.w4_linear(w.id, d["x"].ptr, o.ptr, R)  # noqa: E731
        assert e.workspace_bytes() == 0
        stream = C.c_void_p(e.stream)

        def refused():
            for call in (scan, product):
                with pytest.raises(MmfError, match="before the capture"):
                    call()
            e.w4_linear(w.id, d["x"].ptr, o.ptr, 2)  # needs none

        graph, ge = captured(hip, stream, refused)
        assert hip.hipGraphLaunch(ge, stream) == 0
        e.sync()
        assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(graph) == 0
        scan(), product()
        e.sync()
        want_y, want_o, size = y.get(), o.get(), e.workspace_bytes()
        assert size > 0
        graphs = [captured(hip, stream, scan), captured(hip, stream, product)]
        for step in range(4):
            for b in (y, o):
                z = np.zeros(b.shape, f)
                e._chk(e.lib.mmf_upload(e.h, b.ptr, z.ctypes.data_as(C.c_void_p), z.nbytes))
            for _, ge in graphs[::1 if step % 2 else -1]:
                assert hip.hipGraphLaunch(ge, stream) == 0
            e.sync()
            assert (y.get() == want_y).all() and (o.get() == want_o).all(), step
            product(), scan()
            e.sync()
        assert e.workspace_bytes() == size
        for g, ge in graphs:
            assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(g) == 0
    finally:
        e.close()


def test_layer_in_a_graph(eng):  # noqa: F811
    """The layer's step captured once and replayed between eager work: every replay equals the eager
    calls on the same buffers bit for bit."""
    hip = hip_graphs()
    rng = np.random.default_rng(22)
    L, E = (Layer(eng, np.random.default_rng(23), 128, 256, 16, 4, 8, 8) for _ in range(2))
    L.run(8), E.run(8)  # workspaces
    eng.sync()
    stream = C.c_void_p(eng.stream)
    graph, ge = captured(hip, stream, lambda: L.run(8))
    for step in range(4):
        x = rng.standard_normal((8, 128)).astype(np.float32)
        for layer in (L, E):
            eng._chk(eng.lib.mmf_upload(eng.h, layer.b["x"].ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
        assert hip.hipGraphLaunch(ge, stream) == 0
        E.run(8)
        eng.sync()
        for k in ("x", "res", "y", "codes"):
            a, b = L.b[k].get(), E.b[k].get()
            assert (a.view(np.uint8) == b.view(np.uint8)).all(), (step, k)
        assert (L.d_state.get() == E.d_state.get()).all() and (L.d_conv.get() == E.d_conv.get()).all()
    assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(graph) == 0

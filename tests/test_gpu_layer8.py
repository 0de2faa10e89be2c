"""The operators of a linear attention layer with 8-bit weights (8-bit products, attention with a decay for each head,
norms around a block) and of its logits (token log probabilities) against plain numpy in 64 bits: sizes on both sides of
every tile, odd strides and addresses, all types, empty and one-row sequences, carried states, captured graphs.

U = 2^-24 is fp32's half step; an output of type t is off by half a step of its type more.
"""
import ctypes as C

import numpy as np
import pytest

from test_gpu_layer import BF16, F16, F32, FLOATS, HALF, I8, U, Rows, captured, close, coded, hip_graphs, out_rows, silu, value
from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu

ACT = {"none": 0, "sigmoid": 1, "silu": 2}


# ---- 8-bit products -------------------------------------------------------------------------


def run_w8(eng, rng, rows, K, N, out_t=F32, bias=True, exact=True, padx=0, offx=0, pado=0, offo=0, ends=False):  # noqa: F811
    print(f"w8 rows={rows} K={K} N={N} out={out_t} bias={bias} exact={exact} {padx, offx, pado, offo}", flush=True)
    f = np.float32
    if ends:  # the largest products that there are
        q, x = np.full((N, K), -128, np.int8), rng.choice(np.array([-128, 127], np.int8), (rows, 1)).repeat(K, 1)
    else:
        q, x = rng.integers(-128, 128, (N, K)).astype(np.int8), rng.integers(-128, 128, (rows, K)).astype(np.int8)
    # exact: powers of two and small multiples of them, so that every step but the sum's one rounding is exact
    ws = (2.0 ** rng.integers(-9, -3, N) if exact else 0.01 * (0.5 + rng.random(N))).astype(f)
    xs = (2.0 ** rng.integers(-5, 0, rows) if exact else 0.02 + 0.03 * rng.random(rows)).astype(f)
    b = (rng.integers(-1000, 1000, N) / 16 if exact else rng.standard_normal(N)).astype(f) if bias else None
    wid = eng.register_w8(q, ws)
    assert eng.w8_shape(wid) == (N, K)
    X, O = Rows(eng, x, I8, padx, offx), out_rows(eng, (rows, N), out_t, pado, offo)
    S, B = Rows(eng, xs[None], F32, 0, offo), Rows(eng, b[None], F32, 0, offx) if bias else None
    eng.w8_linear(wid, X.ptr, S.ptr, O.ptr, rows, bias=B.ptr if bias else None, out_dtype=out_t, ldx=X.ld, ldo=O.ld)
    eng.sync()
    got = value(O.get(), out_t)
    # float32 products of integers in halves of the inputs would round: 64 bits hold every sum
    sums = np.concatenate([x[i:i + 64].astype(np.float64) @ q.T.astype(np.float64) for i in range(0, rows, 64)])
    if exact:
        want = (sums.astype(f).astype(np.float64) * xs[:, None] * ws + (b if bias else 0)).astype(f)  # one rounding of the sum of both
        ref = value(coded(want, out_t), out_t)
        assert (got == ref).all(), (np.argwhere(got != ref)[:3], got[got != ref][:3], ref[got != ref][:3])
    else:  # the sum, its product with xs, the last product and sum: three roundings
        mag = np.abs(sums) * xs[:, None] * ws
        close(got, sums * xs[:, None] * ws + (b if bias else 0), 2.001 * U * mag + U * (mag + (np.abs(b) if bias else 0)), out_t, "w8")
    eng.w8_release(wid)


W8_SHAPES = [(1, 1, 1), (1, 64, 16), (1, 2048, 70), (2, 77, 33), (3, 128, 17), (5, 129, 40), (8, 300, 100), (15, 96, 31),
             (16, 1031, 70), (17, 256, 48), (21, 160, 129), (31, 64, 65), (32, 500, 64), (33, 500, 65), (64, 384, 200),
             (65, 130, 16), (100, 1031, 133), (128, 640, 256), (129, 320, 257), (130, 640, 257), (255, 127, 300)]


@pytest.mark.parametrize("out_t", FLOATS)
@pytest.mark.parametrize("i", range(len(W8_SHAPES)))
def test_w8_layouts(eng, i, out_t):  # noqa: F811
    rows, K, N = W8_SHAPES[i]
    rng = np.random.default_rng(i * 3 + out_t)
    run_w8(eng, rng, rows, K, N, out_t, bias=i % 2 == 0)
    run_w8(eng, rng, rows, K, N, out_t, bias=i % 2 == 1, padx=1 + i % 7, offx=1 + i % 5, pado=i % 4, offo=1)
    run_w8(eng, rng, rows, K, N, out_t, padx=-K % 16, pado=-N % 16)  # aligned rows of any length


@pytest.mark.parametrize("out_t", FLOATS)
@pytest.mark.parametrize("rows,K,N", [(300, 256, 144), (257, 1000, 300), (513, 192, 1100), (1030, 70, 40), (90, 4100, 8001),
                                      (700, 2000, 2100), (300, 6912, 520), (2050, 640, 700)])
def test_w8_many_rows(eng, rows, K, N, out_t):  # noqa: F811
    rng = np.random.default_rng(rows + out_t)
    run_w8(eng, rng, rows, K, N, out_t, padx=3, pado=1)
    run_w8(eng, rng, rows, K, N, out_t, bias=False, padx=-K % 16)
    run_w8(eng, rng, rows, K, N, out_t, exact=False)


@pytest.mark.parametrize("out_t", FLOATS)
def test_w8_rounding(eng, out_t):  # noqa: F811
    rng = np.random.default_rng(17 + out_t)
    for rows, K, N in ((1, 2048, 130), (4, 6912, 48), (24, 1031, 70), (70, 512, 100), (300, 640, 160)):
        run_w8(eng, rng, rows, K, N, out_t, exact=False, bias=rows != 4)


def test_w8_largest_sums(eng):  # noqa: F811
    """Sums that reach the ends of 32 bits, in every kernel: 131071 inputs of -128 at weights of -128."""
    rng = np.random.default_rng(18)
    for rows in (1, 20, 70, 300):
        run_w8(eng, rng, rows, 131071, 33, ends=True, padx=1)


def test_w8_long_rows_and_many(eng):  # noqa: F811
    rng = np.random.default_rng(40)
    run_w8(eng, rng, 1, 12000, 40)
    run_w8(eng, rng, 3, 9999, 17, padx=5)
    run_w8(eng, rng, 66000, 160, 64, padx=1)
    run_w8(eng, rng, 1_050_000, 3, 2)  # more rows than one launch takes


def test_w8_scales_without_a_number(eng):  # noqa: F811
    """A row whose scale is NaN (a row without a number before its norm) has no outputs, and leaves the others alone."""
    rng = np.random.default_rng(41)
    for rows in (3, 40, 200):
        q, x = rng.integers(-128, 128, (50, 70)).astype(np.int8), rng.integers(-128, 128, (rows, 70)).astype(np.int8)
        xs = np.ones(rows, np.float32)
        xs[1], x[1] = np.nan, 0
        wid = eng.register_w8(q, np.ones(50, np.float32))
        X, S, O = Dev(eng, x), Dev(eng, xs), Dev(eng, shape=(rows, 50))
        eng.w8_linear(wid, X.ptr, S.ptr, O.ptr, rows)
        eng.sync()
        got, want = O.get(), x.astype(np.float32) @ q.T.astype(np.float32)
        keep = np.arange(rows) != 1
        assert np.isnan(got[1]).all() and (got[keep] == want[keep]).all()
        eng.w8_release(wid)


def test_w8_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    q, s = np.zeros((4, 32), np.int8), np.ones(4, np.float32)
    wid = eng.register_w8(q, s)
    x, xs, o = Dev(eng, np.zeros((2, 32), np.int8)), Dev(eng, np.ones(2, np.float32)), Dev(eng, shape=(2, 4))
    for kw, why in ((dict(out_dtype=I8), "out_dtype"), (dict(ldx=31), "stride"), (dict(ldo=3), "stride")):
        with pytest.raises(MmfError, match=why):
            eng.w8_linear(wid, x.ptr, xs.ptr, o.ptr, 2, **kw)
    with pytest.raises(MmfError, match="null"):
        eng.w8_linear(wid, x.ptr, None, o.ptr, 2)
    with pytest.raises(MmfError, match="overlaps"):
        eng.w8_linear(wid, x.ptr, xs.ptr, xs.ptr, 2)
    with pytest.raises(MmfError, match="131071"):
        eng.register_w8(np.zeros((1, 131072), np.int8), np.ones(1, np.float32))
    with pytest.raises(ValueError):
        eng.register_w8(q, np.ones(5, np.float32))
    eng.w8_linear(wid, None, None, None, 0)
    eng.w8_release(wid)
    with pytest.raises(MmfError, match="released"):
        eng.w8_linear(wid, x.ptr, xs.ptr, o.ptr, 2)
    with pytest.raises(MmfError, match="invalid w8_id"):
        eng.w8_shape(10 ** 6)


# ---- attention with a decay for each head -----------------------------------------------------


def decay_ref(q, k, v, a, state, lens, scale):
    """(out, its bound, state, its bound) in 64 bits, step by step. q, k, v [rows, H, D], a [rows, H] log decays.

    With A the state of the terms' magnitudes, a step's update rounds decay, product and sum (3 U of A, carried on by the
    decays). A sum over 64 rows at once rounds up to 64 times, and one over Dk as often as it has terms, with the scale's, the
    output's and a decay's own: (Dk + 100) U of the sum of magnitudes."""
    rows, H, Dk = q.shape
    Dv = v.shape[2]
    out, bound = np.zeros((rows, H, Dv)), np.zeros((rows, H, Dv))
    new, err = np.zeros((len(lens), H, Dk, Dv)), np.zeros((len(lens), H, Dk, Dv))
    with np.errstate(invalid="ignore", over="ignore"):
        keep = np.exp(a.astype(np.float64))[:, :, None, None]
        kv, r = None, 0
        for s, n in enumerate(lens):
            S = state[s].astype(np.float64) if state is not None else np.zeros((H, Dk, Dv))
            A, e = np.abs(S), np.zeros_like(S)
            for p in range(r, r + n):
                kv = k[p].astype(np.float64)[:, :, None] * v[p].astype(np.float64)[:, None, :]
                e = keep[p] * e + 3 * U * (keep[p] * A + np.abs(kv))
                S, A = keep[p] * S + kv, keep[p] * A + np.abs(kv)
                qq = q[p].astype(np.float64)[:, :, None]
                out[p] = scale * (qq * S).sum(1)
                bound[p] = scale * (np.abs(qq) * (e + (Dk + 100) * U * A)).sum(1)
            new[s], err[s] = S, e + (64 + 16) * U * A
            r += n
    return out, bound, new, err


# A 16-bit output's own matrix products take the state and the weights of the rows in two bf16 parts, 2^-16 of each.
PARTS = {F32: 0.0, BF16: 2.0 ** -15, F16: 2.0 ** -15}


def run_decay(eng, rng, t, lens, H, Dk, Dv, q_heads=0, k_heads=0, v_heads=0, decay=True, gates=True, state=True, pads=(0,) * 5,  # noqa: F811
              offs=(0,) * 5, seqs=None, log_decay=None, data=None):
    print(f"decay t={t} lens={lens if len(lens) < 20 else len(lens)} H={H} Dk={Dk} Dv={Dv} {q_heads, k_heads, v_heads} "
          f"{decay, gates, state} {pads, offs}", flush=True)
    rows, n, f = sum(lens), len(lens), np.float32
    heads = [q_heads or H, k_heads or H, v_heads or H]
    data = data or [coded(rng.standard_normal((rows, h * D)), t) for h, D in zip(heads, (Dk, Dk, Dv))]
    d = (np.log1p(-2.0 ** -rng.uniform(1, 10, H)) if log_decay is None else np.broadcast_to(log_decay, H)).astype(f) if decay else None
    g = np.log(rng.uniform(0.2, 1.0, (rows, H)) ** 0.3).astype(f) if gates else None
    st = rng.standard_normal((n, H, Dk, Dv)).astype(f) if state else None
    Q, K, V = (Rows(eng, x, t, pads[i], offs[i]) for i, x in enumerate(data))
    O = out_rows(eng, (rows, H * Dv), t, pads[3], offs[3])
    D = Rows(eng, d[None], F32, 0, offs[0]) if decay else None
    G = Rows(eng, g, F32, pads[4], offs[4]) if gates else None
    S = Rows(eng, st.reshape(1, -1), F32, 0, offs[4]) if state else None
    scale = f(Dk ** -0.5)
    q, k, v = (value(x, t).reshape(rows, h, -1).repeat(H // h, 1) for x, h in zip(data, heads))
    a = np.zeros((rows, H)) + (d.astype(np.float64) if decay else 0) + (g.astype(np.float64) if gates else 0)
    want, bound, new, err = decay_ref(q, k, v, a, st, lens, float(scale))
    eng.decay_attention(O.ptr, Q.ptr, K.ptr, V.ptr, rows, H, Dk, Dv, decay=D.ptr if D else None, gates=G.ptr if G else None,
                        state=S.ptr if S else None, lens=None if seqs else lens, seqs=seqs or 1, q_heads=q_heads, k_heads=k_heads,
                        v_heads=v_heads, dtype=t, ldo=O.ld, ldq=Q.ld, ldk=K.ld, ldv=V.ld, ldg=G.ld if G else 0)
    eng.sync()
    got = value(O.get(), t).reshape(want.shape)
    mag = bound / ((Dk + 100) * U)  # at least the sum of magnitudes
    close(got, want, bound + PARTS[t] * mag, t, "decay")
    if state:
        S = S.get().reshape(new.shape)
        for s, m in enumerate(lens):
            if not m:
                assert (S[s] == st[s]).all(), "state of an empty sequence"
        off = np.abs(S - new)
        assert (off <= err + U * np.abs(new) + 1e-37).all() or not np.isfinite(new).all(), (off - err).max()
        return got, S
    return got, None


DECAY_SHAPES = [(1, 1, 1), (2, 16, 16), (3, 5, 7), (2, 31, 33), (1, 32, 64), (2, 63, 65), (1, 64, 128), (2, 72, 111), (1, 100, 32),
                (1, 127, 129), (2, 128, 128), (1, 129, 31), (1, 160, 96), (1, 256, 256), (1, 255, 200)]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("i", range(len(DECAY_SHAPES)))
def test_decay_heads(eng, i, t):  # noqa: F811
    H, Dk, Dv = DECAY_SHAPES[i]
    rng = np.random.default_rng(i * 3 + t)
    run_decay(eng, rng, t, [1], H, Dk, Dv)
    run_decay(eng, rng, t, [1] * 5, H, Dk, Dv, seqs=5, pads=(1, 2, 0, 3, 1), offs=(1, 0, 3, 1, 2))
    run_decay(eng, rng, t, [3, 0, 1, 20, 0, 40, 9], H, Dk, Dv, pads=(3, 1, 2, 0, 5), offs=(1, 3, 1, 5, 2))
    run_decay(eng, rng, t, [70], H, Dk, Dv, state=False, gates=False, pads=(8, 8, 8, 8, 0))
    run_decay(eng, rng, t, [130], H, Dk, Dv, decay=False)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("n", [2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 513, 1000])
def test_decay_lengths(eng, n, t):  # noqa: F811
    rng = np.random.default_rng(n * 3 + t)
    run_decay(eng, rng, t, [n], 2, 48, 40, gates=n % 2 == 0)
    run_decay(eng, rng, t, [n, 0, 1, n // 2], 1, 128, 64, pads=(0, 4, 0, 1, 3))
    run_decay(eng, rng, t, [n], 1, 64, 128, state=False, decay=n % 3 > 0)


@pytest.mark.parametrize("t", FLOATS)
def test_decay_shared_heads(eng, t):  # noqa: F811
    rng = np.random.default_rng(100 + t)
    for lens in ([1] * 3, [90, 40], [300]):
        run_decay(eng, rng, t, lens, 6, 32, 48, q_heads=1, k_heads=1)
        run_decay(eng, rng, t, lens, 6, 48, 32, k_heads=2, v_heads=3, pads=(1, 2, 3, 4, 5))
        run_decay(eng, rng, t, lens, 4, 64, 64, q_heads=2, k_heads=4, v_heads=1)


@pytest.mark.parametrize("t", FLOATS)
def test_decay_many_sequences(eng, t):  # noqa: F811
    rng = np.random.default_rng(110 + t)
    run_decay(eng, rng, t, [int(n) for n in rng.integers(0, 5, 600)], 1, 16, 24)  # several tables of sequences
    run_decay(eng, rng, t, [1] * 500, 2, 32, 32)
    run_decay(eng, rng, t, [1] * 500, 2, 32, 32, seqs=500)
    run_decay(eng, rng, t, [12] * 300, 1, 16, 16, seqs=300)
    run_decay(eng, rng, t, [700] + [1, 0, 2] * 90 + [500, 400], 1, 32, 32)
    run_decay(eng, rng, t, [64] * 10, 2, 64, 64, seqs=10)


@pytest.mark.parametrize("t", FLOATS)
def test_decay_range(eng, t):  # noqa: F811
    """Decays that forget within a row, that forget nothing over the whole length, and that grow."""
    rng = np.random.default_rng(120 + t)
    for log_decay in (0.0, -1e-6, -0.5, -20.0, -1000.0, 0.01):
        run_decay(eng, rng, t, [200, 1, 70], 2, 32, 48, gates=False, log_decay=log_decay)


@pytest.mark.parametrize("t", FLOATS)
def test_decay_forgets(eng, t):  # noqa: F811
    """A log decay of -infinity starts the sequence anew: outputs and state as from that row on, also within a tile, and the
    decays after it keep their digits."""
    rng = np.random.default_rng(130 + t)
    H, Dk, Dv, n, f = 2, 40, 33, 150, np.float32
    q, k, v = (coded(rng.standard_normal((n, H * D)), t) for D in (Dk, Dk, Dv))
    g = (-0.2 * rng.random((n, H))).astype(f)
    for at in (0, 1, 63, 64, 77, 149):
        print(f"decay forgets t={t} at={at}", flush=True)
        gi = g.copy()
        gi[at] = -np.inf
        Q, K, V, G = Rows(eng, q, t), Rows(eng, k, t), Rows(eng, v, t), Rows(eng, gi, F32)
        S, O = Dev(eng, np.ones((1, H, Dk, Dv), f)), out_rows(eng, (n, H * Dv), t)
        eng.decay_attention(O.ptr, Q.ptr, K.ptr, V.ptr, n, H, Dk, Dv, gates=G.ptr, state=S.ptr, dtype=t)
        eng.sync()
        qq, kk, vv = (value(x[at:], t).reshape(n - at, H, -1) for x in (q, k, v))
        want, bound, new, err = decay_ref(qq, kk, vv, gi[at:], None, [n - at], Dk ** -0.5)
        mag = bound / ((Dk + 100) * U)
        close(value(O.get()[at:], t).reshape(want.shape), want, bound + PARTS[t] * mag, t, "after")
        assert (np.abs(S.get() - new) <= err + U * np.abs(new)).all()


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("which", ["q", "k", "v", "gates"])
def test_decay_rows_without_a_number(eng, which, t):  # noqa: F811
    """An infinity or NaN leaves the rows before it, other sequences and other heads their bits; of q it stays in its row, of v in
    its column."""
    rng = np.random.default_rng(140 + t)
    H, Dk, Dv, lens, f = 2, 40, 48, [100, 30], np.float32
    n = sum(lens)
    clean = {"q": rng.standard_normal((n, H * Dk)), "k": rng.standard_normal((n, H * Dk)), "v": rng.standard_normal((n, H * Dv))}
    gates = (-0.2 * rng.random((n, H))).astype(f)

    def run(x, g):
        T = {m: Rows(eng, coded(a, t), t) for m, a in x.items()}
        S, O, G = Dev(eng, np.ones((2, H, Dk, Dv), f)), out_rows(eng, (n, H * Dv), t), Rows(eng, g, F32)
        eng.decay_attention(O.ptr, T["q"].ptr, T["k"].ptr, T["v"].ptr, n, H, Dk, Dv, gates=G.ptr, state=S.ptr, lens=lens, dtype=t)
        eng.sync()
        return value(O.get(), t).reshape(n, H, Dv), S.get()

    o0, s0 = run(clean, gates)
    assert np.isfinite(o0).all() and np.isfinite(s0).all()
    for at in (0, 5, 37, 63, 64, 99):
        for bad in (np.nan, np.inf, -np.inf):
            if which == "gates" and bad != bad or which != "gates":
                print(f"no number t={t} {which} at={at} {bad}", flush=True)
                x, g = {m: a.copy() for m, a in clean.items()}, gates.copy()
                if which == "gates":
                    g[at, 1] = bad
                else:
                    x[which][at, (Dk if which != "v" else Dv) + 7] = bad  # of the second head
                o, s = run(x, g)
                assert (o[:, 0] == o0[:, 0]).all() and (s[:, 0] == s0[:, 0]).all(), "the other head"
                assert (o[100:] == o0[100:]).all() and (s[1] == s0[1]).all(), "the other sequence"
                assert (o[:at] == o0[:at]).all(), "rows before"
                if which == "q":
                    assert not np.isfinite(o[at, 1]).any() and (o[at + 1:] == o0[at + 1:]).all() and (s == s0).all()
                elif which == "v":
                    others = np.arange(Dv) != 7
                    assert not np.isfinite(o[at:100, 1, 7]).any() and not np.isfinite(s[0, 1, :, 7]).any()
                    assert (o[:, 1, others] == o0[:, 1, others]).all() and (s[:, 1][..., others] == s0[:, 1][..., others]).all()
                elif which == "k":
                    assert not np.isfinite(o[at:100, 1]).any() and not np.isfinite(s[0, 1, 7]).any()
                else:
                    assert not np.isfinite(o[at:100, 1]).any() and not np.isfinite(s[0, 1]).any()


def test_decay_carries_its_state(eng):  # noqa: F811
    """A prompt and then single tokens give what the whole sequence gives."""
    rng = np.random.default_rng(150)
    T, H, Dk, Dv, f = 150, 2, 32, 64, np.float32
    q, k, v = (rng.standard_normal((T, H * D)).astype(f) for D in (Dk, Dk, Dv))
    g = (-0.1 * rng.random((T, H))).astype(f)
    want, bound, new, err = decay_ref(*(x.reshape(T, H, -1) for x in (q, k, v)), g, None, [T], Dk ** -0.5)
    Q, K, V, G, O = Dev(eng, q), Dev(eng, k), Dev(eng, v), Dev(eng, g), Dev(eng, shape=(T, H * Dv))
    S, r = Dev(eng, np.zeros((1, H, Dk, Dv), f)), 0
    for n in (100, 1, 1, 30, 1, 17):
        eng.decay_attention(O.ptr + 4 * r * H * Dv, Q.ptr + 4 * r * H * Dk, K.ptr + 4 * r * H * Dk, V.ptr + 4 * r * H * Dv, n, H,
                            Dk, Dv, gates=G.ptr + 4 * r * H, state=S.ptr)
        r += n
    eng.sync()
    close(O.get().reshape(want.shape), want, bound, F32, "pieces")
    assert (np.abs(S.get() - new) <= err + 5 * 80 * U * np.abs(new) + 1e-6).all()


def test_decay_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    p = [Dev(eng, np.zeros((4, 64), np.float32)).ptr for _ in range(8)]
    ok = dict(rows=4, heads=4, Dk=16, Dv=16)
    for kw, why in ((dict(heads=0), "heads"), (dict(Dk=257), "256"), (dict(Dv=0), "256"), (dict(q_heads=3), "divide"),
                    (dict(lens=[1, 2]), "sum to the rows"), (dict(seqs=3), "divide"), (dict(ldk=63), "stride"),
                    (dict(gates=p[4], ldg=3), "stride"), (dict(dtype=I8), "dtype"), (dict(state=p[1]), "overlaps")):
        with pytest.raises(MmfError, match=why):
            eng.decay_attention(p[0], p[1], p[2], p[3], **{**ok, **kw})
    with pytest.raises(MmfError, match="overlaps"):
        eng.decay_attention(p[0], p[0], p[2], p[3], **ok)
    with pytest.raises(MmfError, match="null"):
        eng.decay_attention(p[0], None, p[2], p[3], **ok)
    eng.decay_attention(None, None, None, None, 0, 4, 16, 16, lens=[0, 0])
    eng.sync()


# ---- norms around a block -----------------------------------------------------------------------


def block_ref(b, x, gate, act, w_post, w_pre, channels, scale, eps):
    """h in 64 bits before its rounding; y, codes' real values and scales of h rounded to fp32."""
    f = np.float64
    with np.errstate(all="ignore"):
        p = b.astype(f)
        if w_post is not None:
            p = p / np.sqrt((p * p).mean(1, keepdims=True) + f(np.float32(eps))) * w_post
        if gate is not None:
            g = gate.astype(f)
            p = p * {0: g, 1: 1 / (1 + np.exp(-g)), 2: silu(g)}[act]
        h = p * (1.0 if channels is None else channels.astype(f)) * f(np.float32(scale)) + (0 if x is None else x.astype(f))
        y = h.astype(np.float32).astype(f)
        if w_pre is not None:
            y = y / np.sqrt((y * y).mean(1, keepdims=True) + f(np.float32(eps))) * w_pre
        m = np.maximum(np.abs(y).max(1, keepdims=True), 1e-5)
    return h, y, y * 127.0 / m, (m / 127.0)[:, 0]


def run_block(eng, rng, t, rows, cols, x=True, gate="silu", post=True, pre=True, channels=True, h=True, y=True, codes=True,  # noqa: F811
              scale=0.7, pads=(0,) * 6, offs=(0,) * 6, in_place=None, eps=1e-6):
    print(f"block t={t} rows={rows} cols={cols} x={x} gate={gate} post={post} pre={pre} {channels, h, y, codes} {pads, offs} "
          f"{in_place}", flush=True)
    f = np.float32
    data = {"b": rng.standard_normal((rows, cols)), "x": rng.standard_normal((rows, cols)) * np.where(rng.random(cols) < 0.02, 30, 2),
            "gate": rng.standard_normal((rows, cols)) * 2}
    have = {"b": True, "x": x, "gate": gate != "none"}
    data = {k: coded(v, t) if have[k] else None for k, v in data.items()}
    params = {k: (1 + 0.1 * rng.standard_normal(cols)).astype(f) if on else None
              for k, on in (("w_post", post), ("w_pre", pre), ("channels", channels))}
    act = {"none": 0, "plain": 0, "sigmoid": 1, "silu": 2}[gate]
    T = {k: Rows(eng, v, t, pads[i], offs[i]) if v is not None else None for i, (k, v) in enumerate(data.items())}
    P = {k: Rows(eng, v[None], F32, 0, offs[0]) if v is not None else None for k, v in params.items()}
    H, Y = out_rows(eng, (rows, cols), t, pads[3], offs[3]), out_rows(eng, (rows, cols), t, pads[4], offs[4])
    Q, S = out_rows(eng, (rows, cols), I8, pads[5], offs[5]), out_rows(eng, (rows, 1), F32)
    if in_place:
        H = T[in_place]
    at = lambda o: o.ptr if o else None  # noqa: E731
    ld = lambda o: o.ld if o else 0  # noqa: E731
    eng.block_norm_q8(Q.ptr if codes else None, S.ptr if codes else None, T["b"].ptr, rows, cols, x=at(T["x"]), gate=at(T["gate"]),
                      act=act, w_post=at(P["w_post"]), w_pre=at(P["w_pre"]), channels=at(P["channels"]), scale=scale,
                      h=H.ptr if h else None, y=Y.ptr if y else None, eps=eps, dtype=t, ldb=T["b"].ld, ldx=ld(T["x"]),
                      ldgate=ld(T["gate"]), ldh=H.ld, ldy=Y.ld, ldcodes=Q.ld)
    eng.sync()
    v = {k: value(a, t) if a is not None else None for k, a in data.items()}
    hw, yw, real, sw = block_ref(v["b"], v["x"], v["gate"], act, params["w_post"], params["w_pre"], params["channels"], scale, eps)
    # h: one rounding to fp32, then the type's. What follows is taken of that fp32 number, which differs by a step (2 U) only
    # where the 64-bit value, itself off by some 2^-48, lies that near to a tie: y and the codes' real values by as much.
    got_h = H._in(H.dev.get()) if in_place else H.get()
    if h:
        close(value(got_h, t), hw, 1.001 * U * np.abs(hw), t, "h")
    if y:
        close(value(Y.get(), t), yw, 3.1 * U * np.abs(yw), t, "y")
    if codes:
        q, s = Q.get().astype(np.float64), S.get()[:, 0]
        assert (np.abs(q - real) <= 0.5 + 127 * 4.1 * U).all(), np.abs(q - real).max()
        assert np.mean(np.abs(q - real) > 0.5 + 1e-9) < 1e-4  # and hardly anywhere
        assert (np.abs(s - sw) <= 3.1 * U * sw).all()


BLOCK_COLS = [1, 3, 7, 64, 100, 255, 256, 257, 511, 512, 513, 1024, 1031, 2048, 2050, 2560, 4095, 4096, 4097, 5632, 6912, 8192, 8200,
              16384, 16391, 32768, 32769, 65536, 65537, 70000]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("cols", BLOCK_COLS)
def test_block_lengths(eng, cols, t):  # noqa: F811
    rng = np.random.default_rng(cols + t)
    run_block(eng, rng, t, 5, cols)
    run_block(eng, rng, t, 3, cols, gate="plain", pads=(1, 2, 3, 5, 1, 2), offs=(1, 3, 5, 2, 1, 3))
    run_block(eng, rng, t, 1, cols, gate="none", y=False)
    run_block(eng, rng, t, 2, cols, gate="sigmoid", codes=False, in_place="x")


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("cols", [100, 2048, 40000, 70001])
def test_block_forms(eng, cols, t):  # noqa: F811
    """Every part left out, and h in the place of each input."""
    rng = np.random.default_rng(cols + t)
    for kw in (dict(x=False), dict(post=False), dict(pre=False), dict(channels=False), dict(post=False, pre=False, channels=False, gate="none"),
               dict(h=False), dict(h=False, codes=False), dict(y=False, codes=False), dict(in_place="b"), dict(in_place="gate"),
               dict(in_place="x", y=False), dict(x=False, gate="none", scale=-1.5)):
        run_block(eng, rng, t, 3, cols, **kw)


@pytest.mark.parametrize("t", FLOATS)
def test_block_many_rows(eng, t):  # noqa: F811
    rng = np.random.default_rng(4 + t)
    for rows, cols in ((1000, 70), (700, 1030), (2100, 256), (600, 2560)):
        run_block(eng, rng, t, rows, cols, pads=(2, 0, 4, 0, 3, 1))


def test_block_special_rows(eng):  # noqa: F811
    """Zero rows keep the smallest scale; an infinity or NaN anywhere has the scale NaN and codes 0 for its row alone; gates far out
    saturate."""
    rng = np.random.default_rng(9)
    for cols in (300, 70000):
        rows, f = 9, np.float32
        b, x, g = (rng.standard_normal((rows, cols)).astype(f) for _ in range(3))
        b[0] = x[0] = 0
        b[1], x[1] = b[1] * f(1e30), x[1] * f(1e30)
        b[2], x[2] = b[2] * f(1e-30), x[2] * f(1e-30)
        b[3, 7], x[4, 299], g[5, 0], b[6, 5] = np.inf, np.nan, np.nan, -np.inf
        g[7, ::2], g[7, 1::2] = 1e4, -1e4
        w = np.ones(cols, f)
        D = {k: Dev(eng, v) for k, v in dict(b=b, x=x, g=g, w=w).items()}
        Q, S, H, Y = out_rows(eng, (rows, cols), I8), out_rows(eng, (rows, 1), F32), *(out_rows(eng, (rows, cols), F32) for _ in range(2))
        eng.block_norm_q8(Q.ptr, S.ptr, D["b"].ptr, rows, cols, x=D["x"].ptr, gate=D["g"].ptr, act=2, w_post=D["w"].ptr, w_pre=D["w"].ptr,
                          h=H.ptr, y=Y.ptr)
        eng.sync()
        hw, yw, real, sw = block_ref(b, x, g, 2, w, w, None, 1.0, 1e-6)
        q, s = Q.get(), S.get()[:, 0]
        bad, fine = [3, 4, 5, 6], [0, 1, 2, 7, 8]
        assert np.isnan(s[bad]).all() and (q[bad] == 0).all()
        assert (q[0] == 0).all() and s[0] == f(1e-5 / 127.0)
        assert (np.abs(s[fine] - sw[fine]) <= 3.1 * U * sw[fine]).all()
        close(H.get()[fine], hw[fine], U * 1.001 * np.abs(hw[fine]), F32, "h")
        close(Y.get()[fine], yw[fine], 3.1 * U * np.abs(yw[fine]), F32, "y")


def test_block_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    p = [Dev(eng, np.zeros((4, 64), np.float32)).ptr for _ in range(6)]
    for args, kw, why in (((p[0], p[1], None, 4, 64), {}, "null"), ((p[0], None, p[2], 4, 64), {}, "go together"),
                          ((None, None, p[2], 4, 64), {}, "no output"), ((p[0], p[1], p[2], 4, 64), dict(act=1), "gate"),
                          ((p[0], p[1], p[2], 4, 64), dict(act=3), "act"), ((p[0], p[1], p[2], 4, 64), dict(y=p[2]), "overlaps"),
                          ((p[0], p[1], p[2], 4, 64), dict(h=p[2] + 4), "overlaps"), ((p[0], p[1], p[2], 4, 64), dict(ldx=9), "stride")):
        with pytest.raises(MmfError, match=why):
            eng.block_norm_q8(*args, **kw)
    eng.block_norm_q8(None, None, None, 0, 64)
    eng.sync()


# ---- log probabilities ------------------------------------------------------------------------------


def logp_ref(x, ids, T):
    """(log probabilities of ids, entropies, all log probabilities, their bounds) in 64 bits.

    z = (x - m) / T has three roundings (difference, 1 / T, product); an exponential its exponent's two and two of its own, of
    weight p; the sums some 50 additions; the logarithm two of its own and the difference one."""
    with np.errstate(all="ignore"):
        z = (x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)) / np.float64(np.float32(T))
        e = np.exp(z)
        s = e.sum(1, keepdims=True)
        lp, p = z - np.log(s), e / s
        az = np.where(p > 0, np.abs(z), 0)
        log_err = U * ((p * (5 * az + 4)).sum(1, keepdims=True) + 50 + 3 * np.log(s))
        lp_err = log_err + U * (3 * np.abs(z) + 2 * np.abs(lp))
        ent = np.log(s)[:, 0] + (p * az).sum(1)
        ent_err = log_err[:, 0] * (1 + (p * az).sum(1)) + U * (p * az * (5 * az + 55)).sum(1) + 2 * U * ent
    return lp[np.arange(len(x)), ids], ent, lp, lp_err, ent_err


def run_logp(eng, rng, t, x, top, T=1.0, pad=0, off=0, ids=None, some=True):  # noqa: F811
    rows, V = x.shape
    print(f"logprobs t={t} rows={rows} V={V} top={top} T={T} pad={pad} off={off}", flush=True)
    x = coded(x, t)
    v = value(x, t)
    ids = rng.integers(0, V, rows) if ids is None else ids
    X, I = Rows(eng, x, t, pad, off), Dev(eng, ids.astype(np.int64))
    L, E = out_rows(eng, (rows, 1), F32), out_rows(eng, (rows, 1), F32)
    TI, TL = Dev(eng, np.full((rows, max(top, 1)), -7, np.int64)), Dev(eng, np.zeros((rows, max(top, 1)), np.float32))
    eng.token_logprobs(X.ptr, rows, V, ids=I.ptr if some else None, logprobs=L.ptr if some else None, entropy=E.ptr if some else None,
                       top=top, top_ids=TI.ptr if top else None, top_logprobs=TL.ptr if top else None, temperature=T, dtype=t, ld=X.ld)
    eng.sync()
    want, ent, lp, lp_err, ent_err = logp_ref(v, ids, T)
    if some:
        close(L.get()[:, 0], want, lp_err[np.arange(rows), ids], F32, "logprobs")
        close(E.get()[:, 0], ent, ent_err, F32, "entropy")
    if top:
        order = np.argsort(-v, axis=1, kind="stable")[:, :top]
        got = TI.get()
        assert (got == order).all(), (np.argwhere(got != order)[:3], got[got != order][:5], order[got != order][:5])
        r = np.arange(rows)[:, None]
        close(TL.get(), lp[r, order], lp_err[r, order], F32, "top log probabilities")


LOGP_V = [1, 2, 5, 63, 64, 65, 257, 1000, 4095, 4096, 4097, 8193, 16384, 16385, 32000, 32767, 32768, 32769, 50000, 131073]


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V", LOGP_V)
def test_logprobs_lengths(eng, V, t):  # noqa: F811
    rng = np.random.default_rng(V + t)
    x = 3 * rng.standard_normal((3, V))
    run_logp(eng, rng, t, x, min(V, 20))
    run_logp(eng, rng, t, x, min(V, 64), T=0.7, pad=3, off=1)
    run_logp(eng, rng, t, x[:1], min(V, 1), T=1.5)
    run_logp(eng, rng, t, x, 0)
    run_logp(eng, rng, t, x, min(V, 3), some=False)


@pytest.mark.parametrize("t", FLOATS)
def test_logprobs_many_rows(eng, t):  # noqa: F811
    rng = np.random.default_rng(160 + t)
    run_logp(eng, rng, t, 2 * rng.standard_normal((1500, 333)), 7, pad=1)
    run_logp(eng, rng, t, 2 * rng.standard_normal((300, 4100)), 64)
    run_logp(eng, rng, t, 2 * rng.standard_normal((70, 70000)), 64)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V", [50, 5000, 32000, 100000])
def test_logprobs_ties_and_masks(eng, V, t):  # noqa: F811
    """Equal logits go by the lower id, however many they are; -infinity leaves tokens out, but for one or a few too."""
    rng = np.random.default_rng(V + t)
    top = 20
    x = np.zeros((9, V))
    x[1] = rng.integers(-3, 4, V)  # thousands of equal ones
    x[2] = -np.inf
    x[2, [V - 1, V // 2, 3]] = (0.5, 1.5, 1.5)
    x[3] = np.sort(rng.standard_normal(V))
    x[4] = np.sort(rng.standard_normal(V))[::-1]
    x[5] = np.where(rng.random(V) < 0.5, -0.0, 0.0)  # equal
    x[6] = -np.inf
    x[6, V // 3] = -3.0
    x[7] = -1e30 if t != F16 else -6e4
    x[7, 7] = 30.0
    x[8, ::7] = 1.0
    ids = np.array([V - 1, 0, 3, V - 1, V // 2, 1, V // 3, 7, 7])
    run_logp(eng, rng, t, x, top, ids=ids)
    run_logp(eng, rng, t, x, 1, ids=ids, T=2.0)
    run_logp(eng, rng, t, x, 50, ids=ids, T=0.5, off=1, pad=1)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V", [50, 5000, 32000, 100000])
def test_logprobs_rows_without_a_number(eng, V, t):  # noqa: F811
    rng = np.random.default_rng(V + t)
    x = rng.standard_normal((6, V))
    x[0] = -np.inf  # no token can come
    x[1, V // 2] = np.nan
    x[2, V - 1] = np.inf
    x[3] = -np.inf
    x[3, 5] = np.nan
    x[4, [2, V - 2]] = np.nan
    ids = np.array([3, 3, 3, 3, 3, -1])  # and the last row's id is none
    X, I = Rows(eng, coded(x, t), t), Dev(eng, ids.astype(np.int64))
    L, E = out_rows(eng, (6, 1), F32), out_rows(eng, (6, 1), F32)
    TI, TL = Dev(eng, np.zeros((6, 4), np.int64)), Dev(eng, np.zeros((6, 4), np.float32))
    for bad in (V, -1, 2 ** 40, -2 ** 63):
        ids[5] = bad
        I = Dev(eng, ids.astype(np.int64))
        eng.token_logprobs(X.ptr, 6, V, ids=I.ptr, logprobs=L.ptr, entropy=E.ptr, top=4, top_ids=TI.ptr, top_logprobs=TL.ptr, dtype=t)
        eng.sync()
        lp, ent, ti, tl = L.get()[:, 0], E.get()[:, 0], TI.get(), TL.get()
        assert lp[0] == -np.inf and ent[0] == 0 and (ti[0] == np.arange(4)).all() and (tl[0] == -np.inf).all()
        assert np.isnan(lp[1:]).all() and np.isnan(ent[1:5]).all() and np.isfinite(ent[5]) and np.isnan(tl[1:5]).all()
        assert ti[1, 0] == V // 2 and ti[2, 0] == V - 1 and (ti[3] == [5, 0, 1, 2]).all() and (ti[4, :2] == [2, V - 2]).all()
        assert np.isfinite(tl[5]).all()


def test_logprobs_refusals(eng):  # noqa: F811
    from matmulfreellmcpu_amd import MmfError
    p = [Dev(eng, np.zeros((4, 64), np.float32)).ptr for _ in range(6)]
    ok = dict(ids=p[1], logprobs=p[2])
    for kw, why in ((dict(V=0), "vocabulary"), (dict(V=2 ** 20 + 1), "vocabulary"), (dict(top=65), "top"), (dict(V=3, top=4), "top"),
                    (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e-39), "temperature"), (dict(ld=63), "stride"),
                    (dict(logprobs=None), "go together"), (dict(top=2), "need"), (dict(ids=None, logprobs=None), "no output"),
                    (dict(entropy=p[2]), "overlaps"), (dict(entropy=p[0]), "overlaps"), (dict(ids=p[1] + 4), "aligned"), (dict(dtype=I8), "dtype")):
        with pytest.raises(MmfError, match=why):
            eng.token_logprobs(p[0], **{**dict(rows=4, V=64), **ok, **kw})
    eng.token_logprobs(None, 0, 64)
    eng.sync()


@pytest.mark.parametrize("name,mode", [("tiny", 0), ("small", 1), ("small", 2)])
def test_score_is_forward_and_logprobs(blobs, name, mode):
    """The model's own score: the log probabilities of its forward's logits, without their copy."""
    from matmulfreellmcpu_amd import Engine, MmfError
    e = Engine(0)
    try:
        e.load_blob(blobs(name), mode)
        ids = np.random.default_rng(3).integers(0, e.cfg.vocab_size, 37)
        logits = e.forward(ids)[:-1]
        want, ent, lp, lp_err, ent_err = logp_ref(logits, ids[1:], 1.0)
        got, gent, ti, tl = e.score(ids, top=5)
        n = len(want)
        close(got, want, lp_err[np.arange(n), ids[1:]], F32, "score")
        close(gent, ent, ent_err, F32, "entropy")
        order = np.argsort(-logits, axis=1, kind="stable")[:, :5]
        assert (ti == order).all()
        close(tl, np.take_along_axis(lp, order, 1), np.take_along_axis(lp_err, order, 1), F32, "top")
        again = e.score(ids)
        assert (again[0] == got).all() and (again[1] == gent).all()
        assert (e.forward(ids)[:-1] == logits).all()
        for bad in (dict(ids=ids[:1]), dict(ids=ids, top=65), dict(ids=[0, -1])):
            with pytest.raises(MmfError):
                e.score(**bad)
    finally:
        e.close()


# ---- together -----------------------------------------------------------------------------------------


class W8:
    def __init__(self, eng, rng, N, K):  # noqa: F811
        q, s = rng.integers(-127, 128, (N, K)).astype(np.int8), (0.02 / np.sqrt(K) * (0.5 + rng.random(N))).astype(np.float32)
        self.id, self.w = eng.register_w8(q, s), q * s[:, None].astype(np.float64)


class Layer:
    """A layer of linear attention with 8-bit weights on device buffers: the projection of queries, keys, values and gate,
    attention, its gated norm's codes, the output projection, the norms around it, an MLP matrix, and the logits' scores."""

    def __init__(self, eng, rng, hidden, heads, Dk, Dv, V, seqs, rows):  # noqa: F811
        self.eng, self.hd, self.H, self.Dk, self.Dv, self.V, self.seqs = eng, hidden, heads, Dk, Dv, V, seqs
        self.n, self.o = heads * (2 * Dk + 2 * Dv), heads * Dv
        self.w = {"qkvg": W8(eng, rng, self.n, hidden), "out": W8(eng, rng, hidden, self.o), "lm": W8(eng, rng, V, hidden)}
        f = np.float32
        self.host = {k: (1 + 0.1 * rng.standard_normal(n)).astype(f) for k, n in
                     (("norm", hidden), ("mix", self.o), ("post", hidden), ("pre", hidden))}
        self.host["decay"] = np.log1p(-2.0 ** -rng.uniform(2, 8, heads)).astype(f)
        self.p = {k: Dev(eng, v) for k, v in self.host.items()}
        self.state = np.zeros((seqs, heads, Dk, Dv))
        self.d_state = Dev(eng, self.state.astype(f))
        z = lambda n, t=f: Dev(eng, np.zeros((rows, n), t))  # noqa: E731
        self.b = dict(x=z(hidden), c=z(hidden, np.int8), s=z(1), qkvg=z(self.n), a=z(self.o), ac=z(self.o, np.int8), y=z(hidden), h=z(hidden),
                      hc=z(hidden, np.int8), logits=z(V), ids=z(1, np.int64), lp=z(1), ent=z(1), ti=z(3, np.int64), tl=z(3))

    def run(self, rows, lens=None):
        e, b, p, H, Dk, Dv, n = self.eng, self.b, self.p, self.H, self.Dk, self.Dv, self.n
        e.add_rmsnorm_q8(b["c"].ptr, b["s"].ptr, b["x"].ptr, p["norm"].ptr, rows, self.hd)
        e.w8_linear(self.w["qkvg"].id, b["c"].ptr, b["s"].ptr, b["qkvg"].ptr, rows)
        at = b["qkvg"].ptr
        e.decay_attention(b["a"].ptr, at, at + 4 * H * Dk, at + 8 * H * Dk, rows, H, Dk, Dv, decay=p["decay"].ptr, state=self.d_state.ptr,
                          lens=lens, seqs=self.seqs, ldq=n, ldk=n, ldv=n)
        e.block_norm_q8(b["ac"].ptr, b["s"].ptr, b["a"].ptr, rows, self.o, gate=at + 4 * H * (2 * Dk + Dv), act=2, w_post=p["mix"].ptr, ldgate=n)
        e.w8_linear(self.w["out"].id, b["ac"].ptr, b["s"].ptr, b["y"].ptr, rows)
        e.block_norm_q8(b["hc"].ptr, b["s"].ptr, b["y"].ptr, rows, self.hd, x=b["x"].ptr, w_post=p["post"].ptr, w_pre=p["pre"].ptr, scale=0.5,
                        h=b["h"].ptr)
        e.w8_linear(self.w["lm"].id, b["hc"].ptr, b["s"].ptr, b["logits"].ptr, rows)
        e.token_logprobs(b["logits"].ptr, rows, self.V, ids=b["ids"].ptr, logprobs=b["lp"].ptr, entropy=b["ent"].ptr, top=3, top_ids=b["ti"].ptr,
                         top_logprobs=b["tl"].ptr)

    def check(self, rows, lens, x, ids):
        """Step by step on the device's own inputs: codes flip at a half by the rounding of what came before."""
        b, h, H, Dk, Dv = {k: v.get()[:rows] for k, v in self.b.items()}, self.host, self.H, self.Dk, self.Dv
        real, s = block_ref(x, None, None, 0, None, h["norm"], None, 1.0, 1e-6)[2:]
        assert (np.abs(b["c"] - real) <= 0.5 + 1e-4).all()
        qkvg = (b["c"].astype(np.float64) * s[:, None]) @ self.w["qkvg"].w.T
        near(b["qkvg"], qkvg, 1e-6, "projection")
        q, k, v, g = np.split(b["qkvg"], np.cumsum([H * Dk, H * Dk, H * Dv]), 1)
        a, bound, self.state, err = decay_ref(q.reshape(rows, H, Dk), k.reshape(rows, H, Dk), v.reshape(rows, H, Dv),
                                              np.broadcast_to(h["decay"], (rows, H)), self.state, lens, Dk ** -0.5)
        close(b["a"].reshape(a.shape), a, bound + 1e-5 * np.abs(a).max(), F32, "attention")
        near(self.d_state.get(), self.state, 1e-5, "state")
        self.state = self.d_state.get().astype(np.float64)
        real, s = block_ref(b["a"], None, g, 2, h["mix"], None, None, 1.0, 1e-6)[2:]
        assert (np.abs(b["ac"] - real) <= 0.5 + 1e-4).all()
        near(b["y"], (b["ac"].astype(np.float64) * s[:, None]) @ self.w["out"].w.T, 1e-6, "output")
        hw, _, real, s = block_ref(b["y"], x, None, 0, h["post"], h["pre"], None, 0.5, 1e-6)
        near(b["h"], hw, 1e-6, "residual")
        assert (np.abs(b["hc"] - real) <= 0.5 + 1e-4).all()
        near(b["logits"], (b["hc"].astype(np.float64) * s[:, None]) @ self.w["lm"].w.T, 1e-6, "logits")
        want, ent, lp, lp_err, ent_err = logp_ref(b["logits"], ids, 1.0)
        close(b["lp"][:, 0], want, lp_err[np.arange(rows), ids], F32, "log probabilities")
        assert (b["ti"] == np.argsort(-b["logits"], axis=1, kind="stable")[:, :3]).all()


def near(got, want, tol, what):
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= tol, f"{what}: {off:.2e}"


def test_layer_prompt_then_tokens(eng):  # noqa: F811
    rng = np.random.default_rng(21)
    lens = [37, 1, 90, 5]
    L = Layer(eng, rng, 200, 3, 32, 48, 500, 4, sum(lens))
    for rows, ls in ((sum(lens), lens), (4, None), (4, None)):
        x, ids = rng.standard_normal((rows, 200)).astype(np.float32), rng.integers(0, 500, rows)
        for k, v in (("x", x), ("ids", ids.astype(np.int64))):
            eng._chk(eng.lib.mmf_upload(eng.h, L.b[k].ptr, v.ctypes.data_as(C.c_void_p), v.nbytes))
        L.run(rows, ls)
        eng.sync()
        L.check(rows, ls or [1] * 4, x, ids)


def test_layer_in_a_graph(eng):  # noqa: F811
    """Prompts and single tokens captured once and replayed between eager work: every replay equals the eager calls bit for bit."""
    hip = hip_graphs()
    for rows, lens in ((8, None), (300, [170, 0, 1, 99, 30, 0, 0, 0])):
        rng = np.random.default_rng(22)
        L, E = (Layer(eng, np.random.default_rng(23), 128, 2, 32, 64, 300, 8, rows) for _ in range(2))
        L.run(rows, lens), E.run(rows, lens)  # workspaces
        eng.sync()
        stream = C.c_void_p(eng.stream)
        graph, ge = captured(hip, stream, lambda: L.run(rows, lens))
        for step in range(4):
            x = rng.standard_normal((rows, 128)).astype(np.float32)
            for layer in (L, E):
                eng._chk(eng.lib.mmf_upload(eng.h, layer.b["x"].ptr, x.ctypes.data_as(C.c_void_p), x.nbytes))
            assert hip.hipGraphLaunch(ge, stream) == 0
            E.run(rows, lens)
            eng.sync()
            for k in ("a", "h", "hc", "logits", "lp", "ent", "ti", "tl"):
                a, b = L.b[k].get(), E.b[k].get()
                assert (a.view(np.uint8) == b.view(np.uint8)).all(), (step, k)
            assert (L.d_state.get() == E.d_state.get()).all()
        assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(graph) == 0

"""The linear attention layer's operators where offsets pass 32 bits, at the edges of their launch plans, in captured graphs
that share the workspace, and in two contexts at once, against plain numpy in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_layer8 as layer8
from test_gpu_layer import F16, F32, FLOATS, SENTINEL, STORE, U, Rows, captured, close, coded, hip_graphs, out_rows, value
from test_gpu_layer8 import PARTS, W8, decay_ref, logp_ref, run_block, run_decay, run_logp, run_w8
from test_gpu_parity import Dev, eng  # noqa: F401  (module fixture)

pytestmark = pytest.mark.gpu


# ---- rows far apart ---------------------------------------------------------------------------


class Far:
    """As Rows, in an arena of rows `step` bytes apart that all of a call's row tensors lie side by side in."""

    arena, step, at = None, 0, 0

    @classmethod
    def open(cls, eng, rows, step):  # noqa: F811
        cls.arena, cls.step, cls.at = Dev(eng, shape=(rows, step), dtype=np.uint8), step, 0

    def __init__(self, eng, a, t):  # noqa: F811
        self.eng, self.t, (self.rows, self.cols) = eng, t, a.shape
        host = np.full((self.rows, (self.cols * a.itemsize + 191) // 64 * 64), SENTINEL, np.uint8)
        self.host = host
        self._in(host)[:] = a
        self.start = Far.arena.ptr + Far.at
        self.ptr, self.ld = self.start + 64, Far.step // a.itemsize
        Far.at += host.shape[1]
        assert Far.at <= Far.step
        for r in range(self.rows):
            eng._chk(eng.lib.mmf_upload(eng.h, self.start + r * Far.step, host[r].ctypes.data_as(C.c_void_p), host.shape[1]))

    def _in(self, a):
        return a[:, 64:64 + self.cols * np.dtype(STORE[self.t]).itemsize].view(STORE[self.t])

    def get(self):
        got = np.empty_like(self.host)
        for r in range(self.rows):
            self.eng._chk(self.eng.lib.mmf_download(self.eng.h, got[r].ctypes.data_as(C.c_void_p), self.start + r * Far.step, got.shape[1]))
        around = got.copy()
        self._in(around)[:] = self._in(self.host)
        assert (around == self.host).all(), "memory around the tensor was written"
        return self._in(got).copy()


@pytest.fixture
def far(eng, monkeypatch):  # noqa: F811
    """Opens an arena for the row tensors of layer8's runs; arrays of one row or column stay as they are."""
    def rows(e, a, t, pad=0, off=0):
        return Far(e, a, t) if min(a.shape) > 1 else Rows(e, a, t, pad, off)

    def out(e, shape, t, pad=0, off=0):
        a = np.empty(shape, STORE[t])
        a.view(np.uint8)[...] = SENTINEL
        return rows(e, a, t, pad, off)

    monkeypatch.setattr(layer8, "Rows", rows)
    monkeypatch.setattr(layer8, "out_rows", out)
    yield lambda n, step: Far.open(eng, n, step)
    Far.arena = None


MANY, FEW = (200, 2 ** 26), (16, 2 ** 29)  # rows, bytes from one to the next: 12.5 and 8 GiB


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("shape,K,N", [(FEW, 200, 70), (MANY, 300, 130), (MANY, 130, 4700), (MANY, 70, 32768)])
def test_w8_rows_far_apart(eng, far, shape, K, N, t):  # noqa: F811
    far(*shape)
    run_w8(eng, np.random.default_rng(N), shape[0], K, N, t)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("lens", [[1] * 16, [200], [90, 0, 110], [67, 1, 132]])
def test_decay_rows_far_apart(eng, far, lens, t):  # noqa: F811
    far(*(FEW if len(lens) == 16 else MANY))
    run_decay(eng, np.random.default_rng(len(lens)), t, lens, 2, 64, 33)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("cols", [100, 10000, 40000])
def test_block_rows_far_apart(eng, far, cols, t):  # noqa: F811
    far(*MANY)
    run_block(eng, np.random.default_rng(cols), t, MANY[0], cols)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("V", [1000, 40000])
def test_logprobs_rows_far_apart(eng, far, V, t):  # noqa: F811
    far(*MANY)
    rng = np.random.default_rng(V)
    run_logp(eng, rng, t, 2 * rng.standard_normal((MANY[0], V)), 5)


def test_decay_states_past_4_gib(eng):  # noqa: F811
    """Only the last of 280 sequences have rows: their states of 16 MiB each lie past 4 GiB, and those before them, which
    hold anything, are not touched."""
    rng, f = np.random.default_rng(1), np.float32
    H, Dk, Dv, seqs, lens = 64, 256, 256, 280, [1, 2, 150]
    n, rows = H * Dk * Dv, sum(lens)
    S, first = Dev(eng, shape=(seqs, n)), seqs - len(lens)
    st = rng.standard_normal((len(lens), H, Dk, Dv)).astype(f)
    mark = np.full(64, 7.25, f)
    before = S.ptr + 4 * n * first - mark.nbytes
    eng._chk(eng.lib.mmf_upload(eng.h, before, mark.ctypes.data_as(C.c_void_p), mark.nbytes))
    eng._chk(eng.lib.mmf_upload(eng.h, S.ptr + 4 * n * first, st.ctypes.data_as(C.c_void_p), st.nbytes))
    q, k, v = (rng.standard_normal((rows, H * D)).astype(f) for D in (Dk, Dk, Dv))
    a = np.log1p(-2.0 ** -rng.uniform(2, 8, H)).astype(f)
    Q, K, V, A, O = Dev(eng, q), Dev(eng, k), Dev(eng, v), Dev(eng, a), Dev(eng, shape=(rows, H * Dv))
    eng.decay_attention(O.ptr, Q.ptr, K.ptr, V.ptr, rows, H, Dk, Dv, decay=A.ptr, state=S.ptr, lens=[0] * first + lens)
    eng.sync()
    got, gs, around = O.get().reshape(rows, H, Dv), np.empty_like(st), np.empty_like(mark)
    for to, at in ((gs, S.ptr + 4 * n * first), (around, before)):
        eng._chk(eng.lib.mmf_download(eng.h, to.ctypes.data_as(C.c_void_p), at, to.nbytes))
    assert (around == mark).all()
    heads = [0, 31, 63]  # (of 64, for the time the reference takes)
    pick = lambda x, D: x.reshape(rows, H, D)[:, heads]  # noqa: E731
    want, bound, new, err = decay_ref(pick(q, Dk), pick(k, Dk), pick(v, Dv), np.broadcast_to(a[heads], (rows, 3)), st[:, heads], lens, Dk ** -0.5)
    close(got[:, heads], want, bound, F32, "decay")
    assert (np.abs(gs[:, heads] - new) <= err + U * np.abs(new)).all()


# ---- launch plans -----------------------------------------------------------------------------


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (60, 70), (96, 128), (90, 128), (96, 131), (128, 128), (120, 60), (256, 256), (200, 129)])
def test_decay_tiles_of_each_width(eng, Dk, Dv, t):  # noqa: F811
    """Sequences of several tiles, of one, and of a row, at every width and evenness of a head."""
    run_decay(eng, np.random.default_rng(Dk + Dv), t, [300, 1, 0, 129, 45], 2, Dk, Dv)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("Dk,Dv", [(64, 96), (60, 70), (96, 128), (90, 127), (128, 72), (120, 130), (160, 136), (200, 129)])
def test_decay_tiles_of_many_heads(eng, Dk, Dv, t):  # noqa: F811
    """As above, of many heads that share their queries and keys."""
    run_decay(eng, np.random.default_rng(Dk + Dv), t, [300, 1, 0, 40], 68, Dk, Dv, q_heads=17, k_heads=34)


@pytest.mark.parametrize("t", FLOATS)
def test_decay_states_of_growing_heads(eng, t):  # noqa: F811
    """Log decays above 0 whose sum over a tile passes fp32, of a state that is 0 until the last rows: all results are finite."""
    H, D, n, f = 2, 32, 400, np.float32
    rng = np.random.default_rng(5)
    for log_decay in (0.5, 1.0, 2.0):
        print(f"growth t={t} {log_decay}", flush=True)
        q, k, v = (coded(rng.standard_normal((n, H * D)), t) for _ in range(3))
        k[:n - 30] = 0
        Q, K, V, A = Rows(eng, q, t), Rows(eng, k, t), Rows(eng, v, t), Dev(eng, np.full(H, log_decay, f))
        S, O = Dev(eng, np.zeros((1, H, D, D), f)), out_rows(eng, (n, H * D), t)
        eng.decay_attention(O.ptr, Q.ptr, K.ptr, V.ptr, n, H, D, D, decay=A.ptr, state=S.ptr, dtype=t)
        eng.sync()
        qq, kk, vv = (value(x, t).reshape(n, H, D) for x in (q, k, v))
        want, bound, new, err = decay_ref(qq, kk, vv, np.full((n, H), f(log_decay), np.float64), None, [n], D ** -0.5)
        mag = bound / ((D + 100) * U)
        over = np.abs(want) > 65000 if t == F16 else np.zeros(want.shape, bool)
        got = value(O.get(), t).reshape(want.shape)
        assert not np.isfinite(got[np.abs(want) > 66000]).any() or t != F16
        # An exponent of up to 30 * log_decay rounds its exponential by as many half steps more; the state's bound counts
        # 80 U of its magnitudes already.
        close(np.where(over, 0, got), np.where(over, 0, want), bound + (PARTS[t] + 60 * U) * mag, t, "growth")
        assert (np.abs(S.get() - new) <= 1.75 * err + U * np.abs(new)).all()


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("rows", [3, 256])
@pytest.mark.parametrize("units", [256, 512, 1024, 2048, 4096])
def test_logprobs_plans(eng, units, rows, t):  # noqa: F811
    """Vocabularies that a block's registers just hold, and one more, of few rows and of many."""
    rng = np.random.default_rng(units + rows)
    V = units * (4 if t == F32 else 8)
    for n in (V - 1, V, V + 1):
        run_logp(eng, rng, t, 3 * rng.standard_normal((rows, n)), 7)


@pytest.mark.parametrize("T", [1e-38, 1e-6, 1e30])
@pytest.mark.parametrize("V", [50, 40000])
def test_logprobs_temperatures(eng, V, T):  # noqa: F811
    """The smallest temperature leaves all to the largest logit, whose z of 0 it may not turn into a NaN."""
    rng = np.random.default_rng(V)
    run_logp(eng, rng, F32, 0.2 * rng.standard_normal((5, V)), 3, T=T)


@pytest.mark.parametrize("t", FLOATS)
@pytest.mark.parametrize("waves", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 17, 32])
def test_block_many_rows_of_each_width(eng, waves, t):  # noqa: F811
    """More rows than the chip has blocks for, with blocks of every number of waves, and of two vectors a thread."""
    rng, V = np.random.default_rng(waves), 4 if t == F32 else 8
    cols = waves * 64 * V
    for rows, n in ((4100 if waves == 1 else 1100, cols), (520, cols - 3)):
        run_block(eng, rng, t, rows, n, gate=["silu", "none", "plain", "sigmoid"][waves % 4], y=waves % 2 == 0)


# ---- graphs and contexts ------------------------------------------------------------------------


class Work:
    """A long attention and log probabilities of a vocabulary of two parts, both of which use the workspace."""

    def __init__(self, e, seed):
        rng, f = np.random.default_rng(seed), np.float32
        self.e, self.T, self.H, self.D, self.V, self.R = e, 600, 2, 64, 40000, 6
        x = rng.standard_normal((self.T, 3 * self.H * self.D)).astype(f)
        self.x, self.a = Dev(e, x), Dev(e, np.full(self.H, -0.05, f))
        self.logits, self.ids = Dev(e, (3 * rng.standard_normal((self.R, self.V))).astype(f)), Dev(e, rng.integers(0, self.V, self.R))
        self.outs = [Dev(e, np.zeros(s, t)) for s, t in (((self.T, self.H * self.D), f), ((self.R,), f), ((self.R,), f),
                                                          ((self.R, 9), np.int64), ((self.R, 9), f))]

    def attention(self):
        n, at = self.H * self.D, self.x.ptr
        self.e.decay_attention(self.outs[0].ptr, at, at + 4 * n, at + 8 * n, self.T, self.H, self.D, self.D, decay=self.a.ptr, ldq=3 * n,
                               ldk=3 * n, ldv=3 * n)

    def logprobs(self):
        o = [b.ptr for b in self.outs]
        self.e.token_logprobs(self.logits.ptr, self.R, self.V, ids=self.ids.ptr, logprobs=o[1], entropy=o[2], top=9, top_ids=o[3], top_logprobs=o[4])

    def clear(self):
        for b in self.outs:
            z = np.zeros(b.shape, b.dtype)
            self.e._chk(self.e.lib.mmf_upload(self.e.h, b.ptr, z.ctypes.data_as(C.c_void_p), z.nbytes))

    def get(self):
        self.e.sync()
        return [b.get() for b in self.outs]


def same(a, b):
    return all((x.view(np.uint8) == y.view(np.uint8)).all() for x, y in zip(a, b))


def test_workspace_in_graphs():
    """The workspace's first use is refused under capture, and leaves the capture alone; two graphs that share it replay in
    turn with eager calls between them."""
    from matmulfreellmcpu_amd import Engine, MmfError
    e, hip = Engine(0), hip_graphs()
    try:
        w = Work(e, 60)
        stream = C.c_void_p(e.stream)
        assert e.workspace_bytes() == 0

        def refused():
            for call in (w.attention, w.logprobs):
                with pytest.raises(MmfError, match="before the capture"):
                    call()

        graph, ge = captured(hip, stream, lambda: (refused(), e.token_logprobs(w.logits.ptr, w.R, 30000, entropy=w.outs[2].ptr, ld=w.V)))
        assert hip.hipGraphLaunch(ge, stream) == 0
        e.sync()
        assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(graph) == 0
        w.attention(), w.logprobs()
        want, size = w.get(), e.workspace_bytes()
        assert size > 0
        graphs = [captured(hip, stream, w.attention), captured(hip, stream, w.logprobs)]
        for step in range(4):
            w.clear()
            for _, ge in graphs[::1 if step % 2 else -1]:
                assert hip.hipGraphLaunch(ge, stream) == 0
            assert same(w.get(), want), step
            w.logprobs(), w.attention()
            assert same(w.get(), want), step
        assert e.workspace_bytes() == size
        for g, ge in graphs:
            assert hip.hipGraphExecDestroy(ge) == 0 and hip.hipGraphDestroy(g) == 0
    finally:
        e.close()


def test_two_contexts_at_once():
    """Calls of two contexts whose streams run side by side: each has its own workspace."""
    from matmulfreellmcpu_amd import Engine
    engines = [Engine(0), Engine(0)]
    try:
        works = [Work(e, 61 + i) for i, e in enumerate(engines)]
        want = []
        for w in works:
            w.attention(), w.logprobs()
            want.append(w.get())
            w.clear()
        for _ in range(10):
            for w in works:
                w.attention(), w.logprobs()
        assert all(same(w.get(), x) for w, x in zip(works, want))
        w8 = [W8(e, np.random.default_rng(70), 50, 40) for e in engines]
        engines[0].w8_release(w8[0].id)
        assert engines[1].w8_shape(w8[1].id) == (50, 40)
    finally:
        for e in engines:
            e.close()


def test_score_of_a_large_vocabulary(tmp_path):
    """The score of a model whose rows of logits are cut into parts."""
    from matmulfreellmcpu_amd import Engine, make_blob
    path = str(tmp_path / "wide.blob")
    make_blob(path, vocab=40001, hidden=64, layers=1)
    e = Engine(0)
    try:
        e.load_blob(path, 0)
        ids = np.random.default_rng(4).integers(0, 40001, 9)
        logits = e.forward(ids)[:-1]
        want, ent, lp, lp_err, ent_err = logp_ref(logits, ids[1:], 1.0)
        got, gent, ti, _ = e.score(ids, top=4)
        close(got, want, lp_err[np.arange(8), ids[1:]], F32, "score")
        close(gent, ent, ent_err, F32, "entropy")
        assert (ti == np.argsort(-logits, axis=1, kind="stable")[:, :4]).all()
    finally:
        e.close()

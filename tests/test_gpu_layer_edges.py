"""The layer operators at the edges of their launch plans, against plain numpy in 64 bits."""
import numpy as np
import pytest

from test_gpu_layer import F32, FLOATS, I8, run_norm, run_w4
from test_gpu_parity import eng  # noqa: F401  (module fixture)

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

"""`token_logprobs` on rows where the everyday tolerance shows nothing: rows sure of one token.  Definitions in 64 bits; u = 2^-24."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests.test_gpu_logprobs import U, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols,apart", [(64, 1024, 512), (64, 5000, 2048), (300, 5000, 2048), (300, 12000, 4096), (3, 32768, 1024), (20, 32768, 2048)])
def test_rows_sure_of_one_token(eng, rows, cols, apart, bf16):
    # Two tokens a row, the rest masked: first the smaller one, then, so many columns behind it that one thread meets both, one
    # 8 to 11 above it.  The larger term is within 4 u of 1 (the exponential of a rounding), the smaller within as much of
    # itself, and one addition: log S, and so the log probability, within 8 u of the 64-bit value, the entropy within 4 u more.
    rng = np.random.default_rng(cols)
    x = np.full((rows, cols), -np.inf, np.float32)
    at = rng.integers(0, cols - apart, rows)
    if cols == 32768:
        at = rng.integers(0, 1000, rows)
    gap = orc.from_bf16(orc.to_bf16(np.linspace(8.0, 11.05, rows).astype(np.float32))) if bf16 else np.linspace(8.0, 11.05, rows).astype(np.float32)
    x[np.arange(rows), at], x[np.arange(rows), at + apart] = 0.0, gap
    _, got = run(eng, x, at + apart, 1.0, 2, bf16)
    g = gap.astype(np.float64)
    log = -np.log1p(np.exp(-g))
    ent = -log * np.exp(log) - np.exp(log - g) * (log - g)
    assert np.all(np.abs(got[0] - log) <= 8 * U), float(np.abs(got[0] - log).max() / U)
    assert np.all(np.abs(got[1] - ent) <= 12 * U), float(np.abs(got[1] - ent).max() / U)
    assert np.all(np.abs(got[4][:, 0] - log) <= 8 * U)
    assert np.all(got[0] <= 0) and np.all(got[1] >= 0)

"""`attention_pages` where a result hangs on more than F32's everyday range: large scores, sums over thousands of tiles.
Definitions in 64 bits; u = 2^-24."""
import numpy as np
import pytest

from metalium_rs_b200 import BF16, PageShape
from oracle import oracle as orc
from tests.test_gpu_pages import U, tables, up, up_i32

pytestmark = pytest.mark.gpu


def half_step(x):
    """Half a BF16 step at x: 2^-8 of the power of two below it."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -126))) - 8)


@pytest.mark.parametrize("o_bf16", [True, False])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 192, 256])
def test_large_scores_of_f32_queries(eng, d, o_bf16):
    # Two positions a sequence whose scores, about 500 each, come from one channel each and differ by less than 1: an error of the
    # scores is an error of the result.  A score is one product of a query's three parts, each exact, joined by at most eight F32
    # operations: within 8 u of it; the weights by that and 16 u of their functions, numerator and denominator alike.
    rng = np.random.default_rng(d)
    n, heads, page = 40, 4, 16
    q = np.zeros((n, heads, d), np.float32)
    q[:, :, 3] = rng.uniform(28, 32, (n, heads))
    q[:, :, d - 2] = q[:, :, 3] + rng.uniform(-0.06, 0.06, (n, heads))
    table, pages = tables(rng, [2] * n, page)
    k, v = np.zeros((pages * page, d), np.float32), np.zeros((pages * page, d), np.float32)
    first = table[:, 0] * page
    k[first, 3] = k[first + 1, d - 2] = 16.0
    v[first] = orc.from_bf16(orc.to_bf16(rng.uniform(0.5, 1.0, (n, d)).astype(np.float32)))
    v[first + 1] = -v[first]
    iq, _ = up(eng, q.reshape(n, -1), False)
    ik, iv = up(eng, k, True)[0], up(eng, v, True)[0]
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, np.ones(n), 1, n)
    out, _ = eng.attention_pages(PageShape(heads, 1, d, page), (iq, (0, 0), (n, heads * d)), ik, iv, it, ip, 1.0, bf16=o_bf16)
    got = (orc.from_bf16(eng.download_bf16(out)) if o_bf16 else eng.download(out)).astype(np.float64).reshape(n, heads, d)
    a, b = 16 * q[:, :, 3].astype(np.float64), 16 * q[:, :, d - 2].astype(np.float64)
    want = np.tanh((a - b) / 2)[:, :, None] * v[first][:, None, :].astype(np.float64)
    tol = 2 * (8 * U * np.maximum(a, b) + 16 * U)[:, :, None] * np.abs(v[first])[:, None, :]
    if o_bf16:
        tol = tol + 2.0 ** -16 * np.abs(v[first])[:, None, :]                     # a weight's two parts
        tol = tol + half_step(np.abs(want) + tol)
    off = np.abs(got - want)
    assert np.all(off <= tol), float((off / tol).max())
    for i in (iq, ik, iv, it, ip, out):
        eng.free(i)


@pytest.mark.parametrize("d", [64, 128])
def test_a_long_mean_is_the_nearest_bf16(eng, d):
    # Zero queries: a result is the mean of about 32,000 values, every other one 2^-9 of the size of its neighbour (512 sequences over
    # the same pages: every warp sums a run of hundreds of tiles).  Weights and their sum are exact, a sum of sixteen values is within
    # 4 u; each of T tiles' additions to the running sum rounds to nearest, an error of at most u of it that is as often up as
    # down: eight standard deviations of T of them are 8 sqrt(T / 3) u, and the division and the joins of a sequence's runs,
    # 16 at most, are one each.  What remains is the result's own half step.
    rng = np.random.default_rng(d)
    n, page, longest = 512, 64, 32768
    lengths = longest - np.arange(n)
    ik = eng.zeros_dram((longest, d), BF16)[0]
    v = rng.uniform(0.5, 1.5, (longest, d)).astype(np.float32)
    v[1::2] *= np.float32(2.0 ** -9)
    iv, v = up(eng, v, True)
    table = np.broadcast_to(np.arange(longest // page, dtype=np.int32), (n, longest // page))
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, lengths - 1, 1, n)
    iq = eng.zeros_dram((n, d), BF16)[0]
    out, _ = eng.attention_pages(PageShape(1, 1, d, page), (iq, (0, 0), (n, d)), ik, iv, it, ip, 0.125, bf16=True)
    got = orc.from_bf16(eng.download_bf16(out)).astype(np.float64)
    want = np.cumsum(v.astype(np.float64), 0)[lengths - 1] / lengths[:, None]
    tol = (8 * np.sqrt(longest / 16 / 3) + 32) * U * want
    assert np.all(np.abs(got - want) <= half_step(want) + tol), int((np.abs(got - want) > half_step(want) + tol).sum())
    for i in (ik, iv, it, ip, iq, out):
        eng.free(i)

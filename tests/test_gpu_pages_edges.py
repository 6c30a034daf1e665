"""`attention_pages` where a result hangs on more than F32's everyday range: large scores, sums over thousands of tiles, scores
that leave the type's range, infinities and NaN among the attended values.  Definitions in 64 bits; u = 2^-24."""
import numpy as np
import pytest

from metalium_rs_b200 import BF16, BOOL, PageShape
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


def rows_and_pages(eng, q, k, v, scale, c_bf16, o_bf16, width):
    """The result of `attention_rows` and of `attention_pages`, [heads, d], for one sequence of whole positions, one key/value head."""
    heads, d = q.shape
    n, page = len(k), 16
    iq, ik, iv = up(eng, q, False)[0], up(eng, k, c_bf16)[0], up(eng, v, c_bf16)[0]
    mask = eng.upload_bits(np.zeros((1, n), np.uint32), 1, n, BOOL)
    one, _ = eng.attention_rows((iq, ik, iv, mask), [((h, 0), (0, 0), (0, 0)) for h in range(heads)], (1, d, n, d), scale)
    table = np.zeros((1, max(n // page, width)), np.int32)
    table[0, :n // page] = np.arange(n // page)
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, [n - 1], 1, 1)
    flat, _ = eng.reshape(iq, 1, heads * d)
    two, _ = eng.attention_pages(PageShape(heads, 1, d, page), (flat, (0, 0), (1, heads * d)), ik, iv, it, ip, scale, bf16=o_bf16)
    a = eng.download(one).reshape(heads, d)
    b = (orc.from_bf16(eng.download_bf16(two)) if o_bf16 else eng.download(two)).reshape(heads, d)
    for i in (iq, ik, iv, mask, one, it, ip, flat, two):
        eng.free(i)
    return a, b


@pytest.mark.parametrize("c_bf16,o_bf16", [(True, False), (True, True), (False, False)])
@pytest.mark.parametrize("width", [0, 3000])
@pytest.mark.parametrize("n", [32, 320])
def test_a_score_beyond_the_type_s_range(eng, n, width, c_bf16, o_bf16):
    # A product of 1e30 times a scale of 1e10 is infinite in F32: NaN, as the composition's steps give; to -inf it is weight 0.
    rng = np.random.default_rng(n)
    q, k = np.zeros((2, 64), np.float32), rng.standard_normal((n, 64)).astype(np.float32) * np.float32(1e-10)
    q[:, 0], q[:, 1], k[:, 0] = [2.0 ** 50, -2.0 ** 50], 1.0, 0.0
    k[n - 3, 0] = 2.0 ** 50
    v = rng.standard_normal((n, 64)).astype(np.float32)
    a, b = rows_and_pages(eng, q, k, v, 1e10, c_bf16, o_bf16, width)
    assert np.isnan(a[0]).all() and np.isfinite(a[1]).all()
    assert np.isnan(b[0]).all()
    # scores within 4, weights by (64 + 24) u of them and of their functions; the result's own step
    assert np.all(np.abs(a[1] - b[1]) <= 4 * 88 * 8 * U * np.abs(v).max() + (2.0 ** -8 if o_bf16 else U) * np.abs(a[1]))


@pytest.mark.parametrize("c_bf16", [True, False])
@pytest.mark.parametrize("length", [16, 40])
def test_a_score_beyond_the_type_s_range_at_a_sequence_s_end(eng, length, c_bf16):
    # The same for sequences that one warp sums whole, the infinite score the last of its last tile.
    rng = np.random.default_rng(length)
    n, page = 600, 16
    table, pages = tables(rng, [length] * n, page)
    q, k = np.ones((n, 64), np.float32), rng.standard_normal((pages * page, 64)).astype(np.float32) * np.float32(1e-12)
    q[:, 0], k[:, 0] = 2.0 ** 50, 0.0
    k[table[:, (length - 1) // page] * page + (length - 1) % page, 0] = 2.0 ** 50
    iq, ik = up(eng, q, False)[0], up(eng, k, c_bf16)[0]
    iv = up(eng, rng.standard_normal((pages * page, 64)).astype(np.float32), c_bf16)[0]
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, np.full(n, length - 1), 1, n)
    out, _ = eng.attention_pages(PageShape(1, 1, 64, page), (iq, (0, 0), (n, 64)), ik, iv, it, ip, 1e10)
    assert np.isnan(eng.download(out)).all()
    for i in (iq, ik, iv, it, ip, out):
        eng.free(i)


@pytest.mark.parametrize("c_bf16,o_bf16", [(True, False), (True, True), (False, False)])
@pytest.mark.parametrize("heads,d", [(1, 32), (8, 64), (3, 96), (11, 128), (2, 192), (4, 256)])
@pytest.mark.parametrize("n,width", [(32, 0), (320, 0), (320, 3000), (4096, 0)])
def test_infinite_and_nan_values(eng, n, width, heads, d, c_bf16, o_bf16):
    # What the composition's steps make of values that are no numbers: an infinity stays one, +inf beside -inf and a NaN are NaN,
    # and so is an infinity whose weight is 0.  The other columns are as if there were none.
    rng = np.random.default_rng(n + d)
    q, k, v = ((rng.standard_normal(s) * f).astype(np.float32) for s, f in (((heads, d), 0.3), ((n, d), 0.3), ((n, d), 1.0)))
    k = orc.from_bf16(orc.to_bf16(k)) if c_bf16 else k
    v = orc.from_bf16(orc.to_bf16(v)) if c_bf16 else v
    v[3, 0], v[n - 1, 1], v[n // 2, 5] = np.inf, -np.inf, np.nan
    v[5, 9], v[n - 2, 9] = np.inf, -np.inf                      # both in one column
    v[16, 11], v[17, 11] = np.inf, np.inf
    v[n // 2, 30] = np.inf
    if not c_bf16:
        v[9, 13] = np.finfo(np.float32).max                     # the largest value is one like the others
    a, b = rows_and_pages(eng, q, k, v, 0.5, c_bf16, o_bf16, width)
    assert np.isposinf(a[:, [0, 11, 30]]).all() and np.isneginf(a[:, 1]).all() and np.isnan(a[:, [5, 9]]).all()
    assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b))
    fin = np.isfinite(a)
    assert np.array_equal(np.sign(a[~fin]), np.sign(b[~fin]), equal_nan=True)
    # each form's scores: (d + 24) u of sum |q k|, and 2^-21 of it for operands in parts; its weights by that, numerator and
    # denominator; the sums n / 16 + 32 roundings; a weight's own parts; the result's step
    size = np.broadcast_to(np.where(np.isfinite(v), np.abs(v), 0).max(0), a.shape)
    mass = float((np.abs(q) @ np.abs(k).T).max()) * 0.5
    tol = (4 * ((d + 24) * U + 2.0 ** -21) * (mass + 1) + 4 * (n / 16 + 32) * U + (2.0 ** -16 if o_bf16 else 2.0 ** -20)) * size
    tol = tol + (2.0 ** -8 if o_bf16 else U) * (np.abs(a) + tol)
    with np.errstate(invalid="ignore"):
        assert np.all((np.abs(a - b) <= tol)[fin])


def test_an_infinite_value_behind_a_weight_of_zero(eng):
    # its product is NaN; behind the sequence's last position, or before its window, it is not read
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((2, 64), (64, 64), (64, 64)))
    q[:, 4] = 1.0
    k[10, 4] = -np.inf
    v[10, 2] = np.inf
    for c_bf16 in (True, False):
        a, b = rows_and_pages(eng, q, k, v, 0.25, c_bf16, False, 0)
        assert np.isnan(a[:, 2]).all() and np.array_equal(np.isnan(a), np.isnan(b))

"""`token_logprobs` and its gradient on rows where the everyday tolerance shows nothing: rows sure of one token, rows masked by the
type's lowest values, rows far from zero, padding rows.  Definitions in 64 bits; u = 2^-24.

What a row's results are held to goes by the terms that carry weight: with m the row's largest y, a term e^(y - m) is within
6 u |y - m| + 8 u of itself, which weighted by the term is below 12 u; the additions of a row of up to 32,768 are within 512 u;
so log sum, entropy (another factor |y - m|, weighted) and a log probability are within 600 u (1 + |entropy|) and 6 u |y - m| of the
token's own, whatever |m|, and only lse, which holds m itself, by 4 u |m| more."""
import numpy as np
import pytest

from oracle import oracle as orc
from tests.test_gpu_logprobs import U, grad64, logits, run, up, up_i32

pytestmark = pytest.mark.gpu


def weighted(eng, x, ids, scale=1.0, top=0, bf16=False):
    x, got = run(eng, x, ids, scale, top, bf16)
    n, cols = x.shape
    y = x.astype(np.float64) * np.float64(np.float32(scale))
    m = y.max(1)
    z = y - m[:, None]
    p = np.exp(z)
    s = p.sum(1)
    p /= s[:, None]
    log = z - np.log(s)[:, None]
    ent = -np.where(p > 0, p * log, 0).sum(1)
    spread = np.where(p > 0, p * -z, 0).sum(1)
    sums = 600 * U * (1 + ent + spread)
    r = np.arange(n)
    token = np.where(ids < 0, 0.0, log[r, np.maximum(ids, 0)])
    own = np.where(ids < 0, 0.0, -z[r, np.maximum(ids, 0)])
    assert np.all(np.abs(got[0] - token) <= sums + 6 * U * own), (got[0], token)
    assert np.all(np.abs(got[1] - ent) <= sums), (got[1], ent)
    assert np.all(np.abs(got[2] - (m + np.log(s))) <= sums + 4 * U * np.abs(m)), (got[2], m + np.log(s))
    if top:
        best = np.argsort(-x.astype(np.float64), 1, kind="stable")[:, :top]
        assert np.array_equal(got[3], best)
        assert np.all(np.abs(got[4] - np.take_along_axis(log, best, 1)) <= sums[:, None] + 6 * U * -np.take_along_axis(z, best, 1))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(9, 40), (9, 1000), (9, 3001), (300, 3001), (300, 20011), (9, 32768)])
def test_rows_masked_by_the_type_s_lowest_values(eng, rows, cols, bf16):
    rng = np.random.default_rng(cols)
    x = logits(rng, rows, cols)
    low = orc.from_bf16(np.array([0xFF7F], np.uint16))[0] if bf16 else np.finfo(np.float32).min
    for i, mask in enumerate((-3.0e38, low, -1.0e30, -1.0e31, -2.0e9)):
        live = rng.random(cols) < 0.2
        live[cols // 2] = True
        x[i] = np.where(live, x[i], mask)
    x[5], x[6], x[7] = low, -1.0e30, -1.0e31                # nothing left: all alike
    x[8], x[8, 1] = -3.0e38, -2.9e38
    ids = np.full(rows, cols // 2)
    for top in (0, min(20, cols)):
        weighted(eng, x, ids, 1.0, top, bf16)


@pytest.mark.parametrize("rows,cols", [(8, 100), (8, 3000), (300, 3000), (300, 12000), (2, 32768)])
def test_rows_far_from_zero_keep_their_differences(eng, rows, cols):
    # In 1e8 .. 4e8, where F32's step is 8 to 32, and beyond: three largest and ten next to them, the others far below.
    rng = np.random.default_rng(rows + cols)
    base = np.array([1.0e6, -1.0e6, 1.2e8, -1.2e8, 4.0e8, 3.0e12, -3.0e12, 2.0e30])
    x = np.empty((rows, cols), np.float32)
    scale = 0.25
    for i in range(rows):
        b = np.float32(base[i % len(base)])
        step = np.spacing(np.abs(b))
        at = rng.permutation(cols)
        x[i] = b - 4000 * step
        x[i, at[:3]] = b
        x[i, at[3:13]] = b - step
        x[i, at[13:30]] = b - 2 * step
    ids = x.argmax(1)
    ids[1::2] = [int(np.flatnonzero(r == r.max() - np.spacing(np.abs(r.max())))[0]) if (r == r.max() - np.spacing(np.abs(r.max()))).any() else 0
                 for r in x[1::2]]
    weighted(eng, x, ids, scale, 5)
    weighted(eng, x, ids, 1.0)


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


# ------------------------------------------------------------------------------------------------ the gradient
def gradient(eng, x, ids, g, h, scale, bf16, o_bf16):
    n, cols = x.shape
    ix, x = up(eng, x, bf16)
    ii = up_i32(eng, ids, n, 1)
    (lp, _), (en, _), (ls, _) = eng.token_logprobs(ix, ii, scale)
    ig = eng.upload(g.astype(np.float32).reshape(n, 1), n, 1)
    ih = None if h is None else eng.upload(h.astype(np.float32).reshape(n, 1), n, 1)
    out, _ = eng.token_logprobs_backward(ix, ii, ls, None if h is None else en, ig, ih, scale, o_bf16)
    got = orc.from_bf16(eng.download_bf16(out)) if o_bf16 else eng.download(out)
    lse, ent = eng.download(ls)[:, 0], eng.download(en)[:, 0]
    for i in [ix, ii, lp, en, ls, ig, out] + ([] if ih is None else [ih]):
        eng.free(i)
    return x, got.astype(np.float64), lse, ent


@pytest.mark.parametrize("bf16,o_bf16", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("cols", [5, 33, 1003, 20011])
def test_padding_rows_have_no_gradient_whatever_they_hold(eng, cols, bf16, o_bf16):
    rng = np.random.default_rng(cols)
    x = logits(rng, 8, cols)
    x[1] = np.nan
    x[3, cols // 2] = np.nan
    x[4, 0] = np.inf
    x[5] = -np.inf
    x[6] = np.inf
    ids = np.array([0, -1, cols - 1, -1, -1, -1, -1, -1])
    g = rng.standard_normal(8)
    for h in (None, np.zeros(8)):
        x_, got, lse, ent = gradient(eng, x, ids, g, h, 1.0, bf16, o_bf16)
        assert not got[[1, 3, 4, 5, 6, 7]].any()
        want, tol = grad64(x_[[0, 2]], ids[[0, 2]], lse[[0, 2]], ent[[0, 2]], g.astype(np.float32)[[0, 2]], None, 1.0)
        assert np.all(np.abs(got[[0, 2]] - want) <= tol + (2.0 ** -8 if o_bf16 else 2 * U) * np.abs(want) + 2.0 ** -126)


@pytest.mark.parametrize("bf16,o_bf16", [(False, False), (True, True), (False, True)])
@pytest.mark.parametrize("rows,cols", [(9, 7), (9, 1003), (9, 20011), (400, 257)])
def test_gradient_of_rows_whose_lse_holds_no_log(eng, rows, cols, bf16, o_bf16):
    # From 4096 on F32's step is 2^-11 and more, at 2^20 an eighth: the sum's logarithm, and with it p, is not in lse.  The gradient
    # is that of the definition: p within 600 u, an entropy's factor within 600 u (1 + entropy + its own |log p|).
    rng = np.random.default_rng(rows + cols)
    low = orc.from_bf16(np.array([0xFF7F], np.uint16))[0] if bf16 else np.finfo(np.float32).min
    x = logits(rng, rows, cols)
    x[0], x[1], x[2] = low, -1.0e30, 1.0e30                  # all alike
    x[3] = np.where(np.arange(cols) % 3 == 0, -2.0e6, low)
    x[4] = rng.integers(0, 3, cols) * 2.0 ** 17 + 2.0 ** 21 if bf16 else rng.integers(0, 9, cols) * 0.5 + 3.0e6
    x[5] = -np.inf
    x[5, 2] = -3.0e7
    x[6] = 1.1e6
    x[7] += 8000
    ids = rng.integers(0, cols, rows)
    ids[6] = -1
    g = rng.standard_normal(rows).astype(np.float32)
    for h in (None, rng.standard_normal(rows).astype(np.float32)):
        x_, got, _, _ = gradient(eng, x, ids, g, h, 1.0, bf16, o_bf16)
        y = x_[:8].astype(np.float64)
        z = y - y.max(1, keepdims=True)
        log = z - np.log(np.exp(z).sum(1, keepdims=True))
        p = np.exp(log)
        one = np.arange(cols)[None, :] == ids[:8, None]
        up_ = np.where(ids[:8] >= 0, g[:8], 0.0)[:, None].astype(np.float64)
        want, tol = up_ * (one - p), 600 * U * np.abs(up_) * p
        if h is not None:
            ent = -np.where(p > 0, p * log, 0).sum(1, keepdims=True)
            inner = np.where(p > 0, p * (log + ent), 0)
            want = want - h[:8, None] * inner
            tol = tol + 600 * U * np.abs(h[:8, None]) * p * (1 + ent + np.where(p > 0, -log, 0)) * 2
        tol = tol + (2.0 ** -8 if o_bf16 else 4 * U) * (np.abs(want) + tol) + 4 * U * np.abs(up_) * one + 2.0 ** -126
        off = np.abs(got[:8] - want)
        assert np.all(off <= tol), (np.argwhere(off > tol)[:4], got[:8][off > tol][:4], want[off > tol][:4])

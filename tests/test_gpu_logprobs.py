"""`token_logprobs` and its gradient through the C ABI against their definitions in 64 bits.

Tolerances, u = 2^-24, m the row's largest y = scale x:
  - a term e^(y - m): y's product and the difference are rounded (2 u |y| + u |y - m|), the function is within 8 u.  Weighted by
    the term itself, |y - m| e^(y - m) <= 1 / e: the sum S is within (2 u max|y| + 12 u) S, and its additions within 512 u S
    (at most 256 values a lane of a row of 2^18 and 24 levels above them).  So lse, a log probability (each two roundings
    more) and the entropy, whose T is as S with another factor |y - m| <= max|y| + |m|:
        (2 max|y| + 600) u (1 + |entropy|)  +  4 u |result|.
  - a gradient's p = e^(y - lse) is within (3 |y| + 2 |lse| + 8) u p, its factors within 8 u, the result within half a step
    of its type (2^-8 of a BF16)."""
import numpy as np
import pytest

from metalium_rs_b200 import BF16, I32, SUM, COLS, TtError
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def up(eng, x, bf16):
    if bf16:
        h = orc.to_bf16(x)
        return eng.upload_bf16(h, *x.shape), orc.from_bf16(h)
    return eng.upload(x, *x.shape), x


def up_i32(eng, a, r, c):
    return eng.upload_bits(np.ascontiguousarray(a, dtype=np.int32).view(np.uint32), r, c, I32)


def definition(x, ids, scale, top):
    """(logprob, entropy, lse, columns, their log probabilities), 64 bits, `argmax_row`'s order."""
    y = x.astype(np.float64) * np.float64(np.float32(scale))
    rows = np.arange(len(x))
    with np.errstate(all="ignore"):
        m = y.max(1, keepdims=True)
        e = np.where(np.isneginf(m), 0.0, np.exp(y - m))
        s = e.sum(1, keepdims=True)
        empty = np.isneginf(m[:, 0])
        lse = np.where(empty, -np.inf, m[:, 0] + np.log(s[:, 0]))
        log = np.where(empty[:, None], -np.inf, y - lse[:, None])
        p = np.where(empty[:, None], 0.0, np.exp(log))
        ent = -np.where(p == 0, 0.0, p * log).sum(1)
    lp = np.where(ids < 0, 0.0, log[rows, np.maximum(ids, 0)])
    key = np.where(np.isnan(x), np.inf, x).astype(np.float64)
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), -(key + 0.0), ~np.isnan(x)), axis=1)[:, :top]
    return lp, ent, lse, order, np.take_along_axis(log, order, 1)


def run(eng, x, ids, scale, top, bf16, view=0):
    n, cols = x.shape
    if view:                                       # the rows start `view` rows into a larger buffer
        whole = np.concatenate([np.full((view, cols), 1e30, np.float32), x, np.full((1, cols), 1e30, np.float32)])
        parent, held = up(eng, whole, bf16)
        ix, x = eng.slice_rows(parent, view, n)[0], held[view:view + n]
    else:
        ix, x = up(eng, x, bf16)
    ii = up_i32(eng, ids, n, 1)
    got = eng.token_logprobs(ix, ii, scale, top)
    out = [eng.download(i)[:, 0].astype(np.float64) for i, _ in got[:3]]
    out += [eng.download_bits(got[3][0]).view(np.int32), eng.download(got[4][0]).astype(np.float64)] if top else []
    for i in [ix, ii] + [g for g, _ in got] + ([parent] if view else []):
        eng.free(i)
    return x, out


def check(eng, x, ids, scale=1.0, top=0, bf16=False, view=0):
    x, got = run(eng, x, ids, scale, top, bf16, view)
    want = definition(x, ids, scale, top)
    y = np.abs(x.astype(np.float64) * scale)
    big = np.where(np.isfinite(y), y, 0.0).max(1)
    tol = (2 * big + 600) * U * (1 + np.abs(np.nan_to_num(want[1])))
    for name, g, w in zip(("logprob", "entropy", "lse"), got, want):
        same = (g == w) | (np.isnan(g) & np.isnan(w))
        with np.errstate(invalid="ignore"):
            ok = same | (np.abs(g - w) <= tol + 4 * U * np.abs(w))
        assert ok.all(), (name, g[~ok][:3], w[~ok][:3])
    if top:
        assert np.array_equal(got[3], want[3]), np.argwhere(got[3] != want[3])[:4]
        with np.errstate(invalid="ignore"):
            ok = (got[4] == want[4]) | (np.isnan(got[4]) & np.isnan(want[4])) | (np.abs(got[4] - want[4]) <= tol[:, None] + 4 * U * np.abs(want[4]))
        assert ok.all()


def logits(rng, rows, cols):
    x = rng.standard_normal((rows, cols)).astype(np.float32) * 3
    x[np.arange(rows), rng.integers(0, cols, rows)] = 12
    return x


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [1, 2, 7, 10, 31, 32, 33, 100, 255, 257, 1000, 1023, 1024, 1025, 2049, 4095, 8193, 49152, 50257, 131075])
def test_logprobs_of_any_width(eng, cols, bf16):
    rng = np.random.default_rng(cols)
    rows = 3 if cols > 5000 else 37
    ids = rng.integers(0, cols, rows)
    ids[0], ids[1], ids[2] = 0, cols - 1, -1
    for top in sorted({0, 1, min(5, cols), min(32, cols)}):
        check(eng, logits(rng, rows, cols), ids, 0.8 if top == 5 else 1.0, top, bf16)


@pytest.mark.parametrize("rows,cols", [(1, 49152), (2, 262145), (5, 49152), (40, 32001), (160, 20000), (700, 5003), (3000, 10), (5001, 33), (1500, 1100)])
def test_logprobs_of_any_count_of_rows(eng, rows, cols):
    rng = np.random.default_rng(rows)
    ids = rng.integers(-1, cols, rows)
    check(eng, logits(rng, rows, cols), ids, 1.3, min(cols, 20), rows % 2 == 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(300, 1500), (297, 9999), (296, 10001), (310, 20011), (296, 33000)])
def test_many_rows_with_hard_ones_among_them(eng, rows, cols, bf16):
    # Rows enough to fill the GPU one a block: every eighth is of few values, masked, rising or holds a NaN or an infinity.
    rng = np.random.default_rng(cols)
    x = logits(rng, rows, cols)
    hard = [np.full(cols, -2.5), np.full(cols, -np.inf), np.where(np.arange(cols) == cols - 1, 1.0, -np.inf),
            np.arange(cols) // (cols // 200), np.arange(cols)[::-1] // (cols // 200), rng.integers(-1, 2, cols),
            np.where(np.arange(cols) == cols // 2, np.nan, 0.5), np.where(np.arange(cols) == 1, np.inf, 0.5),
            np.where(rng.random(cols) < 0.999, -3.0e38, 4.0), np.where(np.arange(cols) < cols - 7, -np.inf, 2.0)]
    for i in range(0, rows, 8):
        x[i] = hard[i // 8 % len(hard)]
    ids = rng.integers(-1, cols, rows)
    for top, view in ((20, 0), (32, 3), (0, 1)):
        check(eng, x, ids, 0.9, top, bf16, view)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [33, 1000, 5000, 49153])
def test_equal_values_go_by_the_lower_column(eng, cols, bf16):
    rng = np.random.default_rng(cols)
    x = rng.integers(-2, 3, (6, cols)).astype(np.float32)
    x[0] = 1.0                                              # all equal
    x[1] = np.arange(cols)[::-1] // 3                       # falling: the largest come first
    x[2] = np.arange(cols) // 3                             # rising
    x[3] = np.where(rng.random(cols) < 0.5, 0.0, -0.0)      # the two zeros are one value
    if bf16:
        x[1:3] = np.minimum(x[1:3], 250)
    check(eng, x, rng.integers(0, cols, 6), 1.0, 32, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [5, 40, 3001, 50001])
def test_infinite_and_nan_logits(eng, cols, bf16):
    rng = np.random.default_rng(cols)
    x = logits(rng, 9, cols)
    x[0] = -np.inf                                          # masked altogether
    x[1] = -np.inf
    x[1, cols - 2] = 3.0                                    # one left
    x[2, rng.random(cols) < 0.9] = -np.inf
    x[2, 0] = 1.0
    x[3, cols // 2] = np.nan
    x[4, cols // 2] = np.inf
    x[5] = np.nan
    x[6, :] = -3.0e38                                       # masked by the type's lowest values, not -inf
    x[6, 1] = 2.0
    x[7, :] = -3.0e38
    x[8, cols - 1], x[8, 1] = np.nan, np.nan
    ids = np.array([0, cols - 2, 0, 1, 1, 2, 1, 3, 0])
    check(eng, x, ids, 1.0, min(cols, 32), bf16)
    ids[1:3] = [0, -1]                                      # a masked token: -inf
    x[2, 3] = -np.inf
    check(eng, x, ids, 0.5, 1, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [33, 50257, 4099])
def test_rows_that_start_at_no_vector_s_boundary(eng, cols, bf16):
    rng = np.random.default_rng(5)
    for view in (1, 2, 3):
        check(eng, logits(rng, 3, cols), np.array([0, cols - 1, 7]), 1.0, 20, bf16, view)


def test_large_logits_keep_their_differences(eng):
    x = np.full((3, 3000), 1.0e6, np.float32)
    x[0, 5] += 3
    x[1] = -1.0e6
    x[1, 7] += 2
    x[2] = np.linspace(-1e30, 1e30, 3000)
    check(eng, x, np.array([5, 7, 2999]), 1.0, 5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("cols", [100, 3001, 50001])
@pytest.mark.parametrize("scale", [1.0e-20, 1.0e-6, 1.0e6])
def test_masked_logits_at_the_ends_of_the_scale(eng, cols, bf16, scale):
    rng = np.random.default_rng(cols)
    x = (logits(rng, 5, cols) / np.float32(scale)).astype(np.float32)    # 3e21 at most
    x[:, rng.random(cols) < 0.5] = -np.inf
    x[:, 0] = 0.0
    x[1, 1:] = -np.inf
    check(eng, x, np.array([0, 0, 0, -1, 0]), scale, 20, bf16)


def test_a_token_outside_the_columns_is_reported(fresh_eng):
    e = fresh_eng
    x = np.zeros((3, 10), np.float32)
    ix, ii = e.upload(x, 3, 10), up_i32(e, [10, -2, 4], 3, 1)
    got = e.token_logprobs(ix, ii, 1.0, 2)
    dst = np.empty((3, 1), np.float32)
    with pytest.raises(TtError) as err:
        e.download_into(got[0][0], dst.ctypes.data, 3)
    assert err.value.status == 6
    assert dst[0, 0] == 0 and dst[1, 0] == 0 and abs(dst[2, 0] + np.log(10.0)) <= 16 * U * np.log(10.0)


# ------------------------------------------------------------------------------------------------ the gradient
def grad64(x, ids, lse, ent, g, h, scale):
    scale = np.float64(np.float32(scale))
    y = x.astype(np.float64) * scale
    with np.errstate(all="ignore"):
        z = y - lse[:, None].astype(np.float64)
        z[np.isneginf(lse)] = -np.inf
        p = np.exp(z)
        one = np.arange(x.shape[1])[None, :] == ids[:, None]
        up_ = np.where(ids >= 0, g, 0.0)[:, None]
        out = up_ * (one - p)
        mag = np.abs(up_) * np.maximum(p, np.where(one, np.abs(1 - p), p))
        rel = (3 * np.abs(y) + 2 * np.abs(lse[:, None]) + 8) * U
        tol = np.abs(up_) * p * rel + 8 * U * mag
        if h is not None:
            inner = np.where(p == 0, 0.0, p * (z + ent[:, None]))
            out = out - h[:, None] * inner
            size = np.where(p == 0, 0.0, p * (np.abs(y) + np.abs(lse[:, None]) + np.abs(ent[:, None]) + 1))
            tol = tol + np.abs(h[:, None]) * size * (rel + 8 * U)
        out[np.isneginf(lse)] = 0.0
        tol = np.where(np.isfinite(tol), tol, 0.0)
    return out * scale, tol * scale


def backward(eng, x, ids, g, h, scale, bf16, o_bf16, view=0):
    n, cols = x.shape
    if view:
        parent, held = up(eng, np.concatenate([np.zeros((view, cols), np.float32), x]), bf16)
        ix, x = eng.slice_rows(parent, view, n)[0], held[view:]
    else:
        ix, x = up(eng, x, bf16)
    ii = up_i32(eng, ids, n, 1)
    (lp, _), (en, _), (ls, _) = eng.token_logprobs(ix, ii, scale)
    ig = eng.upload(g.astype(np.float32).reshape(n, 1), n, 1)
    ih = eng.upload(h.astype(np.float32).reshape(n, 1), n, 1) if h is not None else None
    out, dims = eng.token_logprobs_backward(ix, ii, ls, en if h is not None else None, ig, ih, scale, o_bf16)
    assert dims == (n, cols)
    got = orc.from_bf16(eng.download_bf16(out)) if o_bf16 else eng.download(out)
    lse, ent = eng.download(ls)[:, 0], eng.download(en)[:, 0]
    for i in [ix, ii, lp, en, ls, ig, out] + ([ih] if ih else []) + ([parent] if view else []):
        eng.free(i)
    g32, h32 = g.astype(np.float32).astype(np.float64), None if h is None else h.astype(np.float32).astype(np.float64)
    want, tol = grad64(x, ids, lse, ent, g32, h32, scale)
    return got.astype(np.float64), want, tol + (2.0 ** -8 if o_bf16 else 2 * U) * np.abs(want) + 2.0 ** -126


@pytest.mark.parametrize("bf16,o_bf16", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (37, 10), (5, 31), (9, 33), (300, 257), (4, 1023), (3, 4097), (2, 50257), (1, 262145), (2000, 17)])
def test_gradient_is_the_formula_s(eng, rows, cols, bf16, o_bf16):
    rng = np.random.default_rng(rows * cols)
    ids = rng.integers(-1, cols, rows)
    for h in (None, rng.standard_normal(rows)):
        got, want, tol = backward(eng, logits(rng, rows, cols), ids, rng.standard_normal(rows), h, 0.7 if h is None else 1.0, bf16, o_bf16)
        off = np.abs(got - want)
        assert np.all(off <= tol), (float((off / tol).max()), np.argwhere(off > tol)[:3])


@pytest.mark.parametrize("view", [1, 3])
@pytest.mark.parametrize("bf16,o_bf16", [(False, False), (True, True), (True, False), (False, True)])
def test_gradient_of_rows_that_start_at_no_vector_s_boundary(eng, view, bf16, o_bf16):
    rng = np.random.default_rng(view)
    got, want, tol = backward(eng, logits(rng, 5, 1003), np.array([0, 1002, 5, -1, 700]), rng.standard_normal(5), rng.standard_normal(5), 1.0, bf16, o_bf16, view)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("cols", [40, 3001])
def test_gradient_of_masked_rows(eng, cols):
    rng = np.random.default_rng(cols)
    x = logits(rng, 6, cols)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, 4] = 2.0
    x[2, rng.random(cols) < 0.8] = -np.inf
    x[2, 3] = 0.5
    x[3, :] = -3.0e38
    x[3, 9] = 1.0
    x[4, 7] = -np.inf
    ids = np.array([0, 4, 3, 9, 7, -1])                     # row 4: the given token is itself masked
    got, want, tol = backward(eng, x, ids, rng.standard_normal(6), rng.standard_normal(6), 1.0, False, False)
    assert np.isfinite(got).all() and not got[0].any()
    assert np.all(np.abs(got - want) <= tol)
    assert not got[np.isneginf(x) & (np.arange(cols)[None, :] != ids[:, None])].any()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("scale,h", [(1.0, 1.0e10), (1.0, 1.0e30), (1.0e6, 1.0), (1.0e6, 1.0e6), (1.0e-20, 1.0)])
def test_masked_entries_have_no_gradient_whatever_the_factors(eng, scale, h, bf16):
    # 0 times an infinite factor would be NaN
    rng = np.random.default_rng(17)
    x = (logits(rng, 5, 1003) / np.float32(scale)).astype(np.float32)
    x[:, rng.random(1003) < 0.5] = -np.inf
    x[:, [0, 500, 1002]] = 0.0
    x[2, 500] = -3.0e38
    ids = np.array([0, 500, 1002, -1, 0])
    got, want, tol = backward(eng, x, ids, rng.standard_normal(5), np.full(5, h), scale, bf16, False)
    assert np.isfinite(got).all()
    assert not got[np.isneginf(x)].any()
    assert np.all(np.abs(got - want) <= tol)


def test_gradient_against_differences(eng):
    """Central differences of the 64-bit definition: the step's own error is h^2 / 6 of a third derivative below 4."""
    rng = np.random.default_rng(12)
    rows, cols, scale, step = 3, 12, 1.25, 1e-4
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    ids, g, h = np.array([3, 0, 11]), rng.standard_normal(rows), rng.standard_normal(rows)
    got, _, _ = backward(eng, x, ids, g, h, scale, False, False)

    def value(a):
        lp, ent, _, _, _ = definition(a, ids, scale, 0)
        return (g.astype(np.float32) * lp + h.astype(np.float32) * ent).sum()

    x64 = x.astype(np.float64)
    for r in range(rows):
        for c in range(cols):
            a, b = x64.copy(), x64.copy()
            a[r, c] += step
            b[r, c] -= step
            assert abs((value(a) - value(b)) / (2 * step) - got[r, c]) <= 2e-6, (r, c)


def test_gradient_rows_sum_to_zero(eng):
    """Softmax does not see a shift of its row: each row's gradient sums to zero, here on the device's own sum."""
    rng = np.random.default_rng(13)
    x = logits(rng, 16, 2000)
    ix, ii = eng.upload(x, 16, 2000), up_i32(eng, rng.integers(0, 2000, 16), 16, 1)
    (lp, _), (en, _), (ls, _) = eng.token_logprobs(ix, ii)
    one = eng.upload(np.ones((16, 1), np.float32), 16, 1)
    out, _ = eng.token_logprobs_backward(ix, ii, ls, en, one, one)
    total, _ = eng.reduce(out, SUM, COLS)
    # 2000 terms, each within (3 |y| + 2 |lse| + 16) u of itself and their absolute sum below 2 + 2 (|lse| + entropy) < 60
    assert np.abs(eng.download(total)).max() <= 60 * (3 * 12 + 2 * 14 + 16 + 2000) * U
    for i in (ix, ii, lp, en, ls, one, out, total):
        eng.free(i)


def test_results_into_buffers_and_replays(eng):
    rng = np.random.default_rng(14)
    rows, cols, top = 7, 5003, 5
    x = [logits(rng, rows, cols) for _ in range(3)]
    ids = rng.integers(0, cols, rows)
    ix, ii = eng.upload(x[0], rows, cols), up_i32(eng, ids, rows, 1)
    into = [eng.zeros_dram((rows, 1))[0] for _ in range(3)] + [eng.zeros_dram((rows, top), I32)[0], eng.zeros_dram((rows, top))[0]]
    grad = eng.zeros_dram((rows, cols))[0]
    one = eng.upload(np.ones((rows, 1), np.float32), rows, 1)

    def step():
        got = eng.token_logprobs(ix, ii, 1.0, top, into)
        assert [i for i, _ in got] == into
        assert eng.token_logprobs_backward(ix, ii, into[2], into[1], one, one, into=grad)[0] == grad

    def read():
        return [eng.download_bits(i) for i in into + [grad]]

    eager = []
    for a in x:
        eng.write_ptr(ix, a.ctypes.data, a.size)
        step()
        eager.append(read())
    eng.begin_trace()
    step()
    trace = eng.end_trace()
    for a, want in zip(x, eager):
        eng.write_ptr(ix, a.ctypes.data, a.size)
        eng.run_trace(trace)
        assert all(np.array_equal(p, q) for p, q in zip(read(), want))
    eng.release_trace(trace)
    for i in into + [ix, ii, grad, one]:
        eng.free(i)


def test_offsets_behind_32_bits(fresh_eng):
    eng = fresh_eng                                          # its memory goes back with it
    # The last rows of logits of 2^32 elements and a few more, and their gradient.
    rng = np.random.default_rng(18)
    cols, tail = 50257, 5
    rows = 2 ** 32 // cols + tail + 1
    x = orc.to_bf16(logits(rng, tail, cols))
    ids = np.full(rows, -1, np.int32)
    ids[-tail:] = rng.integers(0, cols, tail)
    whole = eng.zeros_dram((rows, cols), BF16)[0]
    last = eng.slice_rows(whole, rows - tail, tail)[0]
    eng.write_ptr(last, x.ctypes.data, x.size, 2)
    eng.sync()
    ii, one = up_i32(eng, ids, rows, 1), eng.upload(np.ones((rows, 1), np.float32), rows, 1)
    got = eng.token_logprobs(whole, ii, 1.0, 3)
    grad, _ = eng.token_logprobs_backward(whole, ii, got[2][0], got[1][0], one, one, bf16=True)
    few, few_ids = eng.upload_bf16(x, tail, cols), up_i32(eng, ids[-tail:], tail, 1)
    want = eng.token_logprobs(few, few_ids, 1.0, 3)
    ends = eng.slice_rows(grad, rows - tail, tail)[0]
    for (a, _), (b, _), width in zip(got, want, (1, 1, 1, 3, 3)):
        a, b = eng.download_bits(a).reshape(rows, width), eng.download_bits(b).reshape(tail, width)
        if a.dtype == np.uint32 and width == 3 and (b < cols).all():
            assert np.array_equal(a[-tail:], b) and np.array_equal(a[0], [0, 1, 2])          # the columns
        else:                                                                                 # summed in another order: few rows share blocks
            assert np.all(np.abs(a[-tail:].view(np.float32) - b.view(np.float32)) <= 24 * (2 * 12 + 600) * U)   # twice, 1 + log 50257
    ones = eng.upload(np.ones((tail, 1), np.float32), tail, 1)
    lse, ent = (eng.slice_rows(got[i][0], rows - tail, tail)[0] for i in (2, 1))
    few_grad, _ = eng.token_logprobs_backward(few, few_ids, lse, ent, ones, ones, bf16=True)
    assert np.array_equal(eng.download_bf16(ends), eng.download_bf16(few_grad))
    for i in [whole, last, ii, one, grad, few, few_ids, ends, ones, few_grad, lse, ent] + [i for i, _ in got + want]:
        eng.free(i)

"""The paged cache through the C ABI: `rope_append_pages` bit for bit against the rotation's separate roundings in NumPy (and
against the trait ops it joins), `attention_pages` against softmax(scale q K^T) V in 64 bits.

Tolerance of the attention, with u = 2^-24 and A = sum_j p_j |v_j| / sum_j p_j of the row and column:
  - a score is an F32 sum of d products in some order: within (d + 8) u scale sum|q k|; operands wider than the tensor cores'
    types are split into parts, whose dropped products are below 2^-21 of scale sum|q k|;
  - its exponential: the argument's roundings are within 6 u |s|, the function within 8 u: together a weight is off by a
    factor 1 + eps, and numerator and denominator by as much each;
  - the sums: every weight is added with at most n / 16 + 32 additions after it (sixteen positions are one step), in both;
  - a weight's own split: 2^-21 for an F32 result, 2^-16 for a BF16 one, which is then rounded by half a step, 2^-8."""
import numpy as np
import pytest

from metalium_rs_b200 import BF16, F32, I32, EltwiseOp, PageShape, TtError, kinds
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def up_i32(eng, a, r, c):
    return eng.upload_bits(np.ascontiguousarray(a, dtype=np.int32).view(np.uint32), r, c, I32)


def up(eng, x, bf16):
    """(buffer, the values it holds): F32 as they are, or rounded to BF16."""
    if bf16:
        h = orc.to_bf16(x)
        return eng.upload_bf16(h, *x.shape), orc.from_bf16(h)
    return eng.upload(x, *x.shape), x


def down(eng, i, bf16):
    return orc.from_bf16(eng.download_bf16(i)) if bf16 else eng.download(i)


def tables(rng, lengths, page, spare=2, width=0):
    """A table of pages drawn without order, -1 where a sequence needs none; and the pool's pages."""
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    t = np.full((len(lengths), max([1, width] + need)), -1, np.int32)
    at = 0
    for s, k in enumerate(need):
        t[s, :k] = order[at:at + k]
        at += k
    return t, len(order)


def row_of(table, page, s, p):
    return table[s, p // page] * page + p % page


# ------------------------------------------------------------------------------------------------ append
def rotate(x, cos, sin, d):
    """x [n, heads d] F32, cos and sin [n, r]: fl(fl(x cos) + fl(swap(x) sin)) on the first r columns of a head."""
    n, r = x.shape[0], cos.shape[1]
    h = x.reshape(n, -1, d).copy()
    lo, hi = h[..., :r // 2].copy(), h[..., r // 2:r].copy()
    swap = np.concatenate([hi, lo], -1)
    h[..., :r] = (h[..., :r] * cos[:, None]).astype(np.float32) + (swap * sin[:, None]).astype(np.float32)
    return h.reshape(n, -1)


def append_case(eng, rng, sequences, positions, heads, kv, d, page, r, x_bf16, c_bf16, o_bf16, keys, lead=0, tail=0, width=0, seq_buf=True):
    sequences, positions = np.asarray(sequences), np.asarray(positions)
    n = len(positions)
    lengths = [int(positions[sequences == s].max(initial=-1)) + 1 for s in range(int(sequences.max()) + 1)]
    table, pages = tables(rng, lengths, page, width=width)
    cols = (heads + 2 * kv) * d
    ix, x = up(eng, rng.standard_normal((n + (1 if lead else 0), lead + cols + tail)).astype(np.float32), x_bf16)
    ik, k0 = up(eng, rng.standard_normal((pages * page, kv * d)).astype(np.float32), c_bf16)
    iv, v0 = up(eng, rng.standard_normal((pages * page, kv * d)).astype(np.float32), c_bf16)
    first = x.shape[0] - n
    x = x[first:, lead:lead + cols]
    span = max(lengths + [1])
    ang = rng.uniform(0, 6.28, (span, max(r, 2) // 2))
    cos = np.concatenate([np.cos(ang), np.cos(ang)], 1).astype(np.float32)
    sin = np.concatenate([-np.sin(ang), np.sin(ang)], 1).astype(np.float32)
    ic, isn = (eng.upload(cos, *cos.shape), eng.upload(sin, *sin.shape)) if r else (None, None)
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, positions, 1, n)
    iq = up_i32(eng, sequences, n, 1) if seq_buf else None
    out, dims = eng.rope_append_pages(PageShape(heads, kv, d, page), (ix, (first, lead), (n, cols)), ic, isn, ip, iq, it, ik, iv, keys=keys, bf16=o_bf16)
    live = positions >= 0
    turned = x[:, :(heads + kv) * d].astype(np.float32)
    if r:
        turned = rotate(turned, cos[np.maximum(positions, 0)], sin[np.maximum(positions, 0)], d)
    cast = lambda a, b: orc.from_bf16(orc.to_bf16(a)) if b else a
    kept = (heads + (kv if keys else 0)) * d
    want = np.where(live[:, None], cast(turned[:, :kept], o_bf16), np.float32(0))
    assert dims == (n, kept)
    wk, wv = k0.copy(), v0.copy()
    for i in np.nonzero(live)[0]:
        at = row_of(table, page, sequences[i], positions[i])
        wk[at] = cast(turned[i, heads * d:], c_bf16)
        wv[at] = cast(x[i, (heads + kv) * d:], c_bf16)
    got = down(eng, out, o_bf16), down(eng, ik, c_bf16), down(eng, iv, c_bf16)
    for i in (ix, ik, iv, it, ip, out) + ((iq,) if iq else ()) + ((ic, isn) if r else ()):
        eng.free(i)
    for name, a, b in zip(("heads", "keys", "values"), got, (want, wk, wv)):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:4])


@pytest.mark.parametrize("x_bf16", [False, True])
@pytest.mark.parametrize("c_bf16", [False, True])
@pytest.mark.parametrize("o_bf16", [False, True])
def test_append_every_type(eng, x_bf16, c_bf16, o_bf16):
    rng = np.random.default_rng(1)
    append_case(eng, rng, [0, 1, 2], [5, 40, 16], 9, 3, 64, 16, 64, x_bf16, c_bf16, o_bf16, False, seq_buf=False)
    append_case(eng, rng, np.repeat([0, 1], 20), list(range(20)) + list(range(7, 27)), 4, 2, 32, 8, 32, x_bf16, c_bf16, o_bf16, True)


@pytest.mark.parametrize("heads,kv,d,page,r,lead,tail", [
    (32, 8, 128, 16, 128, 0, 0),
    (32, 8, 128, 16, 64, 8, 16),     # half of each head rotated, a block inside a wider buffer
    (1, 1, 256, 1, 256, 0, 0),       # pages of one position
    (6, 6, 192, 24, 192, 0, 0),      # pages that are not a power of two
    (8, 8, 96, 20, 96, 3, 2),        # a block that starts at no 16-byte address
    (4, 2, 6, 5, 4, 1, 0),           # narrow odd heads: nothing a vector fits
    (4, 2, 34, 7, 34, 0, 0),
    (4, 2, 40, 7, 24, 0, 0),         # half a rotation of 12 columns
    (12, 4, 32, 128, 0, 0, 0),       # no rotation
    (40, 1, 64, 64, 64, 0, 0),
])
def test_append_head_layouts(eng, heads, kv, d, page, r, lead, tail):
    rng = np.random.default_rng(2)
    seqs = np.array([2, 0, 1, 1, 2, 0, 0])
    pos = np.array([0, page - 1, page, 3 * page + 1, 7, -1, 2 * page])
    for keys in (False, True):
        for x_bf16, c_bf16 in ((True, True), (False, True), (True, False)):
            append_case(eng, rng, seqs, pos, heads, kv, d, page, r, x_bf16, c_bf16, not c_bf16, keys, lead, tail, width=6)


@pytest.mark.parametrize("n", [1, 2, 147, 148, 149, 1000, 5000])
def test_append_prompts_of_any_length(eng, n):
    rng = np.random.default_rng(n)
    seqs = rng.integers(0, 3, n)
    pos = np.empty(n, np.int64)
    for s in range(3):
        pos[seqs == s] = rng.permutation((seqs == s).sum()) + 3      # a sequence's tokens in any order
    pos[rng.random(n) < 0.1] = -1                                    # padding
    append_case(eng, rng, np.append(seqs, [0, 1, 2]), np.append(pos, [0, 1, 2]), 4, 2, 64, 16, 64, True, True, True, n % 2 == 0)


def test_append_is_the_trait_s_ops(eng):
    """The rotation of `rope_blocks` and the writes of `scatter_rows_into`, bit for bit, where a page is a whole sequence."""
    n, heads, kv, d, longest = 3, 9, 3, 64, 32
    rng = np.random.default_rng(4)
    qk, cols = (heads + kv) * d, (heads + 2 * kv) * d
    ix, _ = up(eng, rng.standard_normal((n, cols)).astype(np.float32), True)
    ang = rng.uniform(0, 6.28, (longest, d // 2))
    cos = np.concatenate([np.cos(ang), np.cos(ang)], 1).astype(np.float32)
    sin = np.concatenate([-np.sin(ang), np.sin(ang)], 1).astype(np.float32)
    ic, isn = eng.upload(cos, longest, d), eng.upload(sin, longest, d)
    pos = 17
    caches = [eng.zeros_dram((n * longest, kv * d), bf16=True)[0] for _ in range(4)]
    rows = up_i32(eng, np.arange(n) * longest + pos, 1, n)
    one = up_i32(eng, [pos], 1, 1)
    cs, sn = eng.select_rows(ic, one)[0], eng.select_rows(isn, one)[0]
    rot, _ = eng.rope_blocks((ix, (0, 0), (n, qk)), (cs, (0, 0), (1, d)), (sn, (0, 0), (1, d)), d, False)
    eng.scatter_rows_into(caches[0], rows, (rot, (0, heads * d), (n, kv * d)))
    eng.scatter_rows_into(caches[1], rows, (ix, (0, qk), (n, kv * d)))
    it, ip = up_i32(eng, np.arange(n), n, 1), up_i32(eng, [pos] * n, 1, n)
    got, _ = eng.rope_append_pages(PageShape(heads, kv, d, longest), (ix, (0, 0), (n, cols)), ic, isn, ip, None, it, caches[2], caches[3], keys=True)
    assert np.array_equal(eng.download_bits(got), eng.download_bits(rot))
    for a, b in ((0, 2), (1, 3)):
        assert np.array_equal(eng.download_bf16(caches[a]), eng.download_bf16(caches[b]))
    for i in [ix, ic, isn, rows, one, cs, sn, rot, it, ip, got] + caches:
        eng.free(i)


@pytest.mark.parametrize("d,r", [(64, 32), (20, 4)])
def test_values_and_unrotated_columns_of_one_type_keep_their_bits(eng, d, r):
    """Subnormals, signed zeros, infinities and NaN payloads pass as `scatter_rows_into` passes them."""
    rng = np.random.default_rng(3)
    n, heads, kv = 5, 2, 1
    bits = rng.integers(0, 1 << 16, (n, (heads + 2 * kv) * d)).astype(np.uint16)
    bits[0, -4:] = [0x0001, 0x8000, 0x7F81, 0xFF80]
    ix = eng.upload_bf16(bits, *bits.shape)
    ik, iv = (eng.zeros_dram((16, kv * d), bf16=True)[0] for _ in range(2))
    one, none = np.ones((8, r), np.float32), np.zeros((8, r), np.float32)
    ic, isn = eng.upload(one, 8, r), eng.upload(none, 8, r)
    it, ip, iq = up_i32(eng, [[1, 0]], 1, 2), up_i32(eng, np.arange(n), 1, n), up_i32(eng, np.zeros(n), 1, n)
    out, _ = eng.rope_append_pages(PageShape(heads, kv, d, 8), (ix, (0, 0), bits.shape), ic, isn, ip, iq, it, ik, iv, bf16=True)
    got, k, v = (eng.download_bf16(i) for i in (out, ik, iv))
    keep = np.arange(d) >= r
    assert np.array_equal(v[8:8 + n], bits[:, -d:])
    assert np.array_equal(k[8:8 + n][:, keep], bits[:, heads * d:(heads + 1) * d][:, keep])
    assert np.array_equal(got.reshape(n, heads, d)[:, :, keep], bits[:, :heads * d].reshape(n, heads, d)[:, :, keep])
    for i in (ix, ik, iv, ic, isn, it, ip, iq, out):
        eng.free(i)


@pytest.mark.parametrize("bad", ["position", "below", "sequence", "page", "negative page", "rotation"])
def test_append_reports_a_bad_index_and_writes_nothing_for_it(fresh_eng, bad):
    e = fresh_eng
    rng = np.random.default_rng(5)
    table = np.array([[0, 1], [2, 3]], np.int32)
    pos, seq = [3, 9], [0, 1]
    if bad == "position":
        pos[1] = 16
    if bad == "below":
        pos[1] = -2
    if bad == "sequence":
        seq[1] = 2
    if bad == "page":
        table[1, 1] = 4
    if bad == "negative page":
        table[1, 1] = -1
    rows = 9 if bad == "rotation" else 16
    ix, x = up(e, rng.standard_normal((2, 4 * 32)).astype(np.float32), False)
    ik, iv = e.zeros_dram((32, 32))[0], e.zeros_dram((32, 32))[0]
    ic = e.upload(np.ones((rows, 32), np.float32), rows, 32)
    isn = e.upload(np.zeros((rows, 32), np.float32), rows, 32)
    out, _ = e.rope_append_pages(PageShape(2, 1, 32, 8), (ix, (0, 0), (2, 128)), ic, isn, up_i32(e, pos, 1, 2), up_i32(e, seq, 1, 2),
                                 up_i32(e, table, 2, 2), ik, iv)
    got = []
    for i in (out, ik, iv):
        dst = np.empty(e.dims_of(i)[0], np.float32)
        with pytest.raises(TtError) as err:
            e.download_into(i, dst.ctypes.data, dst.size)
        assert err.value.status == 6                       # DOMAIN, with the data copied before the wait
        got.append(dst)
    assert np.array_equal(got[0], np.stack([x[0, :64], np.zeros(64, np.float32)]))
    assert np.array_equal(got[1][3], x[0, 64:96]) and np.array_equal(got[2][3], x[0, 96:])
    assert not np.delete(got[1], 3, 0).any() and not np.delete(got[2], 3, 0).any()


# ------------------------------------------------------------------------------------------------ attention
def attend64(q, k, v, table, page, positions, heads, kv, d, scale, window, o_bf16=False):
    """(result, bound) in 64 bits."""
    n = len(positions)
    out, tol = np.zeros((n, heads * d)), np.zeros((n, heads * d))
    for s in range(n):
        last = positions[s]
        if last < 0:
            continue
        j = np.arange(max(0, last + 1 - window) if window else 0, last + 1)
        rows = table[s, j // page] * page + j % page
        for h in range(heads):
            c = slice((h // (heads // kv)) * d, (h // (heads // kv) + 1) * d)
            K, V, x = k[rows, c].astype(np.float64), v[rows, c].astype(np.float64), q[s, h * d:(h + 1) * d].astype(np.float64)
            z = K @ x * scale
            w = np.exp(z - z.max())
            cols = slice(h * d, (h + 1) * d)
            out[s, cols] = w @ V / w.sum()
            mass = np.abs(K) @ np.abs(x) * abs(scale)
            eps = (d + 8) * U * mass + 2.0 ** -21 * mass + 6 * U * np.abs(z).max() + 8 * U
            share = (w * eps)
            A = w @ np.abs(V) / w.sum()
            tol[s, cols] = (share @ np.abs(V) + share.sum() * A) / w.sum() + A * (2 * (len(j) / 16 + 32) * U + (2.0 ** -16 if o_bf16 else 2.0 ** -21))
    return out, tol + (2.0 ** -8 if o_bf16 else U) * (np.abs(out) + tol)


def attention_case(eng, rng, lengths, heads, kv, d, page, q_bf16, c_bf16, o_bf16, window=0, lead=0, scale=None, spread=1.0, poison=True, width=0):
    n = len(lengths)
    positions = np.asarray(lengths) - 1
    table, pages = tables(rng, lengths, page, width=width)
    cols = heads * d
    iq, q = up(eng, (rng.standard_normal((n, lead + cols)) * spread).astype(np.float32), q_bf16)
    q = q[:, lead:]
    k = rng.standard_normal((pages * page, kv * d)).astype(np.float32)
    v = rng.standard_normal((pages * page, kv * d)).astype(np.float32)
    if poison:                                               # what no live position names must not be read into a result
        dead = np.ones(pages * page, bool)
        for s, last in enumerate(positions):
            for p in range(max(0, last + 1 - window) if window else 0, last + 1):
                dead[row_of(table, page, s, p)] = False
        k[dead] = np.nan
        v[dead] = np.inf
    ik, k = up(eng, k, c_bf16)
    iv, v = up(eng, v, c_bf16)
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, positions, 1, n)
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, dims = eng.attention_pages(PageShape(heads, kv, d, page), (iq, (0, lead), (n, cols)), ik, iv, it, ip, scale, window=window, bf16=o_bf16)
    assert dims == (n, cols)
    got = down(eng, out, o_bf16).astype(np.float64)
    for i in (iq, ik, iv, it, ip, out):
        eng.free(i)
    want, tol = attend64(q, k, v, table, page, positions, heads, kv, d, np.float64(np.float32(scale)), window, o_bf16)
    off = np.abs(got - want)
    assert np.all(off <= tol), (float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(~(off <= tol))[:4])
    assert not got[positions < 0].any()


LENGTHS = [1, 2, 0, 15, 16, 17, 63, 64, 65, 127, 130, 300, 0, 700]


@pytest.mark.parametrize("c_bf16", [True, False])
@pytest.mark.parametrize("q_bf16,o_bf16", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("heads,kv,d,page", [(9, 3, 64, 16), (4, 2, 32, 8), (6, 6, 96, 24), (8, 1, 128, 20), (3, 1, 192, 64), (2, 2, 256, 7)])
def test_attention_every_type_and_head_width(eng, heads, kv, d, page, q_bf16, o_bf16, c_bf16):
    attention_case(eng, np.random.default_rng(d), LENGTHS, heads, kv, d, page, q_bf16, c_bf16, o_bf16)


@pytest.mark.parametrize("c_bf16", [True, False])
@pytest.mark.parametrize("heads,kv,d,page,lengths", [
    (16, 1, 64, 16, [40, 5]),                  # a whole tile of query heads a key/value head
    (17, 1, 64, 16, [40, 5]),                  # one more
    (40, 2, 64, 1, [33, 70]),                  # twenty a key/value head, pages of one position
    (71, 1, 128, 16, [100]),
    (1, 1, 128, 1000, [999, 1, 1000]),         # one page a sequence
    (12, 12, 64, 3, [10] * 40),
])
def test_attention_head_groups_and_pages(eng, heads, kv, d, page, lengths, c_bf16):
    attention_case(eng, np.random.default_rng(heads), lengths, heads, kv, d, page, False, c_bf16, False, width=50)


@pytest.mark.parametrize("c_bf16,q_bf16", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("lengths", [[20011], [5000, 1], [1] * 700, list(range(1, 400, 3)), [0, 0, 9000, 0, 64, 128]])
def test_attention_long_and_many(eng, lengths, c_bf16, q_bf16):
    attention_case(eng, np.random.default_rng(7), lengths, 4, 2, 64, 16, q_bf16, c_bf16, False)


@pytest.mark.parametrize("c_bf16,q_bf16,o_bf16", [(True, True, True), (True, False, False), (False, False, False)])
@pytest.mark.parametrize("heads,kv,d", [(8, 2, 32), (9, 3, 64), (4, 4, 96), (40, 4, 128), (3, 1, 192), (6, 2, 256)])
@pytest.mark.parametrize("lengths", [[7], [300], [0], [1, 0, 200], [1000, 3, 0, 17, 16, 999], [129] * 20])
def test_attention_is_the_same_whatever_the_table_s_width(eng, lengths, heads, kv, d, c_bf16, q_bf16, o_bf16):
    # A table as wide as the longest needs, and one that leaves room for sequences of 30,000 positions: the work is cut otherwise.
    for width in (0, 2000):
        attention_case(eng, np.random.default_rng(len(lengths)), lengths, heads, kv, d, 15, q_bf16, c_bf16, o_bf16, width=width)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 699, 700, 701, 100000])
def test_attention_window(eng, window):
    for c_bf16 in (True, False):
        attention_case(eng, np.random.default_rng(window), LENGTHS, 4, 2, 64, 16, False, c_bf16, False, window=window)


@pytest.mark.parametrize("scale,spread", [(1.0, 3.0), (0.0, 1.0), (-0.5, 1.0), (0.125, 40.0)])
def test_attention_scales(eng, scale, spread):
    for c_bf16 in (True, False):
        attention_case(eng, np.random.default_rng(3), [300, 17], 4, 2, 64, 16, False, c_bf16, False, scale=scale, spread=spread)


@pytest.mark.parametrize("lead", [1, 3, 8])
def test_attention_queries_inside_a_wider_buffer(eng, lead):
    for q_bf16 in (True, False):
        attention_case(eng, np.random.default_rng(lead), [50, 3], 4, 2, 64, 16, q_bf16, True, True, lead=lead)


def one_head(eng, q, k, v, lengths, page=16, c_bf16=True, q_bf16=False, scale=1.0, heads=1):
    n, d = len(lengths), q.shape[1] // heads
    ik, _ = up(eng, k, c_bf16)
    iv, _ = up(eng, v, c_bf16)
    iq, _ = up(eng, q, q_bf16)
    table = np.arange(n * (len(k) // page // n), dtype=np.int32).reshape(n, -1)
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, np.asarray(lengths) - 1, 1, n)
    out, _ = eng.attention_pages(PageShape(heads, k.shape[1] // d, d, page), (iq, (0, 0), q.shape), ik, iv, it, ip, scale)
    got = eng.download(out)
    for i in (ik, iv, iq, it, ip, out):
        eng.free(i)
    return got


@pytest.mark.parametrize("c_bf16,q_bf16", [(True, True), (True, False), (False, False)])
def test_attention_infinite_scores(eng, c_bf16, q_bf16):
    """A key that gives -inf has weight 0; a row of them only is zero (the clamped maximum and sum); +inf and NaN give NaN."""
    rng = np.random.default_rng(9)
    d, n = 64, 48
    q = np.abs(rng.standard_normal((3, d))).astype(np.float32)
    k = rng.standard_normal((3 * n, d)).astype(np.float32)
    v = rng.standard_normal((3 * n, d)).astype(np.float32)
    k[5, 3] = -np.inf                                       # sequence 0: one of its positions
    k[n:2 * n, 7] = -np.inf                                 # sequence 1: all of them
    k[2 * n + 9, 1] = np.nan                                # sequence 2
    got = one_head(eng, q, k, v, [n, n, n], c_bf16=c_bf16, q_bf16=q_bf16)
    half = (lambda a: orc.from_bf16(orc.to_bf16(a)))
    qq, kk, vv = (half(q) if q_bf16 else q), (half(k) if c_bf16 else k), (half(v) if c_bf16 else v)
    live = np.delete(np.arange(n), 5)
    z = kk[live].astype(np.float64) @ qq[0].astype(np.float64)
    w = np.exp(z - z.max())
    want = w @ vv[live].astype(np.float64) / w.sum()
    assert np.all(np.abs(got[0] - want) <= 1e-4 * np.abs(vv).max())     # scores to about 20: (d + 8) u sum|q k| < 1e-4
    assert not got[1].any()
    assert np.isnan(got[2]).all()
    k[:] = 0.0
    k[3, 0] = np.inf
    got = one_head(eng, q, k, v, [n, n, n], c_bf16=c_bf16, q_bf16=q_bf16)
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


def test_attention_equal_scores_average(eng):
    """Zero queries: the mean of the attended values, at lengths around every tile's end."""
    for n in (1, 15, 16, 17, 31, 63, 64, 65, 1000, 4097):
        rng = np.random.default_rng(n)
        pages = -(-n // 16)
        v = rng.integers(-8, 9, (pages * 16, 64)).astype(np.float32)
        k = rng.standard_normal((pages * 16, 64)).astype(np.float32)
        got = one_head(eng, np.zeros((1, 64), np.float32), k, v, [n])
        want = v[:n].astype(np.float64).mean(0)
        # the weights are exactly 1, the sum of small integers exact: one division
        assert np.all(np.abs(got[0] - want) <= 4 * U * np.abs(want)), n


@pytest.mark.parametrize("bad", ["page", "negative page", "position", "below"])
def test_attention_reports_a_bad_index(fresh_eng, bad):
    e = fresh_eng
    rng = np.random.default_rng(6)
    table = np.array([[0, 1], [2, 3]], np.int32)
    pos = [9, 13]
    if bad == "page":
        table[1, 0] = 4
    if bad == "negative page":
        table[1, 0] = -7
    if bad == "position":
        pos[1] = 16
    if bad == "below":
        pos[1] = -2
    iq, q = up(e, rng.standard_normal((2, 32)).astype(np.float32), False)
    ik, k = up(e, rng.standard_normal((32, 32)).astype(np.float32), True)
    iv, v = up(e, rng.standard_normal((32, 32)).astype(np.float32), True)
    out, _ = e.attention_pages(PageShape(1, 1, 32, 8), (iq, (0, 0), (2, 32)), ik, iv, up_i32(e, table, 2, 2), up_i32(e, pos, 1, 2), 0.2)
    got = np.empty((2, 32), np.float32)
    with pytest.raises(TtError) as err:
        e.download_into(out, got.ctypes.data, got.size)
    assert err.value.status == 6
    w0, t0 = attend64(q[:1], k, v, table[:1], 8, [9], 1, 1, 32, np.float64(np.float32(0.2)), 0)
    assert np.all(np.abs(got[0] - w0[0]) <= t0[0])
    if "page" in bad:                                       # the other page's positions, 8 .. 13, are attended
        w1, t1 = attend64(q[1:], k, v, np.array([[3]]), 8, [5], 1, 1, 32, np.float64(np.float32(0.2)), 0)
        assert np.all(np.abs(got[1] - w1[0]) <= t1[0])
    else:
        assert not got[1].any()


def test_results_into_a_buffer_leave_its_other_rows(eng):
    rng = np.random.default_rng(8)
    shape = PageShape(4, 2, 64, 16)
    table, pages = tables(rng, [30, 40], 16)
    ix, _ = up(eng, rng.standard_normal((2, 8 * 64)).astype(np.float32), True)
    ik, _ = up(eng, rng.standard_normal((pages * 16, 128)).astype(np.float32), True)
    iv, _ = up(eng, rng.standard_normal((pages * 16, 128)).astype(np.float32), True)
    it, ip = up_i32(eng, table, *table.shape), up_i32(eng, [29, 39], 1, 2)
    big = eng.upload(np.full((4, 256), 7.0, np.float32), 4, 256)
    mid, _ = eng.slice_rows(big, 1, 2)
    got, _ = eng.rope_append_pages(shape, (ix, (0, 0), (2, 512)), None, None, ip, None, it, ik, iv, into=mid)
    assert got == mid
    new, _ = eng.rope_append_pages(shape, (ix, (0, 0), (2, 512)), None, None, ip, None, it, ik, iv)
    a = eng.download(big)
    assert np.array_equal(a[1:3], eng.download(new)) and np.all(a[[0, 3]] == 7.0)
    eng.attention_pages(shape, (new, (0, 0), (2, 256)), ik, iv, it, ip, 0.125, into=mid)
    one, _ = eng.attention_pages(shape, (new, (0, 0), (2, 256)), ik, iv, it, ip, 0.125)
    a = eng.download(big)
    assert np.array_equal(a[1:3], eng.download(one)) and np.all(a[[0, 3]] == 7.0)
    for i in (ix, ik, iv, it, ip, mid, big, new, one):
        eng.free(i)


def test_append_and_attention_repeat_and_replay_bit_for_bit(eng):
    """The same call twice, and captured and replayed for growing positions, gives the eager bits."""
    rng = np.random.default_rng(11)
    shape, n, steps = PageShape(8, 2, 64, 16), 5, 6
    table, pages = tables(rng, [700, 40, 300, 20, 64], 16)
    cols = 12 * 64
    xs = [orc.to_bf16(rng.standard_normal((n, cols)).astype(np.float32)) for _ in range(steps)]
    k0, v0 = (orc.to_bf16(rng.standard_normal((pages * 16, 128)).astype(np.float32)) for _ in range(2))
    start = np.array([650, -1, 250, 3, 50], np.int32)
    it = up_i32(eng, table, *table.shape)

    def fresh():
        return eng.upload_bf16(k0, *k0.shape), eng.upload_bf16(v0, *v0.shape), up_i32(eng, start, 1, n), eng.upload_bf16(xs[0], n, cols)

    def step(ik, iv, ip, ix):
        q, _ = eng.rope_append_pages(shape, (ix, (0, 0), (n, cols)), None, None, ip, None, it, ik, iv)
        o, _ = eng.attention_pages(shape, (q, (0, 0), (n, 512)), ik, iv, it, ip, 0.125)
        live = eng.eltwise_op(EltwiseOp(kinds.INT_GE_S, 0.0, 0.0), ip)[0]
        one = eng.eltwise_op(EltwiseOp(kinds.BOOL_TO_I32, 0.0, 0.0), live)[0]
        nxt = eng.eltwise_op(EltwiseOp(kinds.INT_ADD, 0.0, 0.0), ip, one)[0]
        eng.copy_into(nxt, ip)
        for i in (q, live, one, nxt):
            eng.free(i)
        return o

    def write(buf, bits):
        eng.write_ptr(buf, bits.ctypes.data, bits.size, 2)
        eng.sync()

    eager = []
    state = fresh()
    for t in range(steps):
        write(state[3], xs[t])
        o = step(*state)
        eager.append(eng.download_bits(o))
        eng.free(o)
    assert np.array_equal(eng.download_bits(state[2])[0].view(np.int32), np.where(start < 0, -1, start + steps))
    second = fresh()
    o = step(*second)                                        # every kernel is loaded
    eng.free(o)
    ip = up_i32(eng, start, 1, n)
    eng.copy_into(ip, second[2])
    eng.begin_trace()
    o = step(*second)
    trace = eng.end_trace()
    for t in range(steps):
        write(second[3], xs[t])
        eng.run_trace(trace)
        assert np.array_equal(eng.download_bits(o), eager[t]), t
    for a, b in zip(state[:2], second[:2]):
        assert np.array_equal(eng.download_bf16(a), eng.download_bf16(b))
    eng.release_trace(trace)
    for i in (it, ip, o) + state + second:
        eng.free(i)


def test_offsets_behind_32_bits(fresh_eng):
    eng = fresh_eng                                          # its memory goes back with it
    # The last pages of pools of 2^32 elements and a few more: the bits of the same call on a small pool.
    rng = np.random.default_rng(15)
    shape, page, n, cols = PageShape(8, 8, 128, 64), 64, 3, 24 * 128
    lengths, count = [100, 64, 3], 4
    x = orc.to_bf16(rng.standard_normal((sum(lengths), cols)).astype(np.float32))
    sequences = np.repeat(np.arange(n), lengths)
    positions = np.concatenate([np.arange(m) for m in lengths])
    small = np.array([[2, 0], [3, -1], [1, -1]], np.int32)
    results = []
    for pages in (count, 2 ** 32 // (page * 1024) + count):
        table = np.where(small < 0, small, small + pages - count)
        ik, iv = (eng.zeros_dram((pages * page, 1024), BF16)[0] for _ in range(2))
        it, ip, js = up_i32(eng, table, *table.shape), up_i32(eng, positions, 1, len(x)), up_i32(eng, sequences, 1, len(x))
        last = up_i32(eng, np.array(lengths) - 1, 1, n)
        ix = eng.upload_bf16(x, *x.shape)
        q, _ = eng.rope_append_pages(shape, (ix, (0, 0), x.shape), None, None, ip, js, it, ik, iv)
        o, _ = eng.attention_pages(shape, (q, (0, 0), (n, 1024)), ik, iv, it, last, 0.09)
        tail, _ = eng.slice_rows(ik, (pages - count) * page, count * page)
        results.append((eng.download_bits(o), eng.download_bf16(tail)))
        for i in (ik, iv, it, ip, js, last, ix, q, o, tail):
            eng.free(i)
    assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
    assert np.abs(results[0][0].view(np.float32)).max() > 0.01


def test_two_engines_at_once(eng, fresh_eng):
    # Calls of two engines in turn, nothing waited for between them, are each engine's own.
    rng = np.random.default_rng(16)
    shape, lengths = PageShape(4, 2, 64, 16), [900, 33, 400]
    table, pages = tables(rng, lengths, 16)
    sides = []
    for e in (eng, fresh_eng):
        q, k, v = (rng.standard_normal((r, c)).astype(np.float32) for r, c in ((3, 256), (pages * 16, 128), (pages * 16, 128)))
        ids = [e.upload(a, *a.shape) for a in (q, k, v)] + [up_i32(e, table, *table.shape), up_i32(e, np.array(lengths) - 1, 1, 3)]
        alone, _ = e.attention_pages(shape, (ids[0], (0, 0), (3, 256)), *ids[1:], 0.125)
        sides.append((e, ids, e.download_bits(alone), alone))
    for _ in range(20):
        outs = [e.attention_pages(shape, (ids[0], (0, 0), (3, 256)), *ids[1:], 0.125)[0] for e, ids, _, _ in sides]
        for (e, _, want, _), o in zip(sides, outs):
            assert np.array_equal(e.download_bits(o), want)
            e.free(o)
    for e, ids, _, alone in sides:
        for i in ids + [alone]:
            e.free(i)

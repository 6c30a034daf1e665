"""The serving operators' host logic without a GPU: engine.cu and engine_serving.cu against the host-only stand-in for the
CUDA runtime, every launch a no-op.  Checked here: result dims, what is refused, results written into a caller's buffer, and
that a refused or failed call leaves no buffer behind."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from metalium_rs_b200 import BF16, F32, I32, CudaEngine, PageShape, TtError, engine

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def fake():
    out = ROOT / "tests" / "_build" / "libb200tt_fake_serving.so"
    out.parent.mkdir(exist_ok=True)
    csrc = ROOT / "metalium_rs_b200" / "csrc"
    srcs = [csrc / "engine.cu", csrc / "engine_serving.cu", ROOT / "tests" / "fake_cuda" / "fake_kernels.cpp",
            ROOT / "tests" / "fake_cuda" / "fake_serving_kernels.cpp"]
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-x", "c++", "-I", str(ROOT / "tests" / "fake_cuda"), "-I", str(csrc),
                    *map(str, srcs), "-o", str(out)], check=True)
    return C.CDLL(str(out))


@pytest.fixture()
def e(fake):
    eng = CudaEngine(0, lib=fake)
    yield eng
    eng.close()


def zeros(e, r, c, elem=F32):
    return e.zeros_dram((r, c), elem)[0]


def refused(call, status=2):
    with pytest.raises(TtError) as err:
        call()
    assert err.value.status == status, err.value


class Cache:
    """3 sequences of up to 4 pages of 8 positions; 4 query heads over 2 key/value heads of 32 columns."""

    def __init__(self, e, elem=BF16, dim=32):
        self.shape = PageShape(4, 2, dim, 8)
        self.keys, self.values = zeros(e, 80, 2 * dim, elem), zeros(e, 80, 2 * dim, elem)
        self.table = zeros(e, 3, 4, I32)
        self.cos, self.sin = zeros(e, 32, dim), zeros(e, 32, dim)
        self.dim = dim

    def append(self, e, n=3, x=None, **over):
        a = dict(qkv=(x, (0, 0), (n, 8 * self.dim)), cos=self.cos, sin=self.sin, positions=over.pop("positions"), sequences=None,
                 page_table=self.table, key_pages=self.keys, value_pages=self.values)
        shape = over.pop("shape", self.shape)
        a.update(over)
        return e.rope_append_pages(shape, **a)

    def attend(self, e, n=3, q=None, **over):
        a = dict(q=(q, (0, 0), (n, 4 * self.dim)), key_pages=self.keys, value_pages=self.values, page_table=self.table,
                 positions=over.pop("positions"), scale=0.2)
        shape = over.pop("shape", self.shape)
        a.update(over)
        return e.attention_pages(shape, **a)


def test_struct_layout():
    assert C.sizeof(engine.PageShape) == 16


def test_append_dims_and_forms(fake, e):
    c = Cache(e)
    x, p = zeros(e, 3, 256, BF16), zeros(e, 1, 3, I32)
    out, dims = c.append(e, x=x, positions=p)
    assert dims == (3, 128) and e.dims_of(out) == ((3, 128), F32)
    assert C.c_uint64.in_dll(fake, "fake_append_rotary").value == 32 and not C.c_uint64.in_dll(fake, "fake_append_sequences").value
    out, dims = c.append(e, x=x, positions=p, keys=True, bf16=True)
    assert dims == (3, 192) and e.dims_of(out)[1] == BF16
    c.append(e, x=x, positions=p, cos=None, sin=None)
    assert C.c_uint64.in_dll(fake, "fake_append_rotary").value == 0
    part = zeros(e, 32, 16)
    c.append(e, x=x, positions=p, cos=part, sin=part)                                       # half of each head rotated
    many, pm = zeros(e, 9, 256, F32), zeros(e, 9, 1, I32)
    c.append(e, n=9, x=many, positions=pm, sequences=pm)                                    # positions as a column
    refused(lambda: c.append(e, n=9, x=many, positions=pm))                                 # nine rows, three sequences
    wide = zeros(e, 4, 300, BF16)
    assert c.append(e, qkv=(wide, (1, 44), (3, 256)), positions=p)[1] == (3, 128)           # a block of a wider buffer
    before = e.device_traffic().launches
    assert c.append(e, n=0, qkv=(zeros(e, 1, 256), (0, 0), (0, 256)), positions=zeros(e, 0, 1, I32))[1] == (0, 128)
    assert e.device_traffic().launches == before


def test_append_refusals(e):
    c = Cache(e)
    x, p = zeros(e, 3, 256, BF16), zeros(e, 1, 3, I32)
    bad = lambda **k: refused(lambda: c.append(e, **{"x": x, "positions": p, **k}))
    for shape in (PageShape(4, 3, 32, 8), PageShape(0, 2, 32, 8), PageShape(4, 0, 32, 8), PageShape(4, 2, 0, 8), PageShape(4, 2, 32, 0),
                  PageShape(4, 2, 32, 7), PageShape(4, 2, 16, 8), PageShape(8, 2, 32, 8)):
        bad(shape=shape)
    bad(qkv=(x, (1, 0), (3, 256)))                                                          # the block leaves its buffer
    bad(qkv=(x, (0, 2**63), (3, 256)))
    bad(qkv=(zeros(e, 3, 256, I32), (0, 0), (3, 256)))
    bad(positions=zeros(e, 1, 4, I32))
    bad(positions=zeros(e, 1, 3, F32))
    bad(sequences=zeros(e, 1, 2, I32))
    bad(key_pages=zeros(e, 80, 64, F32))                                                    # keys F32, values BF16
    bad(key_pages=zeros(e, 72, 64, BF16))                                                   # fewer pages than the values
    bad(key_pages=c.values)                                                                 # one memory for both
    bad(page_table=zeros(e, 3, 4, F32))
    bad(sin=None)
    bad(sin=zeros(e, 32, 30))
    bad(cos=zeros(e, 32, 33), sin=zeros(e, 32, 33))
    bad(cos=zeros(e, 32, 34), sin=zeros(e, 32, 34))                                         # wider than a head
    bad(cos=zeros(e, 32, 32, BF16))
    refused(lambda: c.append(e, x=x, positions=777777), 5)
    packed = e.cast_bfp(zeros(e, 80, 64), 8)[0]
    bad(key_pages=packed)
    own = zeros(e, 80, 64, BF16)
    bad(qkv=(own, (0, 0), (3, 64)), shape=PageShape(0, 1, 32, 8))
    rows = e.slice_rows(c.keys, 0, 80)[0]
    bad(shape=PageShape(1, 1, 16, 8), qkv=(rows, (0, 0), (3, 48)), key_pages=e.reshape(c.keys, 320, 16)[0],
        value_pages=zeros(e, 320, 16, BF16), cos=None, sin=None)                            # the rows lie in the pages


def test_attention_dims_and_refusals(e):
    c = Cache(e)
    q, p = zeros(e, 3, 128), zeros(e, 1, 3, I32)
    out, dims = c.attend(e, q=q, positions=p)
    assert dims == (3, 128) and e.dims_of(out) == ((3, 128), F32)
    assert e.dims_of(c.attend(e, q=q, positions=p, bf16=True, window=5)[0])[1] == BF16
    assert c.attend(e, n=2, q=q, positions=zeros(e, 2, 1, I32))[1] == (2, 128)              # fewer rows than sequences
    bad = lambda **k: refused(lambda: c.attend(e, **{"q": q, "positions": p, **k}))
    bad(n=4)
    bad(positions=zeros(e, 1, 2, I32))
    bad(scale=float("nan"))
    bad(scale=float("inf"))
    bad(shape=PageShape(4, 3, 32, 8))
    bad(shape=PageShape(4, 2, 32, 9))
    bad(value_pages=c.keys)
    narrow = Cache(e, dim=48)
    refused(lambda: narrow.attend(e, q=zeros(e, 3, 192), positions=p))                      # heads of 48 columns
    wide = zeros(e, 2**20, 1, I32)
    bad(page_table=e.reshape(wide, 1, 2**20)[0], n=3)                                       # one sequence, three rows
    refused(lambda: c.attend(e, q=31337, positions=p), 5)


def test_results_into_a_buffer(e):
    c = Cache(e)
    x, p = zeros(e, 3, 256, BF16), zeros(e, 1, 3, I32)
    dst = zeros(e, 3, 128)
    count = e.device_traffic().pool_in_use
    assert c.append(e, x=x, positions=p, into=dst) == (dst, (3, 128))
    assert c.attend(e, q=dst, positions=p, into=(got := zeros(e, 3, 128))) == (got, (3, 128))
    e.free(got)
    assert e.device_traffic().pool_in_use == count                                         # no buffer was made
    refused(lambda: c.append(e, x=x, positions=p, into=zeros(e, 3, 127)))
    refused(lambda: c.append(e, x=x, positions=p, into=dst, bf16=True))
    refused(lambda: c.attend(e, q=dst, positions=p, into=dst))                              # over its own queries
    refused(lambda: c.attend(e, q=dst, positions=p, into=e.reshape(dst, 3, 128)[0]))        # a view of them
    long = zeros(e, 4, 127)
    refused(lambda: c.attend(e, q=zeros(e, 3, 128), positions=p, into=e.slice_rows(long, 1, 3)[0]))
    off = e.slice_rows(zeros(e, 160, 3), 1, 128)[0]                                         # 12 bytes into its parent
    refused(lambda: c.attend(e, q=zeros(e, 3, 128), positions=p, into=e.reshape(off, 3, 128)[0]))
    refused(lambda: c.attend(e, q=zeros(e, 3, 128), positions=p, into=999999), 5)


def test_logprob_dims_and_refusals(e):
    x, ids = zeros(e, 5, 100), zeros(e, 5, 1, I32)
    got = e.token_logprobs(x, ids)
    assert [d for _, d in got] == [(5, 1)] * 3 and all(e.dims_of(i) == ((5, 1), F32) for i, _ in got)
    got = e.token_logprobs(zeros(e, 5, 100, BF16), e.reshape(ids, 1, 5)[0], 0.5, 32)
    assert [e.dims_of(i) for i, _ in got[3:]] == [((5, 32), I32), ((5, 32), F32)]
    for k in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-21), dict(top=33)):
        refused(lambda: e.token_logprobs(x, ids, **k))
    refused(lambda: e.token_logprobs(zeros(e, 5, 4), ids, top=5))
    refused(lambda: e.token_logprobs(zeros(e, 5, 100, I32), ids))
    refused(lambda: e.token_logprobs(x, zeros(e, 4, 1, I32)))
    refused(lambda: e.token_logprobs(x, zeros(e, 5, 1)))
    refused(lambda: e.token_logprobs(zeros(e, 5, 0), ids))
    into = [zeros(e, 5, 1), 0, zeros(e, 5, 1), 0, 0]
    got = e.token_logprobs(x, ids, top=2, into=into)
    assert got[0][0] == into[0] and got[2][0] == into[2] and got[1][0] not in into
    floats = zeros(e, 5, 2)
    held = e.device_traffic().pool_in_use
    refused(lambda: e.token_logprobs(x, ids, into=[0, into[0], into[0], 0, 0]))             # two results, one memory
    refused(lambda: e.token_logprobs(x, ids, top=2, into=[0, 0, 0, floats, 0]))           # columns are I32
    assert e.device_traffic().pool_in_use == held                                          # the results made before the refusal went back


def test_logprob_backward_dims_and_refusals(e):
    x, ids, row = zeros(e, 5, 100), zeros(e, 5, 1, I32), zeros(e, 5, 1)
    assert e.token_logprobs_backward(x, ids, row, None, row)[1] == (5, 100)
    out = e.token_logprobs_backward(x, ids, row, row, row, row, 1.0, True)[0]
    assert e.dims_of(out) == ((5, 100), BF16)
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, row, row), 5)              # an entropy gradient without the entropies
    refused(lambda: e.token_logprobs_backward(x, ids, zeros(e, 4, 1), None, row))
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, zeros(e, 5, 1, I32)))
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, row, scale=0.0))
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, row, into=x))              # over the logits
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, row, bf16=True, into=zeros(e, 5, 100)))


def test_widths_and_scales_beyond_the_kernels_are_refused(e):
    c = Cache(e)
    d = 65535
    heads = 2**31 // d + 1                                                                  # columns behind 31 bits (of no rows)
    wide = zeros(e, 0, (heads + 2) * d, BF16)
    refused(lambda: e.rope_append_pages(PageShape(heads, 1, d, 1), (wide, (0, 0), (0, (heads + 2) * d)), None, None, zeros(e, 0, 1, I32), None,
                                        c.table, zeros(e, 0, d, BF16), zeros(e, 0, d, BF16)))
    q, p = zeros(e, 3, 128), zeros(e, 1, 3, I32)
    c.attend(e, q=q, positions=p, scale=-1e20)
    for scale in (1.1e20, -1.1e20, float("-inf")):
        refused(lambda: c.attend(e, q=q, positions=p, scale=scale))
    x, ids, row = zeros(e, 5, 100), zeros(e, 5, 1, I32), zeros(e, 5, 1)
    for scale in (1e-20 * 1.01, 1e6):
        e.token_logprobs(x, ids, scale)
        e.token_logprobs_backward(x, ids, row, None, row, scale=scale)
    refused(lambda: e.token_logprobs(x, ids, 1.1e6))
    refused(lambda: e.token_logprobs_backward(x, ids, row, None, row, scale=1.1e6))


def test_a_failed_launch_leaves_no_result(fake, e):
    c = Cache(e)
    x, q, p, ids, row = zeros(e, 3, 256, BF16), zeros(e, 3, 128), zeros(e, 1, 3, I32), zeros(e, 3, 1, I32), zeros(e, 3, 1)
    held = e.device_traffic().pool_in_use
    fail = C.c_int.in_dll(fake, "fake_serving_fail")
    fail.value = 1
    try:
        for call in (lambda: c.append(e, x=x, positions=p), lambda: c.attend(e, q=q, positions=p), lambda: e.token_logprobs(q, ids, top=3),
                     lambda: e.token_logprobs_backward(q, ids, row, None, row)):
            refused(call)
            assert e.device_traffic().pool_in_use == held
    finally:
        fail.value = 0


def test_out_of_memory_part_way_gives_back_what_was_made(fake):
    for at in (3, 4, 5):
        with CudaEngine(0, lib=fake, fail_alloc_at=at) as e:
            x, ids = zeros(e, 5, 100), zeros(e, 5, 1, I32)
            held = e.device_traffic().pool_in_use
            refused(lambda: e.token_logprobs(x, ids, top=4), 1)
            assert e.device_traffic().pool_in_use == held


def test_the_calls_are_captured_into_a_trace(e):
    c = Cache(e)
    x, p, ids = zeros(e, 3, 256, BF16), zeros(e, 1, 3, I32), zeros(e, 3, 1, I32)
    e.begin_trace()
    q, _ = c.append(e, x=x, positions=p)
    o, _ = c.attend(e, q=q, positions=p)
    e.token_logprobs(o, ids, top=3)
    t = e.end_trace()
    assert len(e.trace_ops(t)) == 3
    e.run_trace(t)
    e.release_trace(t)


def test_calls_as_words(fake, e):
    """Every call as words is the call with its arguments: results, dims and refusals; other words are refused."""
    w, u64 = (C.c_uint64 * 19)(), C.c_uint64
    send = lambda call, n, *words: fake.b200_serving_call(e._e, C.c_int32(call), w, u64(n)) if not w.__setitem__(slice(0, len(words)), words) else None  # noqa: E731
    for call, n in ((-1, 19), (4, 12), (0, 18), (1, 19), (2, 17), (3, 11)):
        assert send(call, n) == 2
    assert fake.b200_serving_call(e._e, C.c_int32(0), None, u64(19)) == 2
    c = Cache(e)
    x, p, q = zeros(e, 3, 256, BF16), zeros(e, 1, 3, I32), zeros(e, 3, 128)
    at = C.addressof(c.shape)
    assert send(0, 19, at, x, 0, 0, 3, 256, c.cos, c.sin, p, 0, c.table, c.keys, c.values, 1, 1, 0, 0, 0, 0) == 0
    assert (w[17], w[18]) == (3, 192) and e.dims_of(w[16]) == ((3, 192), BF16)
    half = int(np.float32(0.5).view(np.uint32))
    assert send(1, 17, at, q, 0, 0, 3, 128, c.keys, c.values, c.table, p, 7, half, 0, q, 0, 0, 0) == 2   # into one of the operands
    out = zeros(e, 3, 128)
    assert send(1, 17, at, q, 0, 0, 3, 128, c.keys, c.values, c.table, p, 7, half, 0, out, 0, 0, 0) == 0
    assert (w[14], w[15], w[16]) == (out, 3, 128)
    logits, ids, row = zeros(e, 5, 100), zeros(e, 5, 1, I32), zeros(e, 5, 1)
    assert send(2, 16, logits, ids, half, 4, 0, 0, row, 0, 0) == 0
    assert w[11] == row and [e.dims_of(w[i])[0] for i in (9, 10, 12, 13)] == [(5, 1), (5, 1), (5, 4), (5, 4)] and (w[14], w[15]) == (5, 1)
    assert send(2, 16, logits, ids, half, 4, 31337, 0, 0, 0, 0) == 5
    assert send(3, 12, logits, ids, row, row, row, row, half, 1, 0) == 0
    assert e.dims_of(w[9]) == ((5, 100), BF16) and (w[10], w[11]) == (5, 100)
    got = e.token_logprobs(logits, ids, top=3, into=[row])                                  # the others are new
    assert got[0][0] == row and len(got) == 5
    with pytest.raises(ValueError):
        e.token_logprobs(logits, ids, into=[0] * 6)
    from metalium_rs_b200.engine import BlockArg
    block = BlockArg(q, (u64 * 2)(0, 0), (u64 * 2)(3, 128))
    assert e.attention_pages(c.shape, block, c.keys, c.values, c.table, p, 0.5)[1] == (3, 128)

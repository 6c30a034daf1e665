"""`LlamaPagedDecode`'s bookkeeping without a GPU: the pool's pages, slots that come and go, what a failed call leaves behind.  The
engine is the host-only one, every launch a no-op."""
import numpy as np
import pytest

from metalium_rs_b200 import I32, workloads as W
from tests.test_serving_host import e, fake  # noqa: F401 (fixtures)

CFG = W.LlamaConfig(layers=2, hidden=64, heads=2, kv_heads=1, head_dim=64, ff=128, vocab=256)


def decode(e, batch, max_len, pages, page_size, seq=32, prompts=2):  # noqa: F811
    pre = W.LlamaPrefill(e, CFG, W.llama_weights(CFG, seed=3), prompts, seq)
    ids = e.upload_bits(np.zeros((1, prompts * seq), np.int32), 1, prompts * seq, I32)
    return pre, ids, W.LlamaPagedDecode(e, CFG, pre.w, batch, max_len=max_len, pages=pages, page_size=page_size)


def test_a_prefill_the_pool_has_no_room_for_takes_nothing(e):  # noqa: F811
    pre, ids, paged = decode(e, 3, 64, pages=3, page_size=16)
    held = e.device_traffic().pool_in_use
    with pytest.raises(MemoryError, match=r"4 pages.*\[2, 0\].*3 spare"):
        pre.forward(ids, cache=paged, slots=[2, 0])
    assert sorted(paged.spare) == [0, 1, 2] and (paged.tables == -1).all() and e.device_traffic().pool_in_use == held
    with pytest.raises(ValueError, match="slot 1"):
        paged.reserve_all([0, 1], [16, 65])
    for slots in ([0, 0], [3], [-1]):
        with pytest.raises(ValueError, match="each once"):
            paged.reserve_all(slots, [1] * len(slots))
    assert len(paged.spare) == 3
    pre.forward(ids, cache=paged, slots=[2, 0], lengths=[32, 16])
    assert not paged.spare and (paged.tables >= 0).sum(1).tolist() == [1, 0, 2]
    paged.finish(2)
    paged.finish(0)
    assert sorted(paged.spare) == [0, 1, 2]


def test_a_prefill_into_a_running_sequence_is_refused(e):  # noqa: F811
    pre, ids, paged = decode(e, 3, 64, pages=12, page_size=16)
    lg, am = pre.forward(ids, cache=paged, slots=[1, 0], lengths=[20, 30])
    paged.begin([1, 0], am, [20, 30])
    before = paged.tables.copy()
    with pytest.raises(ValueError, match=r"\[1\]"):
        pre.forward(ids, cache=paged, slots=[2, 1])
    assert np.array_equal(paged.tables, before) and paged.lengths.tolist() == [30, 20, -1]
    paged.finish(1)
    pre.forward(ids, cache=paged, slots=[2, 1])


def test_a_step_takes_its_pages_at_once_or_names_the_slots(e):  # noqa: F811
    pre, ids, paged = decode(e, 4, 10, pages=5, page_size=4)
    paged.begin([0, 1, 3], [5, 6, 7], [0, 0, 0])
    writes = lambda: e.device_traffic().h2d_calls  # noqa: E731
    before = writes()
    for _ in range(4):
        paged.step()
    assert writes() - before == 1 and paged.held.tolist() == [1, 1, 0, 1]       # three first pages, one table
    with pytest.raises(MemoryError, match=r"3 pages.*\[0, 1, 3\].*2 spare"):
        paged.step()
    assert len(paged.spare) == 2 and paged.lengths.tolist() == [4, 4, -1, 4] and paged.held.tolist() == [1, 1, 0, 1]
    paged.finish(1)
    before = writes()
    for _ in range(4):
        paged.step()
    assert writes() - before == 1 and paged.lengths.tolist() == [8, -1, -1, 8] and len(paged.spare) == 1
    with pytest.raises(MemoryError, match=r"2 pages.*\[0, 3\].*1 spare"):
        paged.step()
    paged.finish(0)
    for _ in range(2):
        paged.step()
    with pytest.raises(ValueError, match=r"\[3\] hold 10 positions"):               # in the middle of its third page
        paged.step()
    assert paged.lengths.tolist() == [-1, -1, -1, 10] and paged.held.tolist() == [0, 0, 0, 3]
    paged.finish(3)
    assert sorted(paged.spare) == [0, 1, 2, 3, 4] and (paged.tables == -1).all()


def test_a_call_without_a_shape_is_refused(e, fake):  # noqa: F811
    import ctypes as C
    words = (C.c_uint64 * 19)(*[0] * 19)
    for call, n in ((0, 19), (1, 17)):
        assert fake.b200_serving_call(e._e, C.c_int32(call), words, C.c_uint64(n)) == 2

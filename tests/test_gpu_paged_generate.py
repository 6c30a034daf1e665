"""The paged cache's operators run together, as a model uses them: `LlamaPagedDecode` against `LlamaDecode` (sequences in
lockstep over dense caches), prompts of several lengths prefilled into pages, slots that come and go, the captured step, and
the loss's fused form in the training step.  Logits are held to the 2e-2 that the cached steps of the dense cache are held to
(two orders of summation around a dozen BF16 roundings a layer)."""
import numpy as np
import pytest

from metalium_rs_b200 import I32, workloads as W
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

CFG = W.LlamaConfig(layers=3, hidden=576, heads=9, kv_heads=3, head_dim=64, ff=1536, vocab=2048)


def _i32(eng, a, r, c):
    return eng.upload_bits(np.ascontiguousarray(a, dtype=np.int32).view(np.uint32), r, c, I32)


@pytest.fixture(scope="module")
def weights(eng):
    pre = W.LlamaPrefill(eng, CFG, W.llama_weights(CFG, seed=11), 2, 32)
    return pre.w


def free(eng, out):
    for i in out.values():
        eng.free(i)


@pytest.mark.parametrize("page_size", [16, 5])
def test_paged_steps_are_the_dense_steps(eng, weights, page_size):
    steps, top = 40, 5
    ids = orc.integers(0x91, 1, (steps, 2), CFG.vocab)
    dense = W.LlamaDecode(eng, CFG, weights, 2, max_len=64)
    paged = W.LlamaPagedDecode(eng, CFG, weights, 3, max_len=64, pages=30, page_size=page_size, top=top)
    dense.reset(ids[0])
    paged.begin([2, 0], ids[0], [0, 0])                     # slot 1 stays idle
    worst = 0.0
    for t in range(steps):
        dense.set_ids(ids[t])
        paged._set(paged.ids, [2, 0], ids[t])
        lg, am = dense.step()
        out = paged.step()
        a, b = eng.download(lg), eng.download(out["logits"])[[2, 0]]
        worst = max(worst, float(np.abs(a - b).max()))
        choice = eng.download_bits(out["argmax"]).view(np.int32)[:, 0]
        b = eng.download(out["logits"]).astype(np.float64)
        log = b - np.log(np.exp(b - b.max(1, keepdims=True)).sum(1, keepdims=True)) - b.max(1, keepdims=True)
        assert np.array_equal(choice, b.argmax(1))
        # F32 logits of at most a few units, 2048 columns: 600 roundings of 2^-24 and the entropy's factor
        assert np.abs(eng.download(out["logprob"])[:, 0] - log.max(1)).max() <= 1e-4
        assert np.abs(eng.download(out["entropy"])[:, 0] + (np.exp(log) * log).sum(1)).max() <= 4e-4
        assert np.array_equal(eng.download_bits(out["top_ids"]).view(np.int32), np.argsort(-b, 1, kind="stable")[:, :top])
        eng.free(lg); eng.free(am)
        free(eng, out)
    assert worst <= 2e-2, worst
    assert list(paged.lengths) == [steps, -1, steps] and eng.download_bits(paged.pos).view(np.int32)[:, 0].tolist() == [steps, -1, steps]
    for l in range(CFG.layers):                             # the rows are the dense cache's, to a BF16 step
        for dense_c, paged_c in ((dense.kc[l], paged.kc[l]), (dense.vc[l], paged.vc[l])):
            d = orc.from_bf16(eng.download_bf16(dense_c)).reshape(2, 64, -1)
            p = orc.from_bf16(eng.download_bf16(paged_c))
            for i, s in enumerate((2, 0)):
                rows = paged.tables[s, np.arange(steps) // page_size] * page_size + np.arange(steps) % page_size
                assert np.max(np.abs(p[rows] - d[i, :steps])) <= 2.0 ** -6 * np.abs(d).max()


@pytest.mark.parametrize("seq", [32, 128])
def test_prompts_of_several_lengths_prefill_into_pages(eng, weights, seq):
    lengths, slots, more = [seq, seq - 13, 1], [3, 0, 2], 6
    ids = orc.integers(0x92, 2, (3, seq), CFG.vocab)
    pre = W.LlamaPrefill(eng, CFG, W.llama_weights(CFG, seed=11), 3, seq)
    paged = W.LlamaPagedDecode(eng, CFG, pre.w, 4, max_len=seq + 16, pages=40, page_size=8)
    ii = _i32(eng, ids.reshape(1, -1), 1, 3 * seq)
    lg, am = pre.forward(ii, cache=paged, lengths=lengths, slots=slots)
    whole, amw = pre.forward(ii, all_positions=True)
    every = eng.download(whole).reshape(3, seq, -1)
    got = eng.download(lg)
    assert max(np.abs(got[b] - every[b, lengths[b] - 1]).max() for b in range(3)) <= 2e-2
    held = {int(p) for p in paged.tables[paged.tables >= 0]}
    spare = [p for p in range(40) if p not in held]
    for l in range(CFG.layers):                             # rows of no prompt are as they were: zero
        for buf in (paged.kc[l], paged.vc[l]):
            rows = orc.from_bf16(eng.download_bf16(buf)).reshape(40, 8, -1)
            assert not rows[spare].any()
            for s, n in zip(slots, lengths):
                flat = rows[paged.tables[s][paged.tables[s] >= 0]].reshape(-1, rows.shape[-1])
                assert flat[:n].any(1).all() and not flat[n:].any()
    # the prompts continued, against the same tokens stepped through a dense cache from their first token
    paged.begin(slots, am, lengths)
    choice = eng.download_bits(am).view(np.int32)[:, 0]
    stepped = W.LlamaDecode(eng, CFG, pre.w, 1, max_len=-(-(seq + 16) // 32) * 32)
    outs = []
    fed = [list(ids[b, :lengths[b]]) + [int(choice[b])] for b in range(3)]
    for _ in range(more):
        out = paged.step()
        outs.append(eng.download(out["logits"])[slots])
        nxt = eng.download_bits(out["argmax"]).view(np.int32)[slots, 0]
        for b in range(3):
            fed[b].append(int(nxt[b]))
        free(eng, out)
    for b in range(3):
        stepped.reset(np.array(fed[b][:1], np.int32))
        for t in range(lengths[b] + more):
            stepped.set_ids(np.array([fed[b][t]], np.int32))
            l1, a1 = stepped.step()
            if t >= lengths[b]:
                assert np.abs(eng.download(l1)[0] - outs[t - lengths[b]][b]).max() <= 2e-2, (b, t)
            eng.free(l1); eng.free(a1)
    with pytest.raises(ValueError):
        pre.forward(ii, cache=paged, lengths=[seq + 1, 1, 1])
    with pytest.raises(ValueError):
        pre.forward(ii, cache=paged, slots=[0, 0, 1])
    with pytest.raises(ValueError):
        pre.forward(ii, lengths=lengths)
    for i in (ii, lg, am, whole, amw):
        eng.free(i)


def test_slots_come_and_go_and_pages_return(eng, weights):
    paged = W.LlamaPagedDecode(eng, CFG, weights, 2, max_len=48, pages=4, page_size=8)
    alone = []
    for first in (7, 1900):                                 # each sequence by itself, ten steps
        paged.begin([0], [first], [0])
        run = []
        for _ in range(10):
            out = paged.step()
            run.append(eng.download(out["logits"])[0])
            free(eng, out)
        alone.append(np.stack(run))
        paged.finish(0)
        assert len(paged.spare) == 4
    paged.begin([1], [1900], [0])
    both = []
    for t in range(14):
        if t == 4:
            paged.begin([0], [7], [0])                      # the other starts four steps later
        out = paged.step()
        both.append(eng.download(out["logits"]))
        free(eng, out)
        if t == 9:
            paged.finish(1)
    assert max(np.abs(both[t][1] - alone[1][t]).max() for t in range(10)) <= 2e-2
    assert max(np.abs(both[t + 4][0] - alone[0][t]).max() for t in range(10)) <= 2e-2
    assert len(paged.spare) == 2 and paged.lengths.tolist() == [10, -1]
    paged.reserve(1, 16)
    with pytest.raises(MemoryError):
        paged.reserve(1, 17)
    with pytest.raises(ValueError):
        paged.reserve(0, 49)
    assert (paged.tables[1] >= 0).sum() == 2                # the refused reservation took nothing
    eng.sync()


def test_a_captured_paged_step_is_the_eager_one(eng, weights):
    def start():
        d = W.LlamaPagedDecode(eng, CFG, weights, 3, max_len=64, pages=20, page_size=4, top=3)
        d.begin([0, 2], [3, 77], [0, 0])
        return d
    eager, traced = start(), start()
    want = []
    for _ in range(12):
        out = eager.step()
        want.append([eng.download_bits(out[k]) for k in ("logits", "argmax", "logprob", "entropy", "top_ids", "top_logprobs")])
        free(eng, out)
    out = traced.capture()
    for t in range(12):
        traced.replay()
        got = [eng.download_bits(out[k]) for k in ("logits", "argmax", "logprob", "entropy", "top_ids", "top_logprobs")]
        live = [0, 2]
        assert all(np.array_equal(a[live], b[live]) for a, b in zip(got, want[t])), t
    assert traced.lengths.tolist() == eager.lengths.tolist() == [12, -1, 12]
    eng.release_trace(traced.trace)
    free(eng, out)


def test_the_training_step_with_the_fused_loss(eng):
    """`MlpStep(fused_loss=True)`: the loss and every gradient are the composition's.  Both form z's gradient (p - 1[label]) / n
    from logits of a few units: within 64 roundings of 1 / n each, and the products that follow keep that relative to the sums
    of absolute values, bounded here through the largest entry times the number of rows."""
    rng = np.random.default_rng(21)
    n, h = 96, 128
    w1, w2 = (rng.standard_normal((784, h)) * 0.05).astype(np.float32), (rng.standard_normal((h, 10)) * 0.1).astype(np.float32)
    b1, b2 = np.zeros(h, np.float32), np.zeros(10, np.float32)
    x, labels = rng.standard_normal((n, 784)).astype(np.float32), rng.integers(0, 10, n)
    got = []
    for fused in (False, True):
        m = W.MlpStep(eng, w1, b1, w2, b2, lr=0.1, fused_loss=fused)
        ix, il = eng.upload(x, n, 784), _i32(eng, labels, n, 1)
        l0 = eng.device_traffic().launches
        out = m.step(ix, il, n, keep=True)
        launches = eng.device_traffic().launches - l0
        got.append({k: eng.download(v) for k, v in out.items()} | {"launches": launches, "w1": eng.download(m.w1)})
        for i in list(out.values()) + [ix, il, m.w1, m.b1, m.w2, m.b2]:
            eng.free(i)
    a, b = got
    u = 2.0 ** -24
    assert abs(a["loss"] - b["loss"]).max() <= 64 * u * 3
    assert np.abs(a["dz"] - b["dz"]).max() <= 64 * u / n
    for k, other in (("dw2", np.maximum(x @ w1, 0)), ("db2", np.ones(1)), ("dw1", x)):
        assert np.abs(a[k] - b[k]).max() <= 64 * u * max(1.0, np.abs(other).max()) * (1 if k != "dw1" else 10 * np.abs(w2).max()), k
    assert b["launches"] <= a["launches"] - 5

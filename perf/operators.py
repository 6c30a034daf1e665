"""The serving and scoring operators as they are measured: cases, inputs, the plain form, and the 64-bit definition.

Four operators of a decoder's step over a paged key/value cache:
  append              rotate a projection's query and key heads and store keys and values into the cache's pages
  attention           one new token a sequence over its pages
  logprobs            log probabilities of given tokens, entropy and the largest alternatives of each row
  logprobs_backward   their gradient with respect to the logits
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------ cases
def _append(name, batch, new, past, heads, kv_heads, dim, page, rotary, x, cache, out, keys):
    return {"name": name, "op": "append", "batch": batch, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "rotary": rotary, "x": x, "cache": cache, "out": out, "keys": keys}


def _attention(name, batch, shortest, longest, idle, heads, kv_heads, dim, page, window, q, cache, out):
    return {"name": name, "op": "attention", "batch": batch, "shortest": shortest, "longest": longest, "idle": idle,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "q": q, "cache": cache, "out": out}


def _logprobs(name, rows, vocab, top, scale, logits):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "scale": scale, "logits": logits}


def _backward(name, rows, vocab, scale, entropy, logits, out):
    return {"name": name, "op": "logprobs_backward", "rows": rows, "vocab": vocab, "scale": scale, "entropy": entropy,
            "logits": logits, "out": out}


def listed():
    return [
        # one generated token of one sequence: the 9 / 3 heads of 64 of the repository's decoder, F32 queries for the attention
        _append("append step 1", 1, 1, 700, 9, 3, 64, 16, 64, "bf16", "bf16", "f32", False),
        # a batch of generated tokens, 32 / 8 heads of 128, half of each head rotated, F32 projections
        _append("append step 96", 96, 1, 1500, 32, 8, 128, 32, 64, "f32", "bf16", "bf16", False),
        # prompts of several lengths padded to 1000 tokens; the rotated keys are kept for the prompt's own attention
        _append("append prompts 8x1000", 8, 1000, 0, 32, 8, 128, 16, 128, "bf16", "bf16", "bf16", True),
        # one sequence, a short chat: latency
        _attention("attention 1x300", 1, 300, 300, 0, 9, 3, 64, 16, 0, "f32", "bf16", "bf16"),
        # an ordinary mixed batch with two idle slots
        _attention("attention 32 mixed", 32, 5, 4100, 2, 32, 8, 128, 16, 0, "bf16", "bf16", "bf16"),
        # one long document: the positions are the only parallel axis
        _attention("attention 1x131001", 1, 131001, 131001, 0, 32, 8, 128, 64, 0, "bf16", "bf16", "bf16"),
        # an F32 cache, F32 in and out, one key/value head a query head, odd pages
        _attention("attention f32 cache", 12, 40, 2500, 0, 8, 8, 96, 24, 0, "f32", "f32", "f32"),
        # the largest: a full serving batch
        _attention("attention 128x8192", 128, 500, 8192, 0, 32, 8, 128, 32, 0, "bf16", "bf16", "bf16"),
        # a sampled token's log probability with five alternatives: one generation step's logits
        _logprobs("logprobs 1x49152", 1, 49152, 5, 1.0, "f32"),
        # scoring: an odd vocabulary in BF16, twenty alternatives
        _logprobs("logprobs 2000x50257", 2000, 50257, 20, 0.8, "bf16"),
        # training: a batch of tokens, log probability alone
        _backward("backward 500x49152", 500, 49152, 1.0, False, "f32", "f32"),
        # training with an entropy bonus, an odd vocabulary, BF16 logits and gradients
        _backward("backward 4000x32001", 4000, 32001, 0.7, True, "bf16", "bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "logprobs", "logprobs_backward"])
    heads, kv_heads, dim = rng.choice([(9, 3, 64), (32, 8, 128), (8, 8, 96), (16, 2, 64), (12, 4, 32), (24, 1, 128), (8, 2, 256), (6, 6, 192)])
    page = rng.choice([8, 16, 20, 32, 48, 64, 128])
    kinds = lambda: rng.choice(["bf16", "bf16", "f32"])  # noqa: E731
    if op == "append":
        new = rng.choice([1, 1, _between(rng, 2, 2000)])
        batch = _between(rng, 1, max(1, min(200, 80_000_000 // (new * (heads + 2 * kv_heads) * dim))))
        return {"op": op, "batch": batch, "new": new, "past": _between(rng, 1, 2000), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": page, "rotary": rng.choice([0, dim // 2, dim, dim]), "x": kinds(), "cache": kinds(), "out": kinds(),
                "keys": new > 1}
    if op == "attention":
        batch = _between(rng, 1, 200)
        cache = kinds()
        longest = _between(rng, 1, max(1, min(140_000, 700_000_000 // (batch * kv_heads * dim * BYTES[cache] // 2))))
        return {"op": op, "batch": batch, "shortest": _between(rng, 1, longest), "longest": longest, "idle": rng.choice([0, 0, 1]) if batch > 2 else 0,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "window": rng.choice([0, 0, 0, _between(rng, 1, 5000)]),
                "q": kinds(), "cache": cache, "out": kinds()}
    vocab = _between(rng, 10, 260_000)
    rows = _between(rng, 1, max(1, min(8000, 100_000_000 // vocab)))
    scale = rng.choice([1.0, 1.0, 0.7, 1.3])
    if op == "logprobs":
        return {"op": op, "rows": rows, "vocab": vocab, "top": min(vocab, rng.choice([0, 1, 5, 20, 32])), "scale": scale, "logits": kinds()}
    return {"op": op, "rows": rows, "vocab": vocab, "scale": scale, "entropy": rng.choice([False, True]), "logits": kinds(), "out": kinds()}


def _spread(lo, hi, count):
    """`count` lengths from `lo` to `hi`: a batch whose sequences differ (the longest is there, alone too)."""
    return np.linspace(hi, lo, count).round().astype(np.int64)


def _visible(case):
    """How many positions each sequence of an attention case attends to."""
    n = _spread(case["shortest"], case["longest"], case["batch"])
    n[len(n) - case["idle"]:] = 0
    return np.minimum(n, case["window"]) if case["window"] else n


def work(case):
    if case["op"] == "append":
        cols = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        new = int(_spread(max(1, case["new"] // 2), case["new"], case["batch"]).sum())
        kept = case["heads"] + (case["kv_heads"] if case["keys"] else 0)
        whole = case["batch"] * case["new"]
        return {"bytes": new * cols * BYTES[case["x"]] + whole * kept * case["dim"] * BYTES[case["out"]]
                + new * 2 * case["kv_heads"] * case["dim"] * BYTES[case["cache"]] + (new * 2 * 4 * case["rotary"] if case["new"] == 1 else 2 * 4 * case["rotary"] * (case["new"] + case["past"])) + whole * 12,
                "flops": new * (case["heads"] + case["kv_heads"]) * case["rotary"] * 3}
    if case["op"] == "attention":
        seen = int(_visible(case).sum())
        row = case["batch"] * case["heads"] * case["dim"]
        return {"bytes": seen * 2 * case["kv_heads"] * case["dim"] * BYTES[case["cache"]] + row * (BYTES[case["q"]] + BYTES[case["out"]]) + seen // case["page"] * 4,
                "flops": 4 * seen * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    if case["op"] == "logprobs":
        return {"bytes": n * BYTES[case["logits"]] + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    return {"bytes": n * (BYTES[case["logits"]] + BYTES[case["out"]]) + case["rows"] * 20, "flops": 8 * n}


# ------------------------------------------------------------------------------------------------ inputs
def _pages(gen, rows, counts, width):
    """A page table [rows, width]: `counts[b]` pages for sequence b, drawn without order from the pool, -1 behind them; and the pool's size."""
    total = int(counts.sum())
    spare = 3 + total // 16
    order = torch.randperm(total + spare, generator=gen, device="cuda")[:total].to(torch.int32)
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    n = torch.from_numpy(counts).cuda()
    table[torch.arange(width, device="cuda")[None, :] < n[:, None]] = order
    return table, total + spare


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda shape, dtype, sigma=1.0: (torch.randn(shape, generator=gen, device="cuda") * sigma).to(DTYPES[dtype])  # noqa: E731
    s = {"case": case}
    if case["op"] == "append":
        batch, new, page, dim = case["batch"], case["new"], case["page"], case["dim"]
        past = _spread(0 if new > 1 else max(0, case["past"] // 3), case["past"], batch)
        fresh = _spread(max(1, new // 2), new, batch)
        ends = past + fresh
        s["table"], pool = _pages(gen, batch, -(-ends // page), int(-(-ends.max() // page)))
        at = torch.arange(new, device="cuda")[None, :]
        position = torch.where(at < torch.from_numpy(fresh).cuda()[:, None], torch.from_numpy(past).cuda()[:, None] + at, -1)
        s["positions"] = position.to(torch.int32).reshape(1, -1)
        s["sequences"] = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(new).reshape(1, -1)
        s["qkv"] = normal((batch * new, (case["heads"] + 2 * case["kv_heads"]) * dim), case["x"])
        s["keys"] = normal((pool * page, case["kv_heads"] * dim), case["cache"])
        s["values"] = normal((pool * page, case["kv_heads"] * dim), case["cache"])
        r = case["rotary"]
        if r:
            angle = torch.arange(int(ends.max()), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
                -2.0 * torch.arange(r // 2, device="cuda", dtype=torch.float64) / r)[None, :]
            s["cos"] = torch.cat([angle.cos(), angle.cos()], 1).float().contiguous()
            s["sin"] = torch.cat([-angle.sin(), angle.sin()], 1).float().contiguous()
        kept = case["heads"] + (case["kv_heads"] if case["keys"] else 0)
        s["out"] = torch.empty((batch * new, kept * dim), dtype=DTYPES[case["out"]], device="cuda")
    elif case["op"] == "attention":
        batch, page, width = case["batch"], case["page"], case["kv_heads"] * case["dim"]
        length = _spread(case["shortest"], case["longest"], batch)
        length[batch - case["idle"]:] = 0
        mix = torch.randperm(batch, generator=gen, device="cuda")
        length = length[mix.cpu().numpy()]
        s["table"], pool = _pages(gen, batch, -(-length // page), int(-(-length.max() // page)))
        s["positions"] = torch.from_numpy(length - 1).cuda().to(torch.int32).reshape(1, -1)
        s["q"] = normal((batch, case["heads"] * case["dim"]), case["q"], 1.5)
        s["keys"] = normal((pool * page, width), case["cache"])
        s["values"] = normal((pool * page, width), case["cache"])
        s["scale"] = 1.0 / math.sqrt(case["dim"])
        s["out"] = torch.empty((batch, case["heads"] * case["dim"]), dtype=DTYPES[case["out"]], device="cuda")
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.0
        likely = torch.randint(0, vocab, (rows, 4), generator=gen, device="cuda")  # a few tokens a row stand out
        x.scatter_(1, likely, 7.0 + 2.0 * torch.randn((rows, 4), generator=gen, device="cuda"))
        s["logits"] = x.to(DTYPES[case["logits"]])
        del x
        other = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        ids = torch.where(torch.rand((rows, 1), generator=gen, device="cuda") < 0.7, likely[:, :1], other)
        column = lambda: torch.empty((rows, 1), device="cuda")  # noqa: E731
        if case["op"] == "logprobs":
            s["ids"] = ids.to(torch.int32)
            s["out"] = [column(), column(), column()]
            if case["top"]:
                s["out"] += [torch.empty((rows, case["top"]), dtype=torch.int32, device="cuda"), torch.empty((rows, case["top"]), device="cuda")]
        else:
            padding = torch.rand((rows, 1), generator=gen, device="cuda") < (0.1 if rows > 4 else 0.0)   # a padded batch
            s["ids"] = torch.where(padding, -1, ids).to(torch.int32)
            lse, entropy = column(), column()
            for a in range(0, rows, 512):
                y = s["logits"][a:a + 512].double() * case["scale"]
                lse[a:a + 512, 0] = torch.logsumexp(y, 1).float()
                p = torch.exp(y - torch.logsumexp(y, 1, keepdim=True))
                entropy[a:a + 512, 0] = (torch.logsumexp(y, 1) - (p * y).sum(1)).float()
            s["lse"], s["entropy"] = lse, entropy
            s["d_logprob"] = torch.where(padding, 0.0, torch.randn((rows, 1), generator=gen, device="cuda"))
            s["d_entropy"] = torch.randn((rows, 1), generator=gen, device="cuda") * 0.1 if case["entropy"] else None
            s["out"] = torch.empty((rows, vocab), dtype=DTYPES[case["out"]], device="cuda")
    return s


_held = {}


def _engine():
    """The process's engine, as a program keeps one."""
    if "engine" not in _held:
        from metalium_rs_b200 import CudaEngine
        _held["engine"] = CudaEngine(0)
    return _held["engine"]


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from metalium_rs_b200 import BF16, F32, I32, PageShape
        eng, elem = _engine(), {torch.bfloat16: BF16, torch.float32: F32, torch.int32: I32}
        adopt = lambda t: eng.adopt(t.data_ptr(), t.shape[0], t.shape[1], elem[t.dtype])  # noqa: E731
        s["id"] = {k: adopt(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if case["op"] == "logprobs":
            s["id"]["out"] = [adopt(t) for t in s["out"]]
        if case["op"] in ("append", "attention"):
            s["shape"] = PageShape(case["heads"], case["kv_heads"], case["dim"], case["page"])
        torch.cuda.synchronize()   # the engine has a stream of its own
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_append(s):
    i, c = s["id"], s["case"]
    _engine().rope_append_pages(s["shape"], (i["qkv"], (0, 0), tuple(s["qkv"].shape)), i.get("cos"), i.get("sin"), i["positions"], i["sequences"],
                                i["table"], i["keys"], i["values"], keys=c["keys"], bf16=c["out"] == "bf16", into=i["out"])
    return {"heads": s["out"], "keys": s["keys"], "values": s["values"]}


def _own_attention(s):
    i, c = s["id"], s["case"]
    _engine().attention_pages(s["shape"], (i["q"], (0, 0), tuple(s["q"].shape)), i["keys"], i["values"], i["table"], i["positions"], s["scale"],
                              window=c["window"], bf16=c["out"] == "bf16", into=i["out"])
    return s["out"]


def _own_logprobs(s):
    i, c = s["id"], s["case"]
    _engine().token_logprobs(i["logits"], i["ids"], c["scale"], c["top"], into=i["out"])
    return s["out"]


def _own_backward(s):
    i, c = s["id"], s["case"]
    _engine().token_logprobs_backward(i["logits"], i["ids"], i["lse"], i["entropy"], i["d_logprob"], i.get("d_entropy"), c["scale"],
                                      bf16=c["out"] == "bf16", into=i["out"])
    return s["out"]


# ------------------------------------------------------------------------------------------------ the plain form
def _plain_append(s):
    c = s["case"]
    n, heads, kv, dim, r = s["qkv"].shape[0], c["heads"], c["kv_heads"], c["dim"], c["rotary"]
    x = s["qkv"].float().view(n, heads + 2 * kv, dim)
    position = s["positions"][0].long()
    there = position >= 0
    p = position.clamp(min=0)
    turn, value = x[:, :heads + kv], x[:, heads + kv:]
    if r:
        swap = torch.cat([turn[..., r // 2:r], turn[..., :r // 2]], -1)
        turn = torch.cat([turn[..., :r] * s["cos"][p][:, None] + swap * s["sin"][p][:, None], turn[..., r:]], -1)
    page = s["table"].long()[s["sequences"][0].long(), p // c["page"]]
    row = (page * c["page"] + p % c["page"])[there]
    s["keys"][row] = turn[there, heads:].reshape(-1, kv * dim).to(s["keys"].dtype)
    s["values"][row] = value[there].reshape(-1, kv * dim).to(s["values"].dtype)
    kept = turn if c["keys"] else turn[:, :heads]
    out = torch.where(there[:, None, None], kept, 0.0).reshape(n, -1).to(DTYPES[c["out"]])
    return {"heads": out, "keys": s["keys"], "values": s["values"]}


def _plain_attention(s):
    c = s["case"]
    batch, heads, kv, dim = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    last = s["positions"][0].long()[:, None]
    at = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    seen = (at[None, :] <= last) & ((at[None, :] > last - c["window"]) if c["window"] else True)
    row = s["table"].long().clamp(min=0)[:, at // c["page"]] * c["page"] + at % c["page"]
    k = s["keys"][row].float().view(batch, -1, kv, dim).permute(0, 2, 3, 1)
    q = s["q"].float().view(batch, kv, heads // kv, dim)
    score = torch.where(seen[:, None, None, :], torch.matmul(q, k) * s["scale"], -math.inf)
    del k
    top = score.max(-1, keepdim=True).values.clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    v = s["values"][row].float().view(batch, -1, kv, dim).permute(0, 2, 1, 3)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    return out.reshape(batch, heads * dim).to(DTYPES[c["out"]])


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    y = x * c["scale"]
    top = y.max(1, keepdim=True).values
    e = torch.exp(y - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.log(total) - (e * (y - top)).sum(1, keepdim=True) / total
    out = [y.gather(1, s["ids"].long()) - lse, entropy, lse]
    if c["top"]:
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
        out += [best.to(torch.int32), y.gather(1, best) - lse]
    return out


def _plain_backward(s):
    c = s["case"]
    y = s["logits"].float() * c["scale"] - s["lse"]
    p = torch.exp(y)
    ids = s["ids"].long()
    one = torch.arange(c["vocab"], device="cuda")[None, :] == ids
    grad = s["d_logprob"] * torch.where(ids >= 0, one.float() - p, 0.0)
    if s["d_entropy"] is not None:
        grad = grad - s["d_entropy"] * p * (y + s["entropy"])
    return (grad * c["scale"]).to(DTYPES[c["out"]])


def run(state):
    op = state["case"]["op"]
    if op == "append":
        return _own_append(state) if own else _plain_append(state)
    if op == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if op == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    return _own_backward(state) if own else _plain_backward(state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "append":
        d, h, g, r = case["dim"], case["heads"], case["kv_heads"], case["rotary"]
        x = s["qkv"].double()
        keys, values = s["keys"].double(), s["values"].double()
        position, sequence = s["positions"].cpu().numpy()[0], s["sequences"].cpu().numpy()[0]
        live = np.nonzero(position >= 0)[0]
        table = s["table"].cpu().numpy()
        row = table[sequence[live], position[live] // case["page"]].astype(np.int64) * case["page"] + position[live] % case["page"]
        t, row = torch.from_numpy(live).cuda(), torch.from_numpy(row).cuda()
        x = x[t]
        if r:
            cos, sin = s["cos"].double()[s["positions"][0].long()[t]], s["sin"].double()[s["positions"][0].long()[t]]
            half = r // 2
            for head in range(h + g):
                lo, hi = x[:, head * d:head * d + half].clone(), x[:, head * d + half:head * d + r].clone()
                x[:, head * d:head * d + half] = lo * cos[:, :half] + hi * sin[:, :half]
                x[:, head * d + half:head * d + r] = hi * cos[:, half:] + lo * sin[:, half:]
        keys[row] = x[:, h * d:(h + g) * d]
        values[row] = x[:, (h + g) * d:]
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        out[t] = x[:, :out.shape[1]]
        return {"heads": out, "keys": keys, "values": values}
    if case["op"] == "attention":
        d, h, g, page = case["dim"], case["heads"], case["kv_heads"], case["page"]
        out = torch.zeros((case["batch"], h * d), dtype=torch.float64, device="cuda")
        for b, last in enumerate(s["positions"][0].tolist()):
            if last < 0:
                continue
            j = torch.arange(max(0, last + 1 - case["window"]) if case["window"] else 0, last + 1, device="cuda")
            row = s["table"][b].long()[j // page] * page + j % page
            k, v = (s[n][row].double().view(len(j), g, d) for n in ("keys", "values"))
            w = torch.softmax(torch.einsum("hrd,jhd->hrj", s["q"][b].double().view(g, h // g, d), k) * s["scale"], -1)
            out[b] = torch.einsum("hrj,jhd->hrd", w, v).reshape(-1)
        return out
    if case["op"] == "logprobs":
        cols = [[], [], [], [], []]
        for a in range(0, case["rows"], 512):
            y = s["logits"][a:a + 512].double() * case["scale"]
            log = torch.log_softmax(y, 1)
            cols[0].append(log.gather(1, s["ids"][a:a + 512].long()))
            cols[1].append(-(log.exp() * log).sum(1, keepdim=True))
            cols[2].append(torch.logsumexp(y, 1, keepdim=True))
            if case["top"]:
                # the order on (value, index) as one whole number: the value's order-preserving 32 bits over the index's complement
                bits = s["logits"][a:a + 512].float().view(torch.int32).long()
                bits = torch.where(bits < 0, -2147483648 - bits, bits)
                key = bits * (1 << 20) + (1 << 20) - 1 - torch.arange(case["vocab"], device="cuda")
                best = (1 << 20) - 1 - torch.topk(key, case["top"], 1).values % (1 << 20)
                cols[3].append(best.to(torch.int32))
                cols[4].append(log.gather(1, best))
        return [torch.cat(col) for col in cols if col]
    out = torch.zeros((case["rows"], case["vocab"]), dtype=torch.float64, device="cuda")
    for a in range(0, case["rows"], 512):
        part = slice(a, a + 512)
        log = s["logits"][part].double() * case["scale"] - s["lse"][part].double()
        ids = s["ids"][part].long()
        g = torch.where(ids >= 0, s["d_logprob"][part].double(), 0.0)
        out[part] = -g * log.exp()
        out[part].scatter_add_(1, ids.clamp(min=0), g)
        if case["entropy"]:
            out[part] -= s["d_entropy"][part].double() * log.exp() * (log + s["entropy"][part].double())
    return out * case["scale"]

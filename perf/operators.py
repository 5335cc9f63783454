"""The serving operators around the block-quantized KV cache, as cases to measure:
writing tokens into the cache and reading them back, reading long prefixes,
attention over the cache (single tokens and prompts), and log probabilities of
given tokens with entropy and top alternatives.

``run`` computes an operator in its plain form (elementary torch operations in
32 bits), or, where ``own`` is true, through the framework's entry points.
Head layouts, widths and vocabularies are those of the framework's model shapes
(32 or 64 query heads over 8 KV heads of 128, heads of 64, vocabularies of
32000 and 128256) and generic odd ones.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SMALLEST = 2.0 ** -126  # a block whose scale would be below the normal range holds zeros


def listed():
    return [
        # one sequence decodes a token inside an open block: latency counts
        dict(name="write_step_1", kind="write", seqs=1, tokens=1, start=777, kv_heads=8, head_dim=128, block=64, dtype="f32"),
        # a serving step of 64 sequences of different lengths
        dict(name="write_step_64", kind="write", seqs=64, tokens=1, start=4003, kv_heads=8, head_dim=128, block=64, dtype="bf16"),
        # prompts of different lengths arrive together
        dict(name="write_prompts_8", kind="write", seqs=8, tokens=8191, start=0, kv_heads=8, head_dim=128, block=64, dtype="bf16"),
        # a 2048-token prefix is moved out of the cache (to another cache, or to compare it)
        dict(name="read_prefix_2048", kind="read", seqs=1, tokens=2048, start=0, kv_heads=8, head_dim=64, block=32, dtype="f32"),
        # a long document's keys and values are read back
        dict(name="read_long_131071", kind="read", seqs=1, tokens=131071, start=0, kv_heads=8, head_dim=128, block=128, dtype="f16"),
        # one sequence decodes after the benchmark's 512-token prompt
        dict(name="attend_step_1", kind="attend", seqs=1, tokens=1, start=512, heads=32, kv_heads=8, head_dim=128, block=64, window=0, dtype="f32"),
        # a serving step of 64 sequences up to 8192 tokens, 8 query heads for each KV head
        dict(name="attend_step_64", kind="attend", seqs=64, tokens=1, start=8191, heads=64, kv_heads=8, head_dim=128, block=64, window=0, dtype="bf16"),
        # one very long sequence: the work has to be split along it
        dict(name="attend_step_131071", kind="attend", seqs=1, tokens=1, start=131071, heads=32, kv_heads=8, head_dim=64, block=128, window=0, dtype="f16"),
        # the benchmark's 512-token prompt with the framework's FP32 activations
        dict(name="attend_prompt_512", kind="attend", seqs=1, tokens=512, start=0, heads=32, kv_heads=8, head_dim=128, block=64, window=0, dtype="f32"),
        # two long prompts of different lengths
        dict(name="attend_prompts_4096", kind="attend", seqs=2, tokens=4096, start=0, heads=32, kv_heads=8, head_dim=128, block=64, window=0, dtype="bf16"),
        # the logits of one decode step of eight sequences
        dict(name="score_step_8", kind="score", rows=8, vocab=128256, top=5, pad=0, dtype="f32"),
        # a prompt's logits, scored token by token
        dict(name="score_prompt_2048", kind="score", rows=2048, vocab=128256, top=20, pad=0, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend", "score", "score"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "score":
        vocab = _spread(rng, 1000, 256000)
        return dict(kind=kind, rows=_spread(rng, 1, min(2048, 262_000_000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), dtype=dtype)
    c = dict(kind=kind, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]), block=rng.choice([16, 32, 64, 128]), dtype=dtype)
    if kind == "write":
        if rng.random() < 0.5:  # a step: one or a few tokens at any position
            c.update(seqs=_spread(rng, 1, 64), tokens=rng.randint(1, 8), start=_spread(rng, 1, 8192))
        else:  # prompts: from the start, or after a shared prefix of whole blocks
            seqs = _spread(rng, 1, 8)
            c.update(seqs=seqs, tokens=_spread(rng, 130, 49152 // seqs), start=rng.choice([0, 0, c["block"] * rng.randint(1, 40)]))
        return c
    if kind == "read":
        seqs = _spread(rng, 1, 32)
        c.update(seqs=seqs, tokens=_spread(rng, 1, 131072 // seqs), start=rng.choice([0, 0, rng.randint(1, 5000)]))
        return c
    group = rng.choice([1, 2, 3, 4, 7, 8])
    c.update(heads=c["kv_heads"] * group, window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]))
    if rng.random() < 0.5:  # a decode step, or the check of a few drafted tokens
        seqs = _spread(rng, 1, 64)
        c.update(seqs=seqs, tokens=rng.choice([1, 1, rng.randint(2, 5)]), start=_spread(rng, 1, min(131072, 524288 // seqs)))
    else:
        seqs = _spread(rng, 1, 4)
        tokens = _spread(rng, 16, 2048)
        start = rng.choice([0, 0, _spread(rng, 1, 16384)])
        while seqs * c["heads"] * tokens * (start + tokens) > 1 << 30:
            start, tokens = start // 2, max(16, tokens * 3 // 4)
        c.update(seqs=seqs, tokens=tokens, start=start)
    return c


def _plan(case):
    """(starts, counts) of the case's sequences: the first has the full size, the others less, by the case alone."""
    rng = random.Random("%(seqs)d %(tokens)d %(start)d" % case)
    few = case["tokens"] <= 8
    starts, counts = [case["start"]], [case["tokens"]]
    for _ in range(case["seqs"] - 1):
        s = rng.randint(case["start"] // 2, case["start"])
        if case["kind"] == "write" and not few:
            s -= s % case["block"]
        starts.append(s)
        counts.append(case["tokens"] if few else rng.randint(max(1, case["tokens"] // 2), case["tokens"]))
    return starts, counts


def _pairs(case):
    """Visible (query, key) pairs of one head, and the keys that any query of a sequence sees."""
    pairs = keys = 0
    w = case["window"]
    for s, n in zip(*_plan(case)):
        pairs += sum(min(s + i + 1, w) for i in range(n)) if w else n * s + n * (n + 1) // 2
        keys += min(s + n, w + n - 1) if w else s + n
    return pairs, keys


def work(case):
    e = SIZE[case["dtype"]]
    if case["kind"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}
    hd, hk = case["head_dim"], case["kv_heads"]
    if case["kind"] == "attend":
        pairs, keys = _pairs(case)
        return {"bytes": 2 * hk * keys * (hd + 4 / case["block"]) + 2 * sum(_plan(case)[1]) * case["heads"] * hd * e, "flops": 4 * pairs * case["heads"] * hd}
    starts, counts = _plan(case)
    t = sum(counts)
    if case["kind"] == "read":
        return {"bytes": 2 * hk * t * (hd * (1 + e) + 4 / case["block"]), "flops": 2 * hk * t * hd}
    # written: the values in, 8 bits out, the newest rows kept; read back: 8 bits in, the values out
    back = sum(n + s % case["block"] for s, n in zip(starts, counts))
    kept = sum(min(n, case["block"]) for n in counts)
    return {"bytes": 2 * hk * hd * (t * (e + 1) + kept * e + back * (1 + e)), "flops": 2 * hk * hd * (4 * t + back)}


def _heads(shape, gen, dtype, dev):
    """Keys or values as a model makes them: normal, with a few wide channels."""
    x = torch.randn(shape, generator=gen, device=dev)
    return (x * (1 + 3 * (torch.rand(shape[-1], generator=gen, device=dev) < 0.05).float())).to(dtype)


def _quantised(x, dims):
    """q and scale of blocks of values (32 bits), one scale over `dims`."""
    top = x.abs().amax(dims, keepdim=True)
    d = top / torch.full_like(top, 127.0)
    d = torch.where(d < SMALLEST, torch.zeros_like(d), d)
    inv = torch.where(d > 0, 1 / d, torch.zeros_like(d))
    return torch.round(x * inv).to(torch.int8), d


def _descriptors(starts, counts, dev):
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    return {"starts": torch.tensor(starts, dtype=torch.int64, device=dev), "offsets": torch.tensor(offsets, dtype=torch.int32, device=dev),
            "total": offsets[-1], "most": max(counts), "end": max(s + n for s, n in zip(starts, counts))}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab + case["pad"]), generator=gen, device=dev) * 2.5
        x[:, :vocab] += 9 * (torch.rand((rows, vocab), generator=gen, device=dev) < 8 / vocab)  # a few likely tokens
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device=dev, dtype=torch.int32)
        x[::8, : vocab // 3] = -math.inf  # rows under a grammar that allows some tokens only
        return {"case": case, "logits": x.to(dtype)[:, :vocab], "tokens": tokens}
    starts, counts = _plan(case)
    block, hk, hd, seqs = case["block"], case["kv_heads"], case["head_dim"], case["seqs"]
    ends = [s + n for s, n in zip(starts, counts)]
    width = max(-(-e // block) for e in ends)
    pages = sum(-(-e // block) for e in ends)
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    slots = torch.randperm(seqs, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros((seqs, width), dtype=torch.int32, device=dev)
    have = torch.tensor([-(-e // block) for e in ends], device=dev)
    table[slots.long()] = torch.where(torch.arange(width, device=dev) < have[:, None],
                                      order[((have.cumsum(0) - have)[:, None] + torch.arange(width, device=dev)).clamp(max=pages - 1)], torch.zeros_like(table))
    st = {"case": case, "slots": slots, "table": table, "batch": _descriptors(starts, counts, dev)}
    for name in ("k", "v"):
        q = torch.empty((1, pages, hk, block, hd), dtype=torch.int8, device=dev)
        step = max(1, (1 << 26) // (hk * block * hd))
        for i in range(0, pages, step):
            q[0, i:i + step] = (torch.randn(q[0, i:i + step].shape, generator=gen, device=dev) * 32).round_().clamp_(-127, 127).to(torch.int8)
        st[name + "_blocks"] = q
        st[name + "_scales"] = (0.5 + torch.rand((1, pages, hk), generator=gen, device=dev)) / 32
    if case["kind"] == "attend":
        st["q"] = torch.randn((st["batch"]["total"], case["heads"], hd), generator=gen, device=dev).to(dtype)
        return st
    if case["kind"] == "read":
        return st
    # what earlier appends left behind: the open block's rows, in the tail and quantized in its page
    first = torch.tensor([s // block for s in starts], device=dev)
    open_rows = torch.tensor([s % block for s in starts], device=dev)
    page = table[slots.long(), first.clamp(max=width - 1)].long()
    rows = torch.arange(block, device=dev)
    ring = ((first[:, None] % 2) * block + rows)
    for name in ("k", "v"):
        st[name] = _heads((st["batch"]["total"], hk, hd), gen, dtype, dev)
        tail = torch.zeros((1, seqs, hk, 2 * block, hd), dtype=dtype, device=dev)
        old = _heads((seqs, block, hk, hd), gen, dtype, dev) * (rows < open_rows[:, None])[:, :, None, None]
        tail[0][slots.long()[:, None], :, ring] = old
        q, d = _quantised(old.float(), (1, 3))
        st[name + "_blocks"][0][page] = q.transpose(1, 2)
        st[name + "_scales"][0][page] = d[:, 0, :, 0]
        st[name + "_tail"] = tail
        st[name + "_tail_max"] = tail.float().abs().amax(-1)
    # which (sequence, block) pairs the append touches, and which tokens stay in the tail
    touched = [(i, b) for i, (s, n) in enumerate(zip(starts, counts)) for b in range(s // block, (s + n - 1) // block + 1)]
    st["touched"] = torch.tensor(touched, dtype=torch.int64, device=dev).t().contiguous()
    kept, at = [], 0
    for i, (s, n) in enumerate(zip(starts, counts)):
        low = max(s, block * ((s + n - 1) // block - 1))
        kept += [(i, at + p - s, p) for p in range(low, s + n)]
        at += n
    st["kept"] = torch.tensor(kept, dtype=torch.int64, device=dev).t().contiguous()
    # the read back covers the whole blocks that the append touched, up to the last token
    st["back"] = _descriptors([s - s % block for s in starts], [n + s % block for s, n in zip(starts, counts)], dev)
    return st


def _token_places(st, b):
    """(sequence, position) of each token of a batch."""
    offsets = b["offsets"].long()
    seq = torch.repeat_interleave(torch.arange(len(offsets) - 1, device=offsets.device), offsets.diff(), output_size=b["total"])
    return seq, b["starts"][seq] + torch.arange(b["total"], device=offsets.device) - offsets[seq]


def _plain_read(st, b):
    block, dtype = st["case"]["block"], DTYPES[st["case"]["dtype"]]
    seq, pos = _token_places(st, b)
    page = st["table"][st["slots"].long()[seq], pos // block].long()

    def values(q, d):
        return (q[0][page, :, pos % block].float() * d[0][page][:, :, None]).to(dtype)

    return values(st["k_blocks"], st["k_scales"]), values(st["v_blocks"], st["v_scales"])


def _plain_write(st):
    block, b = st["case"]["block"], st["batch"]
    seq, blk = st["touched"]
    slots, offsets = st["slots"].long(), b["offsets"].long()
    rows = torch.arange(block, device=seq.device)
    pos = blk[:, None] * block + rows
    start, end = b["starts"][seq][:, None], (b["starts"] + offsets.diff())[seq][:, None]
    new, old = (pos >= start) & (pos < end), pos < start
    token = (offsets[:-1][seq][:, None] + pos - start).clamp(0, b["total"] - 1)
    page = st["table"][slots[seq], blk].long()
    kseq, ktok, kpos = st["kept"]

    def put(x, q, d, tail, tail_max):
        new_rows = torch.where(new[:, :, None, None], x[token].float(), torch.zeros((), device=x.device))
        old_rows = torch.where(old[:, :, None, None], tail[0][slots[seq][:, None], :, pos % (2 * block)].float(), torch.zeros((), device=x.device))
        q8, s = _quantised(new_rows + old_rows, (1, 3))
        q[0][page] = q8.transpose(1, 2)
        d[0][page] = s[:, 0, :, 0]
        tail[0][slots[kseq], :, kpos % (2 * block)] = x[ktok]
        tail_max[0][slots[kseq], :, kpos % (2 * block)] = x[ktok].float().abs().amax(-1)

    put(st["k"], st["k_blocks"], st["k_scales"], st["k_tail"], st["k_tail_max"])
    put(st["v"], st["v_blocks"], st["v_scales"], st["v_tail"], st["v_tail_max"])
    return _plain_read(st, st["back"])


def _plain_attend(st):
    case, b = st["case"], st["batch"]
    block, hk, hd, group = case["block"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    width = -(-b["end"] // block)
    page = st["table"][st["slots"].long(), :width].long()

    def rows(q, d):  # [sequence][KV head][position][dimension]
        x = q[0][page].float() * d[0][page][:, :, :, None, None]
        return x.transpose(1, 2).reshape(len(page), hk, width * block, hd)

    seq, pos = _token_places(st, b)
    within = torch.arange(b["total"], device=pos.device) - b["offsets"].long()[seq]
    q = torch.zeros((len(page), b["most"], hk, group, hd), device=pos.device)
    q[seq, within] = st["q"].float().reshape(-1, hk, group, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(len(page), hk, group * b["most"], hd)
    s = torch.matmul(q, rows(st["k_blocks"], st["k_scales"]).transpose(2, 3)).mul_(1 / math.sqrt(hd))
    s = s.view(len(page), hk, group, b["most"], width * block)
    key = torch.arange(width * block, device=pos.device)
    at = b["starts"][:, None] + torch.arange(b["most"], device=pos.device)
    seen = key <= at[:, :, None]
    if case["window"]:
        seen &= key > at[:, :, None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(len(page), hk, group * b["most"], width * block), rows(st["v_blocks"], st["v_scales"])).view(len(page), hk, group, b["most"], hd)
    o = (o / total).permute(0, 3, 1, 2, 4)[seq, within].reshape(b["total"], case["heads"], hd)
    return o.to(st["q"].dtype)


def _plain_score(st):
    x, k = st["logits"].float(), st["case"]["top"]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    lse = top + log_total
    mean = torch.where(e > 0, e * (x - top), torch.zeros_like(e)).sum(-1, keepdim=True) / total
    out = {"log_prob": (x.gather(1, st["tokens"].long()[:, None]) - lse)[:, 0], "log_sum_exp": lse[:, 0], "entropy": (log_total - mean)[:, 0]}
    if k:
        # value first, then the lower index: one whole number a token
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = bits * (1 << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
        best = torch.topk(key, k, dim=1).values
        ids = 0xFFFFFFFF - (best & 0xFFFFFFFF)
        out["top_ids"] = ids.to(torch.int32)
        out["top_log_probs"] = x.gather(1, ids) - lse
    return out


def _own_cache(st):
    from auratensor_b200.kvblock import BlockKvCache
    return BlockKvCache.wrap(st["k_blocks"], st["v_blocks"], st["k_scales"], st["v_scales"], st["table"],
                             st.get("k_tail"), st.get("v_tail"), st.get("k_tail_max"), st.get("v_tail_max"), dtype=DTYPES[st["case"]["dtype"]])


def _own_batch(st, b):
    from auratensor_b200.kvblock import TokenBatch
    return TokenBatch(st["slots"], b["starts"], b["offsets"], b["total"], b["most"], b["end"])


def run(state):
    kind = state["case"]["kind"]
    if kind == "score":
        if not own:
            return _plain_score(state)
        from auratensor_b200.scoring import LogProbs
        r = LogProbs.of(state["logits"], state["tokens"], state["case"]["top"])
        out = {"log_prob": r.logProb, "log_sum_exp": r.logSumExp, "entropy": r.entropy}
        if state["case"]["top"]:
            out.update(top_ids=r.topIds, top_log_probs=r.topLogProbs)
        return out
    if kind == "attend":
        return _own_cache(state).attention(0, _own_batch(state, state["batch"]), state["q"], window=state["case"]["window"]) if own else _plain_attend(state)
    if kind == "read":
        k, v = _own_cache(state).read(0, _own_batch(state, state["batch"])) if own else _plain_read(state, state["batch"])
        return {"k": k, "v": v}
    if own:
        cache = _own_cache(state)
        cache.append(0, _own_batch(state, state["batch"]), state["k"], state["v"])
        k, v = cache.read(0, _own_batch(state, state["back"]))
    else:
        k, v = _plain_write(state)
    return {"k": k, "v": v, **{n: state[n] for n in ("k_scales", "v_scales", "k_tail", "v_tail", "k_tail_max", "v_tail_max")}}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits, a sequence at a time."""
    st = prepare(case, seed)
    if case["kind"] == "score":
        x = st["logits"].double()
        p = torch.softmax(x, -1)
        logp = torch.log_softmax(x, -1)
        out = {"log_prob": logp[torch.arange(len(x), device=x.device), st["tokens"].long()], "log_sum_exp": torch.logsumexp(x, -1),
               "entropy": -torch.special.xlogy(p, p).sum(-1)}
        if case["top"]:
            out.update(top_ids=None, top_log_probs=torch.sort(logp, dim=-1, descending=True).values[:, : case["top"]] if case["rows"] * case["vocab"] < 1 << 28
                       else torch.topk(logp, case["top"], dim=-1).values)
        return out
    starts, counts = _plan(case)
    block, hd = case["block"], case["head_dim"]
    slots = st["slots"].tolist()

    def values(name, i, n):  # the first n positions of sequence i: [position][KV head][dimension]
        pages = st["table"][slots[i], : -(-n // block)].long()
        x = st[name + "_blocks"][0][pages].double() * st[name + "_scales"][0][pages].double()[:, :, None, None]
        return x.transpose(1, 2).reshape(-1, case["kv_heads"], hd)[:n]

    if case["kind"] == "read":
        return {n: torch.cat([values(n, i, s + c)[s:] for i, (s, c) in enumerate(zip(starts, counts))]) for n in ("k", "v")}
    if case["kind"] == "attend":
        outs, at = [], 0
        group = case["heads"] // case["kv_heads"]
        for i, (s, c) in enumerate(zip(starts, counts)):
            q = st["q"][at:at + c].double()
            k, v = values("k", i, s + c), values("v", i, s + c)
            place, key = torch.arange(s, s + c, device=q.device)[:, None], torch.arange(s + c, device=q.device)
            hidden = key > place
            if case["window"]:
                hidden = hidden | (key <= place - case["window"])
            heads = []
            for h in range(case["heads"]):
                a = (q[:, h] @ k[:, h // group].T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                heads.append(torch.softmax(a, -1) @ v[:, h // group])
            outs.append(torch.stack(heads, 1))
            at += c
        return torch.cat(outs)
    # written: each touched block from its originals, the scale as it is held (32 bits)
    out = {n: st[n].double() for n in ("k_scales", "v_scales", "k_tail", "v_tail", "k_tail_max", "v_tail_max")}
    for name in ("k", "v"):
        back, at = [], 0
        for i, (s, c) in enumerate(zip(starts, counts)):
            low, slot = s - s % block, slots[i]
            tail, tail_max, scales = out[name + "_tail"][0, slot], out[name + "_tail_max"][0, slot], out[name + "_scales"][0]
            new = st[name][at:at + c].double()
            old = tail[:, [p % (2 * block) for p in range(low, s)]].transpose(0, 1)
            x = torch.cat([old, new])
            for j in range(0, len(x), block):
                part = x[j:j + block]
                d = (part.abs().amax((0, 2)) / 127).float().double()
                d[d < SMALLEST] = 0
                scales[st["table"][slot, (low + j) // block]] = d
                back.append(torch.round(part / torch.where(d > 0, d, 1.0)[:, None]) * d[:, None])
            keep = min(c, s + c - max(s, block * ((s + c - 1) // block - 1)))
            ring = [p % (2 * block) for p in range(s + c - keep, s + c)]
            tail[:, ring] = new[c - keep:].transpose(0, 1)
            tail_max[:, ring] = new[c - keep:].abs().amax(-1).T
            at += c
        out[name] = torch.cat(back)
    return {n: out[n] for n in ("k", "v", "k_scales", "v_scales", "k_tail", "v_tail", "k_tail_max", "v_tail_max")}

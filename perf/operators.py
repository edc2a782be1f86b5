"""Operators for serving many sequences over one paged cache, as cases that can be timed and checked: block tables and slot
maps, the write of new keys and values, attention of new tokens, probabilities of logits, verification of drafted tokens.

Sequence lengths follow from the case alone (spread evenly over its range), everything else from the seed: which pages a
sequence holds, queries, keys, values, logits and the random numbers of the verification.  Token ids, positions, slots and
pages are 32-bit words in int32 tensors; -1 is "no slot" / "no page" / "no token".
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1000000.0


# ---------------------------------------------------------------------------------------------- cases

def _plan(name, sequences, cached, drafts, chunks, chunk, page, spare):
    return dict(name=name, op="plan", sequences=sequences, cached_lo=cached[0], cached_hi=cached[1], drafts=drafts, chunks=chunks, chunk=chunk, page=page,
                spare=spare)


def _append(name, rows, heads, kv_heads, head_dim, page, dtype, far):
    return dict(name=name, op="append", rows=rows, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, far=far)


def _attend(name, sequences, fresh, cached, heads, kv_heads, head_dim, page, dtype, window=0):
    return dict(name=name, op="attend", sequences=sequences, fresh_lo=fresh[0], fresh_hi=fresh[1], cached_lo=cached[0], cached_hi=cached[1], heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, window=window)


def _probs(name, rows, vocab, greedy):
    return dict(name=name, op="probs", rows=rows, vocab=vocab, greedy=greedy)


def _verify(name, sequences, drafts, vocab, sampled):
    return dict(name=name, op="verify", sequences=sequences, drafts=drafts, vocab=vocab, sampled=sampled)


def listed():
    return [
        # one token for each of eight chats, and the step taken back: the smallest bookkeeping, latency only
        _plan("plan 8x1", 8, (10, 2000), 0, 0, 0, 16, 64),
        # a loaded server: 496 sequences with four drafted tokens each, 16 with a portion of their prompt
        _plan("plan 512 mixed", 512, (0, 8000), 4, 16, 512, 64, 1024),
        # the keys and values of eight decoded tokens of the SmolLM2-135M shape, all f32: latency
        _append("append 8 f32", 8, 9, 3, 64, 16, "f32", 2000),
        # a portion of 4096 prompt tokens of the Qwen3-8B attention shape into a bf16 cache, far positions
        _append("append 4096 bf16", 4096, 32, 8, 128, 64, "bf16", 120000),
        # four short chats of the SmolLM2-135M shape, a token each, all f32 as its decode step is: the smallest attention
        _attend("attend 4x1 f32", 4, (1, 1), (20, 500), 9, 3, 64, 16, "f32"),
        # 64 chats of very different lengths decoded together, Qwen3-8B shape: reads the cache once
        _attend("attend 64x1 bf16", 64, (1, 1), (100, 8100), 32, 8, 128, 64, "bf16"),
        # 32 sequences with up to four drafted tokens to verify, f16 cache as Tobovik's, small pages
        _attend("attend 32x5 f16", 32, (1, 5), (900, 4000), 32, 8, 128, 16, "f16"),
        # portions of 2048 prompt tokens of four requests, behind what is cached of them: the largest, compute
        _attend("attend 4x2048 bf16", 4, (2048, 2048), (0, 6144), 32, 8, 128, 64, "bf16"),
        # the next token's distribution of four chats, vocabulary of the design benchmarks
        _probs("probs 4x32768", 4, 32768, 1),
        # five rows (one token, four drafts) for each of 64 chats, vocabulary of Qwen3-8B
        _probs("probs 320x151936", 320, 151936, 0),
        # four chats with four drafts each, drafts taken greedily (no distribution of their own)
        _verify("verify 4x4 32768", 4, 4, 32768, False),
        # 64 chats with four drafts each that were drawn from a drafting model's distribution
        _verify("verify 64x4 151936", 64, 4, 151936, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "probs", "verify"])
    if op == "plan":
        s = _log(rng, 1, 512)
        return _drawn(_plan("", s, (0, _log(rng, 20, 8000)), rng.randint(0, 8), rng.randint(0, min(s, 16)), _log(rng, 16, 512), rng.choice([8, 16, 32, 64, 128]),
                            rng.choice([0, s // 2, 4 * s, 1024])))
    if op == "append":
        heads, kv_heads, d = rng.choice([(9, 3, 64), (32, 8, 128), (16, 4, 128), (12, 12, 80), (8, 1, 256)])
        return _drawn(_append("", _log(rng, 1, 4096), heads, kv_heads, d, rng.choice([8, 16, 32, 64, 128]), rng.choice(["f32", "f16", "bf16"]), _log(rng, 10, 200000)))
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        heads, kv_heads, d = rng.choice([(9, 3, 64), (32, 8, 128), (16, 4, 128), (12, 12, 80), (8, 1, 128), (14, 2, 64)])
        page, window = rng.choice([8, 16, 32, 64, 128]), rng.choice([0, 0, 0, _log(rng, 16, 2048)])
        kind = rng.choice(["decode", "decode", "drafts", "chunk", "chunk"])
        if kind == "decode":
            return _drawn(_attend("", _log(rng, 1, 64), (1, 1), (rng.randint(0, 50), _log(rng, 60, 8000)), heads, kv_heads, d, page, dtype, window))
        if kind == "drafts":
            return _drawn(_attend("", _log(rng, 1, 48), (rng.randint(0, 1), rng.randint(2, 9)), (rng.randint(0, 50), _log(rng, 60, 4000)), heads, kv_heads, d, page, dtype,
                                  window))
        most = 2000 if dtype != "f32" else 400
        return _drawn(_attend("", rng.randint(1, 4), (rng.randint(0, 40), _log(rng, 41, most)), (0, _log(rng, 20, 6000 if dtype != "f32" else 1500)), heads, kv_heads, d, page,
                              dtype, window))
    if op == "probs":
        return _drawn(_probs("", _log(rng, 1, 320), rng.choice([_log(rng, 1000, 151936), 32768, 49152, 151936]), rng.randint(0, 2)))
    return _drawn(_verify("", _log(rng, 1, 64), rng.randint(0, 8), rng.choice([_log(rng, 1000, 120000), 32768, 49152]), rng.random() < 0.7))


def _drawn(case):
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- lengths

def _spread(lo, hi, n, stride):
    """n whole numbers from lo to hi, evenly spread, in a mixed order; one alone is hi."""
    return [lo + (hi - lo) * ((i * stride) % n) // (n - 1) for i in range(n)] if n > 1 else [hi]


def _lengths(case):
    """(tokens in the cache, new tokens) of each sequence: what the case says, not the seed."""
    s = case["sequences"]
    cached = _spread(case["cached_lo"], case["cached_hi"], s, 37 if s % 37 else 41)
    if case["op"] == "plan":
        return cached, [case["chunk"] if i % max(1, s // max(1, case["chunks"])) == 0 and i // max(1, s // max(1, case["chunks"])) < case["chunks"] else
                        1 + case["drafts"] for i in range(s)]
    return cached, _spread(case["fresh_lo"], case["fresh_hi"], s, 29 if s % 29 else 31)


def _pages(tokens, page):
    return -(-tokens // page)


def _visible(case):
    """Keys that the rows of each sequence see together, and keys that have to be read for it."""
    pairs, keys, w = 0, 0, case["window"]
    for c, n in zip(*_lengths(case)):
        at = np.arange(c, c + n, dtype=np.int64) + 1
        pairs += int((np.minimum(at, w) if w else at).sum())
        keys += c + n - (max(0, c + 1 - w) if w else 0) if n else 0
    return pairs, keys


def work(case):
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        new = sum(_pages(c + n, case["page"]) - _pages(c, case["page"]) for c, n in zip(cached, fresh))
        # the plan reads cached, fresh, held and writes starts, lengths, held; table entries, free pages; positions and slots; then the way back
        return {"bytes": 4 * (9 * case["sequences"] + 6 * new + 2 * sum(fresh)), "flops": 10 * sum(fresh)}
    if op == "append":
        row = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": case["rows"] * (row * (4 + BYTES[case["dtype"]]) + 8), "flops": 3 * case["rows"] * row}
    if op == "attend":
        pairs, keys = _visible(case)
        rows, b, d = sum(_lengths(case)[1]), BYTES[case["dtype"]], case["head_dim"]
        return {"bytes": b * d * (2 * rows * case["heads"] + 2 * keys * case["kv_heads"]), "flops": 4 * d * case["heads"] * pairs}
    if op == "probs":
        return {"bytes": 8 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    return {"bytes": case["sequences"] * case["vocab"] * (8 if case["sampled"] else 4), "flops": 3 * case["sequences"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape, dtype=torch.float32, gain=1.0):
    return torch.randn(*shape, device="cuda", generator=g).mul_(gain).to(dtype)


def _tables(g, tokens, page, pages, width):
    """A table that holds the pages of `tokens` tokens of each sequence, taken from a shuffled pool, and the rest of the pool."""
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    held = _words([_pages(t, page) for t in tokens])
    first = torch.cumsum(held, 0) - held
    j = torch.arange(width, device="cuda")
    table = torch.where(j < held[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], -1).to(torch.int32)
    used = int(held.sum())
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[:pages - used] = order[used:]
    return table, held, free, pages - used


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        held = sum(_pages(c, case["page"]) for c in cached)
        pages, width = max(1, held + case["spare"]), max(_pages(c + n, case["page"]) for c, n in zip(cached, fresh))
        table, held, free, left = _tables(g, cached, case["page"], pages, width)
        rows, s = sum(fresh), case["sequences"]
        out = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (s + 1, s, rows, rows, 1)]
        return dict(case=case, cached=_words(cached), fresh=_words(fresh), table=table, held=held, free=free, count=_words([left]), rows=rows, out=out)
    if op == "append":
        rows, h, kv, d, page, t = (case[x] for x in ("rows", "heads", "kv_heads", "head_dim", "page", "dtype"))
        pages = 2 * _pages(rows, page) + 1
        # rows of one projection's output, as the fused q|k|v product leaves them
        qkv = _normal(g, rows, (h + 2 * kv) * d)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], 1))
        start = int(torch.randint(0, max(1, case["far"] - rows), (1,), device="cuda", generator=g))
        slots = torch.randperm(pages, device="cuda", generator=g)[:_pages(rows, page)].repeat_interleave(page)[:rows] * page
        slots = (slots + torch.arange(rows, device="cuda") % page).to(torch.int32)
        caches = [_normal(g, pages, page, kv, d, dtype=TYPES[t]) for _ in range(2)]
        return dict(case=case, q=q, k=k, v=v, positions=torch.arange(start, start + rows, dtype=torch.int32, device="cuda"), slots=slots, k_cache=caches[0],
                    v_cache=caches[1], q_out=torch.empty(rows, h, d, dtype=TYPES[t], device="cuda"))
    if op == "attend":
        h, kv, d, page, t = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "dtype"))
        cached, fresh = _lengths(case)
        total = [c + n for c, n in zip(cached, fresh)]
        pages = sum(_pages(n, page) for n in total) + 7
        table = _tables(g, total, page, pages, max(1, max(_pages(n, page) for n in total)))[0]
        rows = max(1, sum(fresh))
        caches = [_normal(g, pages, page, kv, d, dtype=TYPES[t]) for _ in range(2)]
        # queries as peaked as a trained model's: scores with a deviation of 2
        return dict(case=case, q=_normal(g, rows, h, d, dtype=TYPES[t], gain=2.0), k_cache=caches[0], v_cache=caches[1], table=table,
                    starts=_words([0] + list(np.cumsum(fresh))), lengths=_words(total), most=max(1, max(fresh)), keys=max(1, max(total)),
                    out=torch.zeros(rows, h, d, dtype=TYPES[t], device="cuda"))
    if op == "probs":
        rows, v = case["rows"], case["vocab"]
        t = 0.5 + torch.rand(rows, device="cuda", generator=g)
        t[:min(rows, case["greedy"])] = 0.0
        return dict(case=case, logits=_normal(g, rows, v, gain=3.0), temperature=t, out=torch.empty(rows, v, device="cuda"))
    s, n, v = case["sequences"], case["drafts"] + 1, case["vocab"]
    logits = _normal(g, s * n, v, gain=3.0)
    target = torch.softmax(logits, 1)
    draft = torch.softmax(logits.add_(_normal(g, s * n, v, gain=0.7)), 1) if case["sampled"] else None
    noise = torch.rand(s * n, v, device="cuda", generator=g).clamp_(min=1e-20).log_().neg_()
    tokens = ((draft if case["sampled"] else target) / noise).argmax(1).to(torch.int32).roll(1)      # row i's draft is fed as row i + 1
    u = torch.rand(s * n, device="cuda", generator=g)
    out = [torch.empty(k, dtype=torch.int32, device="cuda") for k in (s, s, s * n)]
    return dict(case=case, target=target, draft=draft, tokens=tokens, starts=_words(range(0, s * n + 1, n)), accept=u, sample=torch.rand(s, device="cuda", generator=g),
                out=out)


# ---------------------------------------------------------------------------------------------- the operators, plain

def _plain_plan(s):
    """A step's pages, rows and slots, then the step taken back: its pages return to the pool in the order they came."""
    page, table, held, free, count, rows = s["case"]["page"], s["table"], s["held"].long(), s["free"], s["count"].long(), s["rows"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    need = ((cached + fresh + page - 1) // page - held).clamp(min=0)
    running = need.cumsum(0)
    served = (need == 0) | (running <= count)
    lacking = (running[-1:] - count).clamp(min=0)
    got = torch.where(served, need, 0)
    before = got.cumsum(0) - got
    j = torch.arange(table.shape[1], device="cuda")
    new = (j >= held[:, None]) & (j < (held + got)[:, None])
    table.copy_(torch.where(new, free[(count - 1 - before[:, None] - (j - held[:, None])).clamp(0, free.shape[0] - 1)], table))
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), fresh.cumsum(0)])
    row = torch.arange(rows, device="cuda")
    of = torch.searchsorted(starts[1:], row, right=True)
    position = cached[of] + row - starts[of]
    slots = torch.where(served[of], table[of, (position // page).clamp(max=table.shape[1] - 1)].long() * page + position % page, -1)
    lengths = torch.where(served, cached + fresh, cached)
    # back: what lies behind the cached tokens
    held, count, keep = held + got, count - got.sum(), (cached + page - 1) // page
    gone = (held - keep).clamp(min=0)
    last = gone.cumsum(0)
    give = (j >= keep[:, None]) & (j < held[:, None])
    place = count + last[-1] - 1 - (last - gone)[:, None] - (j - keep[:, None])
    room = torch.cat([free, free.new_zeros(1)])
    room[torch.where(give, place, free.shape[0])] = table
    free.copy_(room[:-1])
    table.masked_fill_(give, -1)
    s["held"].copy_(held - gone)
    s["count"].copy_(count + last[-1:])
    return tuple(x.to(torch.int32) for x in (starts, lengths, position, slots, lacking)) + (table, s["held"], free, s["count"])


def _rotated(x, positions):
    half = x.shape[2] // 2
    angle = positions.double()[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * n, a * n + b * c], 2)


def _plain_append(s):
    k, v, t = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1), s["k_cache"].dtype
    at = s["slots"].long()
    k[at] = _rotated(s["k"], s["positions"]).to(t)
    v[at] = s["v"].to(t)
    return _rotated(s["q"], s["positions"]).to(t), s["k_cache"], s["v_cache"]


def _plain_attend(s):
    case, q, t = s["case"], s["q"], s["q"].dtype
    page, d, kv, most, keys = case["page"], case["head_dim"], case["kv_heads"], s["most"], s["keys"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    fresh = starts[1:] - starts[:-1]
    j = torch.arange(keys, device="cuda")
    slot = s["table"].long().clamp(min=0)[:, j // page] * page + j % page                             # [S, keys]
    k, v = (s[x].flatten(0, 1)[slot].float() for x in ("k_cache", "v_cache"))
    i = torch.arange(most, device="cuda")
    live = i < fresh[:, None]
    row = torch.where(live, starts[:-1, None] + i, 0)                                                 # [S, most]
    x = q[row].float().unflatten(2, (kv, -1))                                                         # [S, most, kv, g, d]
    score = torch.einsum("snkgd,slkd->skgnl", x, k).mul_(d ** -0.5)
    at = (lengths - fresh)[:, None] + i
    seen = j <= at[..., None]
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -torch.inf)
    w = (score - score.amax(-1, keepdim=True)).exp_()
    y = torch.einsum("skgnl,slkd->snkgd", w, v) / w.sum(-1).permute(0, 3, 1, 2)[..., None]
    out = torch.zeros(q.shape[0] + 1, *q.shape[1:], dtype=t, device="cuda")
    out[torch.where(live, row, q.shape[0])] = y.flatten(2, 3).to(t)
    return out[:-1]


def _plain_probs(s):
    l, t = s["logits"], s["temperature"][:, None]
    e = ((l - l.amax(1, keepdim=True)) / t).exp()
    one = torch.arange(l.shape[1], device="cuda") == l.argmax(1, keepdim=True)
    return torch.where(t > 0, e / e.sum(1, keepdim=True), one.float())


def _plain_verify(s):
    p, q, tokens, starts = s["target"], s["draft"], s["tokens"].long(), s["starts"].long()
    n, k = s["case"]["drafts"] + 1, s["case"]["drafts"]
    row = starts[:-1, None] + torch.arange(n, device="cuda")                                          # [S, n]
    d = tokens[row[:, 1:]]
    pd = p[row[:, :k], d].double()
    qd = q[row[:, :k], d].double() if q is not None else torch.ones_like(pd)
    good = s["accept"][row[:, :k]].double() * qd < pd
    accepted = good.long().cumprod(1).sum(1)
    last = starts[:-1] + accepted
    w = p[last].double()
    drop = (accepted < k)[:, None]
    if q is not None:
        rest = (w - q[last].double()).clamp_(min=0)
    else:
        rest = w.clone()
        rest.scatter_(1, tokens[(last + 1).clamp(max=tokens.shape[0] - 1)][:, None], 0)
    w = torch.where(drop & (rest.sum(1, keepdim=True) > 0), rest, w)
    c = w.cumsum(1)
    pick = torch.searchsorted(c, s["sample"].double()[:, None] * c[:, -1:], right=True)[:, 0]
    top = w.shape[1] - 1 - (w > 0).flip(1).int().argmax(1)
    pick = torch.minimum(pick, top)
    i = torch.arange(n, device="cuda")
    fed = torch.cat([d, d.new_zeros(d.shape[0], 1)], 1)
    out = torch.where(i < accepted[:, None], fed, torch.where(i == accepted[:, None], pick[:, None], -1))
    return accepted.int(), pick.int(), out.flatten().int()


PLAIN = {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend, "probs": _plain_probs, "verify": _plain_verify}


# ---------------------------------------------------------------------------------------------- the operators, the framework's

def _own(s):
    from meganeura_b200 import ops
    op = s["case"]["op"]
    if op == "plan":
        step = ops.PagedStep(*s["out"])
        ops.paged_plan(s["cached"], s["fresh"], s["table"], s["held"], s["free"], s["count"], s["case"]["page"], s["rows"], step=step)
        ops.paged_trim(s["cached"], s["table"], s["held"], s["free"], s["count"], s["case"]["page"])
        return tuple(step) + (s["table"], s["held"], s["free"], s["count"])
    if op == "append":
        return ops.paged_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], theta=THETA, q_out=s["q_out"]), s["k_cache"], s["v_cache"]
    if op == "attend":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], s["most"], window=s["case"]["window"], out=s["out"])
    if op == "probs":
        return ops.token_probs(s["logits"], s["temperature"], out=s["out"])
    return ops.verify_drafts(s["target"], s["draft"], s["tokens"], s["starts"], s["accept"], s["sample"], out=s["out"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits

def _exact_plan(s):
    page, rows, s0 = s["case"]["page"], s["rows"], {k: s[k].cpu().numpy().astype(np.int64) for k in ("cached", "fresh", "table", "held", "free", "count")}
    table, held, pool = s0["table"], s0["held"], list(s0["free"][:s0["count"][0]])
    starts, lengths, positions, slots, wanted = [0], [], [], [], 0
    pages = len(pool)
    for i, (c, n) in enumerate(zip(s0["cached"], s0["fresh"])):
        need = max(0, _pages(c + n, page) - held[i])
        wanted += need
        fine = need == 0 or wanted <= pages
        if fine:
            for _ in range(need):
                table[i, held[i]] = pool.pop()
                held[i] += 1
        for at in range(c, c + n):
            positions.append(at)
            slots.append(table[i, at // page] * page + at % page if fine else -1)
        starts.append(starts[-1] + n)
        lengths.append(c + n if fine else c)
    back = []
    for i, c in enumerate(s0["cached"]):
        keep = _pages(c, page)
        back += [int(x) for x in table[i, keep:held[i]]]
        table[i, keep:held[i]] = -1
        held[i] = min(held[i], keep)
    free = s0["free"].copy()
    pool += back[::-1]
    free[:len(pool)] = pool
    assert len(slots) == rows
    return tuple(np.array(x, np.int32) for x in (starts, lengths, positions, slots, [max(0, wanted - pages)], table, held, free, [len(pool)]))


def _exact_rotate(x, positions):
    x, d = x.double(), x.shape[-1]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] / THETA ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_append(s):
    k, v = s["k_cache"].double(), s["v_cache"].double()
    page = k.shape[1]
    at = s["slots"].long()
    k[at // page, at % page] = _exact_rotate(s["k"], s["positions"])
    v[at // page, at % page] = s["v"].double()
    return _exact_rotate(s["q"], s["positions"]), k, v


def _exact_attend(s):
    case = s["case"]
    g, out = case["heads"] // case["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (c, n) in enumerate(zip(*_lengths(case))):
        if n == 0:
            continue
        pages = s["table"][i, :_pages(c + n, case["page"])].long()
        k, v = (s[x][pages].flatten(0, 1)[:c + n].double() for x in ("k_cache", "v_cache"))
        q = s["q"][first:first + n].double()
        ahead = torch.arange(c + n, device="cuda")[None] - torch.arange(c, c + n, device="cuda")[:, None]
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        for h in range(case["heads"]):
            score = (q[:, h] @ k[:, h // g].T / math.sqrt(case["head_dim"])).masked_fill(hidden, -math.inf)
            out[first:first + n, h] = torch.softmax(score, 1) @ v[:, h // g]
        first += n
    return out


def _exact_probs(s):
    out = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i, t in enumerate(s["temperature"].tolist()):
        row = s["logits"][i].double()
        if t > 0:
            out[i] = torch.softmax(row / t, 0)
        else:
            out[i, int((row == row.max()).nonzero()[0, 0])] = 1
    return out


def _exact_verify(s):
    starts, n = s["starts"].tolist(), s["case"]["drafts"] + 1
    tokens, accept, sample = s["tokens"].tolist(), s["accept"].double().tolist(), s["sample"].double().tolist()
    counts, picks, outs = [], [], []
    for i, u in enumerate(sample):
        kept = []
        while len(kept) < n - 1:
            row, d = starts[i] + len(kept), tokens[starts[i] + len(kept) + 1]
            if not accept[row] * (float(s["draft"][row, d]) if s["draft"] is not None else 1.0) < float(s["target"][row, d]):
                break
            kept.append(d)
        row = starts[i] + len(kept)
        w = whole = s["target"][row].double().cpu().numpy()
        if len(kept) < n - 1:
            if s["draft"] is not None:
                w = np.maximum(w - s["draft"][row].double().cpu().numpy(), 0)
            else:
                w = w.copy()
                w[tokens[row + 1]] = 0
            w = w if w.any() else whole
        c = np.cumsum(w)
        pick = min(int(np.count_nonzero(c <= u * c[-1])), int(np.flatnonzero(w)[-1]))
        counts.append(len(kept))
        picks.append(pick)
        outs += kept + [pick] + [-1] * (n - 1 - len(kept))
    return tuple(np.array(x, np.int32) for x in (counts, picks, outs))


EXACT = {"plan": _exact_plan, "append": _exact_append, "attend": _exact_attend, "probs": _exact_probs, "verify": _exact_verify}


def exact(case, seed):
    state = prepare(case, seed)
    return EXACT[case["op"]](state)

"""Operators for serving with 8-bit integers, as cases that can be timed and checked: rows of activations (or of weights) quantized with a
scale each, products of such rows, new keys and values into a paged cache of 8-bit codes with a scale for each block of tokens and head, and
attention over such a cache.

Lengths and sizes follow from the case alone, everything else from the seed.  Positions, slots and pages are 32-bit words in int32 tensors; -1 is "no slot" /
"no page".  Codes are returned as the values that they stand for, in a type of 16 bits: a value next to the border of two codes may have either, as the
scale's last bit has it.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1000000.0
LEAST = 2.0 ** -100                 # rows and blocks whose largest value is below are zeros


# ---------------------------------------------------------------------------------------------- cases

def _quantize(name, rows, k, dtype):
    return dict(name=name, op="quantize", rows=rows, k=k, dtype=dtype)


def _linear(name, rows, k, n, dtype, addend=False):
    return dict(name=name, op="linear", rows=rows, k=k, n=n, dtype=dtype, addend=addend)


def _append(name, sequences, fresh, cached, heads, kv_heads, head_dim, page, block, src, dtype, pad=0):
    return dict(name=name, op="append", sequences=sequences, fresh_lo=fresh[0], fresh_hi=fresh[1], cached_lo=cached[0], cached_hi=cached[1], heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, block=block, src=src, dtype=dtype, pad=pad)


def _attend(name, sequences, fresh, cached, heads, kv_heads, head_dim, page, block, dtype, window=0):
    return dict(name=name, op="attend", sequences=sequences, fresh_lo=fresh[0], fresh_hi=fresh[1], cached_lo=cached[0], cached_hi=cached[1], heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, block=block, dtype=dtype, window=window)


def listed():
    return [
        # the activations of eight chats in front of a projection of width 4096: latency
        _quantize("quantize 8x4096", 8, 4096, "bf16"),
        # a prompt portion's activations in front of the down projection of a model of width 4096
        _quantize("quantize 2048x12288", 2048, 12288, "bf16"),
        # one token through the gate projection of the SmolLM2-135M shape, all f32 as its decode step is
        _linear("linear 1x576x1536", 1, 576, 1536, "f32"),
        # eight chats decoded together, gate and up projection of the Qwen3-8B shape: the weights are read once
        _linear("linear 8x4096x24576", 8, 4096, 24576, "bf16"),
        # an odd portion of a prompt and an odd number of columns, with the residual stream
        _linear("linear 203x1536x4100", 203, 1536, 4100, "f16", True),
        # a prompt portion through the up projection of a model of width 4096: the largest product
        _linear("linear 2048x4096x12288", 2048, 4096, 12288, "bf16"),
        # the keys and values of eight decoded tokens of the SmolLM2-135M shape in the middle of their blocks: latency
        _append("append 8x1", 8, (1, 1), (20, 2000), 9, 3, 64, 16, 16, "f32", "f16"),
        # portions of eight prompts of the Qwen3-8B shape, and rows that a step padded
        _append("append 8x512", 8, (480, 544), (0, 30000), 32, 8, 128, 64, 64, "bf16", "bf16", 17),
        # four short chats of the SmolLM2-135M shape, a token each: the smallest attention
        _attend("attend 4x1", 4, (1, 1), (20, 500), 9, 3, 64, 16, 16, "f16"),
        # 64 chats of very different lengths decoded together, Qwen3-8B shape: reads the cache once
        _attend("attend 64x1", 64, (1, 1), (100, 8100), 32, 8, 128, 64, 64, "bf16"),
        # 32 sequences with up to four drafted tokens to verify, small pages
        _attend("attend 32x5", 32, (1, 5), (900, 4000), 32, 8, 128, 16, 16, "f16"),
        # portions of 2048 prompt tokens of four requests, behind what is cached of them: the largest, compute
        _attend("attend 4x2048", 4, (2048, 2048), (0, 6144), 32, 8, 128, 64, 32, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "append", "append", "attend", "attend", "attend"])
    if op == "quantize":
        return _drawn(_quantize("", _log(rng, 1, 4096), _log(rng, 16, 12288), rng.choice(["f32", "f16", "bf16"])))
    if op == "linear":
        rows, k = _log(rng, 1, 2048), 16 * _log(rng, 4, 768)
        return _drawn(_linear("", rows, k, min(_log(rng, 16, 24576), 2048 * 4096 * 12288 // (rows * k)), rng.choice(["f32", "f16", "bf16", "bf16"]), rng.random() < 0.3))
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    if op == "append":
        heads, kv_heads, d = rng.choice([(9, 3, 64), (32, 8, 128), (16, 4, 128), (12, 12, 80), (8, 1, 256)])
        dtype = rng.choice(["f16", "bf16"])
        most = _log(rng, 1, 512)
        return _drawn(_append("", _log(rng, 1, 4096 // max(64, most)), (rng.randint(0, most), most), (rng.randint(0, 50), _log(rng, 60, 30000)), heads, kv_heads, d, page, block,
                              rng.choice(["f32", dtype]), dtype, rng.choice([0, rng.randint(1, 40)])))
    dtype = rng.choice(["f16", "bf16"])
    heads, kv_heads, d = rng.choice([(9, 3, 64), (32, 8, 128), (16, 4, 128), (12, 12, 80), (8, 1, 128), (14, 2, 64)])
    window = rng.choice([0, 0, 0, _log(rng, 16, 2048)])
    kind = rng.choice(["decode", "decode", "drafts", "chunk", "chunk"])
    if kind == "decode":
        return _drawn(_attend("", _log(rng, 1, 64), (1, 1), (rng.randint(0, 50), _log(rng, 60, 8000)), heads, kv_heads, d, page, block, dtype, window))
    if kind == "drafts":
        return _drawn(_attend("", _log(rng, 1, 48), (rng.randint(0, 1), rng.randint(2, 9)), (rng.randint(0, 50), _log(rng, 60, 4000)), heads, kv_heads, d, page, block, dtype,
                              window))
    return _drawn(_attend("", rng.randint(1, 4), (rng.randint(0, 40), _log(rng, 41, 2000)), (0, _log(rng, 20, 6000)), heads, kv_heads, d, page, block, dtype, window))


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
    return _spread(case["cached_lo"], case["cached_hi"], s, 37 if s % 37 else 41), _spread(case["fresh_lo"], case["fresh_hi"], s, 29 if s % 29 else 31)


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
    if op == "quantize":
        return {"bytes": case["rows"] * (case["k"] * (BYTES[case["dtype"]] + 1) + 4), "flops": 3 * case["rows"] * case["k"]}
    if op == "linear":
        m, k, n, b = case["rows"], case["k"], case["n"], BYTES[case["dtype"]]
        return {"bytes": m * k * b + n * k + 4 * n + m * n * b * (2 if case["addend"] else 1), "flops": 2 * m * n * k}
    if op == "append":
        cached, fresh = _lengths(case)
        rows, d, kv, b = sum(fresh), case["head_dim"], case["kv_heads"], case["block"]
        blocks = sum(_pages(c + n, b) - c // b for c, n in zip(cached, fresh) if n)
        # rows read and written, a scale per block and head each way
        return {"bytes": rows * d * ((case["heads"] + 2 * kv) * BYTES[case["src"]] + case["heads"] * BYTES[case["dtype"]] + 2 * kv) + 8 * rows + 16 * blocks * kv,
                "flops": 6 * rows * d * (case["heads"] + 2 * kv)}
    pairs, keys = _visible(case)
    rows, d = sum(_lengths(case)[1]), case["head_dim"]
    return {"bytes": 2 * d * 2 * rows * case["heads"] + 2 * keys * case["kv_heads"] * d + 8 * (keys // case["block"]) * case["kv_heads"], "flops": 4 * d * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape, dtype=torch.float32, gain=1.0):
    return torch.randn(*shape, device="cuda", generator=g).mul_(gain).to(dtype)


def _table(g, tokens, page, pages, width):
    """A table that holds the pages of `tokens` tokens of each sequence, taken from a shuffled pool."""
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    held = _words([_pages(t, page) for t in tokens])
    first = torch.cumsum(held, 0) - held
    j = torch.arange(width, device="cuda")
    return torch.where(j < held[:, None], order[(first[:, None] + j).clamp(max=pages - 1)], -1).to(torch.int32)


def _activations(g, rows, k, dtype):
    """Rows as a model's hidden states are: rows of different size, a few channels far larger than the others."""
    x = _normal(g, rows, k)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 10.0, 1.0)
    return x.to(dtype)


def _codes(g, pages, page, block, kv_heads, d):
    """A cache's codes and scales as normal keys of a deviation of about 1 leave them: the largest of a block is 127 or so."""
    codes = torch.empty(pages, page, kv_heads, d, dtype=torch.int8, device="cuda")
    for part in codes.split(max(1, (1 << 27) // (page * kv_heads * d))):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g).mul_(127 / 3.7).round_().clamp_(-127, 127))
    scales = torch.exp(0.1 * torch.randn(pages, page // block, kv_heads, device="cuda", generator=g)) * (3.7 / 127)
    return codes, scales


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    if op == "quantize":
        return dict(case=case, x=_activations(g, case["rows"], case["k"], TYPES[case["dtype"]]),
                    codes=torch.empty(case["rows"], case["k"], dtype=torch.int8, device="cuda"), scales=torch.empty(case["rows"], device="cuda"),
                    values=torch.empty(case["rows"], case["k"], dtype=torch.bfloat16 if case["dtype"] == "bf16" else torch.float16, device="cuda"))
    if op == "linear":
        m, k, n, t = case["rows"], case["k"], case["n"], TYPES[case["dtype"]]
        w = torch.randn(n, k, device="cuda", generator=g).mul_(0.02)
        w_scales = w.abs().amax(1) / 127
        return dict(case=case, x=_activations(g, m, k, t), w=(w / w_scales[:, None]).round_().clamp_(-127, 127).to(torch.int8), w_scales=w_scales,
                    addend=_normal(g, m, n, dtype=t) if case["addend"] else None, codes=torch.empty(m, k, dtype=torch.int8, device="cuda"),
                    scales=torch.empty(m, device="cuda"), out=torch.empty(m, n, dtype=t, device="cuda"))
    h, kv, d, page, block, t = (case[x] for x in ("heads", "kv_heads", "head_dim", "page", "block", "dtype"))
    cached, fresh = _lengths(case)
    total = [c + n for c, n in zip(cached, fresh)]
    if op == "append":
        # the pages of the step alone: those in front of a sequence's first new token are not touched
        gone = [c // page * page for c in cached]
        pages = sum(_pages(n - z, page) for n, z in zip(total, gone)) + 2
        width = max(1, max(_pages(n - z, page) for n, z in zip(total, gone)))
        table = _table(g, [n - z for n, z in zip(total, gone)], page, pages, width)
        rows = sum(fresh) + case["pad"]
        of = torch.repeat_interleave(torch.arange(len(fresh), device="cuda"), _words(fresh).long())
        first = torch.cumsum(_words(fresh), 0) - _words(fresh)
        at = torch.arange(sum(fresh), device="cuda") - first[of]
        local = _words([c - z for c, z in zip(cached, gone)])[of] + at
        slots = torch.full((max(1, rows),), -1, dtype=torch.int32, device="cuda")
        slots[:sum(fresh)] = (table[of, local // page].long() * page + local % page).to(torch.int32)
        positions = torch.zeros(max(1, rows), dtype=torch.int32, device="cuda")
        positions[:sum(fresh)] = (_words(cached)[of] + at).to(torch.int32)
        rows = max(1, rows)
        # rows of one projection's output, as the fused q|k|v product leaves them
        qkv = _normal(g, rows, (h + 2 * kv) * d, dtype=TYPES[case["src"]])
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kv * d, kv * d], 1))
        k_cache, k_scales = _codes(g, pages, page, block, kv, d)
        v_cache, v_scales = _codes(g, pages, page, block, kv, d)
        return dict(case=case, q=q, k=k, v=v, positions=positions, slots=slots, k_cache=k_cache, v_cache=v_cache, k_scales=k_scales, v_scales=v_scales,
                    q_out=torch.empty(rows, h, d, dtype=TYPES[t], device="cuda"), values=torch.empty(2, pages, page // block, block, kv, d, dtype=TYPES[t], device="cuda"))
    pages = sum(_pages(n, page) for n in total) + 7
    table = _table(g, total, page, pages, max(1, max(_pages(n, page) for n in total)))
    rows = max(1, sum(fresh))
    k_cache, k_scales = _codes(g, pages, page, block, kv, d)
    v_cache, v_scales = _codes(g, pages, page, block, kv, d)
    # queries as peaked as a trained model's: scores with a deviation of 2
    return dict(case=case, q=_normal(g, rows, h, d, dtype=TYPES[t], gain=2.0), k_cache=k_cache, v_cache=v_cache, k_scales=k_scales, v_scales=v_scales, table=table,
                starts=_words([0] + list(np.cumsum(fresh))), lengths=_words(total), most=max(1, max(fresh)), keys=max(1, max(total)),
                out=torch.zeros(rows, h, d, dtype=TYPES[t], device="cuda"))


# ---------------------------------------------------------------------------------------------- the operators, plain

def _plain_codes(x):
    """Rows of whole numbers from -127 to 127, as f32, and their scales."""
    top = x.abs().amax(1)
    scale = torch.where(top < LEAST, 0, top / 127)
    inverse = torch.where((scale > 0) & (scale < torch.inf), 1 / scale, 0)
    return (x * inverse[:, None]).round_().clamp_(-127, 127), scale


def _plain_quantize(s):
    codes, scale = _plain_codes(s["x"].float())
    return torch.mul(codes, scale[:, None], out=s["values"]), scale


def _plain_linear(s):
    codes, scale = _plain_codes(s["x"].float())
    y = (codes @ s["w"].float().T) * scale[:, None] * s["w_scales"]
    if s["addend"] is not None:
        y += s["addend"].float()
    return y.to(s["out"].dtype)


def _rotated(x, positions):
    half = x.shape[2] // 2
    angle = positions.double()[:, None] * THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * c - b * n, a * n + b * c], 2)


def _plain_store(cache, scales, x, slots, block):
    """Rows x [rows, kv, d] into their slots; what their blocks hold already is kept, in the blocks' new scales."""
    kv, d = x.shape[1:]
    codes, old = cache.view(-1, block, kv, d), scales.view(-1, kv)
    blocks = codes.shape[0]
    live = slots >= 0
    of = torch.where(live, slots.long() // block, blocks)                                             # one more block for rows without a slot
    at = torch.where(live, slots.long() % block, 0)
    top = torch.zeros(blocks + 1, kv, device="cuda").scatter_reduce_(0, of[:, None].expand(-1, kv), x.abs().amax(2), "amax")[:-1]
    written = torch.zeros(blocks + 1, block, dtype=torch.bool, device="cuda")
    written[of, at] = True
    written = written[:-1]
    touched = written.any(1)[:, None]
    old = torch.where(written[:, :1], 0, old)
    new = torch.where(touched, torch.maximum(old, torch.where(top < LEAST, 0, top / 127)), old)
    fine = (new > 0) & (new < torch.inf)
    ratio = torch.where(fine, old / new, 0)
    held = touched & ~written & ~written[:, :1]
    moved = (codes.float() * ratio[:, None, :, None]).round_()
    codes.copy_(torch.where(held[..., None, None], moved, codes.float()).to(torch.int8))
    inverse = torch.where(fine, 1 / new, 0)
    whole = (x[live] * inverse[of[live]][:, :, None]).round_().clamp_(-127, 127)
    codes[of[live], at[live]] = whole.to(torch.int8)
    scales.view(-1, kv).copy_(new)


def _values(s):
    out, block = s["values"], s["case"]["block"]
    for i, x in enumerate("kv"):
        torch.mul(s[x + "_cache"].unflatten(1, (-1, block)), s[x + "_scales"][:, :, None, :, None], out=out[i])
    return out


def _plain_append(s):
    block = s["case"]["block"]
    _plain_store(s["k_cache"], s["k_scales"], _rotated(s["k"], s["positions"]), s["slots"], block)
    _plain_store(s["v_cache"], s["v_scales"], s["v"].float(), s["slots"], block)
    return _rotated(s["q"], s["positions"]).to(s["q_out"].dtype), _values(s)


def _plain_attend(s):
    case, q, t = s["case"], s["q"], s["q"].dtype
    page, block, d, kv, most, keys = case["page"], case["block"], case["head_dim"], case["kv_heads"], s["most"], s["keys"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    fresh = starts[1:] - starts[:-1]
    j = torch.arange(keys, device="cuda")
    slot = s["table"].long().clamp(min=0)[:, j // page] * page + j % page                             # [S, keys]
    k, v = (s[x + "_cache"].flatten(0, 1)[slot].float().mul_(s[x + "_scales"].flatten(0, 1)[slot // block][..., None]) for x in "kv")
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


PLAIN = {"quantize": _plain_quantize, "linear": _plain_linear, "append": _plain_append, "attend": _plain_attend}


# ---------------------------------------------------------------------------------------------- the operators, the framework's

def _own(s):
    from meganeura_b200 import ops
    op = s["case"]["op"]
    if op == "quantize":
        ops.quantize_rows(s["x"], out=(s["codes"], s["scales"]))
        return torch.mul(s["codes"], s["scales"][:, None], out=s["values"]), s["scales"]
    if op == "linear":
        ops.quantize_rows(s["x"], out=(s["codes"], s["scales"]))
        return ops.matmul_int8(s["codes"], s["scales"], s["w"], s["w_scales"], addend=s["addend"], out=s["out"])
    if op == "append":
        q = ops.paged_append_int8(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], theta=THETA, q_out=s["q_out"])
        return q, _values(s)
    return ops.paged_attention_int8(s["q"], s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["table"], s["starts"], s["lengths"], s["most"],
                                    window=s["case"]["window"], out=s["out"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits

def _exact_row_codes(x):
    x = x.double()
    scale = x.abs().max(1, keepdim=True).values / 127.0
    return torch.round(x / scale), scale


def _exact_quantize(s):
    codes, scale = _exact_row_codes(s["x"])
    return codes * scale, scale[:, 0]


def _exact_linear(s):
    codes, scale = _exact_row_codes(s["x"])
    y = (codes * scale) @ (s["w"].double() * s["w_scales"].double()[:, None]).T
    return y if s["addend"] is None else y + s["addend"].double()


def _exact_rotate(x, positions):
    x, d = x.double(), x.shape[-1]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] / THETA ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d))
    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_store(cache, scales, x, slots, block):
    """Block by block: the held tokens' codes in the larger scale, then the new ones'; the cache's values."""
    kv, d = x.shape[1:]
    codes, scale = cache.reshape(-1, block, kv, d).double(), scales.reshape(-1, kv).double()
    rows = {}
    for r, slot in enumerate(slots.tolist()):
        if slot >= 0:
            rows.setdefault(slot // block, []).append((slot % block, r))
    for b, placed in rows.items():
        at, r = ([p[i] for p in placed] for i in (0, 1))
        new = x[r].abs().amax((0, 2)) / 127.0
        if 0 in at:
            was = torch.zeros_like(new)
        else:
            was = scale[b].clone()
        scale[b] = torch.maximum(was, new)
        if 0 not in at:
            held = [i for i in range(block) if i not in at]
            codes[b, held] = torch.round(codes[b, held] * (was / scale[b])[None, :, None])
        codes[b, at] = torch.round(x[r] / scale[b][None, :, None])
    return (codes * scale[:, None, :, None]).view(cache.shape[0], -1, block, kv, d)


def _exact_append(s):
    block = s["case"]["block"]
    k = _exact_store(s["k_cache"], s["k_scales"], _exact_rotate(s["k"], s["positions"]), s["slots"], block)
    v = _exact_store(s["v_cache"], s["v_scales"], s["v"].double(), s["slots"], block)
    return _exact_rotate(s["q"], s["positions"]), torch.stack([k, v])


def _exact_attend(s):
    case = s["case"]
    g, out = case["heads"] // case["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for i, (c, n) in enumerate(zip(*_lengths(case))):
        if n == 0:
            continue
        pages = s["table"][i, :_pages(c + n, case["page"])].long()
        k, v = ((s[x + "_cache"][pages].unflatten(1, (-1, case["block"])).double() * s[x + "_scales"][pages].double()[:, :, None, :, None]).flatten(0, 2)[:c + n] for x in "kv")
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


EXACT = {"quantize": _exact_quantize, "linear": _exact_linear, "append": _exact_append, "attend": _exact_attend}


def exact(case, seed):
    return EXACT[case["op"]](prepare(case, seed))

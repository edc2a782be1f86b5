"""Plain restatements, in 64 bits and sequence by sequence, of the operators over a paged cache and of what follows them:
block tables and slots, the write of new keys and values, attention, probabilities, verification of drafts."""
import math

import numpy as np


def plan(cached, fresh, table, held, free_pages, count, page_size, rows):
    """(starts, lengths, positions, slots, lacking, table, held, count) behind mgq_paged_plan; the arguments stay as they are."""
    table, held, pages = table.copy(), held.copy(), len(free_pages)
    count = min(int(count), pages)
    top, wanted, given = count, 0, 0
    starts, lengths, positions, slots = [0], [], np.zeros(rows, np.int64), np.full(rows, -1, np.int64)
    for s in range(len(cached)):
        begin = starts[-1]
        end = min(begin + int(fresh[s]), rows)
        after = -(-(int(cached[s]) + end - begin) // page_size)
        have = min(int(held[s]), table.shape[1])
        narrow = after > table.shape[1]
        need = 0 if narrow else max(0, after - have)
        wanted += need
        served = not narrow and (need == 0 or wanted <= count)
        if served:
            for i in range(need):
                table[s, have + i] = free_pages[top - 1 - given]
                given += 1
            held[s] = have + need
        for r in range(begin, end):
            at = int(cached[s]) + r - begin
            positions[r] = at
            if served and 0 <= table[s, at // page_size] < pages:
                slots[r] = int(table[s, at // page_size]) * page_size + at % page_size
        starts.append(end)
        lengths.append(int(cached[s]) + (end - begin if served else 0))
    return np.array(starts), np.array(lengths), positions, slots, max(0, wanted - count), table, held, count - given


def trim(lengths, table, held, free_pages, count, page_size):
    """(table, held, free_pages, count) behind mgq_paged_trim."""
    table, held, free_pages = table.copy(), held.copy(), free_pages.copy()
    back = []
    for s in range(len(lengths)):
        have = min(int(held[s]), table.shape[1])
        keep = min(have, -(-int(lengths[s]) // page_size))
        back += [int(p) for p in table[s, keep:have]]
        table[s, keep:have] = -1
        if keep < have:
            held[s] = keep
    count = min(int(count), len(free_pages))
    for i, page in enumerate(back):
        free_pages[count + len(back) - 1 - i] = page
    return table, held, free_pages, count + len(back)


def rotate(x, positions, theta):
    """x [rows, heads, d], half-split pairs."""
    half = x.shape[2] // 2
    angle = positions.astype(np.float64)[:, None] * theta ** (-np.arange(half) / half)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([a * c - b * s, a * s + b * c], 2)


def gather(cache, pages_of, length):
    """(rows [length, kv_heads, d], which of them exist) of one sequence; cache [pages, page_size, kv_heads, d]."""
    page_size = cache.shape[1]
    j = np.arange(length)
    page = pages_of[j // page_size]
    there = (page >= 0) & (page < cache.shape[0])
    return cache[np.where(there, page, 0), j % page_size], there


def attention(q, k_cache, v_cache, table, starts, lengths, scale, window=0):
    """(out, sum of weight * |value|, largest sum of |q k| * scale per row), all f64; rows that belong to nobody are NaN."""
    q = q.astype(np.float64)
    rows, heads, d = q.shape
    kv_heads = k_cache.shape[2]
    out, size, reach = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((rows, heads))
    for s in range(len(lengths)):
        r0, r1 = min(int(starts[s]), rows), min(int(starts[s + 1]), rows)
        n, length = r1 - r0, min(int(lengths[s]), table.shape[1] * k_cache.shape[1])
        if n <= 0:
            continue
        (k, there), (v, _) = (gather(c, table[s].astype(np.int64), length) for c in (k_cache, v_cache))
        k, v = k.astype(np.float64), v.astype(np.float64)
        for i in range(n):
            at = length - n + i
            seen = there & (np.arange(length) <= at)
            if window:
                seen &= np.arange(length) > at - window
            for h in range(heads):
                o = h * kv_heads // heads
                if not seen.any():
                    out[r0 + i, h] = 0
                    continue
                x = k[seen, o] @ q[r0 + i, h] * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[r0 + i, h] = w @ v[seen, o]
                size[r0 + i, h] = w @ np.abs(v[seen, o])
                reach[r0 + i, h] = (np.abs(k[seen, o]) @ np.abs(q[r0 + i, h])).max() * abs(scale)
    return out, size, reach


def probs(logits, temperature):
    out = np.zeros(logits.shape)
    for r, row in enumerate(logits.astype(np.float64)):
        row = np.where(np.isnan(row), -np.inf, row)
        m = row.max()
        if m == -np.inf:
            continue
        if not temperature[r] > 0:
            out[r, int(np.argmax(row))] = 1
        elif m == np.inf:
            out[r] = (row == m) / (row == m).sum()
        else:
            e = np.exp((row - m) / float(temperature[r]))
            out[r] = e / e.sum()
    return out


def mass(p):
    p = p.astype(np.float64)
    return np.where((p > 0) & np.isfinite(p), p, 0.0)


def verify(target, draft, tokens, starts, accept, sample):
    rows, vocab = target.shape
    counts, picks, out = [], [], np.full(rows, -2, np.int64)
    for s in range(len(starts) - 1):
        r0 = min(int(starts[s]), rows)
        n = max(min(int(starts[s + 1]), rows), r0) - r0
        if n == 0:
            counts.append(0)
            picks.append(-1)
            continue
        kept = 0
        while kept < n - 1:
            row, d = r0 + kept, int(tokens[r0 + kept + 1])
            if not 0 <= d < vocab or not float(accept[row]) * (1.0 if draft is None else float(draft[row, d])) < float(target[row, d]):
                break
            kept += 1
        row = r0 + kept
        w = mass(target[row])
        if kept < n - 1:
            if draft is None:
                rest = w.copy()
                if 0 <= tokens[row + 1] < vocab:
                    rest[tokens[row + 1]] = 0
            else:
                rest = np.maximum(w - mass(draft[row]), 0)
            if rest.sum() > 0:
                w = rest
        c = np.cumsum(w)
        if c[-1] > 0:
            u = float(sample[s])
            u = min(max(u, 0.0), 1.0) if not math.isnan(u) else 0.0
            pick = min(int(np.count_nonzero(c <= u * c[-1])), int(np.flatnonzero(w)[-1]))
        else:
            pick = -1
        counts.append(kept)
        picks.append(pick)
        out[r0:r0 + n] = [int(t) for t in tokens[r0 + 1:r0 + 1 + kept]] + [pick] + [-1] * (n - 1 - kept)
    return np.array(counts), np.array(picks), out

"""Plain restatements of the paged key-value cache's operators, in NumPy: loops
over tokens, pages and heads, and 64-bit floating point where numbers are
computed (the float32 quotients of the summaries' and queries' codes are part
of their definition)."""

import numpy as np


def plan(past, fresh, table, free_pages, cursor, page, tokens):
    table = table.copy()
    requests, cols = table.shape
    slots, who, where = [], [], []
    starts, lengths, first = [0], [], []
    at, open_ = cursor, True
    for r in range(requests):
        p, m = int(past[r]), int(fresh[r])
        fits = p >= 0 and m >= 0 and -(-(p + m) // page) <= cols
        need = -(-(p + m) // page) - -(-p // page) if fits else 0
        ok = fits
        if fits and need:
            # a request that the list cannot serve closes it for the later ones
            open_ = open_ and 0 <= at and at + need <= len(free_pages)
            ok = open_
            if ok:
                have = -(-p // page)
                table[r, have:have + need] = free_pages[at:at + need]
        first.append(-1 if not ok else at if need else 0)
        if ok and need:
            at += need
        for i in range(max(m, 0)):
            who.append(r)
            pid = int(table[r, (p + i) // page]) if ok else -1
            where.append(p + i if ok else -1)
            slots.append(pid * page + (p + i) % page if pid >= 0 else -1)
        starts.append(len(who))
        lengths.append(p + m if ok else p)
    pad = [-1] * max(0, tokens - len(who))
    cut = [np.array((x + pad)[:tokens]) for x in (slots, who, where)]
    return dict(slots=cut[0].astype(np.int64), requests=cut[1].astype(np.int32),
                positions=cut[2].astype(np.int32), starts=np.array(starts, np.int32),
                lengths=np.array(lengths, np.int32), first=np.array(first, np.int32),
                cursor=np.array([at], np.int32), table=table)


def codes(x):
    """int8 codes of the sum over the first axis of x [m, d] (float32), the
    largest |x| and the largest |sum| that they are measured by."""
    f = np.float32
    top = np.abs(x).max() if x.size else f(0)
    if not np.isfinite(x).all() or not top > f(1e-30):
        return np.zeros(x.shape[1], np.int8), top, 0
    total = np.rint(x * (f(127) / top)).astype(np.int64).sum(0)
    peak = int(np.abs(total).max())
    if peak == 0:
        return np.zeros(x.shape[1], np.int8), top, 0
    return np.rint(total.astype(f) * (f(127) / f(peak))).astype(np.int8), top, peak


def summary(keys):
    """(codes, scale) of one page and head, keys [page, d] (float32)."""
    if not np.isfinite(keys).all():
        return np.zeros(keys.shape[1], np.int8), np.float32(np.inf)
    c, top, peak = codes(keys)
    return c, np.float32(float(top) * peak / (127.0 * 127.0 * len(keys)))


def select(q, summaries, scales, table, requests, positions, page, n, first, last):
    """q [tokens, q_heads, d] (float32) -> int32 [tokens, heads, n]."""
    pages, heads, d = summaries.shape
    group = q.shape[1] // heads
    out = np.full((len(q), heads, n), -1, np.int32)
    cap = float(np.finfo(np.float32).max)
    for t in range(len(q)):
        r, pos = int(requests[t]), int(positions[t])
        if not 0 <= r < len(table) or pos < 0:
            continue
        own = pos // page
        for h in range(heads):
            c = codes(q[t, h * group:(h + 1) * group])[0].astype(np.int64)
            found = []
            for b in range(min(own + 1, table.shape[1])):
                p = int(table[r, b])
                if not 0 <= p < pages:
                    continue
                s = scales[p, h]
                if b < first or b > own - last:
                    score = np.inf
                elif not np.isfinite(s):
                    score = cap
                else:
                    dot = np.float32((c * summaries[p, h].astype(np.int64)).sum())
                    with np.errstate(over="ignore"):
                        score = min(max(float(dot * s), -cap), cap)
                found.append((-score, b))
            best = sorted(b for _, b in sorted(found)[:n])
            out[t, h, :len(best)] = best
    return out


def attend(q, keys, values, table, requests, positions, scale, blocks=None):
    """float64 (out, lse, weight) of [tokens, q_heads, d]; weight is the
    attention of |v|, the size of the terms that out sums, and reach the
    largest sum of |q_i k_i| of a row times scale."""
    pages, heads, page, d = keys.shape
    tokens, q_heads = q.shape[:2]
    group = q_heads // heads
    out = np.zeros((tokens, q_heads, d))
    weight = np.zeros((tokens, q_heads, d))
    lse = np.full((tokens, q_heads), -np.inf)
    reach = np.zeros((tokens, q_heads, 1))
    count = np.zeros((tokens, q_heads, 1))
    for t in range(tokens):
        r, pos = int(requests[t]), int(positions[t])
        if not 0 <= r < len(table) or pos < 0:
            continue
        for h in range(heads):
            ks, vs = [], []
            listed = range(table.shape[1]) if blocks is None else blocks[t, h]
            for b in listed:
                b = int(b)
                if not 0 <= b < table.shape[1]:
                    continue
                p, seen = int(table[r, b]), min(page, pos + 1 - b * page)
                if 0 <= p < pages and seen > 0:
                    ks.append(keys[p, h, :seen])
                    vs.append(values[p, h, :, :seen].T)
            if not ks:
                continue
            k, v = np.concatenate(ks).astype(np.float64), np.concatenate(vs).astype(np.float64)
            for g in range(h * group, (h + 1) * group):
                x = q[t, g].astype(np.float64)
                s = k @ x * scale
                top = s.max()
                e = np.exp(s - top)
                lse[t, g] = top + np.log(e.sum())
                out[t, g] = e @ v / e.sum()
                weight[t, g] = e @ np.abs(v) / e.sum()
                reach[t, g] = (np.abs(k) @ np.abs(x)).max() * scale
                count[t, g] = len(k)
    return out, lse, weight, reach, count

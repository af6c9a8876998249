"""Plain restatements, in NumPy and 64 bits, of the operators that keep a paged
key-value cache within a budget: loops over requests, heads and keys."""

import math

import numpy as np

import kv_oracle


def frequencies(rotated, base=10000.0, scaling=None, factor=1.0, context=1.0):
    """(radians a position of each pair, factor of the rotated values)"""
    out, gain = [], 1.0
    if scaling == "base":
        base = base * factor ** (rotated / (rotated - 2.0))
    for i in range(rotated // 2):
        f = 1.0 / base ** (2.0 * i / rotated)
        if scaling == "linear":
            f /= factor
        if scaling == "ramp":
            turns = context / (2.0 * math.pi / f)
            w = 0.0 if turns <= 1 else 1.0 if turns >= 32 else (turns - 1.0) / 31.0
            f = w * f + (1.0 - w) * f / factor
        out.append(f)
    if scaling == "ramp":
        gain = 1.0 + 0.1 * math.log(factor)
    return np.array(out), gain


def rotate(x, positions, freq, gain, layout, norm=None, eps=0.0):
    """x [tokens, heads, dim] float64 -> (y, size): size bounds the terms that each
    value sums."""
    x = np.array(x, np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * norm
    y, size = x.copy(), np.abs(x)
    n = len(freq)
    angle = np.maximum(positions, 0).astype(np.float64)[:, None] * freq
    c, s = np.cos(angle) * gain, np.sin(angle) * gain
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + n)
        u, v = x[:, :, a], x[:, :, b]
        y[:, :, a] = u * c[:, None, i] - v * s[:, None, i]
        y[:, :, b] = v * c[:, None, i] + u * s[:, None, i]
        size[:, :, a] = size[:, :, b] = gain * (np.abs(u) + np.abs(v))
    return y, size


def weigh(q, keys, table, starts, positions, lse, mass, scale, decay=1.0):
    """float64 (mass, err): err weighs each term by what its float32 score may be
    off by, in units of 2^-24."""
    pages, heads, page, d = keys.shape
    group = q.shape[1] // heads
    out, err = mass.astype(np.float64), np.zeros(mass.shape)
    tokens, most = len(q), table.shape[1] * page
    for r in range(len(table)):
        a, b = min(max(0, starts[r]), tokens), min(starts[r + 1], tokens)
        if b <= a:
            continue
        first, last = int(positions[a]), min(int(positions[b - 1]), most - 1)
        for h in range(heads):
            for p in range(last + 1):
                before = decay * out[r, h, p] if p < first and decay != 0 else 0.0
                pid = int(table[r, p // page])
                got = off = 0.0
                if 0 <= pid < pages:
                    k = keys[pid, h, p % page].astype(np.float64)
                    see = [t for t in range(a, b) if positions[t] >= p]
                    x = q[see, h * group:(h + 1) * group].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        s = x @ k * scale
                        e = np.exp(s - lse[see, h * group:(h + 1) * group])
                        reach = np.abs(x) @ np.abs(k) * scale
                        w = e * ((d + 4) * reach + 4 * (np.abs(s) + np.abs(lse[see, h * group:(h + 1) * group])) + 16)
                    got, off = e.sum(), w.sum() + len(see) * group * e.sum()
                out[r, h, p] = before + got
                err[r, h, p] = off + 2 * abs(before) + 2 * abs(got)
    return out, err


def keep(mass, lengths, n, first, recent, above):
    requests, heads, slots = mass.shape
    out = np.full((requests, heads, n), -1, np.int32)
    for r in range(requests):
        length = min(int(lengths[r]), slots)
        if length <= above:
            continue
        for h in range(heads):
            always = [p for p in range(length) if p < first or p >= length - recent]
            rest = [p for p in range(length) if first <= p < length - recent]
            # greatest first, the lowest position among equal ones, NaN at the end
            rest.sort(key=lambda p: (np.isnan(mass[r, h, p]),
                                     0.0 if np.isnan(mass[r, h, p]) else -float(mass[r, h, p]), p))
            out[r, h] = sorted(always + rest[:n - len(always)])
    return out


def compact(keys, values, summaries, scales, table, lengths, kept, free_pages, cursor, mass=None):
    """Everything after it, as a dict (the inputs stay as they are); summaries None:
    none are kept."""
    pages, heads, page, d = keys.shape
    requests, _, n = kept.shape
    old_k, old_v, old_m = keys, values, mass
    keys, values, free = keys.copy(), values.copy(), free_pages.copy()
    mass = None if mass is None else mass.copy()
    if summaries is not None:
        summaries, scales = summaries.copy(), scales.copy()
    lengths_out = np.array(lengths, np.int32)
    at, taken, open_ = 0, 0, True
    cut = []
    for r in range(requests):
        length = int(lengths[r])
        if not (length > n and -(-length // page) <= table.shape[1] and kept[r, 0, 0] >= 0):
            continue
        gives = list(range(-(-n // page), -(-length // page)))
        at += len(gives)
        if gives:
            # one whose pages find no room closes the list for the later ones
            open_ = open_ and cursor <= len(free) and at <= cursor
            if not open_:
                continue
            free[cursor - at:cursor - at + len(gives)] = table[r, gives]
            taken = at
        cut.append(r)
        lengths_out[r] = n
    for r in cut:
        for h in range(heads):
            for j in range(n):
                s = int(kept[r, h, j])
                p, to = int(table[r, s // page]), int(table[r, j // page])
                if mass is not None:
                    mass[r, h, j] = old_m[r, h, s]
                if not (0 <= p < pages and 0 <= to < pages):
                    continue
                keys[to, h, j % page] = old_k[p, h, s % page]
                values[to, h, :, j % page] = old_v[p, h, :, s % page]
        for h in range(heads):
            for b in range(n // page):
                to = int(table[r, b])
                moved = any(kept[r, h, j] != j for j in range(b * page, (b + 1) * page))
                if summaries is not None and moved and 0 <= to < pages:
                    summaries[to, h], scales[to, h] = kv_oracle.summary(keys[to, h].astype(np.float32))
    return dict(keys=keys, values=values, summaries=summaries, scales=scales, mass=mass,
                free=free, cursor=np.array([cursor - taken], np.int32), lengths=lengths_out)

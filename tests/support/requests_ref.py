"""Plain restatements of charlotte_amd.serving's operators of a step over several
requests, in 64 bits and whole numbers (test infrastructure)."""

import math

import numpy as np

NONE = 0xFFFFFFFF
WHOLE = 1 << 40


def page_plan(past, counts, held, table, free, free_count, rows, page_tokens, pages):
    """Lists of ints (table a list of rows, free the stack's words), all left as they are; a dict of what the call writes."""
    table, free, stride = [list(r) for r in table], list(free), len(table[0])
    top, n = min(free_count, pages), len(past)
    starts = [sum(counts[:r]) for r in range(n + 1)]
    need = [-(-(p + c) // page_tokens) for p, c in zip(past, counts)]
    here = [min(h, stride) for h in held]
    fits = [(counts[r] == 0 or starts[r + 1] <= rows) and need[r] <= stride for r in range(n)]
    for r in range(n):
        for j in range(need[r], here[r]) if fits[r] else ():
            if top < pages:
                free[top] = table[r][j]
                top += 1
    there, wanted, after, granted = top, 0, list(held), [0] * n
    for r in range(n):
        takes = max(0, need[r] - here[r]) if fits[r] else 0
        wanted += takes
        if not fits[r] or (takes and wanted > there):
            continue
        for j in range(here[r], need[r]):
            top -= 1
            table[r][j] = free[top]
        after[r], granted[r] = need[r], counts[r]
    slots, positions = [NONE] * rows, [0] * rows
    for r in range(n):
        for i in range(starts[r], min(starts[r + 1], rows)):
            at = past[r] + i - starts[r]
            positions[i] = at & 0xFFFFFFFF
            if granted[r] and table[r][at // page_tokens] < pages:
                slots[i] = table[r][at // page_tokens] * page_tokens + at % page_tokens
    return {"table": table, "free": free, "free_count": top, "held": after, "granted": granted,
            "starts": [min(s, NONE) for s in starts], "slots": slots, "positions": positions}


def residual_norm(x, y, w, gate, v, a, b, epsilon):
    """r and n of rows [rows, width] in 64 bits, and how far f32 may be. A sum of squares rounds at most 35 times (a
    product, 10 sums in a thread, 6 in a wave, 16 over the waves, its mean), half of that in the root's reciprocal, which
    rounds twice more; a product of it and of a weight, a gate or a scale once each."""
    u = 2.0 ** -24
    x = np.asarray(x, np.float64)
    a, b, epsilon = (float(np.float32(t)) for t in (a, b, epsilon))

    def root(z):
        return np.sqrt((z * z).mean(-1, keepdims=True) + epsilon)

    r, off = a * x, u * np.abs(a * x)
    if y is not None:
        z, steps = np.asarray(y, np.float64), 0
        if w is not None:
            z, steps = z / root(z) * w, 35 / 2 + 2 + 2
        if gate is not None:
            z, steps = z * gate, steps + 1
        off = off + u * (steps * np.abs(b * z) + np.abs(r) + np.abs(b * z))
        r = r + b * z
    if v is None:
        return r, None, off, None
    size = root(r)
    n = r / size * v
    moved = np.sqrt((off * off).mean(-1, keepdims=True)) / size
    return r, n, off, np.abs(v) / size * off + np.abs(n) * (moved + (35 / 2 + 4) * u)


def weights(logits, temperature):
    """(order, weights in it) of one row, as whole numbers; None where it has no token."""
    x = np.asarray(logits, np.float32).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    x = x[order]
    if x[0] == -np.inf:
        return None
    if x[0] == np.inf:
        return order, np.where(x == np.inf, WHOLE, 0)
    with np.errstate(over="ignore"):
        w = np.floor(np.exp(np.maximum((x - x[0]) / temperature, -100.0)) * WHOLE).astype(np.int64)
    return order, np.where(x == -np.inf, 0, w)


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """(token, its weight, the kept tokens' weight) of one row."""
    t, p, m, u = (float(np.float32(z)) for z in (temperature, top_p, min_p, uniform))
    greedy = not t >= 1e-6
    found = weights(logits, 1.0 if greedy else t)
    if found is None:
        return -1, 0, 1
    order, w = found
    n = 1 if greedy else min(top_k, len(w)) if top_k > 0 else len(w)
    w = w[:n]
    if p < 1:
        running = np.cumsum(w)
        least = math.ceil(max(p, 0.0) * float(running[-1]))
        w = w[:max(1, int(np.searchsorted(running, least)) + 1)]
    least = math.ceil(min(m, 1.0) * WHOLE) if m > 0 else 0
    w = w[:max(1, int((w >= least).sum()))]
    running = np.cumsum(w)
    total = int(running[-1])
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    at = total * int(u * 2.0 ** 31) >> 31
    place = int(np.searchsorted(running, at, side="right"))
    return int(order[place]), int(w[place]), total

"""Plain restatement of sampling with limits and of the walk over drafted tokens, on the CPU in 64 bits (test
infrastructure only), from the definitions in include/dsqg.h."""

import math


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability, margin) of one row of Python floats; the margin is how far u times the kept mass is
    from the nearest running sum and the nucleus from its nearest border, in shares of their masses."""
    cand = [(x, i) for i, x in enumerate(row) if x == x and x != -math.inf]
    if not cand:
        return -1, -math.inf, 1.0
    order = sorted(cand, key=lambda e: (-e[0], e[1]))
    if not temperature > 0:
        return order[0][1], 0.0, 1.0
    top = order[0][0]

    def weight(x):
        return 1.0 if x == top else math.exp((x - top) / temperature) if math.isfinite(top) else 0.0

    if top_k > 0:
        order = order[:top_k]
    margin = 1.0
    if top_p < 1:
        total = math.fsum(weight(x) for x, _ in order)
        limit, run, kept = max(top_p, 0.0) * total, 0.0, []
        for x, i in order:
            if kept:  # (the first stays whatever the limit)
                margin = min(margin, abs(run - limit) / total)
            if run > limit:
                break
            kept.append((x, i))
            run += weight(x)
        order = kept
    order = [(x, i) for x, i in order if weight(x) >= min(min_p, 1.0)]
    total = math.fsum(weight(x) for x, _ in order)
    at, run = max(u, 0.0) * total, 0.0
    pick = None
    for x, i in sorted(order, key=lambda e: e[1]):
        run += weight(x)
        margin = min(margin, abs(run - at) / total)
        if pick is None and run > at:
            pick = (x, i)
    if pick is None:  # u of 1 and more: the last that has a weight
        pick = max(((x, i) for x, i in order if weight(x) > 0), key=lambda e: e[1])
    return pick[1], math.log(weight(pick[0])) - math.log(total), margin


def walk(tokens, parents, picks, count=None):
    """(path, next) of one tree."""
    count = len(tokens) if count is None else min(count, len(tokens))
    if count <= 0:
        return [], -1
    path = [0]
    while True:
        kids = [j for j in range(path[-1] + 1, count) if parents[j] == path[-1] and tokens[j] == picks[path[-1]]]
        if not kids:
            return path, picks[path[-1]]
        path.append(kids[0])

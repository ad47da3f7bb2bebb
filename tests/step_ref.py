"""Plain forms of what a serving step has around its layers, on the host and in 64 bits."""
import numpy as np


def plan(lengths, news, table, free, taken, page, tokens, shift=None):
    """(offsets, lengths, slots, positions, taken, table) of lists, one request and one token after the other."""
    table = [list(row) for row in table]
    offsets, slots, positions = [0], [], []
    for s, (length, more) in enumerate(zip(lengths, news)):
        for x in range(length, length + more):
            if x % page == 0:
                table[s][x // page] = free[taken]
                taken += 1
            slots.append(table[s][x // page] * page + x % page)
            positions.append(x + (shift[s] if shift else 0))
        offsets.append(offsets[-1] + more)
    behind = tokens - offsets[-1]
    return offsets, [a + b for a, b in zip(lengths, news)], slots + [-1] * behind, positions + [0] * behind, taken, table


def trim(lengths, keep, table, free, taken, page):
    """(lengths, free, taken), from the last page of the last request on."""
    lengths, free = list(lengths), list(free)
    for s in reversed(range(len(lengths))):
        while lengths[s] > max(keep[s], 0):
            lengths[s] -= 1
            if lengths[s] % page == 0:
                taken -= 1
                free[taken] = table[s][lengths[s] // page]
    return lengths, free, taken


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, softcap=0.0):
    """(token, probability, how near a border a rule or the random number comes, as a share of the whole) of a row of float64."""
    order = np.argsort(-row, kind="stable")  # (NaN comes last)
    order = order[row[order] > -np.inf]
    if not len(order):
        return -1, 0.0, 1.0
    if not temperature > 0:
        return int(order[0]), 1.0, 1.0
    if top_k > 0:
        order = order[:top_k]
    x = row[order]
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if softcap:
            x = softcap * np.tanh(x / softcap)
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / temperature)) if np.isfinite(x[0]) else (x == x[0]).astype(np.float64)
    near = 1.0
    if top_p < 1:
        through = np.cumsum(w)
        target = top_p * through[-1]
        near = min(near, np.abs(through - target).min() / through[-1])
        count = int(np.searchsorted(through, target, side="left")) + 1
        order, w = order[:count], w[:count]
    if min_p > 0:
        near = min(near, np.abs(w[w < 1] - min(min_p, 1.0)).min(initial=1.0))  # (a share of one is one exactly on both sides)
        order, w = order[w >= min(min_p, 1.0)], w[w >= min(min_p, 1.0)]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    through = np.cumsum(w)
    target = u * through[-1]
    near = min(near, np.abs(through[:-1] - target).min(initial=np.inf) / through[-1])
    at = min(int(np.searchsorted(through, target, side="right")), len(w) - 1)
    return int(order[at]), w[at] / through[-1], near

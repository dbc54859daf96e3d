"""Trees of drafted tokens, sampling and acceptance, restated in numpy for the tests: masks as sets, weights in 64 bits, the order of a
vocabulary by sorting it.  Test infrastructure only."""
from __future__ import annotations

import math

import numpy as np


def ancestors(parents) -> list:
    """Of one sequence: the set of rows that each row sees."""
    seen = []
    for i, p in enumerate(parents):
        seen.append({i} | (seen[p] if 0 <= p < i else set()))
    return seen


def masks(sets, words: int) -> np.ndarray:
    out = np.zeros((len(sets), words), np.uint32)
    for i, s in enumerate(sets):
        for j in s:
            out[i, j // 32] |= np.uint32(1 << (j % 32))
    return out.view(np.int32)


def seen(sets, length: int, window: int) -> np.ndarray:
    """bool [rows, length]: the tokens that each row of a sequence sees, whose last len(sets) tokens are its rows."""
    n, out = len(sets), np.zeros((len(sets), length), bool)
    for i, s in enumerate(sets):
        # in order: context, then the row's tokens of the tree; the window has the last ones
        places = list(range(max(0, length - n))) + sorted(length - n + j for j in s if j < n)
        places = places[-window:] if window else places
        out[i, [p for p in places if p >= 0]] = True
    return out


def attention(q, keys, values, scale: float, see):
    """q [rows, group, D] of one key head, see [rows, tokens], float64 -> (out, weights, scores)."""
    with np.errstate(all="ignore"):
        s = np.where(see[:, None], np.einsum("ngd,td->ngt", q, keys) * scale, -np.inf)
        top = np.max(s, -1, keepdims=True, initial=-np.inf)
        e = np.where(see[:, None], np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        total = e.sum(-1, keepdims=True)
        p = np.where(total == 0, 0, e / np.where(total == 0, 1, total))
        out = np.zeros(q.shape)
        for i in range(len(q)):
            out[i] = p[i][:, see[i]] @ values[see[i]]
    return out, p, s


def sample(x: np.ndarray, u: float, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, its share of what stays, how far u is from the next border between two tokens, of the draw or of top-p) of one row of logits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    most = x.max()
    if most == -np.inf:
        return -1, 0.0, math.inf
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0]), 1.0, math.inf
    with np.errstate(all="ignore"):
        y = np.where(x == most, 0.0, (x - most) / temperature)
        y = np.where(np.isnan(y), -np.inf, y)  # (minus infinity weighs nothing, however high the temperature)
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(y[order])
    edge = math.inf
    if top_p < 1:
        front = np.concatenate([[0.0], np.cumsum(w)[:-1]]) / w.sum()
        n = max(1, int((front < top_p).sum()))
        edge = float(np.abs(front[1:] - top_p).min(initial=math.inf)) if top_p > 0 else math.inf
        order = order[:n]
    if min_p > 0:
        order = order[y[order] >= math.log(min(min_p, 1.0))]
    order = np.sort(order)
    w = np.exp(y[order])
    upto = np.cumsum(w)
    at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), int(np.nonzero(w)[0][-1]))
    edge = min(edge, float(np.abs(upto / upto[-1] - u)[:-1].min(initial=math.inf)))
    return int(order[at]), float(w[at] / upto[-1]), edge


def walk(parents, tokens, sampled) -> list:
    """The path of one sequence: its rows from the root on."""
    if not len(parents):
        return []
    path = [0]
    while sampled[path[-1]] >= 0:
        child = [i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == sampled[path[-1]]]
        if not child:
            break
        path.append(child[0])
    return path

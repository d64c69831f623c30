"""Float64 statements of the operators of speculative decoding, on the CPU, one sequence and one node at a time, and the bounds their kernels are held to."""
import math

import numpy as np


def ancestors(parents):
    """[n, n]: node j is an ancestor of node i, or i itself; depths."""
    n = len(parents)
    sees, depth = np.zeros((n, n), bool), np.zeros(n, int)
    for i, p in enumerate(parents):
        assert -1 <= p < i
        if p >= 0:
            sees[i] = sees[p]
            depth[i] = depth[p] + 1
        sees[i, i] = True
    return sees, depth


def visible(parents, prefix, window):
    anc, depth = ancestors(parents)
    sees = np.concatenate([np.ones((len(parents), prefix), bool), anc], 1)
    if window:
        place = np.concatenate([np.arange(prefix), prefix + depth])
        sees &= (prefix + depth)[:, None] - place[None, :] < window
    return sees


def attention(q, k, v, parents, prefix, n_kv, window=0, sinks=None, scale=None):
    """q [n, H, D], k / v [prefix + n, n_kv, D] in float64 -> (out [n, H, D], how far f32 arithmetic may be off it, per element).

    The bound: a score is a sum of D products in f32, |error| <= D 2^-24 scale sum |q k| =: e, and its exponential is off by 2 e + 2^-21 relative (the argument
    and 2^x itself); so is a weight's share of the denominator.  Sums over n keys add n 2^-24 at most.  Weights enter the products in two bf16 terms
    (bf16 results, 2^-16) or in three (f32 results, 2^-24).  All of it relative to sum w |v|."""
    n, heads, dim = q.shape
    scale = scale or 1.0 / math.sqrt(dim)
    sees = visible(parents, prefix, window)
    out, off = np.zeros((n, heads, dim)), np.zeros((n, heads, dim))
    for i in range(n):
        at = np.nonzero(sees[i])[0]
        for h in range(heads):
            kk, vv = k[at, h // (heads // n_kv)], v[at, h // (heads // n_kv)]
            x = scale * (kk @ q[i, h])
            top = max(x.max(), sinks[h]) if sinks is not None else x.max()
            w = np.exp(x - top)
            total = w.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0)
            out[i, h] = (w / total) @ vv
            e = dim * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(q[i, h])).max() + 2.0 ** -22 * np.abs(x).max()
            off[i, h] = (4 * e + 2.0 ** -20 + 2 * len(at) * 2.0 ** -24) * ((w / total) @ np.abs(vv))
    return out, off


def accept(tokens, parents, picks):
    """(path, next token) of one sequence."""
    if not len(parents):
        return [], -1
    path = [0]
    while True:
        at = path[-1]
        child = [i for i in range(at + 1, len(parents)) if parents[i] == at and tokens[i] == picks[at]]
        if not child:
            return path, int(picks[at])
        path.append(child[0])


def pick(row):
    """The greedy sample: the last maximum, NaN counting as -inf."""
    row = np.where(np.isnan(row), -np.inf, row)
    return int(len(row) - 1 - np.argmax(row[::-1]))


def random_parents(rng, n, kind="mixed"):
    if n == 0:
        return []
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":
        return [-1 if rng.random() < 0.4 else int(rng.integers(-1, i)) if i else -1 for i in range(n)]
    return [-1] + [i - 1 if rng.random() < 0.5 else int(rng.integers(0, i)) for i in range(1, n)]

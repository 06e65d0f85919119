"""Plain forms of decoding with drafted tokens and of sampling, in 64 bits."""
from __future__ import annotations

import numpy as np


def make_tree(rng, n: int, reach: int = 5, roots: float = 0.0) -> list:
    """Parents of n nodes, each among the `reach` nodes before it; others are roots too with that probability."""
    return [-1 if i == 0 or rng.random() < roots else int(rng.integers(max(0, i - reach), i)) for i in range(n)]


def depths(parents) -> list:
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def seen(parents, past: int, window: int = 0) -> np.ndarray:
    """[n, past + n]: the rows that each node sees."""
    n, depth = len(parents), depths(parents)
    out = np.zeros((n, past + n), bool)
    for t in range(n):
        out[t, max(0, past + depth[t] + 1 - window) if window else 0:past] = True
        a = t
        while a >= 0 and (not window or depth[t] - depth[a] < window):
            out[t, past + a] = True
            a = parents[a]
    return out


def rotate(x: np.ndarray, positions, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [n, h, d] by the tables' rows [position][d / 2]."""
    h = x.shape[-1] // 2
    c, s = cos[positions][:, None].astype(np.float64), sin[positions][:, None].astype(np.float64)
    a, b = x[..., :h].astype(np.float64), x[..., h:].astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def norm(x: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, visible: np.ndarray) -> np.ndarray:
    """q [n, hq, d] over keys, values [m, hkv, d], visible [n, m]; what a node does not see takes no part."""
    n, hq, d = q.shape
    hkv = keys.shape[1]
    out = np.empty((n, hq, d))
    for t in range(n):
        at = np.nonzero(visible[t])[0]
        k = np.repeat(keys[at].astype(np.float64), hq // hkv, axis=1)
        v = np.repeat(values[at].astype(np.float64), hq // hkv, axis=1)
        s = np.einsum("hd,mhd->hm", q[t].astype(np.float64), k) / np.sqrt(d)
        p = np.exp(s - s.max(1, keepdims=True))
        out[t] = np.einsum("hm,mhd->hd", p / p.sum(1, keepdims=True), v)
    return out


def accept(parents, tokens, sampled):
    """(path, next) of one sequence's walk."""
    path = [0]
    while True:
        want = sampled[path[-1]]
        more = [t for t in range(len(parents)) if parents[t] == path[-1] and tokens[t] == want and want >= 0]
        if not more:
            return path, want
        path.append(more[0])


def sample(x: np.ndarray, u: float, temperature: float, top_k: int, top_p: float, min_p: float):
    """(token, probability, distance of u from the next border) of one row."""
    x = x.astype(np.float64)
    n = len(x)
    temperature, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if temperature == 0:
        return int(np.argmax(x)), 1.0, 1.0
    w = np.exp((x - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < n:
        order = order[:top_k]
    if top_p < 1:
        run = np.cumsum(w[order])
        order = order[:max(1, int(((run - w[order]) < top_p * run[-1]).sum()))]
    index = np.sort(order[w[order] >= min_p])
    run = np.cumsum(w[index])
    j = min(int(np.searchsorted(run, u * run[-1], side="right")), len(index) - 1)
    return int(index[j]), float(w[index[j]] / run[-1]), float(np.abs(run / run[-1] - u).min())

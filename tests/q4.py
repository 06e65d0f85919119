"""Plain forms of the 4-bit operators for the tests: the cache's format in numpy
float32 (whose operations round as the format's do) and the attention in 64 bits."""
from __future__ import annotations

import numpy as np

GROUP = 32


def hold(x: np.ndarray) -> np.ndarray:
    """The values that rows [..., d] stand for once held in 4 bits, bit for bit."""
    g = np.asarray(x, np.float32).reshape(-1, GROUP)
    lo, hi = g.min(1), g.max(1)
    low = lo.astype(np.float16).astype(np.float32)
    step = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(step > 0, np.float32(1) / step, np.float32(0))
    code = np.clip(np.rint((g - low[:, None]) * inv[:, None]), 0, 15).astype(np.uint8)  # (a whole number: no zero has a sign)
    return (low[:, None] + step[:, None] * code.astype(np.float32)).astype(np.float32).reshape(np.shape(x))


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, causal: bool = True, window: int = 0) -> np.ndarray:
    """q [s, hq, d]: the queries of the last s of the rows keys, values [n, hkv, d]; float64."""
    s, hq, d = q.shape
    n, hkv = keys.shape[:2]
    pos = np.arange(n - s, n)[:, None]
    key = np.arange(n)[None, :]
    hidden = (key > pos) if causal else np.zeros((s, n), bool)
    if window:
        hidden = hidden | (key + window <= pos)
    out = np.empty((s, hq, d))
    for h in range(hq):
        k, v = keys[:, h * hkv // hq].astype(np.float64), values[:, h * hkv // hq].astype(np.float64)
        sc = q[:, h].astype(np.float64) @ k.T / np.sqrt(d)
        sc[hidden] = -np.inf
        p = np.exp(sc - sc.max(1, keepdims=True))
        out[:, h] = (p / p.sum(1, keepdims=True)) @ v
    return out

"""The paged 4-bit cache in 64-bit numpy, from its definition: the 4-bit values,
the norm and rotation, and attention under a window with sinks."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def exponent_range(prec: str):
    return (-23, 13) if prec in ("f16", "int8") else (-64, 64)


def quantize(x: np.ndarray, prec: str) -> np.ndarray:
    """Values (..., 128), rounded to f32 first, as the 4 bits keep them."""
    x = x.astype(np.float32).astype(np.float64)
    b = x.reshape(*x.shape[:-1], 4, 32)
    m = np.abs(b).max(-1, keepdims=True)
    lo, hi = exponent_range(prec)
    with np.errstate(divide="ignore", invalid="ignore"):
        frac, e = np.frexp(m)                     # m = frac 2^e, frac in [0.5, 1)
    e = np.where(frac * 8 > 7, e - 2, e - 3)      # smallest e with m <= 7 2^e
    e = np.clip(e, lo, hi)
    t = np.minimum(np.abs(b) / np.exp2(e), 6.0)
    # nearest level; of two equally near ones the one with the even index
    d = np.abs(t[..., None] - LEVELS)
    order = [0, 2, 4, 6, 1, 3, 5, 7]
    i = np.array(order)[np.argmin(d[..., order], -1)]
    return (np.sign(b) * LEVELS[i] * np.exp2(e)).reshape(x.shape)


def norm_rope(x: np.ndarray, gain: np.ndarray, cos: np.ndarray, sin: np.ndarray, eps: float) -> np.ndarray:
    """x (rows, heads, 128), cos and sin (rows, 64)."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    c, s = cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    lo, hi = y[..., :64], y[..., 64:]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


def rope_tables(n: int, theta: float, dtype):
    """The decoder's tables: f32 angles, cosine and sine rounded to the
    activation dtype (a torch dtype), as float64."""
    import torch

    inv = (1.0 / np.power(theta, np.arange(0, 128, 2) / 128.0)).astype(np.float32)
    a = np.arange(n, dtype=np.float32)[:, None] * inv[None]
    out = []
    for f in (np.cos, np.sin):
        t = torch.from_numpy(f(a.astype(np.float64)).astype(np.float32)).to(dtype)
        out.append(t.double().numpy())
    return out


def visible(n_keys: int, positions: np.ndarray, window: int, sinks: int) -> np.ndarray:
    j, p = np.arange(n_keys)[None], np.asarray(positions)[:, None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, positions, window: int = 0, sinks: int = 0):
    """q (rows, nh, 128) at positions over k, v (keys, nkv, 128)."""
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    rep = q.shape[1] // k.shape[1]
    seen = visible(k.shape[0], positions, window, sinks)
    out = np.empty_like(q)
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // rep].T / np.sqrt(128.0)
        s[~seen] = -np.inf
        s -= s.max(-1, keepdims=True)
        p = np.exp(s)
        vv = v[:, h // rep]
        with np.errstate(invalid="ignore"):
            out[:, h] = (p / p.sum(-1, keepdims=True)) @ np.where(seen.any(0)[:, None], vv, 0.0)
    return out

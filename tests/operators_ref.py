"""Plain 64-bit forms of the shared-prefix, weights, eviction and rotary
operators, and the error bounds of the kernels against them (test code only).

Bounds. With u = eps / 2 of the element type (one rounding), w = 2^-24 (one
fp32 rounding), D the head size and n a row's tokens:
  scores        products of 16-bit values are exact in fp32, their sums are off
                by at most D w sum |q_d k_d|; scaling and the exponent's
                arithmetic round numbers of at most |s| + 32 a few times
                (s in log2 units): ds = scale log2e D w sum |q k| + 8 (|s| + 32) w
  probability   relative: dp = 2 ln2 ds (its score and the normaliser) + 16 w
  output        u |o| + (dp + p_err + (n + 64) w) sum p |v|, and in fp16 what
                probabilities below its smallest normal lose, n 2^-25 max |v|;
                p_err: the probabilities' rounding for the matrix units, u^2
                for two terms
  weight        (dp + (columns + 4) w) of the sum, and w of the total
"""
from __future__ import annotations

import math

import numpy as np
import torch

W = 2.0 ** -24
LOG2E = 1.4426950408889634


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def row_cache(pool_t: torch.Tensor, layer: int, pages, n: int) -> np.ndarray:
    """Row's cache [heads, n, dim] in 64 bits from a host copy of a pool."""
    t = pool_t[torch.as_tensor(list(pages), dtype=torch.int64), layer].double().numpy()
    h, d = t.shape[1], t.shape[3]
    return t.transpose(1, 0, 2, 3).reshape(h, -1, d)[:, :n]


def attend(q, k, v, scale, dtype, p_err=None, valid=None):
    """q [t, Hq, D] (the last t positions), k/v [Hkv, n, D], all float64 ->
    out [t, Hq, D], its bound, probabilities [t, Hq, n], their relative bound."""
    t, hq, d = q.shape
    hkv, n, _ = k.shape
    ratio = hq // hkv
    u = half_step(dtype)
    p_err = u * u if p_err is None else p_err
    kk, vv = np.repeat(k, ratio, axis=0), np.repeat(v, ratio, axis=0)
    s = np.einsum("thd,hnd->thn", q, kk) * (scale * LOG2E)
    mag = np.einsum("thd,hnd->thn", np.abs(q), np.abs(kk)) * (scale * LOG2E)
    hidden = np.arange(n)[None, :] > (n - t + np.arange(t))[:, None]
    if valid is not None:
        hidden = hidden | ~valid[None, :]
    s = np.where(hidden[:, None, :], -np.inf, s)
    top = s.max(-1, keepdims=True) if n else np.zeros((t, hq, 1))
    dead = ~np.isfinite(top)
    e = np.exp2(s - np.where(dead, 0.0, top))
    total = e.sum(-1, keepdims=True)
    p = np.where(total > 0, e / np.where(total > 0, total, 1.0), 0.0)
    shown = np.where(hidden[:, None, :], 0.0, mag)
    ds = (D_err(d) * shown + 8 * (np.abs(np.where(np.isfinite(s), s, 0.0)) + 32) * W).max(
        -1, initial=0.0)
    dp = 2 * math.log(2) * ds + 16 * W                       # [t, hq]
    out = np.einsum("thn,hnd->thd", p, vv)
    mass = np.einsum("thn,hnd->thd", p, np.abs(vv))
    tol = u * np.abs(out) + (dp[..., None] + p_err + (n + 64) * W) * mass
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -25 * (np.abs(vv).max(1, initial=0.0)[None] if n else 0.0)
        tol = tol + 2.0 ** -25      # the output's own subnormals
    return out, tol, p, dp


def D_err(d: int) -> float:
    return d * W


def add_weights(w_old, p, dp, q_len, window, ratio):
    """w_old [Hkv, n] -> new weights and their bound, from p [q_len, Hq, n]."""
    t, hq, n = p.shape
    seen = p[max(0, t - window):]
    err = dp[max(0, t - window):]
    cols = seen.shape[0] * ratio
    g = seen.reshape(seen.shape[0], hq // ratio, ratio, n)
    eg = err.reshape(seen.shape[0], hq // ratio, ratio, 1)
    got = g.sum((0, 2))
    tol = (g * eg).sum((0, 2)) + (cols + 4) * W * got
    old = np.array(w_old, dtype=np.float64)
    old[:, n - q_len:] = 0.0
    # a probability below 2^-126 of the largest is 0 in fp32
    return old + got, tol + 2 * W * np.abs(old + got) + 2.0 ** -120


def choose(w, keep, sinks, recent):
    """Indices that stay of w [n] (float32), in order."""
    n = len(w)
    keep = min(keep, n)
    if keep >= n:
        return np.arange(n)
    lo = min(sinks, keep)
    rec = min(recent, keep - lo)
    mid = np.arange(lo, n - rec)
    vals = np.where(np.isnan(w[mid]), -np.inf, w[mid].astype(np.float64))
    isnan = np.isnan(w[mid])
    order = np.lexsort((mid, -vals, isnan))
    best = mid[order[:keep - lo - rec]]
    return np.sort(np.concatenate([np.arange(lo), best, np.arange(n - rec, n)])).astype(np.int64)


def rotate(x, pos, freq, scale, interleave):
    """x [t, H, D] float64 rotated at pos [t]; freq [R / 2]."""
    r = 2 * len(freq)
    ang = np.asarray(pos, dtype=np.float64)[:, None] * np.asarray(freq)[None, :]
    c, s = np.cos(ang)[:, None, :] * scale, np.sin(ang)[:, None, :] * scale
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleave else (slice(0, r // 2), slice(r // 2, r))
    y = np.array(x, dtype=np.float64)
    xa, xb = np.array(x[..., a], dtype=np.float64), np.array(x[..., b], dtype=np.float64)
    y[..., a] = xa * c - xb * s
    y[..., b] = xb * c + xa * s
    mag = np.zeros_like(y)
    mag[..., a] = mag[..., b] = (np.abs(xa) + np.abs(xb)) * abs(scale)
    return y, mag

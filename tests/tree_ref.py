"""Drafted trees in 64 bits: helpers of their tests (test code only)."""
from __future__ import annotations

import math

import numpy as np
import torch


def random_tree(rng, n: int, fan: int, roots: int = 1) -> list:
    """Parents of n tokens: the first `roots` follow the cache, each other one token of
    the `fan` before it."""
    return [-1 if i < roots else int(rng.integers(max(0, i - fan), i)) for i in range(n)]


def ancestors(parents) -> np.ndarray:
    """[n, n]: whether token i sees drafted token j."""
    sees = np.zeros((len(parents), len(parents)), dtype=bool)
    for i in range(len(parents)):
        j = i
        while j >= 0:
            sees[i, j] = True
            j = parents[j]
    return sees


def random_pages(rng, lens, page_size: int, spare: int = 3) -> tuple:
    """(page lists of rows of these lengths, pages of the pool)."""
    need = [-(-int(n) // page_size) for n in lens]
    total = sum(need) + spare
    ids = iter(rng.permutation(total).tolist())
    return [[next(ids) for _ in range(n)] for n in need], total


def tokens_of(pool_tensor: torch.Tensor, layer: int, pages, n: int) -> torch.Tensor:
    """A row's n cached tokens [heads, n, dim] of a layer."""
    if not pages:
        return pool_tensor[:0, layer].transpose(0, 1).flatten(1, 2)
    ids = torch.tensor(pages, device=pool_tensor.device)
    return pool_tensor[ids, layer].transpose(0, 1).flatten(1, 2)[:, :n]


def tree_attention_ref(q, k, v, parents, scale: float, dropped=None) -> tuple:
    """o [n, Hq, D] and sum of p |v| (what roundings of p and of scores go with), in 64
    bits: q [n, Hq, D], k and v [Hkv, prefix + n, D], its drafted tokens last. dropped
    (bool [prefix + n]): tokens that nobody sees."""
    n, hq, d = q.shape
    hkv, kv = k.shape[0], k.shape[1]
    hidden = np.zeros((n, kv), dtype=bool)
    hidden[:, kv - n:] = ~ancestors(parents)
    if dropped is not None:
        hidden |= dropped
    hidden = torch.tensor(hidden, device=q.device)
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    mass = torch.empty_like(out)
    for h in range(hq):
        g = h // (hq // hkv)
        s = q[:, h].double() @ k[g].double().t().contiguous() * scale
        p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
        # A masked token has no weight, whatever its V is.
        vals = torch.nan_to_num(v[g].double(), nan=0.0, posinf=0.0, neginf=0.0)
        out[:, h] = p @ vals
        mass[:, h] = p @ vals.abs()
    return out, mass


def check_out(out, ref, mass, what="") -> None:
    """The output's one rounding (half a step), and 2^-12 of sum p |v|: what fp32 sums of
    256 products do to a score below 64 (256 * 2^-24 * 32 = 2^-11 / 2 of a probability, its
    two 16-bit terms 2^-16)."""
    err = (out.double() - ref).abs()
    bound = ref.abs() * (torch.finfo(out.dtype).eps / 2) + mass * 2.0 ** -12
    bad = ~(err <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((err - bound).max()), bad.nonzero()[:4].tolist())

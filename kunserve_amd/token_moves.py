"""Cached tokens that change their place: keep_tokens moves those of a row that stay
together, in place; fork_rows continues rows in page lists of their own.

The reference moves whole blocks alone (LlamaOp.local_copy_blocks,
kunserve/worker.py:818-823).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import numpy as np
import torch

from . import _lib
from .paged_kv import KVPool, PageTable, _i32, _stream_ptr, _upload, csr_from_lists


def keep_tokens(pool: KVPool, table: PageTable, first: Union[int, Sequence[int]], kept,
                weights=None) -> None:
    """Of each row's cached tokens from place first[b] on (one number, or one per row)
    those at first[b] + kept[b][j] stay and come to first[b] + j, in every layer and KV
    head, in place; the row goes on with first[b] + len(kept[b]) tokens, and its last
    pages are the caller's to free once the stream has passed this call. Tokens keep
    the rotary positions they were cached with (AttentionStep(rope_positions=...)).

    kept: per row a rising list, or a device int32 tensor [rows, most kept] with -1
    behind a row's last. An entry of a tensor that is not above its own place j or
    lies past the row's end moves nothing. weights (a KVWeights of the pool) move
    along. The pages from first[b] on must be in one place of the table
    (ValueError). Not for a graph capture, which takes AttentionStep.keep_tokens."""
    n = table.num_seqs
    given = np.asarray(first)
    if given.dtype.kind not in "iu" or given.shape not in ((), (n,)):
        raise ValueError(f"first must be a whole number, or one per row ({n})")
    lens = table.kv_len_host
    out = (given < 0) | (given > lens)
    if out.any():
        bad = int(np.argmax(out))
        raise ValueError(f"row {bad}: first place {int(given.reshape(-1)[bad % given.size])} of "
                         f"{int(lens[bad])} tokens")
    starts = np.empty(n, dtype=np.int32)
    starts[:] = given
    if pool.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("keep_tokens is not for a graph capture: AttentionStep.keep_tokens is")
    moving = np.zeros(n + 1, dtype=np.int32)
    np.cumsum(lens - starts, out=moving[1:])
    ids = table.indices_host if table.indices_host.size else moving   # (there is one)
    if not _lib.call("kunserve_new_pages_private", table.indptr_host.ctypes.data,
                     ids.ctypes.data, moving.ctypes.data, table.kv_len_host.ctypes.data, n,
                     pool.page_size, pool.num_pages):
        raise ValueError("tokens move in place: their pages must be in one place of the table")
    move_tokens(pool, table, None, starts, kept, weights)


def move_tokens(pool: KVPool, table: PageTable, first: Optional[torch.Tensor],
                first_host: np.ndarray, kept, weights) -> None:
    """kunserve_keep_tokens for rows whose pages the caller has checked; first:
    first_host on the device, if it is there."""
    n, device = table.num_seqs, pool.device
    if weights is not None:
        weights.check(pool)
    if isinstance(kept, torch.Tensor):
        if (kept.dtype != torch.int32 or kept.dim() != 2 or kept.shape[0] != n
                or kept.device != device or (kept.shape[1] > 1 and kept.stride(1) != 1)
                or (n > 1 and kept.stride(0) < kept.shape[1])):
            raise ValueError(f"kept must be int32 [{n}, most kept] on {device}, its rows apart and "
                             "contiguous")
        width, stride = kept.shape[1], max(kept.stride(0), kept.shape[1])
    else:
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("lists cannot be captured: kept is to be a device tensor")
        kept = _kept_rows(kept, table.kv_len_host - first_host)
        width = stride = kept.shape[1]
    if n == 0 or width == 0:
        return
    here = None
    if first is None and n <= _lib.FIRST_BY_VALUE:
        first_host = _i32(first_host)
        here = first_host.ctypes.data
        if not isinstance(kept, torch.Tensor):
            kept = _upload(kept, device)
    elif not isinstance(kept, torch.Tensor) and first is None:
        both = _upload(np.concatenate([_i32(first_host), kept.reshape(-1)]), device)
        first, kept = both[:n], both[n:]
    elif first is None:
        first = _upload(_i32(first_host), device)
    elif not isinstance(kept, torch.Tensor):
        kept = _upload(kept, device)
    _lib.call("kunserve_keep_tokens", pool.desc(),
              None if weights is None else ctypes.byref(weights._desc), table.desc(), here,
              None if here is not None else first.data_ptr(), kept.data_ptr(), stride, width,
              _stream_ptr(device))


def _kept_rows(kept: Sequence[Sequence[int]], lens: np.ndarray) -> np.ndarray:
    """Lists of kept places, checked, as an int32 array with -1 behind a row's last."""
    if len(kept) != len(lens):
        raise ValueError(f"{len(lens)} rows but {len(kept)} lists of kept tokens")
    out = np.full((len(kept), max(map(len, kept), default=0)), -1, dtype=np.int32)
    for b, places in enumerate(kept):
        p = np.asarray(places)
        if p.ndim != 1 or (p.size and p.dtype.kind not in "iu"):
            raise ValueError(f"row {b}: kept places are whole numbers")
        if p.size and (p[0] < 0 or p[-1] >= lens[b] or np.any(p[1:] <= p[:-1])):
            raise ValueError(f"row {b}: kept places must rise within its {int(lens[b])} tokens")
        out[b, :p.size] = p
    return out


def fork_rows(pool: KVPool, pages_of_reqs: Sequence[Sequence[int]], kv_lens: Sequence[int],
              pages_out: Sequence[Sequence[int]], weights=None) -> None:
    """Continues each row's kv_lens[b] cached tokens in the page list pages_out[b]: places
    where both lists have the same page stay shared, of every other page the tokens in
    use are copied, in every layer and KV head. Samples or beams of one request: its list
    once for each, pages_out with the whole pages it shares and a page of its own for the
    last tokens; a request that moves: other pages throughout.

    Both lists hold ceil(kv_lens[b] / page_size) pages at least; further ones are not
    touched. A page that is copied to holds no row's cached tokens and is in one place of
    pages_out (ValueError). weights (a KVWeights of the pool) are copied along. Its table
    is built on the host: not for a graph capture."""
    n = len(kv_lens)
    if len(pages_of_reqs) != n or len(pages_out) != n:
        raise ValueError(f"{n} kv lengths but {len(pages_of_reqs)} and {len(pages_out)} page lists")
    if weights is not None:
        weights.check(pool)
    lens = np.asarray(kv_lens)
    if n and (lens.ndim != 1 or lens.dtype.kind not in "iu" or lens.min() < 0
              or lens.max() > 2**31 - 1):
        raise ValueError("kv_lens count tokens: whole numbers, 0 at least")
    if pool.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("fork_rows cannot be captured: its table is built on the host")
    lens = lens.astype(np.int64)
    indptr, indices = csr_from_lists([*pages_of_reqs, *pages_out], np.concatenate([lens, lens]),
                                     pool.page_size, pool.num_pages)
    moves = np.empty((indices.size // 2, 3), dtype=np.int32)
    lens = _i32(lens)
    try:
        count = _lib.call("kunserve_fork_moves", indptr.ctypes.data, indices.ctypes.data,
                          lens.ctypes.data, n, pool.page_size, pool.num_pages,
                          moves.ctypes.data, len(moves))
    except _lib.KunserveError as e:
        if e.code != _lib.EINVAL:
            raise
        raise ValueError(e.detail) from None
    if count == 0:
        return
    here = there = None
    if count <= _lib.MOVES_BY_VALUE:
        here = moves.ctypes.data
    else:
        on_device = _upload(moves[:count], pool.device)
        there = on_device.data_ptr()
    _lib.call("kunserve_copy_pages", pool.desc(),
              None if weights is None else ctypes.byref(weights._desc), here, there, count,
              _stream_ptr(pool.device))

"""What attention says of the cache, and the cache made shorter by it.

KVWeights holds, for every cached token and KV head, the attention weight that
it got so far; steps made with it (AttentionStep(weights=...)) add to it. evict
keeps the heaviest tokens of a request in pages of their own. The reference has
no counterpart: its block manager frees whole requests
(kunserve/block_manager.py:493-500).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Union

import numpy as np
import torch

from . import _lib
from .paged_kv import (KVPool, PageTable, _check_reach, _check_row_map, _i32, _ptr, _stream_ptr,
                       _tensor3, _upload, _upload_packed, csr_from_lists)


class KVWeights:
    """Accumulated attention weights of a pool's tokens: w [num_pages, num_layers,
    num_kv_heads, page_size], float32 with the slots contiguous. A new token's
    weight starts at 0 in the step that appends it, if the step was given these
    weights (learn=False where it is to learn nothing, as where its rows share
    pages); what other steps and ops append keeps the weights that the page's last
    user left until clear. The weights are those of one pool: of its fused views, or of
    the pool after a pmm drop or restore, they are others; copies of pages leave
    them behind.

    score_bytes: what a step may hold in scores that its decode launch leaves for the
    weights, 4 bytes per cached token and query head; rows beyond it have their K
    read twice more (at 1 / 128 of the bytes)."""

    def __init__(self, pool: KVPool, w: Optional[torch.Tensor] = None,
                 score_bytes: int = 256 << 20):
        shape = (pool.num_pages, pool.num_layers, pool.num_kv_heads, pool.page_size)
        if w is None:
            w = torch.zeros(shape, dtype=torch.float32, device=pool.device)
        # Every element in a place of its own: by stride, each dim past the ones below.
        reach, apart = 1, True
        for step, size in sorted(zip(w.stride(), w.shape)):
            apart &= size <= 1 or step >= reach
            reach = max(reach, step * (size - 1) + reach)
        if not apart:
            raise ValueError("weights must not share memory among themselves")
        if (tuple(w.shape) != shape or w.dtype != torch.float32 or w.stride(-1) != 1
                or w.device != pool.device):
            raise ValueError(f"weights must be float32 {shape} on {pool.device} with the slots "
                             "contiguous")
        self.w = w
        self.score_bytes = score_bytes
        self._desc = _lib.KVWeights(w.data_ptr(), w.stride(0), w.stride(1), w.stride(2))

    def check(self, pool: KVPool) -> None:
        shape = (pool.num_pages, pool.num_layers, pool.num_kv_heads, pool.page_size)
        if tuple(self.w.shape) != shape or self.w.device != pool.device:
            raise ValueError(f"the weights {tuple(self.w.shape)} on {self.w.device} are not those "
                             f"of a pool {shape} on {pool.device}")

    def plan(self, q_indptr_host, kv_len_host, num_qo_heads: int, window: int,
             decodes: Optional[Sequence[int]] = None) -> "WeightsPlan":
        """The plan of a step's rows, not yet on the device (WeightsPlan.bind)."""
        if decodes is not None:
            marks = np.asarray(decodes, dtype=bool)
            if marks.shape != (len(kv_len_host),):
                raise ValueError(f"{len(kv_len_host)} rows but {marks.shape} decode marks")
            held = np.cumsum(np.where(marks, np.asarray(kv_len_host, dtype=np.int64), 0))
            decodes = marks.astype(np.int32) + (marks & (4 * num_qo_heads * held > self.score_bytes))
        return WeightsPlan(q_indptr_host, kv_len_host, num_qo_heads, window, self.w.device,
                           upload=False, decodes=decodes)

    def clear(self, pool: KVPool, table: PageTable, q_indptr: torch.Tensor,
              num_tokens: int) -> None:
        """The weights of a step's new tokens become 0 in every layer
        (kunserve_clear_weights): num_tokens of q_indptr's (device int32 [num_seqs +
        1]) rows, the last of the table's."""
        self.check(pool)
        _check_row_map(q_indptr, table.num_seqs + 1, pool.device, "q_indptr")
        _lib.call("kunserve_clear_weights", pool.desc(), ctypes.byref(self._desc), table.desc(),
                  q_indptr.data_ptr(), num_tokens, _stream_ptr(pool.device))

    def add(self, pool: KVPool, layer: int, table: PageTable, q_indptr: torch.Tensor,
            q: torch.Tensor, plan: "WeightsPlan", sm_scale: Optional[float] = None,
            workspace: Optional[torch.Tensor] = None) -> None:
        """add_weights to these weights."""
        add_weights(pool, self, layer, table, q_indptr, q, plan, sm_scale, workspace)


class WeightsPlan:
    """Work of add_weights for a step's rows, computed on the host once per step and
    shared by every layer (kunserve_weights_plan). decodes marks the rows whose
    decode launch leaves its scores for the weights (AttentionStep's) with 1;
    add_weights passes over them, not over other decode rows, marked 2. The workspace
    is laid out by q_indptr, so the kernels read the plan's copy of it."""

    def __init__(self, q_indptr_host: Sequence[int], kv_len_host: Sequence[int],
                 num_qo_heads: int, window: int, device: torch.device, upload: bool = True,
                 decodes: Optional[Sequence[int]] = None):
        qi, kv = _i32(q_indptr_host), _i32(kv_len_host)
        n = len(kv)
        if len(qi) != n + 1:
            raise ValueError("q_indptr must have num_seqs + 1 entries")
        kv_ptr = kv.ctypes.data if n else None
        cap = int(_lib.lib().kunserve_weights_plan_bound(qi.ctypes.data, kv_ptr, n, num_qo_heads,
                                                         window))
        buf = np.empty(max(cap, 4), dtype=np.int32)   # the plan writes what it uses
        self.info = _lib.WeightsPlanInfo()
        self.kv_len_host, self.q_indptr_host = kv, qi.copy()
        marks = None if decodes is None else _i32(decodes)
        if marks is not None and marks.shape != (n,):
            raise ValueError(f"{n} rows but {marks.shape} decode marks")
        _lib.call("kunserve_weights_plan", qi.ctypes.data, kv_ptr, n, num_qo_heads, window,
                  None if marks is None else marks.ctypes.data, buf.ctypes.data, buf.size, ctypes.byref(self.info))
        self.plan_host = buf[: self.info.plan_ints].copy()
        self.plan = self.q_indptr = None
        if upload:
            self.bind(_upload_packed(self.host_arrays(), device))

    def host_arrays(self) -> list:
        return [self.plan_host, self.q_indptr_host]

    def bind(self, dev: Sequence[torch.Tensor]) -> None:
        self.plan = dev[0] if self.info.plan_ints else None
        self.q_indptr = dev[1]

    def workspace_bytes(self) -> int:
        return int(_lib.lib().kunserve_weights_workspace_bytes(ctypes.byref(self.info)))


def add_weights(pool: KVPool, weights: KVWeights, layer: int, table: PageTable,
                q_indptr: torch.Tensor, q: torch.Tensor, plan: WeightsPlan,
                sm_scale: Optional[float] = None,
                workspace: Optional[torch.Tensor] = None) -> None:
    """Adds to `weights` what the last new tokens of every row attend to
    (kunserve_cache_weights): q [num_tokens, Hq, D] after its rotation, the step's
    K in its pages. q_indptr (device int32 [num_seqs + 1]) is that of the plan, whose
    own copy is what the launches read. No page may be in two places of the table
    (ValueError)."""
    weights.check(pool)
    _check_reach(pool.device, q=q)
    if not np.array_equal(plan.kv_len_host, table.kv_len_host):
        raise ValueError("the plan was made for other rows than the table's")
    if not table.pages_private:
        raise ValueError("attention weights need pages that are in one place of the table")
    if q.shape[2] != pool.head_dim:
        raise ValueError(f"q shape {tuple(q.shape)} does not match head_dim {pool.head_dim}")
    _check_row_map(q_indptr, table.num_seqs + 1, pool.device, "q_indptr")
    if q.shape[0] < plan.q_indptr_host[-1]:
        raise ValueError(f"q has {q.shape[0]} tokens, the plan's rows end at "
                         f"{plan.q_indptr_host[-1]}")
    if plan.q_indptr is None:
        raise RuntimeError("weights plan used before its device arrays were bound")
    pool.check_dtype(q)
    scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(pool.head_dim)
    need = plan.workspace_bytes()
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=pool.device)
    qd = _tensor3(q)
    _lib.call("kunserve_cache_weights", pool.desc(), ctypes.byref(weights._desc), layer,
              table.desc(), plan.q_indptr.data_ptr(), ctypes.byref(qd), q.shape[1],
              ctypes.c_float(scale), _ptr(plan.plan), ctypes.byref(plan.info), _ptr(workspace),
              0 if workspace is None else workspace.numel() * workspace.element_size(),
              _stream_ptr(pool.device))


def evict(pool: KVPool, weights: KVWeights, pages_of_reqs: Sequence[Sequence[int]],
          kv_lens: Sequence[int], pages_out: Sequence[Sequence[int]],
          budget: Union[int, Sequence[int]], sinks: int = 4, recent: int = 0) -> torch.Tensor:
    """Shortens the cache of requests to `budget` tokens each (one number, or one
    per request; a request that has no more keeps all): in every layer and KV head
    the first `sinks`, the last `recent` and the heaviest of the tokens between
    stay (equal weights: the lowest index), in their order. Their K, V and weights
    are copied to pages_out, ceil(tokens / page_size) pages per request that are
    no pages of the requests; the old pages are the caller's to free once the
    stream has passed this call.

    Every cached token's weight counts: those appended by steps without the weights
    have to be cleared first (KVWeights).

    The shortened request goes on with min(budget, kv_len) cached tokens, its
    positions where they were (AttentionStep(rope_positions=...)). Returns the
    indices kept, int32 [requests, layers, kv_heads, most kept], -1 behind a
    request's last. The tables are built on the host: not for a graph capture."""
    weights.check(pool)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("evict cannot be captured: its tables are built on the host")
    n = len(kv_lens)
    if len(pages_of_reqs) != n or len(pages_out) != n:
        raise ValueError(f"{n} kv lengths but {len(pages_of_reqs)} and {len(pages_out)} page lists")
    kv = [int(x) for x in kv_lens]
    budget = np.asarray(budget) if n else np.zeros((), dtype=np.int64)
    if budget.dtype.kind not in "iu":
        raise ValueError("budget counts tokens: whole numbers")
    if budget.shape not in ((), (n,)):
        raise ValueError(f"budget must be one number or one per request ({n})")
    budgets = budget.tolist() if budget.shape else [int(budget)] * n
    keep = list(map(min, budgets, kv))   # what stays of the requests
    # a negative length or budget is the least of a request's
    if sinks < 0 or recent < 0 or min(keep, default=0) < 0:
        raise ValueError("budget, kv_lens, sinks and recent must not be negative")
    longest, most = max(kv, default=0), max(keep, default=0)
    limit = 2**31 - 1   # tokens of a request are counted in int32
    if longest > limit:
        raise ValueError(f"a request of over {limit} tokens")
    kept = torch.empty((n, pool.num_layers, pool.num_kv_heads, most), dtype=torch.int32,
                       device=pool.device)
    if most == 0:
        return kept
    # one table: the requests' pages, then those that are filled
    lens = np.array(kv + keep, dtype=np.int64)
    indptr, indices = csr_from_lists([*pages_of_reqs, *pages_out], lens, pool.page_size,
                                     pool.num_pages)
    out = indices[indptr[n]:]
    use = np.zeros(pool.num_pages, dtype=np.int8)
    use[indices[:indptr[n]]] = 1
    if use[out].any():
        raise ValueError(f"page {int(out[use[out] != 0][0])} of pages_out holds tokens of the "
                         "requests")
    use[out] = 2
    if np.count_nonzero(use == 2) != out.size:
        raise ValueError("a page is twice in pages_out")
    tables = _upload(np.concatenate((indptr, lens, indices), dtype=np.int32, casting="unsafe"),
                     pool.device)
    at = tables.data_ptr()
    lengths = at + 4 * (2 * n + 1)
    ids = lengths + 4 * 2 * n
    table = _lib.PageTable(at, ids, lengths, n)
    _lib.call("kunserve_evict", pool.desc(), ctypes.byref(weights._desc), ctypes.byref(table),
              at + 4 * n, ids, lengths + 4 * n, most, longest,
              min(sinks, limit), min(recent, limit), kept.data_ptr(), most,
              _stream_ptr(pool.device))
    return kept

"""Performance cases of the operators around drafted trees of tokens: their
attention, what of them the cache keeps, rows that go on from one another, and
rotary positions on several axes.

Kinds of case
  tree     AttentionStep.run over `layers` layers of a step whose rows verify
           drafted trees (trees=): append of the new K/V, then attention in
           which a drafted token sees the row's cache and its own ancestors.
  keep     AttentionStep.keep_tokens: of every row's drafted tokens the accepted
           ones moved behind its cache, in place, in every layer and KV head.
  shorten  keep_tokens on rows as they are: a rising list of cached tokens
           stays, the same in every layer.
  fork     fork_rows: rows continued in page lists of their own; pages listed
           alike stay shared, of the others the tokens in use are copied.
  axes     rotary_append_kv with a Rotary of several axes: pairs turned by a
           time, a height or a width, and the append of k and v.

Where `own` is false the same is computed by elementary torch operations in 32
bits (angles in 64) on padded rows. Row lengths and trees belong to the case
(its `lens` number); tensors and page tables come from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = torch.device("cuda", 0)


def listed() -> list:
    return [
        # One user's answer with a small draft: bound by latency and launches.
        dict(name="tree_one", kind="tree", layers=8, hq=32, hkv=8, dim=128, page=16, dtype="bf16",
             rows=1, t_lo=8, t_hi=8, fan=3, kv_lo=1500, kv_hi=1500, lens=1),
        # A batch of ragged contexts, each with a tree of its own size.
        dict(name="tree_batch", kind="tree", layers=2, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=32, t_lo=9, t_hi=32, fan=6, kv_lo=256, kv_hi=6000, lens=2),
        # Long documents under trees of 64 with 8 query heads to a KV head, on
        # the default 256-token pages: the largest, as much work as traffic.
        dict(name="tree_wide", kind="tree", layers=2, hq=64, hkv=8, dim=128, page=256,
             dtype="fp16", rows=8, t_lo=64, t_hi=64, fan=10, kv_lo=4000, kv_hi=16000, lens=3),
        # A model without GQA, head size 64.
        dict(name="tree_mha_dim64", kind="tree", layers=4, hq=32, hkv=32, dim=64, page=32,
             dtype="fp16", rows=21, t_lo=5, t_hi=27, fan=4, kv_lo=40, kv_hi=1800, lens=4),
        # The accepted path of one user's tree, in a model of 8 layers.
        dict(name="keep_one", kind="keep", layers=8, hq=32, hkv=8, dim=128, page=16, dtype="bf16",
             rows=1, t_lo=16, t_hi=16, fan=4, kv_lo=1500, kv_hi=1500, lens=5),
        # The same for a batch, every layer of a model.
        dict(name="keep_batch", kind="keep", layers=32, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=64, t_lo=20, t_hi=64, fan=8, kv_lo=30, kv_hi=300, lens=6),
        # Conversations cut to about half behind their first tokens, in place.
        dict(name="shorten_rows", kind="shorten", layers=8, hq=32, hkv=8, dim=128, page=16,
             dtype="fp16", rows=6, keep=500, sinks=100, kv_lo=2000, kv_hi=9000, lens=7),
        # Eight samples of one prompt that ends inside a page of 256: whole
        # pages shared, the last one each sample's own.
        dict(name="fork_samples", kind="fork", layers=32, hkv=8, dim=128, page=256, dtype="bf16",
             rows=8, apart=0, kv_lo=1100, kv_hi=1100, one=True, lens=8),
        # Rows that move to other pages whole.
        dict(name="fork_moves", kind="fork", layers=16, hkv=8, dim=128, page=16, dtype="fp16",
             rows=10, apart=1000, kv_lo=300, kv_hi=3500, one=False, lens=9),
        # Decoding rows of a model that sees images: one position on every axis.
        dict(name="axes_decode", kind="axes", hq=32, hkv=8, dim=128, page=16, dtype="bf16",
             rows=33, q_lo=1, q_hi=1, rotary=128, time=16, height=24, interleave=False,
             theta=1000000.0, far=30000, grid=0, lens=10),
        # Prompt chunks of image patches: a grid of heights and widths.
        dict(name="axes_images", kind="axes", hq=32, hkv=8, dim=128, page=256, dtype="bf16",
             rows=9, q_lo=400, q_hi=512, rotary=128, time=16, height=24, interleave=False,
             theta=1000000.0, far=20000, grid=30, lens=11),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["tree", "tree", "tree", "tree", "keep", "shorten", "fork", "axes"])
    ratio, hkv = rng.choice([(1, 32), (1, 16), (2, 8), (3, 8), (4, 8), (4, 8), (4, 4), (5, 8),
                             (6, 8), (7, 4), (8, 8), (8, 4)])
    dim = rng.choice([64, 128, 128, 128, 256])
    case = dict(kind=kind, hkv=hkv, dim=dim, page=rng.choice([16, 16, 32, 256]),
                dtype=rng.choice(["fp16", "bf16"]), lens=rng.randrange(1 << 20))
    if kind != "fork":
        case["hq"] = ratio * hkv
    if kind == "tree":
        hi, rows, t_hi = _log_int(rng, 40, 16000), _log_int(rng, 1, 64), _log_int(rng, 2, 130)
        # at most about the largest case's products and half its cached bytes
        while rows * hi * hkv * dim * max(ratio * t_hi, 128) > 3.2e10:
            if rows > 1:
                rows = rows * 2 // 3
            else:
                t_hi = max(2, t_hi * 2 // 3)
        case.update(rows=rows, t_lo=rng.choice([1, max(1, t_hi // 4), t_hi]), t_hi=t_hi,
                    fan=rng.choice([1, 3, 10, 200]), kv_lo=rng.choice([0, hi // 4, hi]), kv_hi=hi,
                    layers=rng.choice([1, 2]))
    elif kind == "keep":
        rows, t_hi, layers = _log_int(rng, 1, 64), _log_int(rng, 4, 130), rng.choice([2, 8, 16])
        while rows > 1 and rows * (300 + t_hi) * layers * hkv * dim > 3.2e8:
            rows = rows * 2 // 3
        case.update(rows=rows, t_lo=max(1, t_hi // 4), t_hi=t_hi, fan=rng.choice([3, 10, 40]),
                    kv_lo=0, kv_hi=300, layers=layers)
    elif kind == "shorten":
        hi, rows, layers = _log_int(rng, 64, 16384), _log_int(rng, 1, 12), rng.choice([2, 8, 16])
        while rows > 1 and rows * hi * layers * hkv * dim > 3.2e8:
            rows = rows * 2 // 3
        case.update(rows=rows, kv_lo=max(1, hi // rng.choice([1, 4])), kv_hi=hi,
                    keep=rng.choice([50, 250, 500, 900]), sinks=min(hi // 8, rng.choice([0, 4, 200])),
                    layers=layers)
    elif kind == "fork":
        hi, rows, layers = _log_int(rng, 30, 6000), _log_int(rng, 1, 24), rng.choice([2, 8, 32])
        while rows > 1 and rows * hi * layers * hkv * dim > 3e8:
            rows = rows * 2 // 3
        one = rng.random() < 0.5
        case.update(rows=rows, kv_lo=hi if one else max(1, hi // 4), kv_hi=hi, one=one,
                    apart=rng.choice([0, 0, 100, 500, 1000]), layers=layers)
    else:
        prompt, half = rng.random() < 0.5, rng.choice([dim, dim, dim // 2]) // 2
        q_hi = _log_int(rng, 2, 512) if prompt else 1
        time = rng.randrange(1, half // 2)
        case.update(rows=_log_int(rng, 1, 9 if prompt else 200), q_lo=max(1, q_hi // 2), q_hi=q_hi,
                    rotary=2 * half, time=time, height=(half - time) // 2,
                    interleave=rng.random() < 0.5, theta=rng.choice([10000.0, 1000000.0]),
                    far=_log_int(rng, 600, 1000000), grid=rng.choice([7, 16, 40]) if prompt else 0)
    return case


# ------------------------------------------------ rows, trees and page tables


def _rows(case) -> tuple:
    """(new tokens, cached tokens with them) of every row."""
    rng = np.random.default_rng(case["lens"])
    n, kind = case["rows"], case["kind"]
    if kind == "axes":
        q = rng.integers(case["q_lo"], case["q_hi"] + 1, size=n)
        return q, q + rng.integers(0, 600, size=n)
    kv = rng.integers(case["kv_lo"], case["kv_hi"] + 1, size=n)
    if kind in ("tree", "keep"):
        q = rng.integers(case["t_lo"], case["t_hi"] + 1, size=n)
        return q, kv + q
    return np.zeros(n, np.int64), kv


def _parents(case) -> list:
    """Every row's tree: each drafted token's parent among the row's tokens, -1
    for the first, which follows the cache."""
    rng = np.random.default_rng(case["lens"] + 1)
    return [[-1] + [int(rng.integers(max(0, i - case["fan"]), i)) for i in range(1, n)]
            for n in _rows(case)[0]]


def _kept(case) -> list:
    """Places that stay, counted from the row's first place of choice: the path
    to a drafted token, or a rising list of cached tokens."""
    rng = np.random.default_rng(case["lens"] + 2)
    if case["kind"] == "shorten":
        out = []
        for kv in _rows(case)[1]:
            n = max(0, int(kv) - case["sinks"])
            out.append(np.sort(rng.choice(n, size=n * case["keep"] // 1000, replace=False)))
        return [x.tolist() for x in out]
    out = []
    for parents in _parents(case):
        i, path = int(rng.integers(0, len(parents))), []
        while i >= 0:
            path.append(i)
            i = parents[i]
        out.append(path[::-1])
    return out


def _first(case) -> np.ndarray:
    """The place in its cache that a row's kept places count from."""
    ql, kv = _rows(case)
    return np.minimum(kv, case["sinks"]) if case["kind"] == "shorten" else kv - ql


def _same_pages(case) -> np.ndarray:
    """Leading pages that a fork shares with the row it goes on from: whole
    ones before the page of its last token, less those that lie apart."""
    whole = (_rows(case)[1] - 1) // case["page"]
    return whole - whole * case["apart"] // 1000


def _tables(case, seed: int) -> tuple:
    """Page lists of the rows, those that a fork continues them in, and the
    pages of the pool."""
    kv, page = _rows(case)[1], case["page"]
    need = -(-kv // page)
    fork = case["kind"] == "fork"
    sources = 1 if fork and case["one"] else case["rows"]
    more = need - _same_pages(case) if fork else np.zeros_like(need)
    total = int(need[:sources].sum() + more.sum())
    pages = total + total // 4 + 4
    ids = iter(np.random.default_rng(seed).permutation(pages).tolist())
    take = lambda n: [next(ids) for _ in range(n)]   # noqa: E731
    tables = [take(int(n)) for n in need[:sources]] * (case["rows"] // sources)
    out = [t[:len(t) - int(n)] + take(int(n)) for t, n in zip(tables, more)] if fork else []
    return tables, out, pages


# ---------------------------------------------------------------- prepare


def _padded(lists, width, fill=0, dtype=torch.int64) -> torch.Tensor:
    return torch.tensor([list(x) + [fill] * (width - len(x)) for x in lists], dtype=dtype,
                        device=DEVICE).view(len(lists), width)


def prepare(case, seed: int) -> dict:
    kind, dt, ps = case["kind"], DTYPES[case["dtype"]], case["page"]
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(shape, scale=1.0):
        return torch.empty(shape, dtype=dt, device=DEVICE).normal_(0.0, scale, generator=g)

    ql, kv = _rows(case)
    tables, out_tables, pages = _tables(case, seed)
    layers, tokens = case.get("layers", 1), int(ql.sum())
    shape = (pages, layers, case["hkv"], ps, case["dim"])
    width = max(1, max(len(t) for t in tables))
    s = dict(case=case, tables=tables, out_tables=out_tables, ql=ql.tolist(), kv=kv.tolist(),
             k_pool=normal(shape), v_pool=normal(shape), page_of=_padded(tables, width),
             ql_dev=torch.tensor(ql, device=DEVICE), kv_dev=torch.tensor(kv, device=DEVICE))
    if kind in ("tree", "axes"):
        # Scores have a standard deviation of 2, so rows attend unevenly.
        s.update(q=normal((layers, tokens, case["hq"], case["dim"]), 2.0),
                 k=normal((layers, tokens, case["hkv"], case["dim"])),
                 v=normal((layers, tokens, case["hkv"], case["dim"])))
    if kind in ("tree", "keep"):
        s["parents"] = _parents(case)
    if kind == "tree":
        most = max(s["ql"])
        sees = np.zeros((case["rows"], most, most), dtype=bool)
        for b, parents in enumerate(s["parents"]):
            for i, p in enumerate(parents):
                if p >= 0:
                    sees[b, i] = sees[b, p]
                sees[b, i, i] = True
        s["sees"] = torch.tensor(sees, device=DEVICE)
    elif kind in ("keep", "shorten"):
        kept = _kept(case)
        s.update(first=_first(case).tolist(),
                 kept=_padded(kept, max(1, max(len(x) for x in kept)), -1, torch.int32))
    elif kind == "fork":
        s["out_page_of"] = _padded(out_tables, width)
    elif kind == "axes":
        # A row's tokens from where its text ends: one position on every axis,
        # or the patches of an image, row by row of its grid.
        at = np.random.default_rng(case["lens"] + 1).integers(0, case["far"] + 1, size=len(ql))
        i = np.concatenate([np.arange(n) for n in ql])
        base, grid = np.repeat(at, ql), case["grid"]
        pos = np.stack([base, base + i // grid, base + i % grid] if grid else [base + i] * 3)
        s.update(pos=torch.tensor(pos, dtype=torch.int32, device=DEVICE),
                 q_out=torch.empty_like(s["q"][0]))
    if own:
        _handles(s, case)
    return s


def _sections(case) -> tuple:
    """Pairs turned by the time, the height and the width."""
    return case["time"], case["height"], case["rotary"] // 2 - case["time"] - case["height"]


def _handles(s, case) -> None:
    """What a user of the framework keeps: its pool, the step (made once per
    step and shared by its layers), the frequencies."""
    import kunserve_amd as ks

    s["pool"] = pool = ks.KVPool(s["k_pool"], s["v_pool"])
    if case["kind"] in ("tree", "keep"):
        first = [n - t for t, n in zip(s["ql"], s["kv"])]
        s["step"] = ks.AttentionStep(pool, case["hq"], s["ql"], first, [1] * len(first),
                                     s["tables"], trees=s["parents"])
    elif case["kind"] == "shorten":
        s["table"] = ks.PageTable.from_lists(s["tables"], s["kv"], pool)
    elif case["kind"] == "axes":
        s["table"] = ks.PageTable.from_lists(s["tables"], s["kv"], pool)
        s["q_indptr"] = torch.tensor([0] + np.cumsum(s["ql"]).tolist(), dtype=torch.int32,
                                     device=DEVICE)
        s["rotary"] = ks.Rotary(case["rotary"], case["theta"], interleave=case["interleave"],
                                sections=_sections(case), device=DEVICE)


# -------------------------------------------------------------------- run


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import kunserve_amd as ks

    kind, case = s["case"]["kind"], s["case"]
    if kind == "tree":
        out = [s["step"].run(i, s["q"][i], s["k"][i], s["v"][i]) for i in range(case["layers"])]
        return dict(out=out, k=s["k_pool"], v=s["v_pool"])
    if kind == "axes":
        q = ks.rotary_append_kv(s["pool"], 0, s["table"], s["q_indptr"], s["q"][0], s["k"][0],
                                s["v"][0], s["rotary"], positions=s["pos"], out=s["q_out"])
        return dict(q=q, k=s["k_pool"], v=s["v_pool"])
    if kind == "keep":
        s["step"].keep_tokens(s["kept"])
    elif kind == "shorten":
        ks.keep_tokens(s["pool"], s["table"], s["first"], s["kept"])
    else:
        ks.fork_rows(s["pool"], s["tables"], s["kv"], s["out_tables"])
    return dict(k=s["k_pool"], v=s["v_pool"])


def _run_plain(s):
    kind, case = s["case"]["kind"], s["case"]
    if kind == "tree":
        out = [_tree_plain(s, case, i) for i in range(case["layers"])]
        return dict(out=out, k=s["k_pool"], v=s["v_pool"])
    if kind == "axes":
        return _axes_plain(s, case)
    ps = case["page"]
    if kind == "fork":
        t = torch.arange(max(s["kv"]), device=DEVICE)
        src, dst = (x[:, t // ps] for x in (s["page_of"], s["out_page_of"]))
        b, c = torch.nonzero((t < s["kv_dev"][:, None]) & (src != dst), as_tuple=True)
        old, new = (src[b, c], c % ps), (dst[b, c], c % ps)
    else:
        b, j = torch.nonzero(s["kept"] >= 0, as_tuple=True)
        first = torch.tensor(s["first"], device=DEVICE)[b]
        at = first + s["kept"][b, j]
        old = (s["page_of"][b, at // ps], at % ps)
        new = (s["page_of"][b, (first + j) // ps], (first + j) % ps)
    for pool in (s["k_pool"], s["v_pool"]):
        pool[new[0], :, :, new[1]] = pool[old[0], :, :, old[1]]
    return dict(k=s["k_pool"], v=s["v_pool"])


def _new_tokens(s) -> tuple:
    """(row, place among its new tokens, cache slot) of every new token."""
    ql, kv = s["ql_dev"], s["kv_dev"]
    row = torch.repeat_interleave(torch.arange(len(ql), device=DEVICE), ql,
                                  output_size=s["q"].shape[1])
    i = torch.arange(len(row), device=DEVICE) - (ql.cumsum(0) - ql)[row]
    return row, i, (kv - ql)[row] + i


def _tree_plain(s, case, layer):
    ps, hkv, d = case["page"], case["hkv"], case["dim"]
    ratio, rows = case["hq"] // hkv, case["rows"]
    row, i, at = _new_tokens(s)
    page, slot = s["page_of"][row, at // ps], at % ps
    s["k_pool"][page, layer, :, slot] = s["k"][layer]
    s["v_pool"][page, layer, :, slot] = s["v"][layer]
    # padded rows: keys [rows, heads, tokens, dim], queries [rows, heads, new x ratio, dim]
    n, width = max(s["kv"]), max(s["ql"])
    t = torch.arange(n, device=DEVICE)
    pages = s["page_of"][:, t // ps]
    keys = s["k_pool"][pages, layer, :, t % ps].float().transpose(1, 2)
    values = s["v_pool"][pages, layer, :, t % ps].float().transpose(1, 2).contiguous()
    q = torch.zeros((rows, width, case["hq"], d), device=DEVICE)
    q[row, i] = s["q"][layer].float()
    q = q.view(rows, width, hkv, ratio, d).permute(0, 2, 1, 3, 4).reshape(rows, hkv, -1, d)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) / math.sqrt(d)
    drafted = t - (s["kv_dev"] - s["ql_dev"])[:, None]     # [rows, tokens]
    seen = s["sees"].gather(2, drafted.clamp(0, width - 1)[:, None, :].expand(-1, width, -1))
    seen = torch.where((drafted < 0)[:, None, :], True, seen)
    seen = seen & (t < s["kv_dev"][:, None])[:, None, :]
    # queries past a row's tokens: of no output, kept from 0 / 0
    seen = seen | (torch.arange(width, device=DEVICE) >= s["ql_dev"][:, None])[:, :, None]
    scores = scores.view(rows, hkv, width, ratio, n)
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(rows, hkv, -1, n), values).view(rows, hkv, width, ratio, d)
    return out.permute(0, 2, 1, 3, 4).reshape(rows, width, -1, d)[row, i].to(s["q"].dtype)


def _axes_plain(s, case):
    ps, n = case["page"], case["rotary"]
    f = torch.tensor(case["theta"] ** (-np.arange(0, n, 2, dtype=np.float64) / n), device=DEVICE)
    axis = np.repeat(np.arange(3), _sections(case))
    angle = s["pos"].double()[torch.tensor(axis, device=DEVICE)].t() * f
    cos, sin = (x.float()[:, None, :] for x in (angle.cos(), angle.sin()))

    def rotated(x):
        x, y = x.float(), x.float().clone()
        a, b = (slice(0, n, 2), slice(1, n, 2)) if case["interleave"] else \
            (slice(0, n // 2), slice(n // 2, n))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(s["q"].dtype)

    row, _, at = _new_tokens(s)
    page, slot = s["page_of"][row, at // ps], at % ps
    s["k_pool"][page, 0, :, slot] = rotated(s["k"][0])
    s["v_pool"][page, 0, :, slot] = s["v"][0]
    s["q_out"].copy_(rotated(s["q"][0]))
    return dict(q=s["q_out"], k=s["k_pool"], v=s["v_pool"])


# ------------------------------------------------------------------- work


def work(case) -> dict:
    ql, kv = _rows(case)
    row, tokens = 2 * case["dim"], int(ql.sum())     # bytes of a head's row
    heads, kind = case["hkv"] * case.get("layers", 1), case["kind"]
    if kind == "axes":
        pairs = tokens * (case["hq"] + case["hkv"]) * case["rotary"] // 2
        return {"bytes": 2 * tokens * row * (case["hq"] + 2 * case["hkv"]), "flops": 6 * pairs}
    if kind == "tree":
        # K and V of every cached token once (the new ones from k and v), the
        # new ones written, q read, out written.
        depth = 0
        for parents in _parents(case):
            at = []
            for p in parents:
                at.append(1 if p < 0 else at[p] + 1)
            depth += sum(at)
        pairs = int((ql * (kv - ql)).sum()) + depth
        return {"bytes": heads * 2 * row * (int(kv.sum()) + tokens)
                + case["layers"] * 2 * tokens * case["hq"] * row,
                "flops": 4 * case["hq"] * case["dim"] * pairs * case["layers"]}
    if kind == "fork":
        same = _same_pages(case) * case["page"]
        written = int((kv - same).sum())
        read = int((kv - same)[0]) if case["one"] else written
        return {"bytes": heads * 2 * row * (read + written), "flops": 0}
    # the lists of what stays read, and what changes its place read and written
    kept = _kept(case)
    moved = sum(int((np.array(x, np.int64) != np.arange(len(x))).sum()) for x in kept)
    return {"bytes": 4 * sum(map(len, kept)) + heads * 4 * row * moved, "flops": 0}


# ------------------------------------------------------------------ exact


def exact(case, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "axes":
        return _axes_exact(s, case)
    if case["kind"] != "tree":
        return {name: _moved_exact(s, case, s[name + "_pool"]) for name in ("k", "v")}
    ratio, hkv, outs = case["hq"] // case["hkv"], case["hkv"], []
    for layer in range(case["layers"]):
        out, begin = torch.empty(s["q"].shape[1:], dtype=torch.float64, device=DEVICE), 0
        for table, parents, n in zip(s["tables"], s["parents"], s["kv"]):
            t = len(parents)
            ids, new = torch.tensor(table, device=DEVICE), slice(begin, begin + t)
            begin += t
            # the row's cache [heads, tokens, dim], its drafted tokens last
            k, v = (torch.cat([pool[ids, layer].double().transpose(0, 1)
                               .reshape(hkv, -1, case["dim"])[:, :n - t],
                               x[layer, new].double().transpose(0, 1)], dim=1)
                    for pool, x in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])))
            hidden = np.ones((t, n), dtype=bool)
            hidden[:, :n - t] = False
            for i in range(t):
                j = i
                while j >= 0:
                    hidden[i, n - t + j] = False
                    j = parents[j]
            hidden = torch.tensor(hidden, device=DEVICE)
            for h in range(case["hq"]):
                score = s["q"][layer, new, h].double() @ k[h // ratio].t().contiguous()
                score = (score * case["dim"] ** -0.5).masked_fill(hidden, -math.inf)
                out[new, h] = torch.softmax(score, dim=-1) @ v[h // ratio]
        outs.append(out)
    return dict(out=outs, k=None, v=None)


def _moved_exact(s, case, pool):
    """Copies, row by row: the tokens that come to the places behind `first`."""
    out, ps = pool.double(), case["page"]
    firsts = [0] * case["rows"] if case["kind"] == "fork" else s["first"]
    kept = [range(n) for n in s["kv"]] if case["kind"] == "fork" else _kept(case)
    for table, to, first, places in zip(s["tables"], s["out_tables"] or s["tables"], firsts, kept):
        row = pool[torch.tensor(table, device=DEVICE)].transpose(1, 3).flatten(0, 1)
        row = row[[first + i for i in places]].double()     # [tokens, heads, layers, dim]
        for i in range(len(places)):
            out[to[(first + i) // ps], :, :, (first + i) % ps] = row[i].transpose(0, 1)
    return out


def _axes_exact(s, case):
    ps, n = case["page"], case["rotary"]
    turn = torch.empty((s["pos"].shape[1], n // 2), dtype=torch.complex128, device=DEVICE)
    ends = np.cumsum(_sections(case))
    for j in range(n // 2):
        angle = s["pos"][int(np.searchsorted(ends, j, side="right"))].double() \
            * case["theta"] ** (-2 * j / n)
        turn[:, j] = torch.polar(torch.ones_like(angle), angle)

    def rotated(x):
        y = x.double()
        pairs = y[..., :n].unflatten(-1, (n // 2, 2) if case["interleave"] else (2, n // 2))
        pairs = pairs if case["interleave"] else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        z = (z if case["interleave"] else z.transpose(-1, -2)).flatten(-2)
        return torch.cat([z, y[..., n:]], dim=-1)

    k, at = s["k_pool"].double(), 0
    turned = rotated(s["k"][0])
    for table, t, m in zip(s["tables"], s["ql"], s["kv"]):
        c = torch.arange(m - t, m, device=DEVICE)
        k[torch.tensor(table, device=DEVICE)[c // ps], 0, :, c % ps] = turned[at:at + t]
        at += t
    return dict(q=rotated(s["q"][0]), k=k, v=None)

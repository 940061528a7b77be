"""Performance cases of the operators around a shared and shortened KV cache.

Kinds of case
  shared   AttentionStep.run over `layers` layers of a step of decoding rows
           whose page lists begin with the same pages, share_prefixes=True:
           append of the new K/V, then attention that reads what rows share
           once for all of them.
  weights  AttentionStep.run with weights: the append, the attention, and the
           attention weight that each cached token got added to the cache's
           weights; rows decode one token, or are prompt chunks of which the
           last `window` tokens count.
  evict    evict(): of every row, layer and KV head the heaviest tokens, the
           first and the last ones, moved to pages of their own.
  rotary   rotary_append_kv: q and the new k rotated at positions of their
           own (part of the head, frequencies scaled for long contexts) and
           the append of k and v.

Where `own` is false the same is computed by elementary torch operations in 32
bits (angles in 64) on padded rows. Row lengths belong to the case (its `lens`
number); tensors and page tables come from the seed.
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
        # Four samples of one short prompt, the smallest step that shares
        # anything: bound by latency and launches.
        dict(name="shared_samples", kind="shared", layers=8, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=4, root=1000, group=0, branch=0, tail_lo=3, tail_hi=80, lens=1),
        # A chat batch behind one system prompt, GQA.
        dict(name="shared_chat", kind="shared", layers=4, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=64, root=2048, group=0, branch=0, tail_lo=16, tail_hi=1500,
             lens=2),
        # 128 rows behind one long document, every 16 of them with a question
        # and its samples in common too, on the default 256-token pages: the
        # largest.
        dict(name="shared_document", kind="shared", layers=2, hq=64, hkv=8, dim=128, page=256,
             dtype="fp16", rows=128, root=8192, group=16, branch=1100, tail_lo=64, tail_hi=900,
             lens=3),
        # A model without GQA, head size 64, a prompt that ends inside a page.
        dict(name="shared_mha_dim64", kind="shared", layers=4, hq=32, hkv=32, dim=64, page=32,
             dtype="fp16", rows=21, root=777, group=0, branch=0, tail_lo=1, tail_hi=300, lens=4),
        # One user's decode while the cache learns its tokens' weights.
        dict(name="weights_one_row", kind="weights", layers=8, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=1, q_lo=0, q_hi=0, kv_lo=1500, kv_hi=1500, window=16, lens=5),
        # The same for a batch of ragged contexts.
        dict(name="weights_batch", kind="weights", layers=2, hq=32, hkv=8, dim=128, page=16,
             dtype="bf16", rows=48, q_lo=0, q_hi=0, kv_lo=256, kv_hi=6000, window=16, lens=6),
        # Prompt chunks whose last tokens' attention says what of the prompt
        # to keep.
        dict(name="weights_prompts", kind="weights", layers=1, hq=32, hkv=8, dim=128, page=16,
             dtype="fp16", rows=6, q_lo=300, q_hi=512, kv_lo=1000, kv_hi=4000, window=32, lens=7),
        # One conversation's cache cut to a fifth.
        dict(name="evict_one", kind="evict", layers=8, hkv=8, dim=128, page=16, dtype="bf16",
             rows=1, kv_lo=5000, kv_hi=5000, keep=200, sinks=4, recent=256, lens=8),
        # A batch's caches halved, every layer of a model.
        dict(name="evict_batch", kind="evict", layers=32, hkv=8, dim=128, page=16, dtype="bf16",
             rows=8, kv_lo=700, kv_hi=5000, keep=500, sinks=4, recent=64, lens=9),
        # Decoding rows far into a long context: half of each head rotated,
        # frequencies stretched.
        dict(name="rotary_decode", kind="rotary", hq=32, hkv=8, dim=128, page=16, dtype="bf16",
             rows=33, q_lo=1, q_hi=1, rotary=64, interleave=True, scaling="yarn", theta=10000.0,
             far=100000, lens=10),
        # Prompt chunks, whole heads rotated in halves.
        dict(name="rotary_prompts", kind="rotary", hq=32, hkv=8, dim=128, page=256, dtype="bf16",
             rows=9, q_lo=400, q_hi=512, rotary=128, interleave=False, scaling="llama3",
             theta=500000.0, far=20000, lens=11),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["shared", "shared", "shared", "weights", "weights", "evict", "rotary"])
    ratio, hkv = rng.choice([(1, 32), (1, 16), (2, 8), (3, 8), (4, 8), (4, 8), (4, 4), (5, 8),
                             (6, 8), (7, 4), (8, 8), (8, 4)])
    dim = rng.choice([64, 128, 128, 128, 256])
    case = dict(kind=kind, hkv=hkv, dim=dim, page=rng.choice([16, 16, 32, 256]),
                dtype=rng.choice(["fp16", "bf16"]), lens=rng.randrange(1 << 20))
    if kind != "evict":
        case["hq"] = ratio * hkv
    if kind == "shared":
        root, rows = _log_int(rng, 40, 8192), _log_int(rng, 2, 128)
        hi = _log_int(rng, 2, 1500)
        # at most about a sixth of the largest case's cached tokens x heads
        while rows > 2 and rows * (root + hi) * ratio * hkv * dim > 1.6e9:
            rows = rows * 2 // 3
        group = rng.choice([0, 0, 2, 5, 16])
        case.update(rows=rows, root=root, group=group if group < rows else 0,
                    branch=_log_int(rng, 20, 1500) if 0 < group < rows else 0,
                    tail_lo=rng.choice([1, max(1, hi // 8), hi]), tail_hi=hi,
                    layers=rng.choice([1, 2, 4]))
    elif kind == "weights":
        prompt = rng.random() < 0.3
        hi = _log_int(rng, 40, 4000 if prompt else 8192)
        q_hi = min(hi, _log_int(rng, 2, 512)) if prompt else 0
        rows = _log_int(rng, 1, 12 if prompt else 48)
        # at most the flops of the listed prompts, the bytes of the listed batch
        while rows * hi * hkv * dim * max(1, q_hi * ratio) > (1.2e10 if prompt else 1.2e8):
            rows, hi = max(1, rows * 2 // 3), hi if rows > 1 else hi * 2 // 3
            q_hi = min(q_hi, hi)
        case.update(rows=rows, q_lo=max(1, q_hi // 4) if prompt else 0, q_hi=q_hi,
                    kv_lo=max(q_hi, hi // rng.choice([1, 4, 16]), 1), kv_hi=hi,
                    window=rng.choice([1, 8, 16, 32, 50]), layers=1 if prompt else 2)
    elif kind == "evict":
        hi, rows, layers = _log_int(rng, 64, 16384), _log_int(rng, 1, 12), rng.choice([2, 8, 16])
        while rows > 1 and rows * hi * layers * hkv * dim > 6e8:
            rows = rows * 2 // 3
        recent = rng.choice([0, 16, 100])
        case.update(rows=rows, kv_lo=max(1, hi // rng.choice([1, 4])), kv_hi=hi,
                    keep=rng.choice([100, 250, 500, 900]), sinks=rng.choice([0, 4]),
                    recent=min(recent, hi // 20), layers=layers)
    else:
        prompt = rng.random() < 0.5
        q_hi = _log_int(rng, 2, 512) if prompt else 1
        case.update(rows=_log_int(rng, 1, 9 if prompt else 200), q_lo=max(1, q_hi // 2), q_hi=q_hi,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleave=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                    theta=rng.choice([10000.0, 500000.0]), far=_log_int(rng, 600, 1000000))
    return case


# ---------------------------------------------------- rows and page tables


def _rows(case) -> tuple:
    """(new tokens, cached tokens with them) of every row."""
    rng = np.random.default_rng(case["lens"])
    n = case["rows"]
    if case["kind"] == "shared":
        tail = rng.integers(case["tail_lo"], case["tail_hi"] + 1, size=n)
        return np.ones(n, np.int64), case["root"] + case["branch"] + tail
    if case["kind"] == "rotary":
        q = rng.integers(case["q_lo"], case["q_hi"] + 1, size=n)
        return q, q + rng.integers(0, 600, size=n)
    kv = rng.integers(case["kv_lo"], case["kv_hi"] + 1, size=n)
    if case["kind"] == "evict" or case["q_hi"] == 0:
        return np.ones(n, np.int64), kv
    return np.minimum(rng.integers(case["q_lo"], case["q_hi"] + 1, size=n), kv), kv


def _shared_pages(case) -> tuple:
    """Leading pages that all rows share, and further ones that the rows of a
    group share."""
    if case["kind"] != "shared":
        return 0, 0
    root = case["root"] // case["page"]
    branch = (case["root"] + case["branch"]) // case["page"] - root if case["group"] else 0
    return root, branch


def _kept(case) -> np.ndarray:
    """Tokens that an eviction keeps of every row."""
    kv = _rows(case)[1]
    return np.minimum(kv, np.maximum(kv * case["keep"] // 1000, case["sinks"] + case["recent"]))


def _tables(case, seed: int) -> tuple:
    """Page lists of the rows (and those that an eviction fills), and the
    pages of the pool."""
    kv, page = _rows(case)[1], case["page"]
    root, branch = _shared_pages(case)
    need = -(-kv // page)
    out = -(-_kept(case) // page) if case["kind"] == "evict" else np.zeros_like(need)
    groups = -(-case["rows"] // case["group"]) if branch else 0
    total = int(root + groups * branch + (need - root - branch).sum() + out.sum())
    pages = total + total // 4 + 4
    ids = iter(np.random.default_rng(seed).permutation(pages).tolist())
    take = lambda n: [next(ids) for _ in range(n)]   # noqa: E731
    common, mine = take(root), [take(branch) for _ in range(groups)]
    tables = [common + (mine[b // case["group"]] if branch else [])
              + take(int(n) - root - branch) for b, n in enumerate(need)]
    return tables, [take(int(n)) for n in out], pages


# ---------------------------------------------------------------- prepare


def _padded(lists, width) -> torch.Tensor:
    return torch.tensor([x + [0] * (width - len(x)) for x in lists], device=DEVICE)


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
    s = dict(case=case, tables=tables, out_tables=out_tables, ql=ql.tolist(), kv=kv.tolist(),
             k_pool=normal(shape), v_pool=normal(shape),
             page_of=_padded(tables, max(len(t) for t in tables)),
             ql_dev=torch.tensor(ql, device=DEVICE), kv_dev=torch.tensor(kv, device=DEVICE))
    if kind != "evict":
        # Scores have a standard deviation of 2, so rows attend unevenly.
        s.update(q=normal((layers, tokens, case["hq"], case["dim"]), 2.0),
                 k=normal((layers, tokens, case["hkv"], case["dim"])),
                 v=normal((layers, tokens, case["hkv"], case["dim"])))
    if kind in ("weights", "evict"):
        # Sums of attention weights: a few tokens hold most; one in ten never
        # got any, so ties occur.
        w = torch.empty(shape[:4], device=DEVICE).normal_(0.0, 2.0, generator=g).exp_()
        w *= torch.rand(w.shape, device=DEVICE, generator=g) > 0.1
        s.update(w=w, w_now=w.clone())
    if kind == "evict":
        kept = _kept(case)
        s.update(kept=kept.tolist(), kept_dev=torch.tensor(kept, device=DEVICE),
                 out_page_of=_padded(out_tables, max(1, max(len(t) for t in out_tables))))
    if kind == "rotary":
        # A row's next position has nothing to do with what its cache holds.
        at = np.random.default_rng(case["lens"] + 1).integers(0, case["far"] + 1, size=len(ql))
        pos = np.concatenate([a + np.arange(n) for a, n in zip(at, ql)])
        s.update(pos=torch.tensor(pos, dtype=torch.int32, device=DEVICE),
                 q_out=torch.empty_like(s["q"][0]))
    if own:
        _handles(s, case)
    return s


SCALING = {
    "none": None,
    "linear": dict(rope_type="linear", factor=4.0),
    "ntk": dict(rope_type="ntk", factor=4.0),
    "yarn": dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096),
    "llama3": dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192),
}


def _handles(s, case) -> None:
    """What a user of the framework keeps: its pool, the step (made once per
    step and shared by its layers), the weights, the frequencies."""
    import kunserve_amd as ks

    s["pool"] = pool = ks.KVPool(s["k_pool"], s["v_pool"])
    decode = case.get("q_hi", 0) <= 1
    first = [n if decode else n - t for t, n in zip(s["ql"], s["kv"])]
    if "w" in s:
        s["weights"] = ks.KVWeights(pool, s["w_now"])
    if case["kind"] == "shared":
        s["step"] = ks.AttentionStep(pool, case["hq"], s["ql"], first, [0] * len(first),
                                     s["tables"], share_prefixes=True)
    elif case["kind"] == "weights":
        s["step"] = ks.AttentionStep(pool, case["hq"], s["ql"], first,
                                     [int(not decode)] * len(first), s["tables"],
                                     weights=s["weights"], window=case["window"])
    elif case["kind"] == "rotary":
        s["table"] = ks.PageTable.from_lists(s["tables"], s["kv"], pool)
        s["q_indptr"] = torch.tensor([0] + np.cumsum(s["ql"]).tolist(), dtype=torch.int32,
                                     device=DEVICE)
        s["rotary"] = ks.Rotary(case["rotary"], case["theta"], interleave=case["interleave"],
                                scaling=SCALING[case["scaling"]], device=DEVICE)


# -------------------------------------------------------------------- run


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import kunserve_amd as ks

    kind, case = s["case"]["kind"], s["case"]
    if kind == "evict":
        kept = ks.evict(s["pool"], s["weights"], s["tables"], s["kv"], s["out_tables"], s["kept"],
                        sinks=case["sinks"], recent=case["recent"])
        return dict(kept=kept, k=s["k_pool"], v=s["v_pool"], w=s["w_now"])
    if kind == "rotary":
        q = ks.rotary_append_kv(s["pool"], 0, s["table"], s["q_indptr"], s["q"][0], s["k"][0],
                                s["v"][0], s["rotary"], positions=s["pos"], out=s["q_out"])
        return dict(q=q, k=s["k_pool"], v=s["v_pool"])
    if kind == "weights":
        s["w_now"].copy_(s["w"])   # the weights as the steps before left them
    out = [s["step"].run(i, s["q"][i], s["k"][i], s["v"][i]) for i in range(case["layers"])]
    return dict(out=out, k=s["k_pool"], v=s["v_pool"], **({"w": s["w_now"]} if "w" in s else {}))


def _run_plain(s):
    kind, case = s["case"]["kind"], s["case"]
    if kind == "evict":
        return _evict_plain(s, case)
    if kind == "rotary":
        return _rotary_plain(s, case)
    if kind == "weights":
        s["w_now"].copy_(s["w"])
    out = [_attend_plain(s, case, i) for i in range(case["layers"])]
    return dict(out=out, k=s["k_pool"], v=s["v_pool"], **({"w": s["w_now"]} if "w" in s else {}))


def _new_tokens(s) -> tuple:
    """(row, place among its new tokens, cache slot) of every new token."""
    ql, kv = s["ql_dev"], s["kv_dev"]
    row = torch.repeat_interleave(torch.arange(len(ql), device=DEVICE), ql,
                                  output_size=s["q"].shape[1])
    i = torch.arange(len(row), device=DEVICE) - (ql.cumsum(0) - ql)[row]
    return row, i, (kv - ql)[row] + i


def _attend_plain(s, case, layer):
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
    pos = (s["kv_dev"] - s["ql_dev"])[:, None] + torch.arange(width, device=DEVICE)
    seen = (t[None, None, :] <= pos[:, :, None]) & (t < s["kv_dev"][:, None])[:, None, :]
    scores = scores.view(rows, hkv, width, ratio, n)
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(rows, hkv, -1, n), values).view(rows, hkv, width, ratio, d)
    out = out.permute(0, 2, 1, 3, 4).reshape(rows, width, -1, d)[row, i]
    if "w" in s:
        place = torch.arange(width, device=DEVICE)
        counts = (place < s["ql_dev"][:, None]) & (place >= s["ql_dev"][:, None] - case["window"])
        got = torch.where(counts[:, None, :, None, None], p, 0.0).sum((2, 3))   # [rows, heads, n]
        b, c = torch.nonzero(t < s["kv_dev"][:, None], as_tuple=True)
        page, slot = s["page_of"][b, c // ps], c % ps
        old = s["w_now"][page, layer, :, slot]
        old = torch.where((c >= (s["kv_dev"] - s["ql_dev"])[b])[:, None], 0.0, old)
        s["w_now"][page, layer, :, slot] = old + got[b, :, c]
    return out.to(s["q"].dtype)


def _evict_plain(s, case):
    ps, n, most = case["page"], max(s["kv"]), max(s["kept"])
    t = torch.arange(n, device=DEVICE)
    w = s["w_now"][s["page_of"][:, t // ps], :, :, t % ps].permute(0, 2, 3, 1)
    kv, kept = s["kv_dev"][:, None, None, None], s["kept_dev"][:, None, None, None]
    w = torch.where((t < case["sinks"]) | (t >= kv - case["recent"]), math.inf, w)
    w = torch.where(t < kv, w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :most]
    j = torch.arange(most, device=DEVICE)
    order = torch.where(j < kept, order, n).sort(-1).values     # what is past a row's last: n
    b, layer, h, c = torch.nonzero(order < n, as_tuple=True)
    src = order[b, layer, h, c]
    old = (s["page_of"][b, src // ps], layer, h, src % ps)
    new = (s["out_page_of"][b, c // ps], layer, h, c % ps)
    for pool in (s["k_pool"], s["v_pool"], s["w_now"]):
        pool[new] = pool[old]
    return dict(kept=torch.where(order < n, order, -1).to(torch.int32), k=s["k_pool"],
                v=s["v_pool"], w=s["w_now"])


def _frequencies(case) -> tuple:
    """Angle per position of every rotated pair, in 64 bits, and the factor on
    what is rotated."""
    n, theta = case["rotary"], case["theta"]
    sc = SCALING[case["scaling"]] or dict(rope_type="none")
    s = sc.get("factor", 1.0)
    if sc["rope_type"] == "ntk" and n > 2:
        theta = theta * s ** (n / (n - 2))
    f = theta ** (-np.arange(0, n, 2, dtype=np.float64) / n)
    length = sc.get("original_max_position_embeddings", 0)
    if sc["rope_type"] == "linear":
        return f / s, 1.0
    if sc["rope_type"] == "yarn":
        # dimension at which `turns` rotations fill the original length
        at = lambda turns: n * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(theta))   # noqa: E731
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), n - 1)
        ramp = np.clip((np.arange(n // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        return f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1
    if sc["rope_type"] == "llama3":
        turns = length * f / (2 * math.pi)
        mix = np.clip((turns - sc["low_freq_factor"])
                      / (sc["high_freq_factor"] - sc["low_freq_factor"]), 0, 1)
        return f * (mix + (1 - mix) / s), 1.0
    return f, 1.0


def _rotary_plain(s, case):
    ps, n = case["page"], case["rotary"]
    f, factor = _frequencies(case)
    angle = s["pos"].double()[:, None] * torch.tensor(f, device=DEVICE)
    cos, sin = ((x * factor).float()[:, None, :] for x in (angle.cos(), angle.sin()))

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
    heads = case["hkv"] * case.get("layers", 1)
    if case["kind"] == "evict":
        kept = int(_kept(case).sum())
        # the middle's weights read; kept K, V and weights read and written
        return {"bytes": heads * (4 * int(kv.sum()) + kept * (4 * row + 12)), "flops": 0}
    if case["kind"] == "rotary":
        pairs = tokens * (case["hq"] + case["hkv"]) * case["rotary"] // 2
        return {"bytes": 2 * tokens * row * (case["hq"] + 2 * case["hkv"]), "flops": 6 * pairs}
    root, branch = _shared_pages(case)
    cached = int(kv.sum()) - (case["rows"] - 1) * root * case["page"]
    if branch:
        cached -= (case["rows"] - -(-case["rows"] // case["group"])) * branch * case["page"]
    # K and V of every distinct cached token once (the new ones from k and v),
    # the new ones written, q read, out written.
    total = heads * (2 * cached * row + 2 * tokens * row) \
        + case["layers"] * 2 * tokens * case["hq"] * row
    pairs = int((ql * (kv - ql) + ql * (ql + 1) // 2).sum())
    if case["kind"] == "weights":
        total += heads * 4 * (2 * int((kv - ql).sum()) + tokens)
    return {"bytes": total, "flops": 4 * case["hq"] * case["dim"] * pairs * case["layers"]}


# ------------------------------------------------------------------ exact


def exact(case, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "evict":
        return _evict_exact(s, case)
    if case["kind"] == "rotary":
        return _rotary_exact(s, case)
    ps, hkv = case["page"], case["hkv"]
    ratio, outs = case["hq"] // hkv, []
    w = s["w"].double() if "w" in s else None
    for layer in range(case["layers"]):
        out, begin = torch.empty(s["q"].shape[1:], dtype=torch.float64, device=DEVICE), 0
        for table, t, n in zip(s["tables"], s["ql"], s["kv"]):
            ids, new = torch.tensor(table, device=DEVICE), slice(begin, begin + t)
            begin += t
            # the row's cache [heads, tokens, dim], its new tokens last
            k, v = (torch.cat([pool[ids, layer].double().transpose(0, 1)
                               .reshape(hkv, -1, case["dim"])[:, :n - t],
                               x[layer, new].double().transpose(0, 1)], dim=1)
                    for pool, x in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])))
            ahead = torch.ones((t, n), dtype=torch.bool, device=DEVICE).triu(n - t + 1)
            for h in range(hkv):
                mass = torch.zeros(n, dtype=torch.float64, device=DEVICE)
                for x in range(h * ratio, (h + 1) * ratio):
                    score = s["q"][layer, new, x].double() @ k[h].t().contiguous()
                    score = (score * case["dim"] ** -0.5).masked_fill(ahead, -math.inf)
                    p = torch.softmax(score, dim=-1)
                    out[new, x] = p @ v[h]
                    if w is not None:
                        mass += p[-case["window"]:].sum(0)
                if w is not None:
                    pages = ids[torch.arange(n, device=DEVICE) // ps]
                    place = (pages, layer, h, torch.arange(n, device=DEVICE) % ps)
                    old = w[place]
                    old[n - t:] = 0
                    w[place] = old + mass
        outs.append(out)
    return dict(out=outs, k=None, v=None, **({} if w is None else {"w": w}))


def _evict_exact(s, case):
    """The weights; K and V are copies that go with them."""
    ps, w = case["page"], s["w"].double()
    for table, out_table, n, keep in zip(s["tables"], s["out_tables"], s["kv"], s["kept"]):
        t = np.arange(n)
        here = s["w"][torch.tensor(table, device=DEVICE)].permute(1, 2, 0, 3).flatten(2)[..., :n]
        here = here.cpu().numpy()
        always = (t < case["sinks"]) | (t >= n - case["recent"])
        first = np.lexsort((np.broadcast_to(t, here.shape), -here, np.broadcast_to(~always, here.shape)))
        chosen = np.sort(first[..., :keep], axis=-1)
        got = torch.tensor(np.take_along_axis(here, chosen, -1), device=DEVICE, dtype=torch.float64)
        j = torch.arange(keep, device=DEVICE)
        w[torch.tensor(out_table, device=DEVICE)[j // ps], :, :, j % ps] = got.permute(2, 0, 1)
    return dict(kept=None, k=None, v=None, w=w)


def _rotary_exact(s, case):
    ps, n = case["page"], case["rotary"]
    sc, theta = SCALING[case["scaling"]] or {}, case["theta"]
    kind, factor = sc.get("rope_type"), 1.0
    turn = torch.empty((len(s["pos"]), n // 2), dtype=torch.complex128, device=DEVICE)
    for j in range(n // 2):
        f = theta ** (-2 * j / n)
        if kind == "linear":
            f /= sc["factor"]
        elif kind == "ntk" and n > 2:     # the last pair's wavelength times the factor
            f /= sc["factor"] ** (2 * j / (n - 2))
        elif kind == "yarn":
            length = sc["original_max_position_embeddings"]
            lo, hi = (n / 2 * math.log(length / (b * 2 * math.pi), theta) for b in (32, 1))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
            whole = 1 - min(max((j - lo) / max(hi - lo, 0.001), 0), 1)
            f = f * whole + f * (1 - whole) / sc["factor"]
            factor = 1 + math.log(sc["factor"]) / 10
        elif kind == "llama3":
            wave = 2 * math.pi / f / sc["original_max_position_embeddings"]
            if wave > 1 / sc["low_freq_factor"]:
                f /= sc["factor"]
            elif wave >= 1 / sc["high_freq_factor"]:
                part = (1 / wave - sc["low_freq_factor"]) / (sc["high_freq_factor"]
                                                             - sc["low_freq_factor"])
                f = (1 - part) * f / sc["factor"] + part * f
        angle = s["pos"].double() * f
        turn[:, j] = torch.polar(torch.full_like(angle, factor), angle)

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

"""The operators of a shared and shortened cache as an engine runs them: requests
behind one prompt that learn what they attend to, are shortened, and go on at
their own positions."""
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
from helpers import random_tensor
from kunserve_amd import KVWeights, LlamaOp, Rotary, evict

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, LAYERS, WINDOW = 8, 2, 64, 16, 2, 8
TRIG = 16 * ref.W   # test_gpu_rotary.py


class Request:
    """One request's pages, what its cache holds, and its next position."""

    def __init__(self, pages):
        self.pages, self.cached, self.position = list(pages), 0, 0


def step(op, reqs, q_lens, weights, rotary, seed, share=False):
    """A step of all requests, prompts (several tokens) and decodes (one), every
    layer; checks rotation, append, outputs and weights of each."""
    dev, dtype = op.pool.device, op.pool.dtype
    total = sum(q_lens)
    is_prompt = [int(t > 1) for t in q_lens]
    starts = [r.position for r in reqs]
    first = [r.cached if p else r.cached + 1 for r, p in zip(reqs, is_prompt)]
    s = op.pforward(len(reqs), total, op.max_num_pages, 0, LAYERS, [[1] * t for t in q_lens],
                    first, is_prompt, [r.pages for r in reqs], weights=weights, window=WINDOW,
                    rope_positions=starts, share_prefixes=share)
    freq = rotary.frequencies.cpu().numpy()
    pos = np.concatenate([a + np.arange(t) for a, t in zip(starts, q_lens)])
    for layer in range(LAYERS):
        q, k, v = (random_tensor((total, h, D), dev, seed + 10 * layer + h, 1.5, dtype)
                   for h in (HQ, HKV, HKV + 1))
        v = v[:, :HKV].contiguous()
        q_raw, w_old = q.clone(), None if weights is None else weights.w.cpu().double().numpy()
        out = s.run(layer, q, k, v, rope=rotary)
        torch.cuda.synchronize()
        want, mag = ref.rotate(q_raw.cpu().double().numpy(), pos, freq, rotary.scale, False)
        tol = ref.half_step(dtype) * np.abs(want) + TRIG * mag * 1.001 + 2.0 ** -25
        assert np.all(np.abs(q.cpu().double().numpy() - want) <= tol)
        want_k, mag_k = ref.rotate(k.cpu().double().numpy(), pos, freq, rotary.scale, False)
        kh, vh, qh = op.pool.k.cpu(), op.pool.v.cpu(), q.cpu().double().numpy()
        at = 0
        for r, t in zip(reqs, q_lens):
            n, rows = r.cached + t, slice(at, at + t)
            at += t
            kc, vc = (ref.row_cache(x, layer, r.pages, n) for x in (kh, vh))
            tol = (ref.half_step(dtype) * np.abs(want_k[rows]) + TRIG * mag_k[rows] * 1.001
                   + 2.0 ** -25)
            assert np.all(np.abs(kc[:, n - t:].transpose(1, 0, 2) - want_k[rows]) <= tol)
            assert np.array_equal(vc[:, n - t:].transpose(1, 0, 2), v[rows].cpu().double().numpy())
            o, o_tol, p, dp = ref.attend(qh[rows], kc, vc, 1 / math.sqrt(D), dtype,
                                         p_err=ref.half_step(dtype) if t > 1 else None)
            assert np.all(np.abs(out[rows].cpu().double().numpy() - o) <= o_tol)
            if weights is not None:
                c = np.arange(n)
                where = (np.array(r.pages)[c // PS], layer, slice(None), c % PS)
                new, err = ref.add_weights(w_old[where].T, p, dp, t, WINDOW, HQ // HKV)
                got = weights.w.cpu().double().numpy()[where].T
                assert np.all(np.abs(got - new) <= err)
    for r, t in zip(reqs, q_lens):
        r.cached += t
        r.position += t


def shorten(op, reqs, weights, budget, sinks, recent, free):
    outs = [[free.pop() for _ in range(-(-min(budget, r.cached) // PS))] for r in reqs]
    old = [x.cpu().clone() for x in (op.pool.k, op.pool.v, weights.w)]
    kept = evict(op.pool, weights, [r.pages for r in reqs], [r.cached for r in reqs], outs, budget,
                 sinks, recent).cpu().numpy()
    new = [x.cpu() for x in (op.pool.k, op.pool.v, weights.w)]
    for b, (r, o) in enumerate(zip(reqs, outs)):
        m = min(budget, r.cached)
        t, o, j = np.array(r.pages), np.array(o), np.arange(m)
        for layer in range(LAYERS):
            for h in range(HKV):
                w = old[2][t, layer, h].numpy().reshape(-1)[:r.cached]
                c = ref.choose(w, m, sinks, recent)
                assert np.array_equal(kept[b, layer, h, :m], c)
                for x, y in zip(new, old):
                    assert torch.equal(x[o[j // PS], layer, h, j % PS], y[t[c // PS], layer, h, c % PS])
        r.pages = list(o) + [free.pop() for _ in range(2)]
        r.cached = m


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_requests_are_shortened_and_go_on(device, dtype):
    op = LlamaOp(80, LAYERS, HQ, HKV, PS, D, 256, 1000, 8, 512, 4096, 1, device=device, dtype=dtype)
    for t in (op.pool.k, op.pool.v):
        t.fill_(float("nan"))    # what the pages' last users left
    weights = KVWeights(op.pool)
    weights.w.fill_(float("inf"))
    free = np.random.default_rng(0).permutation(80).tolist()
    rotary = Rotary(32, 10000.0, device=device, scaling=dict(
        rope_type="yarn", factor=4.0, original_max_position_embeddings=64))
    reqs = [Request([free.pop() for _ in range(10)]) for _ in range(2)]
    step(op, reqs, [70, 33], weights, rotary, 100)        # prompts
    step(op, reqs, [1, 40], weights, rotary, 200)         # a decode beside a chunk
    step(op, reqs, [1, 1], weights, rotary, 300)
    shorten(op, reqs, weights, 48, 4, 8, free)
    assert [r.cached for r in reqs] == [48, 48] and [r.position for r in reqs] == [72, 74]
    for i in range(3):
        step(op, reqs, [1, 1], weights, rotary, 400 + 50 * i)
    step(op, reqs, [5, 1], weights, rotary, 600)
    shorten(op, reqs, weights, 20, 2, 4, free)            # a second time
    step(op, reqs, [1, 1], weights, rotary, 700)


def test_shortened_copies_of_a_shared_prompt(device):
    """Requests behind one prompt share its pages until each takes what it needs
    of them to pages of its own; the prompt's pages stay as they were."""
    op = LlamaOp(120, LAYERS, HQ, HKV, PS, D, 256, 1000, 8, 512, 4096, 1, device=device)
    rotary = Rotary(64, 10000.0, device=device)
    free = np.random.default_rng(1).permutation(120).tolist()
    prompt = Request([free.pop() for _ in range(12)])
    weights = KVWeights(op.pool)
    step(op, [prompt], [192], weights, rotary, 10)
    reqs = []
    for _ in range(3):
        r = Request(prompt.pages + [free.pop() for _ in range(2)])
        r.cached = r.position = 192
        reqs.append(r)
    step(op, reqs, [1, 1, 1], None, rotary, 20, share=True)
    step(op, reqs, [1, 3, 1], None, rotary, 30, share=True)
    # what a request appended has no weight yet: this evicts by the prompt's
    for r in reqs:
        for page in r.pages[12:]:
            weights.w[page] = 0
    before = [x[prompt.pages].clone() for x in (op.pool.k, op.pool.v, weights.w)]
    shorten(op, reqs, weights, 64, 4, 8, free)
    for x, y in zip((op.pool.k, op.pool.v, weights.w), before):
        assert torch.equal(x[prompt.pages], y)
    step(op, reqs, [1, 1, 1], weights, rotary, 40)

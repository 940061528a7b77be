"""Steps with decode, prefill and tree rows against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from helpers import random_pool, random_tensor
from kunserve_amd import AttentionStep, Rotary, _lib
from tree_ref import check_out, random_pages, random_tree, tokens_of, tree_attention_ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


class Mixed:
    """Two tree rows between decode and prefill rows; each row as a tree: a prefill row is a
    chain, a decode row one token."""

    def __init__(self, device, dim=128, dtype=BF16, page=16, hq=8, hkv=2, tokens=17, seed=0):
        rng = np.random.default_rng(seed + dim)
        self.dim, self.dtype, self.hq = dim, dtype, hq
        self.sizes = [1, 9, 40, 1, tokens]
        self.flags = [0, 1, 1, 0, 1]
        cached = [300, 500, 64, 76, 1000]
        self.firsts = [c if f else c + 1 for c, f in zip(cached, self.flags)]
        self.trees = [None, random_tree(rng, 9, 3), None, None, random_tree(rng, tokens, 4, 2)]
        self.as_trees = [t if t is not None else list(range(-1, n - 1))
                         for t, n in zip(self.trees, self.sizes)]
        self.lens = [c + n for c, n in zip(cached, self.sizes)]
        self.lists, self.pages = random_pages(rng, self.lens, page)
        total = sum(self.sizes)
        self.q, self.k, self.v = (random_tensor((total, h, dim), device, seed + i, 1.0, dtype)
                                  for i, h in enumerate((hq, hkv, hkv)))
        self.pool = random_pool(self.pages, 1, hkv, page, dim, device, 4, dtype=dtype)

    def step(self, **kw):
        return AttentionStep(self.pool, self.hq, self.sizes, self.firsts, self.flags, self.lists,
                             trees=self.trees, **kw)

    def rows(self):
        at = 0
        for b, n in enumerate(self.sizes):
            yield b, slice(at, at + n)
            at += n

    def check_pool(self, before):
        """The new tokens in their places, every other slot as it was."""
        for t, old, x in zip((self.pool.k, self.pool.v), before, (self.k, self.v)):
            want, page = old.clone(), t.shape[3]
            for b, new in self.rows():
                for i, at in enumerate(range(self.lens[b] - self.sizes[b], self.lens[b])):
                    want[self.lists[b][at // page], 0, :, at % page] = x[new][i]
            assert torch.equal(t, want)

    def check(self, out):
        for b, new in self.rows():
            keys, values = (tokens_of(t, 0, self.lists[b], self.lens[b])
                            for t in (self.pool.k, self.pool.v))
            ref, mass = tree_attention_ref(self.q[new], keys, values, self.as_trees[b],
                                           self.dim ** -0.5)
            if self.trees[b] is not None:
                check_out(out[new], ref, mass, f"row {b}")
            else:
                # Prefill rows round each probability once to 16 bits, by eps / 2 of it at
                # most, and so may the sum that they are divided by.
                err = (out[new].double() - ref).abs()
                eps = torch.finfo(out.dtype).eps
                assert (err <= ref.abs() * eps / 2 + mass * (eps + 2.0 ** -12)).all(), b


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("offset,width", [(4, 4), (0, 12), (4, 8)])
def test_out_of_eight_byte_alignment(device, dim, dtype, offset, width):
    """out needs no more than the prefill rows' launch asks: 8 bytes, strides of 4."""
    m = Mixed(device, dim, dtype)
    want = m.step().run(0, m.q, m.k, m.v)
    m.check(want)
    big = torch.full((len(m.q), m.hq, dim + width), 7.0, dtype=dtype, device=device)
    out = big[..., offset:offset + dim]
    for t in (m.pool.k, m.pool.v):
        t[m.lists[1][500 // 16], :, :, 500 % 16:] = 0
    m.step().run(0, m.q, m.k, m.v, out=out)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert (big == 7).all()   # and nothing beside it was written


@pytest.mark.parametrize("pinned", [False, True])
def test_refused_before_anything_changes(device, pinned):
    m = Mixed(device)
    total = len(m.q)
    before = [t.clone() for t in (m.pool.k, m.pool.v, m.q)]
    big = torch.zeros(total, m.hq, 136, dtype=BF16, device="cpu" if pinned else device)
    if pinned:
        big = big.pin_memory()
    with pytest.raises((ValueError, _lib.KunserveError), match="8-byte aligned"):
        m.step().run(0, m.q, m.k, m.v, out=big[..., 2:130], rope=Rotary(128, device=device))
    torch.cuda.synchronize()
    for shape in ((total,), (total, m.hq), (total - 1, m.hq, 128)):
        with pytest.raises(ValueError, match="out shape"):
            m.step().run(0, m.q, m.k, m.v, out=torch.empty(shape, dtype=BF16, device=device),
                         rope=Rotary(128, device=device))
    torch.cuda.synchronize()
    for t, old in zip((m.pool.k, m.pool.v, m.q), before):
        assert torch.equal(t, old)
    assert not big.any()


@pytest.mark.parametrize("dim,hq,hkv,tokens,columns", [(64, 8, 2, 17, None), (128, 8, 2, 17, None),
                                                       (128, 16, 4, 64, 256), (256, 8, 2, 64, None)])
@pytest.mark.parametrize("page", [4, 8, 16])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_append_within_their_launches(device, dim, hq, hkv, tokens, columns, page, dtype):
    """Decode, prefill and tree launches that each take their rows' k and v from the step."""
    m = Mixed(device, dim, dtype, page, hq, hkv, tokens)
    before = [t.clone() for t in (m.pool.k, m.pool.v)]
    step = m.step()
    assert step._private and (columns is None or step.tree.plan.info.columns == columns)
    out = step.run(0, m.q, m.k, m.v)
    m.check_pool(before)
    m.check(out)
    for t in (m.pool.k, m.pool.v):   # and again, from pages without them
        t.copy_(before[0] if t is m.pool.k else before[1])
    assert torch.equal(step.run(0, m.q, m.k, m.v), out)
    m.check_pool(before)

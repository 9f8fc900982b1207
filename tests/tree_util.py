"""Inputs of the tests of drafted-token steps: rows of given lengths with given trees over a paged cache with shuffled pages."""
import numpy as np
import torch

from oracle import ref_tree as ref


def random_parents(counts, rng, forest=False):
    out = []
    for n in counts:
        for i in range(n):
            out.append(-1 if i == 0 or (forest and rng.random() < 0.2) else int(rng.integers(max(0, i - 9), i)))
    return torch.tensor(out, dtype=torch.int32)


def starts_of(counts):
    return [0] + np.cumsum(counts).tolist()


def tables(ctx, counts, page, rng, extra_cols=1, spare=2):
    """(block table [rows, columns] with the pages of cached tokens and nodes, pages in the pool)."""
    need = [-(-(c + n) // page) for c, n in zip(ctx, counts)]
    pages = sum(need) + spare
    order = rng.permutation(pages).tolist()
    cols = max(need + [0]) + extra_cols
    table = []
    for k in need:
        table.append(order[:k] + [-1] * (cols - k))
        order = order[k:]
    return table, pages


class AttnCase:
    def __init__(self, ctx, counts, hq, hkv, d, page, dtype, seed=0, forest=False, tail=3, scale_q=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.counts, self.starts, self.page = ctx, counts, starts_of(counts), page
        self.T, self.d, self.dtype = self.starts[-1], d, dtype
        self.parents = random_parents(counts, rng, forest)
        self.table, self.pages = tables(ctx, counts, page, rng)
        self.max_nodes = max(counts + [1])
        self.words = (self.max_nodes + 63) // 64
        self.seen = [set(ref.ancestors(self.parents, self.starts[b], i)) for b, n in enumerate(counts) for i in range(n)]
        self.q = (torch.randn(self.T + tail, hq, d, generator=g) * scale_q).to(dtype)       # `tail` tokens behind the last row
        self.k = torch.randn(self.pages, page, hkv, d, generator=g).to(dtype)
        self.v = torch.randn(self.pages, page, hkv, d, generator=g).to(dtype)
        self.scale = ref.scale_of(d)

    def mask(self):
        m = ref.mask_words(self.seen, self.words)
        return torch.cat([m, torch.full((self.q.shape[0] - self.T, self.words), -1, dtype=torch.int64)])

    def reference(self):
        return ref.attn(self.q[:self.T], self.k, self.v, self.ctx, self.starts, self.table, self.seen, self.scale)

    def check(self, out, what="", reference=None):
        o, mag, size, count = reference or self.reference()
        bound = ref.attn_bound(o, mag, size, count, self.d, self.dtype)
        err = (out[:self.T].double().cpu() - o).abs()
        bad = ~(err <= bound)
        assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {torch.nonzero(bad)[0].tolist()}, " \
            f"worst {float((err / bound).max()):.2f} times the bound"


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)

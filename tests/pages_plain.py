"""Plain forms, in 64 bits, of the operators over a paged cache, how far fp32 sums and rounded weights may be off them, and small pools to try them on."""
from __future__ import annotations

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
STEP32 = 2.0 ** -24


class Pool:
    """One layer's pages of some contexts with `keys` tokens each: values N(0, 1), pages in random order, the rows behind a context's tokens and the pages
    that nobody has hold `behind`.  `spare`: elements between two pages, `shift`: elements in front of the first."""

    def __init__(self, keys, kv_heads, size, dtype, page=16, seed=0, behind=float("nan"), spare=0, shift=0, entries=None):
        g = torch.Generator().manual_seed(seed)
        self.kv_heads, self.size, self.page, self.row, self.keys = kv_heads, size, page, 2 * kv_heads * size, list(keys)
        used = [-(-k // page) for k in keys]
        self.n_pages = sum(used) + 2
        order = torch.randperm(self.n_pages, generator=g)
        memory = torch.full((shift + self.n_pages * (page * self.row + spare),), behind, dtype=torch.float32)
        self.memory = memory.to(dtype).cuda()
        self.pool = torch.as_strided(self.memory, (self.n_pages, page, self.row), (page * self.row + spare, self.row, 1), shift)
        entries = max(1, max(used)) if entries is None else entries
        table = torch.full((len(keys), entries), 2 ** 31 - 1, dtype=torch.int32)      # entries that no token needs name no page
        self.rows = []                                                                # each context's rows, as the cache has them
        at = 0
        for i, k in enumerate(keys):
            table[i, :used[i]] = order[at:at + used[i]].int()
            at += used[i]
            rows = torch.randn((k, self.row), generator=g).to(dtype).cuda()
            self.rows.append(rows)
            self.store(table[i], rows, 0)
        self.table = table.cuda()

    def store(self, line, rows, start):
        for t in range(rows.shape[0]):
            self.pool[int(line[(start + t) // self.page]), (start + t) % self.page] = rows[t]

    def k(self, i):
        return self.rows[i].double()[:, :self.kv_heads * self.size].reshape(-1, self.kv_heads, self.size)

    def v(self, i):
        return self.rows[i].double()[:, self.kv_heads * self.size:].reshape(-1, self.kv_heads, self.size)


def attention(q, k, v, start, dtype, rounded):
    """q (tokens, heads, size) against k, v (keys, kv_heads, size): the causal result of tokens at positions start and up, and how far each of its
    elements may be off.  Counted: scores of `size` products in fp32, their rounding as exponents, the exponential (one step), sums over the keys in fp32, the
    weights rounded to the storage type where the products take them so (`rounded`; below the normal numbers of fp16 by half the smallest), the result's rounding."""
    n, heads, size = q.shape
    keys, kv_heads = k.shape[0], k.shape[1]
    g = heads // kv_heads
    out, off = torch.zeros((n, heads, size), dtype=torch.float64, device=q.device), torch.zeros((n, heads, size), dtype=torch.float64, device=q.device)
    for h in range(heads):
        kh, vh, qh = k[:, h // g], v[:, h // g], q[:, h].double()
        for t in range(n):
            m = min(start + t + 1, keys)
            s = (kh[:m] * qh[t]).sum(1) * size ** -0.5
            sizes = (kh[:m].abs() * qh[t].abs()).sum(1) * size ** -0.5
            w = torch.exp(s - s.max())
            w = w / w.sum()
            out[t, h] = w @ vh[:m]
            mean = w @ vh[:m].abs()
            each = 2 * ((size + 3) * STEP32 * float(sizes.max()) + 4 * STEP32 * float(s.abs().max())) + 8 * STEP32 + 2 * m * STEP32
            off[t, h] = each * mean + HALF_STEP[dtype] * out[t, h].abs() + STEP32 * 2.0 ** -100
            if rounded:
                off[t, h] += 2 * HALF_STEP[dtype] * mean
                if dtype == torch.float16:
                    off[t, h] += m * 2.0 ** -25 * vh[:m].abs().max() + 2.0 ** -25
            if dtype == torch.float16:
                off[t, h] += 2.0 ** -25      # results below its normal numbers
    return out, off


def hold(got, want, off, what=""):
    far = ((got.double() - want).abs() / off).max() if got.numel() else torch.tensor(0.0)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    assert float(far) <= 1.0, f"{what}: {float(far):.2f} of what rounding allows"


def logprobs(logits, tokens, n_top):
    """(given, entropy, ids, values) in 64 bits; ties by the lower index, NaN behind everything."""
    x = logits.double()
    p = torch.log_softmax(x, dim=1)
    entropy = -torch.where(p == -torch.inf, 0.0, p.exp() * p).sum(1)
    key = torch.where(torch.isnan(x), -torch.inf, x)
    order = key.sort(dim=1, descending=True, stable=True).indices
    order = order.gather(1, torch.isnan(x).gather(1, order).to(torch.uint8).sort(dim=1, stable=True).indices)
    ids = order[:, :n_top]
    return p.gather(1, tokens.long()[:, None])[:, 0], entropy, ids, p.gather(1, ids)

"""Cases of paged attention whose results show what was read: random ones with
queries drawn apart from the keys, so that every key weighs in, and ones with a
closed form, in which a lost, repeated or wrongly seen key is a whole share of
an output."""
import numpy as np
import torch

import paged_reference as ref

BF = torch.bfloat16
TILE = 32


def pages(rng, lengths, page, extra=3, width_extra=1):
    """(pages of the cache, a table of them in any order)."""
    need = [ref.ceil(max(int(x), 0), page) for x in lengths]
    count = sum(need) + extra
    table = rng.integers(0, count, (len(lengths), max(max(need), 1) + width_extra))
    order, at = rng.permutation(count), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return count, torch.tensor(table.astype(np.int32))


def starts(new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))


def random_case(seed, new, lengths, QH, KVH, HD, page, gate=False, qstd=1.0):
    """On the CPU. One generator makes keys, values and queries in turn."""
    g = torch.Generator().manual_seed(seed)
    count, table = pages(np.random.default_rng(seed), lengths, page)
    T = int(sum(new))
    k, v = (torch.randn(count, page, KVH, HD, generator=g).to(BF) for _ in range(2))
    q = (torch.randn(T, QH, HD, generator=g) * qstd).to(BF)
    return dict(q=q, k=k, v=v, table=table, row_start=starts(new), lengths=torch.tensor(np.array(lengths, np.int32)),
                gate=torch.randn(T, QH, HD, generator=g).to(BF) if gate else None, scale=HD ** -0.5)


# new tokens of the first request, its length, q heads, kv heads, head dim, page
LONG = [(40, 3000, 4, 1, 256, 16), (33, 2500, 2, 2, 128, 32), (70, 2300, 1, 1, 64, 64), (1, 9000, 8, 2, 256, 16), (2, 5000, 3, 1, 64, 16)]
VERY_LONG = (1, 140000, 2, 1, 64, 64)  # more splits than the join keeps maxima of

# new tokens, lengths, q heads, kv heads, head dim, page
SHAPES = [
    ([1], [520], 16, 2, 256, 16), ([5, 3, 1, 8], [5, 100, 64, 700], 16, 4, 128, 16), ([17], [17], 6, 2, 64, 16),
    ([33, 1, 70], [33, 257, 300], 4, 1, 64, 64), ([40], [1000], 16, 2, 256, 64), ([100, 1, 2, 65], [400, 90, 2, 65], 8, 2, 256, 16),
    ([129], [300], 3, 1, 256, 16), ([70, 0, 1], [70, 20, 9], 12, 2, 64, 16), ([260], [261], 2, 2, 64, 16),
    ([1], [4100], 24, 2, 128, 32), ([3, 2], [2500, 5000], 7, 1, 64, 16), ([513, 1], [700, 1500], 2, 1, 128, 32),
]


class Marked:
    """One request of `new` rows over `length` tokens, queries of 0: every key
    seen weighs the same, and channel c of a result is the share of the keys
    that `marks` gives it among those the row sees. Weights and sums are whole
    numbers below 2^24, so that a result is off by the division's, the join's
    and its own rounding alone."""

    def __init__(self, new, length, QH, KVH, HD, page, seed=0, bad=()):
        rng = np.random.default_rng(seed)
        self.new, self.length, self.QH, self.KVH, self.HD, self.page = new, length, QH, KVH, HD, page
        self.count, self.table = pages(rng, [length], page)
        self.good = torch.ones(length, dtype=torch.bool)
        self.place = self.table.clone()  # where the keys' rows are, of bad pages too
        for j in bad:
            self.good[j // page * page:(j // page + 1) * page] = False
            self.table[0, j // page] = [-1, self.count, 2**31 - 1, -2**31][j % 4]

    def values(self, marks, device):
        """Values with a 1 in channel marks[j] of key j, none where that is -1; rows outside the length hold ones."""
        v = torch.ones(self.count, self.page, self.KVH, self.HD, dtype=BF, device=device)
        j = torch.arange(self.length, device=device)
        hot = (marks.to(device)[:, None] == torch.arange(self.HD, device=device)).to(BF)
        v[self.place.to(device)[0, j // self.page].long(), j % self.page] = hot[:, None].expand(-1, self.KVH, -1)
        return v

    def shares(self, marks, seen=None):
        """[new, HD] in 64 bits; `seen` [new, length]: another mask than the operator's."""
        j = torch.arange(self.length)
        if seen is None:
            seen = self.good & (j <= (self.length - self.new + torch.arange(self.new))[:, None])
        hot = (marks[:, None] == torch.arange(self.HD)).double()
        n = seen.double().sum(1, keepdim=True)
        return torch.where(n > 0, seen.double() @ hot / n.clamp(min=1), 0.0)

    TOLERANCE = 2.0 ** -8 + 2.0 ** -18  # relative; a share of 0 is 0

    def tiles(self):
        """Marks of every key tile, as many at a time as there are channels."""
        tile = torch.arange(self.length) // TILE
        for first in range(0, int(tile[-1]) + 1, self.HD):
            yield torch.where((tile >= first) & (tile < first + self.HD), tile - first, -1)

    def last_keys(self):
        """Marks of the last keys and of the first, one channel each."""
        j = torch.arange(self.length)
        yield torch.where(j >= self.length - self.HD, self.length - 1 - j, -1)
        yield torch.where(j < self.HD, j, -1)

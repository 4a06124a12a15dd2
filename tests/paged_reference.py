"""Plain statements of the paged-cache operators in 64 bits (numpy and torch on
the CPU), for the tests."""
import numpy as np
import torch


def ceil(a, b):
    return -(-a // b)


def page_plan(table, cached, lengths, stack, free, page, rows):
    """The round's tables, stack and outputs, request by request; the inputs are left alone."""
    table, stack = table.copy(), [int(x) for x in stack]
    R, width = table.shape
    same = dict(table=table, stack=np.array(stack, dtype=np.int32), row_start=np.zeros(R + 1, np.int32),
                positions=np.zeros(rows, np.int32), slots=np.full(rows, -1, np.int32), free_left=free)
    have, want = [ceil(int(c), page) for c in cached], [ceil(int(x), page) for x in lengths]
    if any(c < 0 or x < 0 or max(h, w) > width for c, x, h, w in zip(cached, lengths, have, want)):
        return dict(same, status=[3, 0])
    given = [int(table[r, j]) for r in range(R) for j in range(want[r], have[r])]
    if free < 0 or free + len(given) > len(stack):
        return dict(same, status=[4, 0])
    new = [max(int(x) - int(c), 0) for c, x in zip(cached, lengths)]
    if sum(new) > rows:
        return dict(same, status=[2, sum(new) - rows])
    take = sum(max(w - h, 0) for w, h in zip(want, have))
    if take > free + len(given):
        return dict(same, status=[1, take - free - len(given)])
    pile = stack[:free] + given
    positions, slots = np.zeros(rows, np.int32), np.full(rows, -1, np.int32)
    start = np.zeros(R + 1, np.int32)
    t = 0
    for r in range(R):
        for j in range(have[r], want[r]):
            table[r, j] = pile.pop()
        for p in range(int(cached[r]), int(lengths[r])):
            positions[t] = p
            at = int(table[r, p // page])
            slots[t] = at * page + p % page if 0 <= at < len(stack) else -1
            t += 1
        start[r + 1] = t
    # entries past the free ones are what they were; those given back and kept are written
    after = list(stack)
    for i in range(free, len(pile)):
        after[i] = pile[i]
    return dict(table=table, stack=np.array(after, dtype=np.int32), row_start=start, positions=positions, slots=slots,
                free_left=len(pile), status=[0, 0])


def head(x, w, eps, freq, positions, pair_axis):
    """(rotated heads, |a| + |b| of each channel's pair) of x [T, heads, head_dim] in float64."""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = freq.shape[0]
    pos = torch.stack([positions[a].double() for a in pair_axis], 1)  # [T, half]
    angle = pos * freq.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
    size = y.abs()
    size[..., :half] = size[..., half:2 * half] = a.abs() + b.abs()
    y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y, size


def attention(q, key_cache, value_cache, table, row_start, lengths, scale, gate=None):
    """(out, bound) in float64. bound: how far a result may be off that forms F32
    scores and sums and BF16 weights and rounds to BF16 once. With A = sum_j p_j
    |v_j|: a weight is off by its rounding, 2^-8 of itself, by twice the score's
    error (HD products and sums of at most sum |q k| scale, 2^-24 each, and as
    much for the maximum), and by the exponential's and the sums' own roundings,
    2^-24 for each of the keys and 64 more; each moves out by that share of A."""
    q, keys, values = q.double(), key_cache.double(), value_cache.double()
    T, QH, HD = q.shape
    pages, page, KVH, _ = keys.shape
    out, off = torch.full_like(q, float("nan")), torch.zeros_like(q)
    for r in range(len(lengths)):
        b, e = int(row_start[r]), int(row_start[r + 1])
        length = max(0, min(int(lengths[r]), table.shape[1] * page))
        entry = table[r].long()
        j = torch.arange(length)
        at = entry[j // page] if length else j
        good = (at >= 0) & (at < pages)
        at = at.clamp(0, pages - 1)
        k, v = keys[at, j % page], values[at, j % page]  # [length, KVH, HD]
        for t in range(b, e):
            seen = good & (j <= length - (e - b) + (t - b))
            n = int(seen.sum())
            if n == 0:
                out[t] = 0
                continue
            for h in range(QH):
                kk, vv = k[seen, h // (QH // KVH)], v[seen, h // (QH // KVH)]
                p = torch.softmax(kk @ q[t, h] * scale, 0)
                out[t, h] = p @ vv
                reach = float((kk.abs() @ q[t, h].abs()).max()) * abs(scale)
                off[t, h] = (p @ vv.abs()) * (2.0 ** -8 + 2 * (HD + 4) * 2.0 ** -24 * reach + (n + 64) * 2.0 ** -24)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, off = out * g, off * g
    return out, off + 2.0 ** -8 * (out.abs() + off) + 1e-37

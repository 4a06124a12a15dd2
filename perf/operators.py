"""Performance cases of the paged-cache operators (cq35.page_plan,
cq35.paged_prepare, cq35.paged_attention): what a round of batched serving runs
beside a model's projections. `run` computes a case either in plain torch
operations or through the library's operators.
"""
from __future__ import annotations

import os
import random
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "catena-models_amd"))

own = False


def _plan(name, **kw):
    return dict(op="plan", name=name, **kw)


def _prepare(name, **kw):
    return dict(op="prepare", name=name, **kw)


def _attention(name, **kw):
    return dict(op="attention", name=name, **kw)


def listed():
    return [
        # a decode round of a few requests: one new token each, latency alone
        _plan("plan: 8 requests decode", requests=8, keys=32768, new=1, mix="decode", page=16, spread=1),
        # a continuous round: decode tokens, prompt chunks, finished requests
        # and rejected drafts that give pages back
        _plan("plan: 500 requests mixed", requests=500, keys=8192, new=512, mix="mixed", page=32, spread=2),
        # many long prompts at once
        _plan("plan: 64 prompts of 2048", requests=64, keys=4096, new=2048, mix="chunk", page=16, spread=3),
        # a decode round at the 35B head counts
        _prepare("prepare: 16 rows", rows=16, q_heads=16, kv_heads=2, head_dim=256, rope=64, axes=1, page=16),
        # an image prompt (time, height and width positions) at the dense head counts
        _prepare("prepare: 777 rows, 3 axes", rows=777, q_heads=8, kv_heads=2, head_dim=256, rope=64, axes=3, page=32),
        # the largest prompt chunk at the 35B head counts
        _prepare("prepare: 8192 rows", rows=8192, q_heads=16, kv_heads=2, head_dim=256, rope=64, axes=1, page=64),
        # one request, one token, a short context: latency
        _attention("attention: 1 x 1 over 520", requests=1, new=1, keys=520, mix="decode", q_heads=16, kv_heads=2,
                   head_dim=256, page=16, gate=True, spread=4),
        # concurrent long-context decode at the 35B head counts
        _attention("attention: 8 x 1 over 32768", requests=8, new=1, keys=32768, mix="decode", q_heads=16, kv_heads=2,
                   head_dim=256, page=32, gate=True, spread=5),
        # drafted tokens of many requests, plain attention heads
        _attention("attention: 32 x 5 over 5000", requests=32, new=5, keys=5000, mix="drafts", q_heads=16, kv_heads=4,
                   head_dim=128, page=16, gate=False, spread=6),
        # a continuous round: decode tokens and prompt chunks together
        _attention("attention: 16 mixed over 4096", requests=16, new=500, keys=4096, mix="mixed", q_heads=8, kv_heads=2,
                   head_dim=256, page=16, gate=True, spread=7),
        # prompts from their first token, small heads
        _attention("attention: 4 prompts of 1000", requests=4, new=1000, keys=1000, mix="chunk", q_heads=8, kv_heads=8,
                   head_dim=64, page=64, gate=False, spread=8),
        # a prompt chunk far into a long context at the 35B head counts
        _attention("attention: 2048 over 32768", requests=1, new=2048, keys=32768, mix="chunk", q_heads=16, kv_heads=2,
                   head_dim=256, page=64, gate=True, spread=9),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["plan", "prepare", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        mix = rng.choice(["decode", "mixed", "chunk"])
        requests = _log(rng, 1, 1000)
        keys = _log(rng, 32, 32768)
        new = 1 if mix == "decode" else min(keys, _log(rng, 2, max(2, 90000 // requests)))
        return dict(op=op, requests=requests, keys=keys, new=new, mix=mix, page=page, spread=rng.randrange(1 << 30))
    head_dim = rng.choice([64, 128, 256, 256])
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    if op == "prepare":
        most = 8192 * 20 * 1024 // (4 * (q_heads + 2 * kv_heads) * head_dim)
        return dict(op=op, rows=_log(rng, 1, min(16384, most)), q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    rope=rng.choice([head_dim // 4, head_dim // 2, head_dim]), axes=rng.choice([1, 3]), page=page)
    mix = rng.choice(["decode", "drafts", "chunk", "mixed"])
    while True:
        requests = _log(rng, 1, 64)
        keys = _log(rng, 16, 32768)
        new = {"decode": 1, "drafts": rng.randint(2, 8)}.get(mix) or min(keys, _log(rng, 16, 2048))
        if (requests * new * keys * q_heads <= 2048 * 32768 * 16 and requests * keys * kv_heads * head_dim <= 1 << 26
                and requests * new * keys * q_heads * head_dim <= 2048 * 30000 * 16 * 256):
            break
    return dict(op=op, requests=requests, new=new, keys=keys, mix=mix, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, gate=rng.random() < 0.5, spread=rng.randrange(1 << 30))


def _lengths(case):
    """(tokens cached before, tokens after) of each request; the first is as long as the case says."""
    rng = random.Random(case["spread"])
    cached, after = [], []
    for r in range(case["requests"]):
        keys = case["keys"] if r == 0 else rng.randint(max(1, case["keys"] // 4), case["keys"])
        if case["mix"] == "mixed":
            n = case["new"] if r == 0 else rng.choice([1, 1, 1, rng.randint(1, case["new"])])
        elif case["mix"] == "chunk":
            n = case["new"] if r == 0 else rng.randint(max(1, case["new"] // 2), case["new"])
        else:
            n = case["new"]
        n = min(n, keys)
        if case["op"] == "plan" and case["mix"] == "mixed" and rng.random() < 0.1:
            # a finished request, or drafts taken back
            cached.append(keys)
            after.append(rng.choice([0, max(0, keys - rng.randint(1, 40))]))
        else:
            cached.append(keys - n)
            after.append(keys)
    return cached, after


def _ceil(a, b):
    return -(-a // b)


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _normal(gen, shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(mean, std, generator=gen).to(dtype)


def _pair_axis(pairs, axes):
    """The axis of each rotated pair: time, height and width in turn, the
    last pairs (those left over by equal thirds) on the time axis."""
    if axes == 1:
        return None
    third = pairs // 3
    return [i % 3 if i < 3 * third else 0 for i in range(pairs)]


def prepare(case, seed):
    rng = np.random.default_rng([seed, 17])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=dict(case))
    P = case["page"]
    if case["op"] == "plan":
        cached, after = _lengths(case)
        width = _ceil(max(max(cached), max(after)), P) + 3
        have = [_ceil(c, P) for c in cached]
        need = sum(max(0, _ceil(a, P) - h) for a, h in zip(after, have))
        pages = sum(have) + need + 7 + len(cached)
        order = rng.permutation(pages).astype(np.int32)
        table = np.full((len(cached), width), -1, dtype=np.int32)
        at = 0
        for r, h in enumerate(have):
            table[r, :h] = order[at:at + h]
            at += h
        stack = np.full(pages, -1, dtype=np.int32)
        stack[:pages - at] = order[at:]
        s.update(table=_dev(table), cached=_dev(np.array(cached, dtype=np.int32)),
                 lengths=_dev(np.array(after, dtype=np.int32)), free_pages=_dev(stack),
                 free_count=_dev(np.array([pages - at], dtype=np.int32)),
                 rows=sum(max(0, a - c) for a, c in zip(after, cached)))
        return s
    QH, KVH, HD = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prepare":
        T, R = case["rows"], case["rope"]
        pages = _ceil(T, P) + 9
        slots = (rng.permutation(pages)[:_ceil(T, P), None] * P + np.arange(P)[None, :]).reshape(-1)[:T]
        # the projections' rows as the model makes them: query and gate of a
        # head side by side
        qg = _normal(gen, (T, QH, 2, HD))
        start = int(rng.integers(0, 200000))
        pos = np.stack([start + np.arange(T), start + np.arange(T) // 32, start + np.arange(T) % 32])[:case["axes"]]
        s.update(q=qg[:, :, 0], k=_normal(gen, (T, KVH, HD)), v=_normal(gen, (T, KVH, HD)),
                 q_weight=_normal(gen, (HD,), 0.02, 1.0, torch.float32),
                 k_weight=_normal(gen, (HD,), 0.02, 1.0, torch.float32),
                 inv_freq=_dev((1e7 ** (-np.arange(0, R, 2) / R)).astype(np.float32)),
                 positions=_dev(pos.astype(np.int32)), slots=_dev(slots.astype(np.int32)),
                 key_cache=_normal(gen, (pages, P, KVH, HD)), value_cache=_normal(gen, (pages, P, KVH, HD)),
                 pair_axis=_pair_axis(R // 2, case["axes"]), eps=1e-6)
        if s["pair_axis"] is not None:
            s["axis_index"] = torch.tensor(s["pair_axis"], device="cuda")
        return s
    cached, after = _lengths(case)
    new = [a - c for a, c in zip(after, cached)]
    T, width = sum(new), _ceil(max(after), P)
    pages = sum(_ceil(a, P) for a in after) + 5
    order = rng.permutation(pages).astype(np.int32)
    table = np.zeros((len(after), width), dtype=np.int32)
    at = 0
    for r, a in enumerate(after):
        table[r, :_ceil(a, P)] = order[at:at + _ceil(a, P)]
        at += _ceil(a, P)
    s.update(q=_normal(gen, (T, QH, HD), 2.0), key_cache=_normal(gen, (pages, P, KVH, HD)),
             value_cache=_normal(gen, (pages, P, KVH, HD)), table=_dev(table),
             row_start=_dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)),
             lengths=_dev(np.array(after, dtype=np.int32)), scale=HD ** -0.5, max_rows=max(new), max_keys=max(after),
             gate=_normal(gen, (T, QH, 2, HD))[:, :, 1] if case["gate"] else None)
    return s


# ------------------------------------------------------------ plain forms


def _plain_plan(s):
    P, T = s["case"]["page"], s["rows"]
    table, stack = s["table"], s["free_pages"]
    R, width = table.shape
    cached, after = s["cached"].long(), s["lengths"].long()
    have, want = (cached + P - 1) // P, (after + P - 1) // P
    new = (after - cached).clamp(min=0)
    row_start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    page_start = torch.cat([new.new_zeros(1), (want - have).clamp(min=0).cumsum(0)])
    gone = (have - want).clamp(min=0)
    gone_start = torch.cat([new.new_zeros(1), gone.cumsum(0)])
    free = s["free_count"].long()
    top = free + gone_start[-1]
    left = top - page_start[-1]
    # the stack with what is given back on it: entry i past the free ones is
    # page i - gone_start[r] of the pages that request r loses
    column = torch.arange(width, device=table.device)
    lost = (column >= want[:, None]) & (column < have[:, None])
    at = torch.where(lost, free + gone_start[:-1, None] + column - want[:, None], stack.numel())
    full = torch.cat([stack, stack.new_zeros(1)])
    full[at.reshape(-1)] = table.reshape(-1)
    # rows
    t = torch.arange(T, device=table.device)
    r = torch.searchsorted(row_start[1:].contiguous(), t, right=True)
    pos = cached[r] + t - row_start[r]
    j = pos // P
    fresh = j >= have[r]
    k = page_start[r] + j - have[r]
    page = torch.where(fresh, full[(top - 1 - k).clamp(0, stack.numel())], table[r, j])
    slots = page * P + pos % P
    flat = torch.cat([table.reshape(-1), table.new_zeros(1)])
    flat[torch.where(fresh, r * width + j, R * width)] = page
    table.copy_(flat[:-1].view(R, width))
    keep = torch.arange(stack.numel(), device=table.device) < left
    stack.copy_(torch.where(keep, full[:-1], stack))
    return (table, stack, row_start.int(), pos.int(), slots.int(), left.int(), torch.zeros_like(left.int()).expand(2))


def _plain_prepare(s):
    c = s["case"]
    half = c["rope"] // 2
    pos = s["positions"].double()
    if s["pair_axis"] is None:
        angle = pos[0][:, None] * s["inv_freq"].double()
    else:
        angle = pos[s["axis_index"]].t() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x.float()
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1).to(torch.bfloat16)

    slots = s["slots"].long()
    page, off = slots // c["page"], slots % c["page"]
    s["key_cache"][page, off] = turned(s["k"], s["k_weight"])
    s["value_cache"][page, off] = s["v"]
    return turned(s["q"], s["q_weight"]), s["key_cache"], s["value_cache"]


def _plain_attention(s):
    c = s["case"]
    P, KVH, HD = c["page"], c["kv_heads"], c["head_dim"]
    G, N, L = c["q_heads"] // KVH, s["max_rows"], s["max_keys"]
    R, T = s["table"].shape[0], s["q"].shape[0]
    j = torch.arange(L, device="cuda")
    page = s["table"].long()[:, j // P]
    k = s["key_cache"][page, j % P].float().permute(0, 2, 3, 1).contiguous()  # [R, KVH, HD, L]
    v = s["value_cache"][page, j % P].float().permute(0, 2, 1, 3).contiguous()
    start, lengths = s["row_start"].long(), s["lengths"].long()
    new = start[1:] - start[:-1]
    i = torch.arange(N, device="cuda")
    q = s["q"][(start[:-1, None] + i).clamp(max=T - 1)].float()  # [R, N, QH, HD]
    q = q.view(R, N, KVH, G, HD).permute(0, 2, 1, 3, 4).reshape(R, KVH, N * G, HD)
    score = torch.matmul(q, k).mul_(s["scale"]).view(R, KVH, N, G, L)
    pos = (lengths - new)[:, None] + i
    hidden = j > pos[..., None]  # [R, N, L]
    score.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(R, KVH, N * G, L), v).view(R, KVH, N, G, HD) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(R, N, KVH * G, HD)
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(start[1:].contiguous(), t, right=True)
    o = o[r, t - start[r]]
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(torch.bfloat16)


def run(state):
    op = state["case"]["op"]
    if own:
        import cq35
        s = state
        if op == "plan":
            p = cq35.page_plan(s["table"], s["cached"], s["lengths"], s["free_pages"], s["free_count"],
                               page_size=s["case"]["page"], rows=s["rows"])
            return s["table"], s["free_pages"], p.row_start, p.positions, p.slots, p.free_left, p.status
        if op == "prepare":
            q = cq35.paged_prepare(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["inv_freq"], s["positions"],
                                   s["slots"], s["key_cache"], s["value_cache"], eps=s["eps"], pair_axis=s["pair_axis"])
            return q, s["key_cache"], s["value_cache"]
        return cq35.paged_attention(s["q"], s["key_cache"], s["value_cache"], s["table"], s["row_start"], s["lengths"],
                                    gate=s["gate"], scale=s["scale"], max_rows=s["max_rows"], max_keys=s["max_keys"])
    return {"plan": _plain_plan, "prepare": _plain_prepare, "attention": _plain_attention}[op](state)


def work(case):
    if case["op"] == "plan":
        cached, after = _lengths(case)
        P = case["page"]
        rows = sum(max(0, a - c) for a, c in zip(after, cached))
        moved = sum(abs(_ceil(a, P) - _ceil(c, P)) for a, c in zip(after, cached))
        return {"bytes": 12 * len(cached) + 8 * rows + 8 * moved + 16, "flops": 0}
    QH, KVH, HD = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "prepare":
        T = case["rows"]
        return {"bytes": T * (4 * QH * HD + 8 * KVH * HD + 4 * case["axes"] + 4) + 8 * HD + 2 * case["rope"],
                "flops": T * (QH + KVH) * (4 * HD + 3 * case["rope"])}
    cached, after = _lengths(case)
    rows = sum(after) - sum(cached)
    seen = sum((a * (a + 1) - c * (c + 1)) // 2 for a, c in zip(after, cached))
    return {"bytes": rows * QH * HD * (6 if case["gate"] else 4) + sum(after) * KVH * HD * 4
            + sum(_ceil(a, case["page"]) for a in after) * 4, "flops": 4 * HD * QH * seen}


# ------------------------------------------------------------ in 64 bits


def _exact_prepare(s):
    c, half = s["case"], s["case"]["rope"] // 2
    axis = s["pair_axis"] or [0] * half
    pos, freq = s["positions"].cpu().numpy().astype(np.float64), s["inv_freq"].cpu().numpy().astype(np.float64)
    angle = torch.from_numpy(np.stack([pos[axis[i]] * freq[i] for i in range(half)], 1)).cuda().unsqueeze(1)
    turn = torch.polar(torch.ones_like(angle), angle)

    def head(x, w):
        x = x.double()
        y = x / (x.square().sum(-1, keepdim=True) / c["head_dim"] + s["eps"]).sqrt() * w.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return y

    key, value = s["key_cache"].double(), s["value_cache"].double()
    slots = s["slots"].long()
    key.view(-1, *key.shape[2:]).index_copy_(0, slots, head(s["k"], s["k_weight"]))
    value.view(-1, *value.shape[2:]).index_copy_(0, slots, s["v"].double())
    return head(s["q"], s["q_weight"]), key, value


def _exact_attention(s):
    c = s["case"]
    P, KVH = c["page"], c["kv_heads"]
    G = c["q_heads"] // KVH
    start, lengths, table = s["row_start"].tolist(), s["lengths"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, length in enumerate(lengths):
        rows = slice(start[r], start[r + 1])
        n = start[r + 1] - start[r]
        pages = table[r, :_ceil(length, P)]
        keys = s["key_cache"][pages].flatten(0, 1)[:length].double()
        values = s["value_cache"][pages].flatten(0, 1)[:length].double()
        late = torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None]
        for h in range(c["q_heads"]):
            x = s["q"][rows, h].double() @ keys[:, h // G].t().contiguous() * s["scale"]
            p = torch.softmax(x.masked_fill(late, -torch.inf), -1)
            out[rows, h] = p @ values[:, h // G].contiguous()
    if s["gate"] is not None:
        out /= 1 + torch.exp(-s["gate"].double())
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return _exact_prepare(s) if case["op"] == "prepare" else _exact_attention(s)

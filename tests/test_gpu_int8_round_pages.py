"""Rounds with projections in 8 bits over pages: what the requests hold after several rounds,
and every context on the way, against the same tokens in one round of their own pool."""
import pytest

import paged_reference
from test_gpu_int8_round import HD, HIDDEN, KVH, PAGE, QH, i32, inputs, ops, pages, say, weights

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def attend(w, s, x, residual, held, after):
    """The round up to its contexts; (contexts, queries, gates, plan)."""
    o, rows = ops(), x.shape[0]
    plan = o.page_plan(s["table"], i32(held), i32(after), s["stack"], s["free"], page_size=PAGE, rows=rows)
    p = o.int8_linear(o.norm_quantize(x, w["norms"][0], residual=residual), w["qkv"])
    qg, kv = p[:, :2 * QH * HD].unflatten(1, (QH, 2, HD)), p[:, 2 * QH * HD:].unflatten(1, (2 * KVH, HD))
    q = o.paged_prepare(qg[:, :, 0], kv[:, :KVH], kv[:, KVH:], w["qn"], w["kn"], w["freq"], plan.positions, plan.slots, s["k"], s["v"])
    ctx = o.paged_attention(q, s["k"], s["v"], s["table"], plan.row_start, i32(after), gate=qg[:, :, 1])
    s["free"] = plan.free_left
    return ctx.cpu(), q.cpu(), qg[:, :, 1].cpu(), plan


def held_tokens(s, r, length):
    """The keys and values of a request in order."""
    at = torch.arange(length)
    entry = s["table"][r].cpu().long()[at // PAGE]
    assert bool(((entry >= 0) & (entry < s["k"].shape[0])).all())
    return s["k"].cpu()[entry, at % PAGE], s["v"].cpu()[entry, at % PAGE]


def test_rounds_against_one():
    w, s = weights(), pages(3)
    held, rows_of, contexts = [0, 0, 0], [[], [], []], [[], [], []]
    for turn, after in enumerate(([40, 7, 0], [41, 8, 130], [42, 0, 131], [43, 21, 132])):
        say("round", turn, held, after)
        x, r, _ = inputs(turn, sum(max(a - b, 0) for a, b in zip(after, held)))
        ctx, _, _, plan = attend(w, s, x, r, held, after)
        assert plan.status.tolist() == [0, 0]
        at = 0
        for i, (a, b) in enumerate(zip(after, held)):
            n = max(a - b, 0)
            if a < b:
                rows_of[i], contexts[i] = rows_of[i][:a], contexts[i][:a]
            rows_of[i] += [(x[t], r[t]) for t in range(at, at + n)]
            contexts[i] += list(ctx[at:at + n])
            at += n
        held = after
    one = pages(3)
    flat = [t for rows in rows_of for t in rows]
    assert [len(rows) for rows in rows_of] == held
    x, r = (torch.stack([t[k] for t in flat]) for k in (0, 1))
    assert x.shape == (sum(held), HIDDEN)
    ctx, q, gate, plan = attend(w, one, x, r, [0, 0, 0], held)
    # a token's keys and values do not depend on what it was computed with
    for i, n in enumerate(held):
        for a, b in zip(held_tokens(s, i, n), held_tokens(one, i, n)):
            assert torch.equal(a, b), i
    want, off = paged_reference.attention(q, one["k"].cpu(), one["v"].cpu(), one["table"].cpu(), plan.row_start.cpu(), held, HD ** -0.5, gate)
    for got in (ctx, torch.stack([t for rows in contexts for t in rows])):
        away = (got.double() - want).abs()
        assert bool((away <= off).all()), (away / off).max()

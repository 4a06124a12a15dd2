"""A round of serving with its projections in 8 bits: norm, projections, pages,
attention, gated feed-forward, vocabulary head and log probabilities, each
operator on what the one in front of it made."""
import threading

import numpy as np
import pytest

import int8_reference as ref
from test_gpu_logprobs import check as check_logprobs

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
HIDDEN, QH, KVH, HD, WIDE, VOCAB, PAGE = 512, 4, 2, 128, 768, 5001, 16


def say(*a):
    print(*a, flush=True)


def ops():
    import cq35
    return cq35


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32)).cuda()


def weights(seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.empty(s, device="cuda").normal_(generator=g)  # noqa: E731
    q8 = lambda n, k: ops().quantize_rows((normal(n, k) * k ** -0.5).to(BF))  # noqa: E731
    return dict(qkv=q8((2 * QH + 2 * KVH) * HD, HIDDEN), o=q8(HIDDEN, QH * HD), up=q8(2 * WIDE, HIDDEN), down=q8(HIDDEN, WIDE),
                head=q8(VOCAB, HIDDEN), norms=[1 + 0.1 * normal(HIDDEN) for _ in range(3)], qn=1 + 0.1 * normal(HD), kn=1 + 0.1 * normal(HD),
                freq=(1e4 ** (-torch.arange(0, 32, 2, device="cuda") / 32)).float())


def pages(requests, width=12):
    return dict(table=torch.full((requests, width), -1, dtype=torch.int32, device="cuda"), stack=torch.arange(64, dtype=torch.int32, device="cuda"),
                free=i32([64]), k=torch.zeros(64, PAGE, KVH, HD, dtype=BF, device="cuda"), v=torch.zeros(64, PAGE, KVH, HD, dtype=BF, device="cuda"))


def run(w, s, x, residual, cached, lengths, tokens, seen=None):
    """The round; `seen` gets every operator's inputs and outputs."""
    o, rows = ops(), x.shape[0]
    note = seen.append if seen is not None else lambda _: None
    plan = o.page_plan(s["table"], cached, lengths, s["stack"], s["free"], page_size=PAGE, rows=rows)
    n = o.norm_quantize(x, w["norms"][0], residual=residual)
    note(("norm", x, residual, w["norms"][0], n))
    p = o.int8_linear(n, w["qkv"])
    note(("linear", n, w["qkv"], p))
    qg, kv = p[:, :2 * QH * HD].unflatten(1, (QH, 2, HD)), p[:, 2 * QH * HD:].unflatten(1, (2 * KVH, HD))
    q = o.paged_prepare(qg[:, :, 0], kv[:, :KVH], kv[:, KVH:], w["qn"], w["kn"], w["freq"], plan.positions, plan.slots, s["k"], s["v"])
    ctx = o.paged_attention(q, s["k"], s["v"], s["table"], plan.row_start, lengths, gate=qg[:, :, 1]).view(rows, QH * HD)
    c = o.quantize_rows(ctx)
    note(("quantize", ctx, c))
    y = o.int8_linear(c, w["o"])
    note(("linear", c, w["o"], y))
    m = o.norm_quantize(y, w["norms"][1], residual=n.summed)
    note(("norm", y, n.summed, w["norms"][1], m))
    both = o.int8_linear(m, w["up"])
    note(("linear", m, w["up"], both))
    g = o.gated_quantize(both[:, :WIDE], both[:, WIDE:])
    note(("gated", both[:, :WIDE], both[:, WIDE:], g))
    z = o.int8_linear(g, w["down"])
    note(("linear", g, w["down"], z))
    e = o.norm_quantize(z, w["norms"][2], residual=m.summed)
    note(("norm", z, m.summed, w["norms"][2], e))
    logits = o.int8_linear(e, w["head"], dtype=F32)
    note(("linear", e, w["head"], logits))
    a = o.token_logprobs(logits, tokens, top=5)
    note(("logprobs", logits, tokens, a))
    return ctx, logits, a.logprobs, a.entropy, a.top_tokens, a.top_logprobs, plan.free_left


def check(kind, *t):
    if kind == "norm":
        x, r, w, n = t
        assert torch.equal(n.summed, (x.float() + r.float()).to(BF))
        ref.check_rows(n.data, n.scale, ref.norm(n.summed, w, 1e-6), ref.NORM_REL)
    elif kind == "linear":
        x, w, out = t
        assert torch.equal(out, ref.linear(x[:2], w, out.dtype))
    elif kind == "quantize":
        ref.check_rows(t[1].data, t[1].scale, t[0].double(), 0.0)
    elif kind == "gated":
        ref.check_rows(t[2].data, t[2].scale, ref.gated(t[0], t[1]), ref.gated_rel(t[0]))
    else:
        check_logprobs(t[0], t[1], 5, t[2])


def inputs(seed, rows):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, r = (torch.empty(rows, HIDDEN, device="cuda").normal_(generator=g).to(BF) for _ in range(2))
    return x, r, torch.randint(VOCAB, (rows, 1), device="cuda", generator=g)


def test_rounds():
    """Prompts and single tokens: every operator against its statement, and the pages' tokens
    against attention over the same tokens in one pool."""
    w, s = weights(), pages(3)
    held = [0, 0, 0]
    for turn, after in enumerate(([40, 7, 0], [41, 8, 130], [42, 0, 131], [43, 21, 132])):
        rows = sum(max(a - b, 0) for a, b in zip(after, held))
        say("round", turn, held, after, rows)
        x, r, t = inputs(turn, rows)
        seen = []
        out = run(w, s, x, r, i32(held), i32(after), t, seen)
        for step in seen:
            check(*step)
        assert bool(torch.isfinite(out[0]).all())
        s["free"], held = out[-1], after


def test_captured_rounds():
    """A decode round as a graph, replayed with eager rounds of another pool between the replays."""
    w = weights()
    s, other = pages(4), pages(4)
    start = [5, 16, 31, 90]
    x, r, t = inputs(1, sum(start))
    for pool in (s, other):
        pool["free"] = run(w, pool, x, r, i32([0] * 4), i32(start), t)[-1].clone()
    x, r, t = inputs(2, 4)
    cached, after = i32(start), i32([n + 1 for n in start])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = run(w, s, x, r, cached, after, t)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(5):
        new = inputs(10 + turn, 4)
        for a, b in zip((x, r, t), new):
            a.copy_(b)
        cached.copy_(i32([n + turn for n in start]))
        after.copy_(i32([n + turn + 1 for n in start]))
        graph.replay()
        torch.cuda.synchronize()
        want = run(w, other, *new[:2], cached, after, new[2])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        s["free"].copy_(got[-1])
        other["free"].copy_(want[-1])


def test_two_threads():
    """Two rounds at once from two threads, on a stream each."""
    w = weights()
    x, r, t = inputs(3, 60)
    want = run(w, pages(2), x, r, i32([0, 0]), i32([40, 20]), t)
    torch.cuda.synchronize()
    results, failed = {}, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    results[k] = run(w, pages(2), x, r, i32([0, 0]), i32([40, 20]), t)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(results[k], want))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed and len(results) == 2, failed

"""Calls of the paged operators as their documentation allows them: workspaces
and outputs of the caller's, results in place, tables shared by requests, caches
laid out in other orders, few and very many heads, empty calls, and numbers in
device memory that make no sense."""
import numpy as np
import pytest

import paged_reference as ref
import test_gpu_paged as base
from paged_cases import random_case
from test_gpu_paged import (BF, KEYS, check_attention, check_plan, check_prepare, i32, ops, plan_case, prepare_case,
                            run_attention, say)

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

steered = base.steered  # both kernels

SPLIT = ([3, 40, 1], [3000, 1000, 2500], 8, 2, 128, 16)


def on_device(s, **kw):
    return dict(s, k=s["k"].cuda(), v=s["v"].cuda(), **kw)


def device_args(s):
    return [s[n].cuda() for n in ("table", "row_start", "lengths")]


def bits(t):
    return t.contiguous().view(torch.int16)


# -------------------------------------------------------- workspace, outputs


def test_workspace_of_the_caller(steered):
    """Of the bytes asked for, holding anything, used again and again."""
    s = on_device(random_case(1, *SPLIT))
    q, dev = s["q"].cuda(), device_args(s)
    rows, QH, HD = q.shape
    for hints in (dict(max_keys=KEYS[0]), dict(max_rows=40, max_keys=max(3000, KEYS[0]))):
        n = ops().paged_attention_workspace(rows, 3, QH, 2, HD, hints.get("max_rows", 0), hints["max_keys"])
        assert n > 0
        want = ops().paged_attention(q, s["k"], s["v"], *dev, **hints)
        around = torch.full((n + 512,), 255, dtype=torch.uint8, device="cuda")  # NaN as floats
        work = around[256:256 + n]
        for _ in range(3):
            got = ops().paged_attention(q, s["k"], s["v"], *dev, workspace=work, **hints)
            assert torch.equal(got, want)
        assert bool((around[:256] == 255).all()) and bool((around[256 + n:] == 255).all())
        with pytest.raises(ops().CQ35Error, match="workspace"):
            ops().paged_attention(q, s["k"], s["v"], *dev, workspace=work[:-1], **hints)
        with pytest.raises(ops().CQ35Error, match="workspace"):
            ops().paged_attention(q, s["k"], s["v"], *dev, workspace=around[8:], **hints)
    check_attention(s, want)


def test_two_graphs_that_share_a_workspace(steered):
    """On one stream, replayed in turn, eager work between."""
    cases = [on_device(random_case(2 + i, *SPLIT)) for i in range(2)]
    dev = [[c["q"].cuda(), *device_args(c)] for c in cases]
    hints = dict(max_keys=max(3000, KEYS[0]))
    n = ops().paged_attention_workspace(44, 3, 8, 2, 128, 0, hints["max_keys"])
    work = torch.zeros(n, dtype=torch.uint8, device="cuda")
    want = [ops().paged_attention(d[0], c["k"], c["v"], *d[1:], **hints) for c, d in zip(cases, dev)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c, d in zip(cases, dev):
        out = torch.zeros_like(d[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops().paged_attention(d[0], c["k"], c["v"], *d[1:], out=out, workspace=work, **hints)
        graphs.append(graph), outs.append(out)
    for turn in range(5):
        for i in (0, 1, 1, 0)[turn % 2:]:
            outs[i].fill_(7)
            graphs[i].replay()
            torch.randn(300, 300, device="cuda").sum().item()
            assert torch.equal(outs[i], want[i])


def test_plan_into_an_earlier_plans_tensors():
    c = plan_case(51, 40, 16, 300)
    dev, p = base.run_plan(c, c["rows"])
    check_plan(c, c["rows"], dev, p)
    other = plan_case(52, 40, 16, 300)
    rows = c["rows"]
    d = dict(table=i32(other["table"]).cuda(), stack=i32(other["stack"]).cuda(), cached=i32(other["cached"]).cuda(),
             lengths=i32(other["lengths"]).cuda(), free=i32([other["free"]]).cuda())
    again = ops().page_plan(d["table"], d["cached"], d["lengths"], d["stack"], d["free"], page_size=16, rows=rows, out=p)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(again, p))
    check_plan(other, rows, d, again)
    with pytest.raises(ops().CQ35Error, match="count left"):
        ops().page_plan(d["table"], d["cached"], d["lengths"], d["stack"], p.free_left, page_size=16, rows=rows, out=p)


# ------------------------------------------------------------------ in place


@pytest.mark.parametrize("HD,QH,KVH,new,length", [(64, 8, 2, 70, 90), (256, 8, 2, 60, 400), (128, 4, 1, 300, 320), (256, 4, 1, 3, 40)])
def test_in_place_beside_non_finite_values(HD, QH, KVH, new, length, steered):
    """Rows that are done again read their queries again, beside rows whose
    results have taken their queries' place."""
    say("in place, non-finite", HD, new, length)
    s = on_device(random_case(HD + new, [new, 2], [length, 50], QH, KVH, HD, 16, True))
    for j, x in ((length - 1, float("nan")), (length - new // 2, float("inf")), (length - new // 3, float("nan"))):
        page, at = int(s["table"][0, j // 16]), j % 16
        s["v"][page, at, :, j % HD] = x
        if x != x:
            s["k"][page, at] = x
    want = run_attention(s)
    both = torch.stack([s["q"], s["gate"]], 2).cuda()
    got = ops().paged_attention(both[:, :, 0], s["k"], s["v"], *device_args(s), gate=both[:, :, 1], out=both[:, :, 0],
                                scale=s["scale"], max_keys=KEYS[0])
    assert torch.equal(bits(got), bits(want)) and torch.equal(both[:, :, 1].cpu(), s["gate"])
    assert bool(torch.isnan(got[new - 1]).any()) and bool(torch.isfinite(got[:new // 2 - 1]).all())


def test_in_place_of_split_rows(steered):
    s = on_device(random_case(9, *SPLIT))
    want = run_attention(s, max_keys=max(3000, KEYS[0]))
    q = s["q"].cuda()
    got = ops().paged_attention(q, s["k"], s["v"], *device_args(s), out=q, max_keys=max(3000, KEYS[0]))
    assert got is q and torch.equal(got, want)


# ------------------------------------------------------------------- tables


def test_requests_that_share_a_table(steered):
    """One row of pages for all requests (a shared prompt): an expanded table."""
    s = on_device(random_case(12, [2, 5, 40], [700, 700, 700], 4, 2, 64, 16))
    s["table"][:] = s["table"][0].clone()
    check_attention(s, run_attention(s))
    want = run_attention(s)
    table = s["table"][:1].cuda().expand(3, -1)
    got = ops().paged_attention(s["q"].cuda(), s["k"], s["v"], table, *device_args(s)[1:], max_keys=KEYS[0])
    assert torch.equal(got, want)


def test_a_table_inside_a_larger_one(steered):
    s = on_device(random_case(13, [2, 40], [90, 200], 4, 2, 64, 16))
    whole = torch.full((2, s["table"].shape[1] + 9), 2**31 - 1, dtype=torch.int32, device="cuda")
    view = whole[:, 4:4 + s["table"].shape[1]]
    view.copy_(s["table"])
    got = ops().paged_attention(s["q"].cuda(), s["k"], s["v"], view, *device_args(s)[1:], max_keys=KEYS[0])
    assert torch.equal(got, run_attention(s))


# ------------------------------------------------------------------- layouts


def relaid(t, order, gap=0):
    """A copy whose dimensions follow each other in memory as `order` says, head_dim innermost."""
    shape = [t.shape[i] for i in order] + [t.shape[3]]
    back = [order.index(i) for i in range(3)] + [3]
    out = torch.empty(*shape[:-1], shape[-1] + gap, dtype=t.dtype, device="cuda")[..., :shape[-1]].permute(*back)
    out.copy_(t)
    return out


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
def test_caches_in_any_order(order, steered):
    """Pages, rows and heads in any order, rows apart."""
    say("order", order)
    for HD, page in ((64, 16), (256, 32)):
        s = random_case(sum(order) + HD, [1, 50, 3], [40, 300, 33], 4, 2, HD, page, True)
        s = dict(s, k=relaid(s["k"], order, 8), v=relaid(s["v"], order, 8))
        check_attention(s, run_attention(s))
        T, slots = 70, np.random.default_rng(1).permutation(s["k"].shape[0] * page)[:70]
        p = prepare_case(3, T, 4, 2, HD, 32, 1)
        before = s["k"].cpu().clone(), s["v"].cpu().clone()
        out = base.run_prepare(p, 2, HD, s["k"], s["v"], slots)
        check_prepare(p, out, s["k"], s["v"], before, slots.tolist(), page)


def test_rows_as_far_apart_as_allowed(steered):
    """Rows of a page 2^26 elements apart, the pages inside them: 2^30 elements a side."""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("not enough memory")
    KVH, page, apart = 2, 16, 1 << 26
    for HD in (64, 256):
        s = random_case(HD, [1, 40], [50, 300], 4, KVH, HD, page)
        count = s["k"].shape[0]
        far = []
        for n in ("k", "v"):
            buffer = torch.empty(page * apart, dtype=BF, device="cuda")
            view = buffer.as_strided((count, page, KVH, HD), (KVH * HD, apart, HD, 1))
            view.copy_(s[n])
            far.append(view)
        s = dict(s, k=far[0], v=far[1])
        check_attention(s, run_attention(s))
        del far


@pytest.mark.parametrize("page", [1024, 65536])
def test_large_pages(page, steered):
    say("pages of", page)
    s = on_device(random_case(page, [1, 40, 2], [page + 30, 700, 33], 4, 1, 64, page))
    check_attention(s, run_attention(s))


# --------------------------------------------------------------------- heads


@pytest.mark.parametrize("QH,KVH,HD", [(40, 1, 64), (300, 1, 128), (512, 2, 64), (96, 32, 256), (33, 33, 128), (1024, 1024, 64), (31, 1, 256)])
def test_head_counts(QH, KVH, HD, steered):
    """Groups of one to several hundred query heads, up to the most of heads."""
    say("heads", QH, KVH, HD)
    few = KVH > 100
    s = on_device(random_case(QH + HD, [2, 1] if few else [3, 1, 20], [40, 3] if few else [100, 700, 60], QH, KVH, HD, 16))
    check_attention(s, run_attention(s))
    T = 19
    p = prepare_case(QH, T, QH, KVH, HD, 32, 1)
    k, v = base.cache_tensors(3, 16, KVH, HD)
    before = k.cpu().clone(), v.cpu().clone()
    slots = np.random.default_rng(2).permutation(48)[:T]
    check_prepare(p, base.run_prepare(p, KVH, HD, k, v, slots), k, v, before, slots.tolist(), 16)


@pytest.mark.parametrize("T", [2047, 4097, 6145, 16390, 20000])
def test_prepare_many_rows(T):
    """Blocks of one to eight rows, the last one short."""
    say("prepare", T)
    s = prepare_case(T, T, 2, 1, 64, 16, 2)
    pages = ref.ceil(T, 16) + 1
    k, v = base.cache_tensors(pages, 16, 1, 64)
    slots = np.random.default_rng(T).permutation(pages * 16)[:T]
    out = base.run_prepare(s, 1, 64, k, v, slots)
    # the cache as a whole, without a loop over its rows
    at = torch.tensor(slots.astype(np.int64))
    want, size = ref.head(s["kv"][:, :1], s["kw"], 1e-6, s["freq"], s["positions"], s["axis"])
    got = k.cpu().view(-1, 1, 64)[at].double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * size + 1e-37).all())
    want, size = ref.head(s["qg"][:, :, :64], s["qw"], 1e-6, s["freq"], s["positions"], s["axis"])
    assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * size + 1e-37).all())
    assert torch.equal(v.cpu().view(-1, 1, 64)[at], s["kv"][:, 1:])


def test_prepare_heads_in_front_of_rows():
    """Queries, keys and values laid out head by head, positions below zero."""
    T, QH, KVH, HD = 60, 6, 2, 128
    s = prepare_case(7, T, QH, KVH, HD, 64, 1)
    s["positions"] = -s["positions"]
    k, v = base.cache_tensors(4, 16, KVH, HD)
    before = k.cpu().clone(), v.cpu().clone()
    turned = lambda x: x.transpose(0, 1).contiguous().cuda().transpose(0, 1)  # noqa: E731
    out = torch.zeros(QH, T, HD, dtype=BF, device="cuda").transpose(0, 1)
    got = ops().paged_prepare(turned(s["qg"][:, :, :HD]), turned(s["kv"][:, :KVH]), turned(s["kv"][:, KVH:]), s["qw"].cuda(),
                              s["kw"].cuda(), s["freq"].cuda(), s["positions"][0].cuda(), i32(np.arange(T)).cuda(), k, v, out=out)
    check_prepare(s, got, k, v, before, list(range(T)), 16)


# ------------------------------------------------------------- empty, senseless


def test_empty_calls():
    s = on_device(random_case(3, [2], [40], 4, 2, 64, 16))
    table, row_start, lengths = device_args(s)
    none = s["q"][:0].cuda()
    assert ops().paged_attention(none, s["k"], s["v"], table, row_start * 0, lengths).shape == (0, 4, 64)
    out = torch.full((2, 4, 64), 3.0, dtype=BF, device="cuda")
    ops().paged_attention(s["q"].cuda(), s["k"], s["v"], table[:0], row_start[:1], lengths[:0], out=out)
    assert bool((out == 3).all())
    w, f = torch.ones(64, device="cuda"), torch.ones(8, device="cuda")
    kv = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    before = s["k"].clone()
    assert ops().paged_prepare(none, kv, kv, w, w, f, lengths[:0], lengths[:0], s["k"], s["v"]).shape == (0, 4, 64)
    assert torch.equal(before, s["k"])
    c = plan_case(3, 5, 16, 100)
    c["lengths"] = np.minimum(c["lengths"], c["cached"])  # nobody grows
    dev, p = base.run_plan(c, 0)
    check_plan(c, 0, dev, p)


def test_row_starts_that_make_no_sense(steered):
    """Descending, overlapping, negative, past the end: rows of no request are
    left alone, nothing outside the output is touched, and requests whose rows
    are in order have their results."""
    rng = np.random.default_rng(4)
    s = on_device(random_case(21, [9, 9, 9, 9], [300, 90, 33, 2000], 4, 2, 128, 16))
    T = s["q"].shape[0]
    around = torch.full((T + 8, 4, 128), 5.0, dtype=BF, device="cuda")
    far = [-2**31, -7, 0, 4, 11, T, T + 3, 2**31 - 1]
    for turn in range(40):
        bad = dict(s, row_start=i32(rng.choice(far, 5)), lengths=i32(rng.choice([-2**31, -1, 0, 5, 300, 2**31 - 1], 4)))
        around.fill_(5)
        run_attention(bad, out=around[4:4 + T])
        assert bool((around[:4] == 5).all()) and bool((around[4 + T:] == 5).all())
        start, inside = bad["row_start"].tolist(), torch.zeros(T, dtype=torch.bool)
        for a, b in zip(start, start[1:]):
            inside[max(a, 0):max(0, min(b, T))] = True
        assert bool((around[4:4 + T][~inside] == 5).all())
    good = dict(s, row_start=i32([9, 18, 18, 9, 9]))  # the second one's rows are gone, the third descends
    around.fill_(5)
    run_attention(good, out=around[4:4 + T])
    alone = dict(s, q=s["q"][9:18], row_start=i32([0, 9]), lengths=s["lengths"][:1], table=s["table"][:1])
    check_attention(alone, around[13:22])


def test_two_equal_slots_hold_one_of_the_rows():
    """Piece by piece of 16 bytes: every piece is one of the two rows'."""
    T, HD = 2, 64
    s = prepare_case(31, T, 1, 1, HD, 16, 1)
    got = []
    for slots in ([3, 7], [3, 3]):
        k, v = base.cache_tensors(1, 16, 1, HD, fill=0.0)
        base.run_prepare(s, 1, HD, k, v, slots)
        got.append((k[0, :, 0].cpu(), v[0, :, 0].cpu()))
    for apart, same in zip(*got):
        a, b, x = (t.view(8, 8) for t in (apart[3], apart[7], same[3]))
        assert all(torch.equal(x[i], a[i]) or torch.equal(x[i], b[i]) for i in range(8))
        assert bool((same[7] == 0).all())


# ------------------------------------------------------------------- padding


def test_padded_rounds_with_an_output_of_the_caller(steered):
    """Rows behind the last request's stay what the caller made them: zeros, so
    that a projection of all rows stays finite, replay after replay."""
    rows, R, QH, HD = 24, 6, 8, 128
    st = base.round_state(seed=5)
    for n in ("qw", "kw", "freq"):
        st[n + "_dev"] = st[n].cuda()
    g = torch.Generator().manual_seed(9)
    qg = torch.full((rows, QH, 2, HD), float("nan"), dtype=BF, device="cuda")
    kv = torch.full((rows, 4, HD), float("nan"), dtype=BF, device="cuda")
    cached, lengths = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    q, out = torch.zeros(rows, QH, HD, dtype=BF, device="cuda"), torch.zeros(rows, QH, HD, dtype=BF, device="cuda")
    w = torch.randn(QH * HD, 64, generator=g).to(BF).cuda()

    def call():
        p = ops().page_plan(st["table"], cached, lengths, st["stack"], st["free"], page_size=st["page"], rows=rows)
        ops().paged_prepare(qg[:, :, 0], kv[:, :2], kv[:, 2:], st["qw_dev"], st["kw_dev"], st["freq_dev"], p.positions, p.slots,
                            st["k"], st["v"], out=q)
        ops().paged_attention(q, st["k"], st["v"], st["table"], p.row_start, lengths, gate=qg[:, :, 1], out=out, max_keys=KEYS[0])
        return p

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = call()
    held = [0] * R
    for turn in range(5):
        to = [h + (turn + r) % 4 for r, h in enumerate(held)]
        n = sum(to) - sum(held)
        qg.fill_(float("nan")), kv.fill_(float("nan"))  # the rows behind are nothing
        qg[:n] = torch.randn(n, QH, 2, HD, generator=g).to(BF).cuda()
        kv[:n] = torch.randn(n, 4, HD, generator=g).to(BF).cuda()
        cached.copy_(i32(held)), lengths.copy_(i32(to))
        out.zero_()
        graph.replay()
        projected = (out.view(rows, -1) @ w).cpu()
        assert p.status.tolist() == [0, 0]
        assert bool(torch.isfinite(projected).all()) and bool((out[n:] == 0).all()) and bool((out[:n] != 0).any())
        st["free"].copy_(p.free_left)
        held = to

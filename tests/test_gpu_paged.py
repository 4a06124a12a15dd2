"""The paged-cache operators on the device against their plain statements in 64
bits (paged_reference.py): sizes from one row up, page edges, strides, rows that
see nothing, pages outside the cache, non-finite values in masked places, other
streams, captured graphs, and rounds of all three together."""
import numpy as np
import pytest

import paged_reference as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def say(*a):
    print(*a, flush=True)


def ops():
    import cq35
    return cq35


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32))


# ------------------------------------------------------------------- plan


def plan_case(seed, requests, page, most, pages_extra=5, width_extra=2):
    """Requests that grow, shrink, finish or stand still."""
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, most + 1, requests)
    kind = rng.integers(0, 5, requests)
    lengths = np.where(kind == 0, cached, np.where(kind == 1, rng.integers(0, most + 1, requests),
                       np.where(kind == 2, 0, cached + rng.integers(1, 20, requests))))
    width = ref.ceil(int(max(cached.max(), lengths.max(), 1)), page) + width_extra
    have = [ref.ceil(int(c), page) for c in cached]
    take = sum(max(ref.ceil(int(x), page) - h, 0) for x, h in zip(lengths, have))
    pages = sum(have) + take + pages_extra
    order = rng.permutation(pages)
    table = rng.integers(-5, 5, (requests, width))
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = order[at:at + h]
        at += h
    stack = rng.integers(-9, 9, pages)
    stack[:pages - at] = order[at:]
    return dict(table=table.astype(np.int32), cached=cached.astype(np.int32), lengths=lengths.astype(np.int32),
                stack=stack.astype(np.int32), free=pages - at, page=page,
                rows=int(np.maximum(lengths - cached, 0).sum()))


def run_plan(c, rows, dev=None, repeat=1, table=None):
    dev = dev or dict(table=i32(c["table"]).cuda() if table is None else table, stack=i32(c["stack"]).cuda(),
                      cached=i32(c["cached"]).cuda(), lengths=i32(c["lengths"]).cuda(), free=i32([c["free"]]).cuda())
    for _ in range(repeat):
        p = ops().page_plan(dev["table"], dev["cached"], dev["lengths"], dev["stack"], dev["free"], page_size=c["page"],
                            rows=rows)
    return dev, p


def check_plan(c, rows, dev, p):
    want = ref.page_plan(c["table"], c["cached"], c["lengths"], c["stack"], c["free"], c["page"], rows)
    assert p.status.tolist() == want["status"]
    assert int(p.free_left) == want["free_left"]
    for name, got in (("table", dev["table"]), ("stack", dev["stack"]), ("row_start", p.row_start),
                      ("positions", p.positions), ("slots", p.slots)):
        assert np.array_equal(got.cpu().numpy(), want[name]), name
    assert int(dev["free"]) == c["free"]
    return want


@pytest.mark.parametrize("seed,requests,page,most", [
    (1, 1, 16, 0), (2, 1, 16, 40), (3, 2, 16, 16), (4, 7, 32, 100), (5, 64, 16, 3000), (6, 255, 64, 500), (7, 256, 16, 20),
    (8, 257, 128, 2000), (9, 1000, 16, 300), (10, 8192, 16, 60), (11, 5461, 32, 40), (12, 3, 65536, 200000),
])
def test_plan(seed, requests, page, most):
    say("plan", seed, requests, page, most)
    c = plan_case(seed, requests, page, most)
    dev, p = run_plan(c, c["rows"], repeat=2)  # with the same count again: the same
    check_plan(c, c["rows"], dev, p)
    dev, p = run_plan(c, c["rows"] + 300)  # rows behind the last request's
    check_plan(c, c["rows"] + 300, dev, p)


def test_plan_table_rows_apart():
    c = plan_case(21, 20, 16, 200)
    whole = torch.full((20, c["table"].shape[1] + 7), -3, dtype=torch.int32, device="cuda")
    view = whole[:, 3:3 + c["table"].shape[1]]
    view.copy_(i32(c["table"]))
    dev, p = run_plan(c, c["rows"], table=view)
    check_plan(c, c["rows"], dev, p)
    assert bool((whole[:, :3] == -3).all()) and bool((whole[:, 3 + c["table"].shape[1]:] == -3).all())


def test_plan_refuses_without_a_change():
    """Each status leaves tables, stack and count as they were and the round empty."""
    say("plan refusals")
    c = plan_case(31, 40, 16, 300, pages_extra=0)
    def outcome(rows=None, **kw):
        d = dict(c, **kw)
        dev, p = run_plan(d, d["rows"] if rows is None else rows)
        return check_plan(d, d["rows"] if rows is None else rows, dev, p)["status"]
    assert outcome() == [0, 0]
    spare = int(c["free"]) - 3
    short = dict(stack=c["stack"][:], free=max(0, c["free"] - 3))
    code = outcome(**short)
    assert code[0] == (1 if code[1] else 0) and (spare >= 0)
    assert outcome(rows=c["rows"] - 1) == [2, 1]
    assert outcome(rows=0) == [2, c["rows"]]
    for name, value in (("cached", -1), ("lengths", -7), ("lengths", 10**9), ("cached", 2**31 - 1)):
        x = c[name].copy()
        x[17] = value
        assert outcome(**{name: x}) == [3, 0]
    assert outcome(free=-1) == [4, 0]
    assert outcome(free=len(c["stack"]) + 1) == [4, 0]


def test_plan_counts_missing_pages():
    c = dict(table=np.zeros((3, 9), np.int32), cached=np.array([0, 16, 5], np.int32), lengths=np.array([33, 17, 16], np.int32),
             stack=np.arange(20, dtype=np.int32)[::-1].copy(), free=1, page=16, rows=45)
    dev, p = run_plan(c, 45)
    assert check_plan(c, 45, dev, p)["status"] == [1, 3]


def test_plan_bad_page_in_the_stack():
    """A page number outside the cache gets no slot."""
    c = dict(table=np.zeros((2, 4), np.int32), cached=np.array([0, 3], np.int32), lengths=np.array([20, 5], np.int32),
             stack=np.array([4, 77, -9, 2, 1], np.int32), free=3, page=16, rows=22)
    dev, p = run_plan(c, 22)
    check_plan(c, 22, dev, p)
    assert p.slots[:20].tolist() == [-1] * 20 and p.slots[20] >= 0


# ---------------------------------------------------------------- prepare


def cache_tensors(pages, page, kvh, hd, layout="rows", fill=None, seed=0):
    """A pair of caches: rows of heads; heads of rows; keys and values of a page side by side."""
    g = torch.Generator().manual_seed(seed)
    if layout == "rows":
        k, v = (torch.empty(pages, page, kvh, hd, dtype=BF, device="cuda") for _ in range(2))
    elif layout == "heads":
        k, v = (torch.empty(pages, kvh, page, hd, dtype=BF, device="cuda").transpose(1, 2) for _ in range(2))
    else:
        whole = torch.empty(pages, 2, page, kvh, hd, dtype=BF, device="cuda")
        k, v = whole[:, 0], whole[:, 1]
    for t in (k, v):
        t.copy_(torch.randn(t.shape, generator=g).to(BF) if fill is None else torch.full(t.shape, fill, dtype=BF))
    return k, v


def prepare_case(seed, T, QH, KVH, HD, rope, axes, far=300000):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = dict(qg=torch.randn(T, QH, 2 * HD, generator=g).mul(torch.rand(T, 1, 1, generator=g) * 4).to(BF),
             kv=torch.randn(T, 2 * KVH, HD, generator=g).to(BF), qw=1 + 0.1 * torch.randn(HD, generator=g),
             kw=1 + 0.1 * torch.randn(HD, generator=g),
             freq=torch.tensor((1e7 ** (-np.arange(0, rope, 2) / rope)).astype(np.float32)),
             positions=i32(rng.integers(0, far, (axes, T))), axis=[i % axes for i in range(rope // 2)])
    return s


def check_prepare(s, out, key_cache, value_cache, before, slots, page, eps=1e-6):
    """Every written head within its bound, everything else untouched. The
    bound: F32 sums of HD squares, a square root, a reciprocal, products and the
    turn's sine and cosine, 2^-19 of both channels of a pair together, and half
    a BF16 step of the result."""
    QH, HD = s["qg"].shape[1], s["kv"].shape[2]
    KVH = s["kv"].shape[1] // 2
    rows = [t for t, x in enumerate(slots) if 0 <= x < key_cache.shape[0] * page]
    for name, x, w, got in (("q", s["qg"][:, :, :HD], s["qw"], out),
                            ("k", s["kv"][:, :KVH], s["kw"], None)):
        want, size = ref.head(x, w, eps, s["freq"], s["positions"], s["axis"])
        if got is None:
            at = [slots[t] for t in rows]
            got = torch.full(want.shape, float("nan"), dtype=torch.float64)
            got[rows] = key_cache.cpu().double()[[a // page for a in at], [a % page for a in at]]
        got = got.cpu().double()
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -19 * size + 1e-37
        bad = ((got - want).abs() > tol)[rows]
        assert not bool(bad.any()), (name, int(bad.sum()), float(((got - want).abs() / tol)[rows].max()))
    k0, v0 = before
    for t in rows:
        k0[slots[t] // page, slots[t] % page] = key_cache.cpu()[slots[t] // page, slots[t] % page]
        v0[slots[t] // page, slots[t] % page] = s["kv"][t, KVH:]
    assert torch.equal(k0, key_cache.cpu()) and torch.equal(v0, value_cache.cpu())


def run_prepare(s, KVH, HD, key_cache, value_cache, slots, out=None, positions=None, **kw):
    qg, kv = s["qg"].cuda(), s["kv"].cuda()
    axes = s["positions"].shape[0]
    return ops().paged_prepare(qg[:, :, :HD], kv[:, :KVH], kv[:, KVH:], s["qw"].cuda(), s["kw"].cuda(), s["freq"].cuda(),
                               s["positions"].cuda() if axes > 1 else s["positions"][0].cuda(), i32(slots).cuda(), key_cache,
                               value_cache, pair_axis=s["axis"] if axes > 1 else None, out=out, **kw)


@pytest.mark.parametrize("T,QH,KVH,HD,rope,axes,page,layout", [
    (1, 16, 2, 256, 64, 1, 16, "rows"), (7, 8, 2, 256, 64, 3, 32, "heads"), (33, 4, 1, 64, 16, 1, 16, "sides"),
    (5, 3, 3, 128, 128, 3, 16, "rows"), (130, 6, 2, 128, 32, 2, 64, "heads"), (9, 1, 1, 256, 256, 4, 16, "sides"),
    (64, 5, 1, 64, 64, 3, 16, "rows"), (1025, 8, 2, 256, 64, 3, 16, "rows"), (1031, 4, 2, 64, 32, 1, 128, "heads"),
])
def test_prepare(T, QH, KVH, HD, rope, axes, page, layout):
    say("prepare", T, QH, KVH, HD, rope, axes, page, layout)
    s = prepare_case(T + HD, T, QH, KVH, HD, rope, axes)
    pages = ref.ceil(T, page) + 3
    k, v = cache_tensors(pages, page, KVH, HD, layout)
    before = k.cpu().clone(), v.cpu().clone()
    slots = np.random.default_rng(T).permutation(pages * page)[:T]
    out = run_prepare(s, KVH, HD, k, v, slots)
    check_prepare(s, out, k, v, before, slots.tolist(), page)


def test_prepare_skips_rows_without_a_slot():
    """Negative slots and slots past the cache: query, key and value left as they were."""
    T, QH, KVH, HD, page = 40, 4, 2, 128, 16
    s = prepare_case(3, T, QH, KVH, HD, 32, 1)
    k, v = cache_tensors(4, page, KVH, HD)
    before = k.cpu().clone(), v.cpu().clone()
    slots = np.arange(T)
    slots[[0, 7, 39]] = -1
    slots[5], slots[6], slots[11], slots[12] = 64, 2**31 - 1, -2**31, 65
    out = torch.full((T, QH, HD), 7.0, dtype=BF, device="cuda")
    run_prepare(s, KVH, HD, k, v, slots, out=out)
    check_prepare(s, out, k, v, before, slots.tolist(), page)
    for t in (0, 5, 6, 7, 11, 12, 39):
        assert bool((out[t] == 7.0).all())


def test_prepare_far_positions():
    """The turn of positions up to 2^31 - 1, the first frequency a radian a token."""
    T = 64
    s = prepare_case(5, T, 2, 1, 64, 64, 1)
    s["positions"] = i32([[0, 1, 2**20, 2**24 + 1, 2**31 - 1, 10**6 + 7, 2**30 + 3, 262143] * 8])
    k, v = cache_tensors(6, 16, 1, 64)
    before = k.cpu().clone(), v.cpu().clone()
    out = run_prepare(s, 1, 64, k, v, np.arange(T))
    check_prepare(s, out, k, v, before, list(range(T)), 16)


def test_prepare_in_place_and_strided_output():
    T, QH, KVH, HD = 50, 6, 2, 64
    s = prepare_case(8, T, QH, KVH, HD, 32, 3)
    k, v = cache_tensors(6, 16, KVH, HD)
    first = run_prepare(s, KVH, HD, k, v, np.arange(T))
    qg, kv = s["qg"].cuda(), s["kv"].cuda()
    gate = qg[:, :, HD:].clone()
    k2, v2 = cache_tensors(6, 16, KVH, HD)
    got = ops().paged_prepare(qg[:, :, :HD], kv[:, :KVH], kv[:, KVH:], s["qw"].cuda(), s["kw"].cuda(), s["freq"].cuda(),
                              s["positions"].cuda(), i32(np.arange(T)).cuda(), k2, v2, pair_axis=s["axis"], out=qg[:, :, :HD])
    assert torch.equal(got, first) and torch.equal(qg[:, :, HD:], gate) and torch.equal(k, k2) and torch.equal(v, v2)


def test_prepare_one_row_repeated():
    """An input of stride 0: one key and value row for every token."""
    T, HD = 20, 64
    s = prepare_case(9, T, 2, 1, HD, 16, 1)
    s["kv"] = s["kv"][:1].expand(T, -1, -1)
    k, v = cache_tensors(2, 16, 1, HD)
    before = k.cpu().clone(), v.cpu().clone()
    kv = s["kv"][:1].contiguous().cuda()
    q = s["qg"].cuda()
    out = ops().paged_prepare(q[:, :, :HD], kv[:, :1].expand(T, 1, HD), kv[:, 1:].expand(T, 1, HD), s["qw"].cuda(),
                              s["kw"].cuda(), s["freq"].cuda(), s["positions"][0].cuda(), i32(np.arange(T)).cuda(), k, v)
    check_prepare(s, out, k, v, before, list(range(T)), 16)


def test_prepare_zero_and_huge_rows():
    """A head of zeros gives zeros (eps), one of huge values whose squares pass
    the type's range gives what the formula does in F32: zeros."""
    T, HD = 3, 64
    s = prepare_case(10, T, 1, 1, HD, 16, 1)
    s["qg"][0] = 0
    s["kv"][0, 0] = 0
    k, v = cache_tensors(1, 16, 1, HD)
    before = k.cpu().clone(), v.cpu().clone()
    out = run_prepare(s, 1, HD, k, v, np.arange(T))
    check_prepare(s, out, k, v, before, list(range(T)), 16)
    assert bool((out[0] == 0).all())


# -------------------------------------------------------------- attention


def attention_case(seed, new, lengths, QH, KVH, HD, page, layout="rows", gate=False, extra=3, qstd=2.0, width_extra=1):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    T = int(sum(new))
    need = [ref.ceil(max(x, 0), page) for x in lengths]
    pages = sum(need) + extra
    k, v = cache_tensors(pages, page, KVH, HD, layout, seed=seed)
    table = rng.integers(0, pages, (len(new), max(max(need), 1) + width_extra))
    order = rng.permutation(pages)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    q = (torch.randn(T, QH, HD, generator=g) * qstd).to(BF)
    return dict(q=q, k=k, v=v, table=i32(table), row_start=i32(np.concatenate([[0], np.cumsum(new)])), lengths=i32(lengths),
                gate=torch.randn(T, QH, HD, generator=g).to(BF) if gate else None, scale=HD ** -0.5)


# The bounds choose the kernel besides the cut: an unknown or a small max_keys
# leaves these sizes with the one for short work, a large one gives chunks of
# more than 32 rows of a KV head to the one for long chunks.
KEYS = [0]


@pytest.fixture(params=[0, 1 << 22], ids=["short", "long"])
def steered(request):
    KEYS[0] = request.param
    yield
    KEYS[0] = 0


def run_attention(s, **kw):
    kw.setdefault("max_keys", KEYS[0])
    return ops().paged_attention(s["q"].cuda(), s["k"], s["v"], s["table"].cuda(), s["row_start"].cuda(), s["lengths"].cuda(),
                                 gate=None if s["gate"] is None else s["gate"].cuda(), scale=s["scale"], **kw)


def check_attention(s, got, rows=None):
    want, tol = ref.attention(s["q"], s["k"].cpu(), s["v"].cpu(), s["table"], s["row_start"], s["lengths"], s["scale"], s["gate"])
    got = got.cpu().double()
    rows = slice(None) if rows is None else rows
    got, want, tol = got[rows], want[rows], tol[rows]
    assert bool(torch.isfinite(got).all())
    off = ((got - want).abs() / tol).max() if got.numel() else 0
    say("  largest error over its bound: %.3f" % float(off))
    assert off <= 1, float(off)


SHAPES = [
    # new tokens, lengths, q heads, kv heads, head dim, page, layout, gate
    ([1], [1], 1, 1, 64, 16, "rows", False),
    ([1], [1], 16, 2, 256, 16, "rows", True),
    ([1], [520], 16, 2, 256, 16, "rows", True),
    ([1] * 5, [1, 15, 16, 17, 300], 8, 2, 256, 16, "heads", True),
    ([1, 1, 1], [31, 33, 1000], 4, 4, 128, 32, "sides", False),
    ([5, 3, 1, 8], [5, 100, 64, 700], 16, 4, 128, 16, "rows", False),
    ([17], [17], 6, 2, 64, 16, "heads", True),
    ([33, 1, 70], [33, 257, 300], 4, 1, 64, 64, "rows", False),
    ([40], [1000], 16, 2, 256, 64, "rows", True),
    ([100, 1, 2, 65], [400, 90, 2, 65], 8, 2, 256, 16, "sides", True),
    ([64], [64], 5, 5, 128, 128, "rows", False),
    ([129], [300], 3, 1, 256, 16, "heads", False),
    ([70, 0, 1], [70, 20, 9], 12, 2, 64, 16, "rows", True),
    ([260], [261], 2, 2, 64, 16, "rows", False),
    ([1], [4100], 24, 2, 128, 32, "rows", True),
    ([3, 2], [2500, 5000], 7, 1, 64, 16, "rows", False),
]


@pytest.mark.parametrize("new,lengths,QH,KVH,HD,page,layout,gate", SHAPES)
def test_attention(new, lengths, QH, KVH, HD, page, layout, gate, steered):
    say("attention", new, lengths, QH, KVH, HD, page, layout, gate)
    s = attention_case(sum(lengths) + HD, new, lengths, QH, KVH, HD, page, layout, gate)
    plain = run_attention(s)
    check_attention(s, plain)
    assert torch.equal(plain, run_attention(s))
    # the bounds steer the launch alone: right ones, and ones that are too small
    check_attention(s, run_attention(s, max_rows=max(new), max_keys=max(lengths)))
    check_attention(s, run_attention(s, max_rows=1, max_keys=1))


def test_attention_rows_that_see_nothing(steered):
    """More new tokens than the request holds, no tokens at all, requests
    without rows: zeros where no key is seen."""
    for HD, new, lengths in ((64, [5, 3, 0, 4], [3, 0, 7, -2]), (256, [40, 1], [30, 0])):
        say("nothing seen", HD, new, lengths)
        s = attention_case(7, new, lengths, 8, 2, HD, 16, gate=True)
        got = run_attention(s)
        check_attention(s, got)
        hidden = [t for r, (n, x) in enumerate(zip(new, lengths)) for t in range(sum(new[:r]), sum(new[:r]) + max(0, n - max(x, 0)))]
        assert hidden and bool((got[hidden] == 0).all())


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", [
    (40, 3000, 4, 1, 256, 16), (33, 2500, 2, 2, 128, 32), (70, 2300, 1, 1, 64, 64), (1, 9000, 8, 2, 256, 16), (2, 5000, 3, 1, 64, 16),
    (1, 140000, 2, 1, 64, 64),  # more splits than the join keeps maxima of
])
def test_attention_long_splits(new, length, QH, KVH, HD, page, steered):
    """Splits of more tiles than a wave keeps places of, with pages outside the
    cache in several of those stretches."""
    say("long splits", new, length, HD)
    s = attention_case(length, [new, 1], [length, 40], QH, KVH, HD, page)
    check_attention(s, run_attention(s, max_rows=new, max_keys=1))
    check_attention(s, run_attention(s, max_rows=new, max_keys=length))
    for j in (0, 1030, 1100, 2100, length - 1):
        s["table"][0, j // page] = -3
    check_attention(s, run_attention(s, max_rows=new, max_keys=1))
    check_attention(s, run_attention(s))


@pytest.mark.parametrize("R,most_new,most,HD,QH,KVH", [(64, 3, 200, 64, 2, 1), (65, 1, 300, 128, 4, 2), (70, 40, 90, 64, 4, 1),
                                                       (300, 2, 100, 64, 2, 2), (1500, 2, 40, 64, 1, 1), (8192, 1, 20, 64, 1, 1)])
def test_attention_many_requests(R, most_new, most, HD, QH, KVH, steered):
    say("many requests", R, most_new, most)
    rng = np.random.default_rng(R)
    new = rng.integers(0, most_new + 1, R).tolist()
    lengths = [int(n + rng.integers(0, most)) for n in new]
    if most_new == 1:
        lengths[3] = 5000  # one that is split
    s = attention_case(R, new, lengths, QH, KVH, HD, 16)
    check_attention(s, run_attention(s))
    check_attention(s, run_attention(s, max_rows=most_new, max_keys=max(lengths)))


def test_attention_leaves_other_rows(steered):
    """Rows behind the last request, in front of the first, and requests whose rows pass the tensor's end."""
    s = attention_case(11, [3, 30], [40, 90], 4, 2, 128, 16, width_extra=80)
    s["q"] = torch.cat([s["q"][:2], s["q"], s["q"][:4]])
    s["row_start"] = s["row_start"] + 2
    out = torch.full(s["q"].shape, 5.0, dtype=BF, device="cuda")
    got = run_attention(s, out=out)
    assert bool((got[:2] == 5).all()) and bool((got[35:] == 5).all())
    want = dict(s, q=s["q"][2:35], row_start=s["row_start"] - 2)
    check_attention(want, got[2:35])
    # a last request whose rows pass the tensor's end: those in it are its first
    s["row_start"][2], s["lengths"][1] = 1000, 995
    got = run_attention(s, out=torch.full(s["q"].shape, 5.0, dtype=BF, device="cuda"))
    assert bool((got[:2] == 5).all())
    check_attention(dict(s, q=s["q"][5:39], row_start=i32([0, 34]), lengths=i32([34]), table=s["table"][1:2]), got[5:39])


def test_attention_bad_pages(steered):
    """Keys of pages outside the cache are not seen; lengths past the table are cut to it."""
    for HD, new in ((64, [1, 6]), (256, [1, 50])):
        say("bad pages", HD, new)
        s = attention_case(13, new, [200, 300], 8, 2, HD, 16)
        s["table"][0, 3], s["table"][0, 12], s["table"][1, 0], s["table"][1, 18] = -1, 10**6, 2**31 - 1, s["k"].shape[0]
        check_attention(s, run_attention(s))
        s["table"][:] = -7
        got = run_attention(s)
        assert bool((got == 0).all())
    s = attention_case(14, [2], [50], 4, 2, 64, 16, width_extra=0)
    cut = dict(s, lengths=i32([64]))
    s["lengths"] = i32([10**9])
    check_attention(cut, run_attention(s))


@pytest.mark.parametrize("HD,new,length,QH", [(64, 3, 40, 4), (256, 9, 70, 16), (128, 80, 130, 8), (256, 40, 40, 4)])
def test_attention_non_finite_values_that_are_not_seen(HD, new, length, QH, steered):
    """NaN and infinities past the length (stale pages) and in later tokens of
    the chunk never reach a row that does not see them."""
    say("non-finite", HD, new, length)
    s = attention_case(17, [new], [length], QH, 2, HD, 32)
    page = s["table"][0]
    clean = {n: s[n].clone() for n in ("k", "v")}
    for j, x in ((length, float("nan")), (length + 1, float("inf")), (length - 1, float("nan")), (length - 2, float("-inf"))):
        if j < page.shape[0] * 32:
            s["k"][int(page[j // 32]), j % 32] = x
            s["v"][int(page[j // 32]), j % 32] = x
    got = run_attention(s)
    check_attention(dict(s, **clean), got, rows=slice(0, new - 2))
    assert bool(torch.isnan(got[new - 1]).all())


@pytest.mark.parametrize("HD,QH,KVH,new,length", [(256, 8, 1, 60, 400), (64, 2, 2, 300, 500), (128, 4, 2, 3, 100)])
def test_attention_non_finite_values_that_are_seen(HD, QH, KVH, new, length, steered):
    """Each channel's infinity or NaN reaches the rows that see it, as the
    formula has it, and no other channel or row."""
    say("non-finite seen", HD, new, length)
    s = attention_case(18, [new], [length], QH, KVH, HD, 16)
    page = s["table"][0]
    start = length - new
    odd = {5: (1, float("nan")), 40: (7, float("inf")), start + new // 2: (9, float("-inf")), start + new // 2 + 1: (11, float("nan"))}
    clean = s["v"].clone()
    for j, (c, x) in odd.items():
        s["v"][int(page[j // 16]), j % 16, :, c] = x
        clean[int(page[j // 16]), j % 16, :, c] = 0
    got = run_attention(s).cpu().double()
    want, tol = ref.attention(s["q"], s["k"].cpu(), clean.cpu(), s["table"], s["row_start"], s["lengths"], s["scale"])
    for t in range(new):
        for j, (c, x) in odd.items():
            if j <= start + t:
                assert bool((torch.isnan(got[t, :, c]) if x != x else got[t, :, c] == x).all()), (t, j, c)
                got[t, :, c] = want[t, :, c]
    assert bool(((got - want).abs() <= tol).all())


def test_attention_extreme_scores(steered):
    """Scores far past the exponential's range, one key that outweighs all
    others, equal scores: finite, and the weights those of the maximum."""
    for QH, new in ((4, 1), (4, 40)):
        s = attention_case(19, [new], [200], QH, 2, 64, 16, qstd=300.0)
        check_attention(s, run_attention(s))
        s["q"].zero_()
        check_attention(s, run_attention(s))
        # rising scores: the running maximum grows at every tile
        s = attention_case(20, [new], [500], QH, 1, 64, 16)
        s["q"][:] = 1.0
        at = torch.arange(500)
        rows = (s["table"][0, at // 16].long(), at % 16)
        s["k"][rows[0].cuda(), rows[1].cuda()] = (at[:, None, None] * 0.01).expand(500, 1, 64).to(BF).cuda()
        check_attention(s, run_attention(s))
        s["k"].neg_()
        check_attention(s, run_attention(s))


def test_attention_negative_and_zero_scale(steered):
    s = attention_case(23, [20], [90], 4, 2, 64, 16)
    for scale in (0.0, -0.125, 0.5):
        s["scale"] = scale
        check_attention(s, run_attention(s))


def test_attention_strided_and_in_place(steered):
    T, QH, HD = 45, 8, 128
    s = attention_case(29, [T], [300], QH, 2, HD, 16, gate=True)
    both = torch.stack([s["q"], s["gate"]], 2).cuda()  # [T, QH, 2, HD]
    dev = [s[n].cuda() for n in ("table", "row_start", "lengths")]
    want = run_attention(s)
    got = ops().paged_attention(both[:, :, 0], s["k"], s["v"], *dev, gate=both[:, :, 1], out=both[:, :, 0], max_keys=KEYS[0])
    assert torch.equal(got, want) and torch.equal(both[:, :, 1].cpu(), s["gate"])
    by_head = s["q"].cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops().paged_attention(by_head, s["k"], s["v"], *dev, gate=both[:, :, 1], max_keys=KEYS[0]), want)
    one = s["q"][:1].cuda().expand(T, -1, -1)  # one query row for every token
    s["q"] = s["q"][:1].expand(T, -1, -1)
    check_attention(s, ops().paged_attention(one, s["k"], s["v"], *dev, gate=both[:, :, 1], max_keys=KEYS[0]))


def test_attention_long_offsets():
    """Cache rows whose element offsets pass 32 bits: 2^17 pages of 64 rows of 2
    heads of 256 are 2^32 elements a side."""
    pages, page, KVH, HD = (1 << 17) + 40, 64, 2, 256
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("not enough memory")
    g = torch.Generator().manual_seed(1)
    k = torch.zeros(pages, page, KVH, HD, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    for new, length, most in ((1, 700, 0), (50, 700, 0), (50, 700, 1 << 22)):
        n = ref.ceil(length, page)
        at = [pages - 1 - 3 * i for i in range(n - 1)] + [1]
        kk, vv = torch.randn(n, page, KVH, HD, generator=g).to(BF), torch.randn(n, page, KVH, HD, generator=g).to(BF)
        k[at], v[at] = kk.cuda(), vv.cuda()
        q = (2 * torch.randn(new, 16, HD, generator=g)).to(BF)
        got = ops().paged_attention(q.cuda(), k, v, i32([at]).cuda(), i32([0, new]).cuda(), i32([length]).cuda(),
                                    max_keys=most)
        small = dict(q=q, k=kk, v=vv, table=i32([list(range(n))]), row_start=i32([0, new]), lengths=i32([length]),
                     scale=HD ** -0.5, gate=None)
        check_attention(small, got)
    # prepare writes there too
    s = prepare_case(2, 3, 4, KVH, HD, 64, 1)
    slots = [pages * page - 1, (pages - 2) * page, 5]
    run_prepare(s, KVH, HD, k, v, slots)
    want, size = ref.head(s["kv"][:, :KVH], s["kw"], 1e-6, s["freq"], s["positions"], s["axis"])
    got = torch.stack([k[x // page, x % page] for x in slots]).cpu().double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * size).all())


# ------------------------------------------------------- streams and graphs


def test_other_stream(steered):
    s = attention_case(37, [9, 1], [200, 900], 8, 2, 128, 16)
    want = run_attention(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run_attention(s, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    with torch.cuda.stream(side):
        got = run_attention(s)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once(steered):
    """Calls on two streams, each with a workspace of its own."""
    cases = [attention_case(41 + i, [7 + 40 * i], [3000], 8, 2, 128, 16) for i in range(2)]
    dev = [[c[n].cuda() for n in ("q", "table", "row_start", "lengths")] for c in cases]
    def call(i):
        q, *rest = dev[i]
        return ops().paged_attention(q, cases[i]["k"], cases[i]["v"], *rest, max_keys=KEYS[0])
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def round_state(page=16, requests=6, QH=8, KVH=2, HD=128, rope=32, pages=120, width=40, seed=1):
    g = torch.Generator().manual_seed(seed)
    k, v = cache_tensors(pages, page, KVH, HD, fill=float("nan"))
    return dict(table=torch.full((requests, width), -1, dtype=torch.int32, device="cuda"),
                stack=torch.randperm(pages, generator=g).int().cuda(), free=i32([pages]).cuda(), k=k, v=v, page=page,
                requests=requests, QH=QH, KVH=KVH, HD=HD, qw=1 + 0.1 * torch.randn(HD, generator=g),
                kw=1 + 0.1 * torch.randn(HD, generator=g),
                freq=torch.tensor((1e4 ** (-np.arange(0, rope, 2) / rope)).astype(np.float32)),
                kept=[[torch.zeros(0, KVH, HD, dtype=BF)] * 2 for _ in range(requests)], cached=[0] * requests, pages=pages)


def run_round(st, qg, kv, cached, lengths, rows):
    """One serving round through the three operators: (attention output, plan)."""
    HD, KVH = st["HD"], st["KVH"]
    p = ops().page_plan(st["table"], cached, lengths, st["stack"], st["free"], page_size=st["page"], rows=rows)
    q = ops().paged_prepare(qg[:, :, 0], kv[:, :KVH], kv[:, KVH:], st["qw_dev"], st["kw_dev"], st["freq_dev"], p.positions,
                            p.slots, st["k"], st["v"])
    out = ops().paged_attention(q, st["k"], st["v"], st["table"], p.row_start, lengths, gate=qg[:, :, 1], max_keys=KEYS[0])
    return out, p, q


def test_rounds_together(steered):
    """Rounds of prompts, single tokens, drafts that are taken back and finished
    requests: each round's attention against one over the tokens kept by hand."""
    say("rounds together")
    st = round_state()
    for n in ("qw", "kw", "freq"):
        st[n + "_dev"] = st[n].cuda()
    rng = np.random.default_rng(5)
    g = torch.Generator().manual_seed(6)
    QH, KVH, HD, R = st["QH"], st["KVH"], st["HD"], st["requests"]
    held = [0] * R
    for turn in range(12):
        want_len = []
        for r in range(R):
            kind = rng.integers(0, 6)
            if held[r] == 0 or kind == 0:
                n = held[r] + int(rng.integers(1, 60))
            elif kind == 1:
                n = max(0, held[r] - int(rng.integers(1, 6)))  # drafts taken back
            elif kind == 2 and turn > 4:
                n = 0
            else:
                n = held[r] + int(rng.integers(1, 5))
            want_len.append(min(n, 300))
        new = [max(a - b, 0) for a, b in zip(want_len, held)]
        rows = sum(new) + int(rng.integers(0, 5))
        say("  round", turn, "held", held, "to", want_len)
        qg, kv = torch.randn(rows, QH, 2, HD, generator=g).to(BF), torch.randn(rows, 2 * KVH, HD, generator=g).to(BF)
        lengths = i32(want_len).cuda()
        out, p, q = run_round(st, qg.cuda(), kv.cuda(), i32(held).cuda(), lengths, rows)
        assert p.status.tolist() == [0, 0]
        st["free"] = p.free_left
        used = [int(x) for r in range(R) for x in st["table"][r, :ref.ceil(want_len[r], st["page"])]]
        free = st["stack"][:int(p.free_left)].tolist()
        assert sorted(used + free) == list(range(st["pages"]))
        t = 0
        for r in range(R):
            st["kept"][r] = [x[:want_len[r]] for x in st["kept"][r]]
            if new[r]:
                at = slice(t, t + new[r])
                pos = torch.arange(held[r], want_len[r])[None].int()
                keys, _ = ref.head(kv[at, :KVH], st["kw"], 1e-6, st["freq"], pos, [0] * st["freq"].shape[0])
                st["kept"][r] = [torch.cat([st["kept"][r][0].double(), keys]), torch.cat([st["kept"][r][1], kv[at, KVH:]])]
                qs, _ = ref.head(qg[at, :, 0], st["qw"], 1e-6, st["freq"], pos, [0] * st["freq"].shape[0])
                n = len(st["kept"][r][0])
                want, tol = ref.attention(qs, st["kept"][r][0][None], st["kept"][r][1][None].double(), i32([[0]]),
                                          i32([0, new[r]]), i32([n]), HD ** -0.5, qg[at, :, 1])
                # the rounded queries and keys move a score by 2^-8 of each of
                # its products twice, a weight by twice that share
                reach = float(qs.abs().sum(-1).max() * st["kept"][r][0].abs().max()) * HD ** -0.5
                slack = 4 * 2.0 ** -8 * min(reach, float(qs.norm(dim=-1).max() * st["kept"][r][0].norm(dim=-1).max()) * HD ** -0.5)
                big = st["kept"][r][1].abs().max()
                assert bool(((out[at].cpu().double() - want).abs() <= tol + slack * big).all())
                # and exactly the operator's own bound from the operator's own queries and keys
                check_attention(dict(q=q[at].cpu(), k=st["k"], v=st["v"], table=st["table"][r:r + 1].cpu(),
                                     row_start=i32([0, new[r]]), lengths=i32([want_len[r]]), scale=HD ** -0.5,
                                     gate=qg[at, :, 1]), out[at])
                t += new[r]
        held = want_len


def test_round_without_pages_does_nothing():
    """A plan that lacks pages leaves the rest of the round without work."""
    st = round_state(pages=4)
    for n in ("qw", "kw", "freq"):
        st[n + "_dev"] = st[n].cuda()
    before = st["k"].clone()
    g = torch.Generator().manual_seed(6)
    qg, kv = torch.randn(100, 8, 2, 128, generator=g).to(BF).cuda(), torch.randn(100, 4, 128, generator=g).to(BF).cuda()
    out, p, _ = run_round(st, qg, kv, i32([0] * 6).cuda(), i32([90, 10, 0, 0, 0, 0]).cuda(), 100)
    assert p.status.tolist() == [1, 3] and int(p.free_left) == 4 and p.row_start.tolist() == [0] * 7
    assert torch.equal(before.view(torch.int16), st["k"].view(torch.int16))


def test_captured_round(steered):
    """A round captured into a graph and replayed with new lengths and rows, the
    program's own work between the replays: the same as eager calls."""
    say("captured round")
    rows, R = 24, 6
    g = torch.Generator().manual_seed(8)
    def fresh():
        st = round_state(seed=3)
        for n in ("qw", "kw", "freq"):
            st[n + "_dev"] = st[n].cuda()
        return st
    eager, graphed = fresh(), fresh()
    qg, kv = torch.zeros(rows, 8, 2, 128, dtype=BF, device="cuda"), torch.zeros(rows, 4, 128, dtype=BF, device="cuda")
    cached, lengths = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
    run_round(graphed, qg, kv, cached, lengths, rows)  # loads the kernels
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, p, _ = run_round(graphed, qg, kv, cached, lengths, rows)
    second = torch.cuda.CUDAGraph()  # another graph over the same cache
    with torch.cuda.graph(second):
        out2, p2, _ = run_round(graphed, qg, kv, cached, lengths, rows)
    held = [0] * R
    for turn in range(6):
        to = [h + (turn + r) % 5 if (turn + r) % 4 else max(0, h - 2) for r, h in enumerate(held)]
        qg.copy_(torch.randn(qg.shape, generator=g).to(BF))
        kv.copy_(torch.randn(kv.shape, generator=g).to(BF))
        cached.copy_(i32(held))
        lengths.copy_(i32(to))
        want, pe, _ = run_round(eager, qg, kv, cached, lengths, rows)
        torch.cuda.synchronize()
        if turn % 2:
            graph.replay()
            got, pg = out, p
        else:
            second.replay()
            got, pg = out2, p2
        torch.cuda.synchronize()
        torch.randn(1000, 1000, device="cuda").sum().item()
        n = int(pe.row_start[-1])
        assert pg.status.tolist() == [0, 0] and all(torch.equal(a, b) for a, b in zip(pg, pe))
        assert torch.equal(got[:n], want[:n]) and torch.equal(graphed["table"], eager["table"])
        eager["free"] = pe.free_left
        graphed["free"].copy_(pg.free_left)
        held = to


def test_two_threads(steered):
    """Calls from two threads, each on a stream of its own."""
    import threading
    s = attention_case(43, [30, 1], [400, 2000], 8, 2, 128, 16)
    dev = [s[n].cuda() for n in ("q", "table", "row_start", "lengths")]
    want = ops().paged_attention(dev[0], s["k"], s["v"], *dev[1:], max_keys=KEYS[0])
    torch.cuda.synchronize()
    bad = []
    def work():
        stream = torch.cuda.Stream()
        for _ in range(20):
            got = ops().paged_attention(dev[0], s["k"], s["v"], *dev[1:], stream=stream, max_keys=KEYS[0])
            stream.synchronize()
            if not torch.equal(got, want):
                bad.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals_on_the_device():
    s = attention_case(47, [2], [40], 4, 2, 64, 16)
    dev = [s[n].cuda() for n in ("q", "table", "row_start", "lengths")]
    call = lambda **kw: ops().paged_attention(*[kw.get(n, x) for n, x in zip(("q", "k", "v", "table", "row_start", "lengths"),
                                              (dev[0], s["k"], s["v"], *dev[1:]))], **kw.get("more", {}))  # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        call(lengths=s["lengths"])
    with pytest.raises(ValueError, match="int32"):
        call(table=dev[1].long())
    with pytest.raises(ValueError, match="contiguous"):
        call(q=dev[0].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="entries"):
        call(row_start=dev[2][:1])
    with pytest.raises(ValueError, match="rows"):
        call(table=dev[1].repeat(2, 1))
    with pytest.raises(ops().CQ35Error, match="16-byte"):
        call(q=torch.zeros(2 * 4 * 64 + 4, dtype=BF, device="cuda")[4:].view(2, 4, 64))
    with pytest.raises(ops().CQ35Error, match="multiples of 8"):
        call(q=torch.zeros(2, 4, 68, dtype=BF, device="cuda")[:, :, :64])
    with pytest.raises(ops().CQ35Error, match="overlap"):
        call(more=dict(out=torch.zeros(1, 4, 64, dtype=BF, device="cuda").expand(2, 4, 64)))
    with pytest.raises(ops().CQ35Error, match="query heads"):
        call(q=torch.zeros(2, 3, 64, dtype=BF, device="cuda"))
    with pytest.raises(ops().CQ35Error, match="head_dim"):
        c = torch.zeros(2, 16, 2, 96, dtype=BF, device="cuda")
        call(q=torch.zeros(2, 4, 96, dtype=BF, device="cuda"), k=c, v=c)
    with pytest.raises(ops().CQ35Error, match="power of two"):
        c = torch.zeros(2, 24, 2, 64, dtype=BF, device="cuda")
        call(k=c, v=c)
    for name in ("q", "k", "table", "row_start", "lengths"):
        with pytest.raises(TypeError, match="tensor"):
            call(**{name: [0]})
    with pytest.raises(TypeError, match="workspace must be a tensor"):
        call(more=dict(workspace=1 << 20))
    with pytest.raises(ValueError, match=r"q must be \(2, 4, 64\)"):
        call(q=torch.zeros(2, 4, 128, dtype=BF, device="cuda"))
    p = prepare_case(1, 3, 4, 2, 64, 32, 1)
    k, v = cache_tensors(4, 16, 2, 64)
    q, kv = p["qg"][:, :, :64].cuda(), p["kv"].cuda()
    args = dict(q_weight=p["qw"].cuda(), k_weight=p["kw"].cuda(), inv_freq=p["freq"].cuda(), positions=i32([0, 1, 2]).cuda(),
                slots=i32([0, 1, 2]).cuda())
    for name in args:
        with pytest.raises(TypeError, match=name + " must be a tensor"):
            ops().paged_prepare(q, kv[:, :2], kv[:, 2:], key_cache=k, value_cache=v, **dict(args, **{name: [0]}))
        with pytest.raises(ValueError, match=name):
            ops().paged_prepare(q, kv[:, :2], kv[:, 2:], key_cache=k, value_cache=v, **dict(args, **{name: args[name].cpu()}))

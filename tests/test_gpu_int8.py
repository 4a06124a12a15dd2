"""8-bit rows and their product on the device against plain statements in 64 bits
(int8_reference.py)."""
import pytest

import int8_reference as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
TYPES = [BF, F32]


def say(*a):
    print(*a, flush=True)


def ops():
    import cq35
    return cq35


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0, dtype=F32):
    return torch.empty(shape, dtype=F32, device="cuda").normal_(0, std, generator=gen(seed)).to(dtype)


def ints(seed, rows, channels):
    g = gen(seed)
    data = torch.randint(-128, 128, (rows, channels), dtype=I8, device="cuda", generator=g)
    scale = torch.rand(rows, device="cuda", generator=g) * 0.1 + 1e-3
    return data, scale


def apart(t, extra, front=0):
    """The same values as a view of a wider tensor of sentinels."""
    rows, channels = t.shape
    whole = torch.full((rows, channels + extra), 77, dtype=t.dtype, device=t.device)
    view = whole[:, front:front + channels]
    view.copy_(t)
    return whole, view


# ------------------------------------------------------------------- rows

SHAPES = [(1, 16), (3, 32), (5, 48), (2, 512), (7, 1008), (1, 2048), (65, 2048), (4, 2064), (3, 4096), (2, 8192), (3, 8208),
          (1, 14336), (2, 32768), (1, 65536), (1001, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_quantize(rows, channels, dtype):
    say("quantize", rows, channels, dtype)
    x = normal(rows + channels, rows, channels, dtype=dtype)
    q = ops().quantize_rows(x)
    assert q.data.shape == x.shape and q.data.dtype == I8 and q.scale.shape == (rows,)
    ref.check_rows(q.data, q.scale, x.double(), 0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, channels, dtype, residual):
    say("norm", rows, channels, dtype, residual)
    x, r = normal(1, rows, channels, dtype=dtype), normal(2, rows, channels, std=3.0, dtype=dtype)
    w = 1 + 0.1 * normal(3, channels)
    q = ops().norm_quantize(x, w, residual=r if residual else None, eps=1e-5)
    h = x if not residual else (x.float() + r.float()).to(dtype)
    assert torch.equal(q.summed, h)
    assert residual or q.summed is x
    ref.check_rows(q.data, q.scale, ref.norm(h, w, 1e-5), ref.NORM_REL)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", SHAPES)
def test_gated(rows, channels, dtype):
    say("gated", rows, channels, dtype)
    both = normal(5, rows, 2 * channels, std=4.0, dtype=dtype)
    gate, up = both[:, :channels], both[:, channels:]
    q = ops().gated_quantize(gate, up)
    ref.check_rows(q.data, q.scale, ref.gated(gate, up), ref.gated_rel(gate))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(8195, 64), (20001, 272), (9001, 2048)])
def test_more_rows_than_waves(rows, channels, dtype):
    """Waves that go on to other rows."""
    say("many rows", rows, channels, dtype)
    x, r = normal(1, rows, channels, dtype=dtype), normal(2, rows, channels, dtype=dtype)
    w = 1 + 0.1 * normal(3, channels)
    q = ops().quantize_rows(x)
    ref.check_rows(q.data, q.scale, x.double(), 0.0)
    h = (x.float() + r.float()).to(dtype)
    q = ops().norm_quantize(x, w, residual=r, summed=r)
    assert torch.equal(r, h)
    ref.check_rows(q.data, q.scale, ref.norm(h, w, 1e-6), ref.NORM_REL)
    q = ops().norm_quantize(x, w)
    ref.check_rows(q.data, q.scale, ref.norm(x, w, 1e-6), ref.NORM_REL)
    q = ops().gated_quantize(x, h)
    ref.check_rows(q.data, q.scale, ref.gated(x, h), ref.gated_rel(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [48, 2048, 6144, 16384])
def test_rows_of_extremes(dtype, channels):
    """Zeros, magnitudes at the ends of the range, single values, values that are not finite."""
    say("extremes", dtype, channels)
    big, small = torch.finfo(dtype).max, 2.0 ** -126
    x = torch.zeros(14, channels, dtype=dtype, device="cuda")
    x[1, 5] = big
    x[2] = -big
    x[3, channels - 1] = small  # below the least magnitude
    x[4, 0] = 127 * small * 2
    x[4, 3] = -63 * small * 2
    x[5, 7], x[5, 8] = float("inf"), 1.0
    x[6, 9] = float("-inf")
    x[7, channels - 1] = float("nan")
    x[8] = 1.0
    x[9, 11] = -3.0
    x[10] = torch.arange(channels, device="cuda") % 255 - 127.0
    x[11, ::2] = 2.0 ** -100
    x[12, 1], x[12, 2] = 2.0 ** 100, 2.0 ** -100
    x[13] = -0.0
    q = ops().quantize_rows(x)
    ref.check_rows(q.data, q.scale, x.double(), 0.0)
    assert torch.equal(q.data[10].double(), x[10].double())  # whole numbers up to 127 stay
    # half to even: the integers' halves under a scale of one
    h = torch.zeros(1, channels, dtype=dtype, device="cuda")
    h[0, :8] = torch.tensor([127, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 3.5])
    assert ops().quantize_rows(h).data[0, :8].tolist() == [127, 0, 2, 2, 0, -2, -2, 4]
    # the norm: a mean square past F32's range gives zeros, what is not finite NaN
    w = torch.ones(channels, device="cuda")
    n = ops().norm_quantize(x, w, eps=1e-6)
    assert bool(torch.isnan(n.scale[[5, 6, 7]]).all()) and bool((n.data[[1, 2, 5, 6, 7, 0, 13]] == 0).all())
    assert n.scale[[0, 1, 2, 13]].tolist() == [0.0] * 4
    ref.check_rows(n.data[8:11], n.scale[8:11], ref.norm(x[8:11], w, 1e-6), ref.NORM_REL)
    none = ops().norm_quantize(x[:1], w, eps=0.0)  # 0 / 0
    assert bool(torch.isnan(none.scale).all()) and bool((none.data == 0).all())
    # a residual that cancels, one that makes infinity
    n = ops().norm_quantize(x[1:3], w, residual=x[1:3])
    assert bool(torch.isnan(n.scale).all()) and bool(torch.isinf(n.summed[1]).all())
    n = ops().norm_quantize(x[8:11], w, residual=-x[8:11])
    assert n.scale.tolist() == [0.0] * 3 and bool((n.data == 0).all())
    # gates far out on either side
    g = torch.zeros(4, channels, dtype=dtype, device="cuda")
    g[0], g[1], g[2, 3], g[3] = 300.0, -300.0, float("inf"), 50.0
    y = ops().gated_quantize(g, torch.full_like(g, 2.0))
    assert y.data[0].eq(127).all() and abs(float(y.scale[0]) * 127 - 600) < 1e-3
    assert float(y.scale[1]) == 0 and bool((y.data[1:3] == 0).all()) and bool(torch.isnan(y.scale[2]))
    assert y.data[3].eq(127).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_apart(dtype):
    """Views of wider tensors, in and out; nothing beside them is touched."""
    say("rows apart", dtype)
    for rows, channels in ((9, 272), (6, 4112), (2, 9008)):
        x, r = normal(1, rows, channels, dtype=dtype), normal(2, rows, channels, dtype=dtype)
        w = 1 + 0.1 * normal(3, channels)
        _, xv = apart(x, 40, 16)
        _, rv = apart(r, 24, 8)
        whole_s, sv = apart(torch.zeros_like(x), 16, 8)
        whole_q, qv = apart(torch.zeros(rows, channels, dtype=I8, device="cuda"), 48, 16)
        scale = torch.zeros(rows + 2, device="cuda")
        n = ops().norm_quantize(xv, w, residual=rv, summed=sv, out=(qv, scale[1:-1]))
        want = ops().norm_quantize(x, w, residual=r)
        assert n.data is qv and n.summed is sv
        assert torch.equal(qv, want.data) and torch.equal(scale[1:-1], want.scale) and torch.equal(sv, want.summed)
        assert bool((whole_q[:, :16] == 77).all()) and bool((whole_q[:, 16 + channels:] == 77).all())
        assert bool((whole_s[:, :8] == 77).all()) and bool((whole_s[:, 8 + channels:] == 77).all())
        assert scale[0] == 0 and scale[-1] == 0
        # in place of the residual, and of the input
        for target in (xv, rv):
            keep = target.clone()
            got = ops().norm_quantize(xv, w, residual=rv, summed=target)
            assert torch.equal(got.data, want.data) and torch.equal(target, want.summed)
            target.copy_(keep)
        got = ops().quantize_rows(xv, out=(qv, scale[1:-1]))
        assert torch.equal(got.data, ops().quantize_rows(x).data)
        # one row for all
        got = ops().gated_quantize(x[:1].expand(rows, channels), rv)
        assert torch.equal(got.data, ops().gated_quantize(x[:1].repeat(rows, 1), r).data)


# ---------------------------------------------------------------- product

PRODUCTS = [(1, 16, 1), (1, 48, 3), (2, 2048, 100), (5, 144, 33), (16, 2048, 512), (17, 1040, 4097), (31, 512, 250), (33, 6144, 128),
            (64, 2048, 1000), (65, 272, 640), (100, 4096, 2048), (128, 80, 127), (129, 3584, 1024), (255, 512, 511), (256, 2048, 4096),
            (257, 1024, 2049), (300, 2048, 9216), (513, 768, 4104), (1000, 1408, 512), (2049, 512, 2304), (4100, 256, 1100),
            (1, 65536, 40), (70, 65536, 70), (300, 16384, 300), (8, 16, 5000), (900, 16, 900), (600, 32, 31)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs", PRODUCTS)
def test_linear(rows, channels, outputs, dtype):
    """Bit for bit: the sums are exact, the roundings those of the definition."""
    say("linear", rows, channels, outputs, dtype)
    x, w = ints(rows, rows, channels), ints(outputs + 7, outputs, channels)
    got = ops().int8_linear(x, w, dtype=dtype)
    assert got.shape == (rows, outputs) and got.dtype == dtype
    assert torch.equal(got, ref.linear(x, w, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs,front", [(2300, 2064, 12300, 0), (2049, 4112, 6200, 8), (1030, 6160, 12501, 0), (700, 1040, 9000, 0),
                                                         (700, 1040, 9003, 3), (520, 16, 20000, 16), (300, 80, 20001, 1), (40, 2048, 30000, 0)])
def test_linear_many_tiles(rows, channels, outputs, front, dtype):
    """More tiles than compute units, of every size: ragged at their ends, in rows of whole lines and not."""
    say("many tiles", rows, channels, outputs, front, dtype)
    x, w = ints(1, rows, channels), ints(2, outputs, channels)
    whole = torch.full((rows, outputs + 2 * front), 77, dtype=dtype, device="cuda")
    got = ops().int8_linear(x, w, out=whole[:, front:front + outputs])
    assert torch.equal(got, ref.linear(x, w, dtype))
    assert bool((whole[:, :front] == 77).all()) and bool((whole[:, front + outputs:] == 77).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs", [(1, 16, 8193), (1, 2048, 12300), (2, 1040, 33000), (7, 4112, 9217), (3, 144, 50001), (16, 304, 8200)])
def test_linear_few_rows_many_outputs(rows, channels, outputs, dtype):
    say("few rows, many outputs", rows, channels, outputs, dtype)
    x, w = ints(1, rows, channels), ints(2, outputs, channels)
    whole = torch.full((rows, outputs + 5), 77, dtype=dtype, device="cuda")
    got = ops().int8_linear(x, w, out=whole[:, :outputs])
    assert torch.equal(got, ref.linear(x, w, dtype))
    assert bool((whole[:, outputs:] == 77).all())


@pytest.mark.parametrize("rows,outputs", [(1, 7), (40, 70), (300, 520)])
def test_linear_sums_at_their_largest(rows, outputs):
    """-128 times -128 over every channel."""
    say("largest sums", rows, outputs)
    x = (torch.full((rows, 65536), -128, dtype=I8, device="cuda"), torch.ones(rows, device="cuda"))
    w = (torch.full((outputs, 65536), -128, dtype=I8, device="cuda"), torch.ones(outputs, device="cuda"))
    assert bool((ops().int8_linear(x, w, dtype=F32) == 2.0 ** 30).all())
    w[0].fill_(127)
    assert bool((ops().int8_linear(x, w, dtype=F32) == -float(128 * 127 * 65536)).all())


@pytest.mark.parametrize("rows,channels,outputs", [(3, 208, 50), (48, 1040, 300), (200, 400, 270), (700, 912, 777)])
def test_linear_of_every_place(rows, channels, outputs):
    """One value of each row and output in turn: a place that is read twice, lost or taken from
    another row shows as a whole number."""
    say("places", rows, channels, outputs)
    k = torch.arange(channels, device="cuda")
    x = ((k[None] * 7 + torch.arange(rows, device="cuda")[:, None] * 13) % 251 - 125).to(I8)
    w = torch.zeros(outputs, channels, dtype=I8, device="cuda")
    n = torch.arange(outputs, device="cuda")
    for step in (0, 1, 5):
        w.zero_()
        at = (n * 11 + step * 37) % channels
        w[n, at] = 1
        got = ops().int8_linear((x, torch.ones(rows, device="cuda")), (w, torch.ones(outputs, device="cuda")), dtype=F32)
        assert torch.equal(got, x[:, at].float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels,outputs", [(1, 272, 100), (20, 528, 333), (150, 1040, 260), (520, 272, 530)])
def test_linear_rows_apart(rows, channels, outputs, dtype):
    """Operands and results inside wider tensors, results at odd addresses too."""
    say("product apart", rows, channels, outputs, dtype)
    x, w = ints(1, rows, channels), ints(2, outputs, channels)
    want = ref.linear(x, w, dtype)
    _, xv = apart(x[0], 48, 32)
    _, wv = apart(w[0], 16, 16)
    for extra, front in ((0, 0), (1, 1), (7, 3), (8, 8), (16, 4)):
        whole, view = apart(torch.zeros(rows, outputs, dtype=dtype, device="cuda"), extra, front)
        assert ops().int8_linear((xv, x[1]), (wv, w[1]), out=view) is view
        assert torch.equal(view, want), (extra, front)
        assert bool((whole[:, :front] == 77).all()) and bool((whole[:, front + outputs:] == 77).all())
    # one row for all of them
    got = ops().int8_linear((xv[:1].expand(rows, channels), x[1][:1].repeat(rows)), (wv, w[1]), dtype=dtype)
    assert torch.equal(got, ref.linear((x[0][:1], x[1][:1]), w, dtype).expand(rows, outputs))


def test_linear_scales_of_all_kinds():
    """Zeros, NaN and infinity stay with their row and output."""
    say("scales")
    for rows in (5, 90, 300):
        x, w = ints(1, rows, 512), ints(2, 130, 512)
        x[1][1], x[1][2], x[1][3] = float("nan"), 0.0, float("inf")
        w[1][7], w[1][9], w[1][100] = 0.0, float("nan"), 1e-30
        got, want = ops().int8_linear(x, w, dtype=F32), ref.linear(x, w, F32)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0, 1, 2), want.nan_to_num(0, 1, 2))


def test_far_rows():
    """Offsets past 32 bits in every operand."""
    say("far rows")
    rows, channels, outputs, step = 5, 512, 3, (1 << 30) + 16
    def far(values, step):
        whole = torch.empty((rows - 1) * step + values.shape[1], dtype=values.dtype, device="cuda")
        view = whole.as_strided(values.shape, (step, 1))
        view.copy_(values)
        return view
    x = ints(1, rows, channels)
    w = ints(2, rows, channels)
    xv = far(x[0], step)
    assert torch.equal(ops().int8_linear((xv, x[1]), w, dtype=BF), ref.linear(x, w, BF))
    assert torch.equal(ops().int8_linear(w, (xv, x[1]), dtype=BF), ref.linear(w, x, BF))
    many = (xv[:1].expand(300, channels), x[1][:1].repeat(300))
    assert torch.equal(ops().int8_linear(many, (xv, x[1]), dtype=BF), ref.linear((x[0][:1], x[1][:1]), x, BF).expand(300, rows))
    del xv, many
    h = normal(3, rows, channels, dtype=BF)
    hv = far(h, step)
    out = far(torch.zeros(rows, channels, dtype=I8, device="cuda"), step)
    want = ops().norm_quantize(h, torch.ones(channels, device="cuda"), residual=h)
    got = ops().norm_quantize(hv, torch.ones(channels, device="cuda"), residual=hv, summed=hv, out=(out, torch.empty(rows, device="cuda")))
    assert torch.equal(got.data, want.data) and torch.equal(got.summed, want.summed)
    del out, got
    y = ops().int8_linear(x, w, out=hv[:, :rows])
    assert torch.equal(y, ref.linear(x, w, BF))


# ------------------------------------------------- streams, graphs, together


def layer(c, s):
    """A layer's norm, feed-forward and next norm, as a round runs them."""
    n = ops().norm_quantize(s["x"], s["norm"], residual=s["residual"])
    both = ops().int8_linear(n, s["w1"])
    g = ops().gated_quantize(both[:, :c], both[:, c:])
    y = ops().int8_linear(g, s["w2"])
    return (n.summed, y, *ops().norm_quantize(y, s["norm"], residual=n.summed))


def layer_state(rows, hidden, c, seed=0):
    return dict(x=normal(seed + 1, rows, hidden, dtype=BF), residual=normal(seed + 2, rows, hidden, dtype=BF), norm=1 + 0.1 * normal(3, hidden),
                w1=ops().quantize_rows(normal(4, 2 * c, hidden, std=hidden ** -0.5, dtype=BF)),
                w2=ops().quantize_rows(normal(5, hidden, c, std=c ** -0.5, dtype=BF)))


@pytest.mark.parametrize("rows", [1, 19, 300])
def test_another_stream(rows):
    say("stream", rows)
    s = layer_state(rows, 512, 768)
    want = layer(768, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(768, s)
    q = ops().quantize_rows(s["x"], stream=side)
    z = ops().int8_linear(q, s["w1"], stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(z, ops().int8_linear(ops().quantize_rows(s["x"]), s["w1"]))


@pytest.mark.parametrize("rows", [1, 40, 600])
def test_captured(rows):
    """A captured layer, replayed over new inputs with eager work between the replays."""
    say("captured", rows)
    c = 768
    s = layer_state(rows, 512, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(c, s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = layer(c, s)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        new = layer_state(rows, 512, c, seed=10 * i)
        s["x"].copy_(new["x"])
        s["residual"].copy_(new["residual"])
        graph.replay()
        torch.cuda.synchronize()
        want = layer(c, dict(s, x=new["x"], residual=new["residual"]))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_products(dtype):
    """Tiles of every size in one graph, LDS of more than 64 KB among them, without a call in front of it."""
    sizes = [(5, 512, 700), (24, 512, 700), (70, 256, 300), (300, 2048, 9216), (1030, 2064, 6300), (2300, 2064, 12300)]
    say("captured products", dtype)
    made = [(ints(r, r, c), ints(o, o, c)) for r, c, o in sizes]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = [ops().int8_linear(x, w, dtype=dtype) for x, w in made]
    for i in range(3):
        for (x, _), _ in made:
            x.copy_(x.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        for g, (x, w) in zip(got, made):
            assert torch.equal(g, ref.linear(x, w, dtype)), (i, g.shape)


@pytest.mark.parametrize("rows", [1, 33])
def test_layer_near_the_exact_products(rows):
    """The layer in 8 bits against its definition in 64 bits: each operator's output follows from
    the one in front of it."""
    say("layer", rows)
    c = 768
    s = layer_state(rows, 512, c)
    n = ops().norm_quantize(s["x"], s["norm"], residual=s["residual"])
    h = (s["x"].float() + s["residual"].float()).to(BF)
    assert torch.equal(n.summed, h)
    ref.check_rows(n.data, n.scale, ref.norm(h, s["norm"], 1e-6), ref.NORM_REL)
    both = ops().int8_linear(n, s["w1"])
    assert torch.equal(both, ref.linear(n[:2], s["w1"], BF))
    g = ops().gated_quantize(both[:, :c], both[:, c:])
    ref.check_rows(g.data, g.scale, ref.gated(both[:, :c], both[:, c:]), ref.gated_rel(both[:, :c]))
    assert torch.equal(ops().int8_linear(g, s["w2"]), ref.linear(g, s["w2"], BF))


def test_empty_calls():
    say("empty")
    x = torch.empty(0, 512, dtype=BF, device="cuda")
    q = ops().quantize_rows(x)
    assert q.data.shape == (0, 512) and q.scale.shape == (0,)
    assert ops().int8_linear(q, ints(1, 30, 512)).shape == (0, 30)
    n = ops().norm_quantize(x, torch.ones(512, device="cuda"), residual=x)
    assert n.data.shape == n.summed.shape == (0, 512)
    assert ops().gated_quantize(x, x).data.shape == (0, 512)


def test_refused_on_the_device():
    """What the torch binding refuses of tensors on the GPU."""
    say("refusals")
    o = ops()
    x, w = normal(1, 4, 64, dtype=BF), torch.ones(64, device="cuda")
    q = o.quantize_rows(x)
    for call, text in [
        (lambda: o.quantize_rows(x.half()), "bfloat16"), (lambda: o.quantize_rows(x[0]), "dimensions"),
        (lambda: o.quantize_rows(x.t()), "contiguous"), (lambda: o.quantize_rows(x, out=(q.data[:3], q.scale[:3])), "out must be"),
        (lambda: o.quantize_rows(x, out=(q.data, q.scale[:3])), "entries"), (lambda: o.quantize_rows(x, out=(q.data.int(), q.scale)), "int8"),
        (lambda: o.norm_quantize(x, w[:63]), "entries"), (lambda: o.norm_quantize(x, w.bfloat16()), "float32"),
        (lambda: o.norm_quantize(x, w, residual=x.float()), "bfloat16"), (lambda: o.norm_quantize(x, w, residual=x[:3]), "residual must be"),
        (lambda: o.norm_quantize(x, w, summed=x.clone()), "summed"), (lambda: o.norm_quantize(x, w, residual=x, summed=x.float()), "bfloat16"),
        (lambda: o.norm_quantize(x, w.cpu()), "GPU"), (lambda: o.gated_quantize(x, x[:, :48]), "up must be"),
        (lambda: o.int8_linear(q, (q.data[:, :48], q.scale)), "channels"), (lambda: o.int8_linear(q, q, dtype=torch.float16), "dtype"),
        (lambda: o.int8_linear(q, q, out=x), "out must be"), (lambda: o.int8_linear(q, (q.data, q.scale[:2])), "entries"),
        (lambda: o.int8_linear((q.data.cpu(), q.scale), q), "GPU"), (lambda: o.int8_linear((q.data.t(), q.scale), q), "contiguous"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    for call, text in [
        (lambda: o.quantize_rows(normal(1, 4, 68)), "multiple of 16"), (lambda: o.quantize_rows(normal(1, 4, 80)[:, 1:65]), "16-byte"),
        (lambda: o.quantize_rows(normal(1, 4, 66)[:, :64]), "multiple of"), (lambda: o.norm_quantize(x, w, eps=-1.0), "eps"),
        (lambda: o.norm_quantize(x, torch.ones(65, device="cuda")[1:]), "16-byte"),
        (lambda: o.quantize_rows(x, out=(q.data[:1].expand(4, 64), q.scale)), "overlap"),
        (lambda: o.int8_linear(q, q, out=torch.zeros(1, 4, device="cuda").expand(4, 4)), "overlap"),
        (lambda: o.quantize_rows(torch.zeros(1, 65552, device="cuda")), "65536"),
    ]:
        with pytest.raises(o.CQ35Error, match=text):
            call()
    for call in (lambda: o.quantize_rows([1.0]), lambda: o.int8_linear(3, q), lambda: o.norm_quantize(x, None)):
        with pytest.raises(TypeError):
            call()

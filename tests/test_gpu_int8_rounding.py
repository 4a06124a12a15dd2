"""Where the roundings of the 8-bit rows lie: integers at exact halves, and gated
values far out, against the definitions in 64 bits."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def say(*a):
    print(*a, flush=True)


def ops():
    import cq35
    return cq35


def mantissas(channels, power):
    """A row for each of the 128 mantissas that a largest magnitude can have in BF16: the
    magnitude, its halves of both signs, and values of all sizes below it."""
    g = torch.Generator().manual_seed(channels)
    a = (torch.arange(128, 256, dtype=torch.float64) * 2.0 ** power)[:, None]
    x = (torch.rand(128, channels, dtype=torch.float64, generator=g) * 2 - 1) * 2.0 ** -torch.randint(12, (128, channels), generator=g)
    x = (x * a).to(BF).double().clamp(-a, a)
    x[:, 3:4], x[:, 5:6], x[:, channels - 2:channels - 1] = -a, a / 2, -a / 2
    return x, a


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("power", [-120, -7, 100, 119])
@pytest.mark.parametrize("channels", [16, 272, 2064, 9008])
def test_integers_of_exact_halves(channels, power, dtype):
    """y (127 / a) of values of 8 bits is a half exactly or at least 2^-16 of itself away from one, so
    that one rounding to F32 decides nothing: every integer is the definition's. 64 bits hold 127 y
    exactly and divide with far less than that."""
    say("halves", channels, power, dtype)
    x, a = mantissas(channels, power)
    q = ops().quantize_rows(x.to(dtype).cuda())
    assert torch.equal(q.data.cpu().double(), torch.round(127 * x / a))
    assert torch.equal(q.scale.cpu(), (a[:, 0] / 127).float())
    assert bool((q.data[:, 5] == 64).all()) and bool((q.data[:, channels - 2] == -64).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_halves_of_a_norm_and_a_gated_product(dtype):
    """The same behind the norm of a row of ones, whose values are its weights, and behind gates so far
    out that their sigmoid is 1."""
    say("halves behind others", dtype)
    x, a = mantissas(272, -7)
    one = torch.ones(1, 272, device="cuda", dtype=dtype)
    want = torch.round(127 * x / a)
    for r in range(128):
        q = ops().norm_quantize(one, x[r].float().cuda(), eps=0.0)
        assert torch.equal(q.data[0].cpu().double(), want[r]), r
    gate = torch.full((128, 272), 128.0, dtype=dtype, device="cuda")
    q = ops().gated_quantize(gate, x.to(dtype).cuda())
    assert torch.equal(q.data.cpu().double(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("channels", [16, 2064, 9008])
def test_gates_far_out(channels, dtype):
    """A row of one gate and one factor: its scale times 127 is the product itself. In half-steps u of
    F32: e^-g is off by 4 (2^t within a step, its correction and their product by 1 each), 1 + e^-g by 1, the
    reciprocal by 2 (a step), two products and the scale's division by 1 each. Gates to where e^-g
    nears 2^126."""
    say("gates", channels, dtype)
    gate = torch.cat([torch.linspace(-87.0, 87.0, 700), torch.tensor([-0.5, -1e-3, 1e-3, 2.0 ** -60, 100.0, 1e4])]).to(dtype)
    up = torch.where(torch.arange(len(gate)) % 2 == 0, 1.0, -2.75).to(dtype)
    up[gate < -40] *= 2.0 ** 60  # the product itself stays far above the least magnitude
    q = ops().gated_quantize(*(t[:, None].expand(-1, channels).contiguous().cuda() for t in (gate, up)))
    y = gate.double() * torch.sigmoid(gate.double()) * up.double()
    off = (q.scale.cpu().double() * 127 / y.abs() - 1).abs() / 2.0 ** -24
    assert off.max() <= 10.1, (off.max(), gate[off.argmax()])
    assert torch.equal(q.data.cpu().double(), (127.0 * y.sign())[:, None].expand(-1, channels))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("channels", [16, 2064, 9008])
def test_norm_of_tiny_rows(channels, dtype):
    """Rows of one power of two: the norm is the weights down to squares of 2^-140, exact in F32's subnormals;
    below 2^-75 the squares are zeros, which eps decides about."""
    say("tiny rows", channels, dtype)
    w = torch.linspace(0.5, 2.0, channels).cuda()
    tiny = torch.tensor([2.0 ** -30, 2.0 ** -60, 2.0 ** -70, 2.0 ** -76, 2.0 ** -100, 0.0], dtype=dtype, device="cuda")
    x = tiny[:, None].expand(-1, channels).contiguous()
    q = ops().norm_quantize(x, w, eps=0.0)
    for r in range(3):
        assert torch.equal(q.data[r].cpu().double(), torch.round(127 * w.cpu().double() / 2))
        assert float(q.scale[r]) == float(torch.tensor(2.0) / 127)
    assert bool(torch.isnan(q.scale[3:]).all()) and bool((q.data[3:] == 0).all())
    q = ops().norm_quantize(x, w, eps=1e-6)
    off = q.scale.cpu().double() * 127 / (tiny.cpu().double() * 2 / (tiny.cpu().double() ** 2 + 1e-6).sqrt()) - 1
    assert off[:5].abs().max() < 8 * 2.0 ** -24 and float(q.scale[5]) == 0  # eps, mean and root, division, two products, the scale


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("channels", [16, 2064, 9008])
def test_gates_at_the_ends_of_the_range(channels, dtype):
    """Gates whose exponent passes F32's range, to the largest number: the product is the gate, or 0."""
    say("largest gates", channels, dtype)
    top = torch.finfo(dtype).max
    gate = torch.tensor([200.0, 2.0 ** 24, 1e30, 1e38, 2.3e38, 2.4e38, 3e38, top], dtype=torch.float64).to(dtype)
    gate = torch.cat([gate, -gate])
    rows = gate[:, None].expand(-1, channels).contiguous().cuda()
    q = ops().gated_quantize(rows, torch.ones_like(rows))
    n = len(gate) // 2
    # the reciprocal of 1 is within a step, the scale rounds
    off = (q.scale[:n].cpu().double() * 127 / gate[:n].double() - 1).abs() / 2.0 ** -24
    assert off.max() <= 3.1, off
    assert bool((q.data[:n] == 127).all())
    assert q.scale[n:].tolist() == [0.0] * n and bool((q.data[n:] == 0).all())
    for x in (float("inf"), float("-inf"), float("nan")):
        rows[1, channels - 1] = x
        q = ops().gated_quantize(rows, torch.ones_like(rows))
        assert bool(torch.isnan(q.scale[1])) and bool((q.data[1] == 0).all())

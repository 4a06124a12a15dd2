"""Log probabilities, entropies and most likely tokens on the device against the
statement in 64 bits (int8_reference.logprobs)."""
import numpy as np
import pytest

import int8_reference as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
TYPES = [BF, F32]
INF = float("inf")


def say(*a):
    print(*a, flush=True)


def ops():
    import cq35
    return cq35


def logits(seed, rows, vocab, dtype, std=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(rows, vocab, device="cuda").normal_(0, std, generator=g).to(dtype)


def tokens(seed, rows, given, vocab):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(vocab, (rows, given), device="cuda", generator=g)


def check(x, t, top, got):
    lp, entropy, best, best_lp = ref.logprobs(x, t, top)
    assert np.array_equal(got.top_tokens.cpu().numpy(), best), "top tokens"
    rows = x.cpu().double().numpy()
    fine = np.isfinite(rows.max(-1))
    g, ge, gt = (a.cpu().double().numpy() for a in (got.logprobs.reshape(lp.shape), got.entropy, got.top_logprobs))
    for a, b in ((g, lp), (ge, entropy), (gt, best_lp)):
        assert np.array_equal(np.isnan(a), np.isnan(b))
        assert np.array_equal(np.isneginf(a), np.isneginf(b))
    if not fine.any():
        return
    xf = x.cpu()[torch.from_numpy(fine)]
    m = rows[fine].max(-1, keepdims=True)
    for a, b, at in ((g, lp, t.cpu().numpy()), (gt, best_lp, best)):
        if a.shape[1] == 0:
            continue
        a, b, at = a[fine], b[fine], at[fine]
        there = np.isfinite(b)
        d = np.where(there, np.take_along_axis(rows[fine], np.clip(at, 0, x.shape[1] - 1), 1) - m, 0.0)
        limit, _ = ref.logprob_limits(xf, d)
        off = np.abs(np.where(there, a, 0.0) - np.where(there, b, 0.0))
        assert (off <= limit).all(), f"off by {off.max():.3g}, allowed {limit[off > limit].min():.3g}"
    _, limit = ref.logprob_limits(xf, np.zeros((len(xf), 1)))
    off = np.abs(ge[fine] - entropy[fine])
    assert (off <= limit).all(), f"entropy off by {off.max():.3g}"


SIZES = [(1, 1, 1, 1), (3, 2, 2, 1), (2, 31, 1, 31), (5, 33, 3, 32), (4, 255, 1, 0), (1, 1000, 0, 7), (7, 4096, 1, 5), (2, 8191, 4, 32),
         (2, 8192, 1, 1), (2, 8193, 1, 20), (1, 16385, 1, 20), (3, 50257, 1, 8), (1, 248320, 1, 20), (4, 248320, 2, 32), (700, 1001, 1, 3),
         (300, 20011, 1, 20), (130, 65537, 1, 1), (1100, 9000, 1, 4)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,given,top", SIZES)
def test_logprobs(rows, vocab, given, top, dtype):
    say("logprobs", rows, vocab, given, top, dtype)
    x, t = logits(rows + vocab, rows, vocab, dtype), tokens(7, rows, given, vocab)
    check(x, t, top, ops().token_logprobs(x, t, top=top))


def shaped(kind, vocab, dtype):
    """Rows in which a selection can go wrong."""
    i = torch.arange(vocab, device="cuda", dtype=torch.float64)
    x = {"equal": lambda: torch.zeros(vocab), "ascending": lambda: i * 1e-3, "descending": lambda: -i * 1e-3,
         "steps": lambda: torch.floor(i / 977) % 7, "late steps": lambda: (i >= vocab - 40).double(),
         "two values": lambda: (i % 3 == 1).double() * 4 - 2, "lowest": lambda: torch.full((vocab,), torch.finfo(dtype).min),
         "lowest but one": lambda: torch.where(i == vocab // 2, 3.0, torch.finfo(dtype).min),
         "masked": lambda: torch.where(i % 50 == 17, torch.sin(i), -INF), "masked but two": lambda: torch.where((i == 3) | (i == vocab - 1), 1.0, -INF),
         "masked front": lambda: torch.where(i > vocab * 0.9, torch.cos(i), -INF), "one peak": lambda: torch.where(i == vocab - 2, 80.0, -80.0),
         "huge": lambda: torch.where(i % 5 == 0, 1e30, -1e30), "zeros of both signs": lambda: torch.where(i % 2 == 0, -0.0, 0.0),
         "strided peaks": lambda: torch.where(i % 256 == 5, 10 + i * 1e-4, torch.sin(i)),
         "run of peaks": lambda: torch.where((i >= 100) & (i < 140), 20.0, 0.0)}[kind]()
    return x.to(device="cuda", dtype=dtype)


KINDS = ["equal", "ascending", "descending", "steps", "late steps", "two values", "lowest", "lowest but one", "masked", "masked but two",
         "masked front", "one peak", "huge", "zeros of both signs", "strided peaks", "run of peaks"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [150, 5003, 40000, 248320])
@pytest.mark.parametrize("top", [1, 32])
def test_rows_of_all_shapes(vocab, top, dtype):
    say("shapes", vocab, top, dtype)
    x = torch.stack([shaped(k, vocab, dtype) for k in KINDS])
    t = tokens(3, len(KINDS), 3, vocab)
    check(x, t, top, ops().token_logprobs(x, t, top=top))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [1, 20])
def test_rows_of_all_shapes_in_one_block_each(top, dtype):
    """So many rows that none is cut: a block goes over many tiles, with the front of some masked for a while."""
    say("one block", top, dtype)
    vocab, rows = 70001, 620
    x = [shaped(k, vocab, dtype) for k in KINDS]
    ordinary = logits(5, 12, vocab, dtype)
    for i, front in enumerate((30, 4096, 4097, 8192, 8200, 16384, 16500, 33000, 40960, 65600, vocab - 21, vocab - 3)):
        ordinary[i, :front] = (-INF, torch.finfo(dtype).min, 0.0)[i % 3]
    x = torch.cat([torch.stack(x), ordinary])
    n = len(x)
    t = tokens(4, n, 2, vocab)
    again = torch.arange(rows, device="cuda") % n
    got = ops().token_logprobs(x[again], t[again], top=top)
    for at in (0, n):
        check(x, t, top, type(got)(*(a[at:at + n] for a in got)))
    assert torch.equal(got.top_tokens, got.top_tokens[:n][again])
    # the order of a row's sums follows from its place within 16 bytes, the same every 8 rows (2 n is a multiple)
    assert 2 * n % 8 == 0
    again = torch.arange(rows, device="cuda") % (2 * n)
    for a in got:
        assert torch.equal(a.view(torch.uint8), a[:2 * n].contiguous()[again].view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("threads", [40, 56, 60, 63, 64, 65])
def test_a_crowd_behind_candidates(threads, dtype):
    """Some candidates in the list, then nearly as many at once as it holds: all the logits of some threads."""
    say("crowd", threads, dtype)
    piece = 16 // dtype.itemsize
    tile = 4 * 256 * piece
    if dtype is F32:
        threads *= 2  # half as many logits each
    n, rows, vocab = 10, 520, 20 * tile
    x = logits(6, n, vocab, dtype, std=0.5)
    g = torch.Generator(device="cuda").manual_seed(threads)
    # few logits above the first tiles' best, fewer than are sorted out at once
    few = 9 * tile + 61 * torch.arange(100, device="cuda")
    x[:, few] = (5 + torch.rand(n, 100, device="cuda", generator=g)).to(dtype)
    for j in range(4):
        at = 16 * tile + j * 256 * piece
        x[:, at:at + threads * piece] = (10 + 4 * torch.rand(n, threads * piece, device="cuda", generator=g)).to(dtype)
    t = tokens(4, n, 1, vocab)
    again = torch.arange(rows, device="cuda") % n
    got = ops().token_logprobs(x[again], t[again], top=20)
    check(x, t, 20, type(got)(*(a[:n] for a in got)))
    for a in got:  # rows of whole 16 bytes: the same bits
        assert torch.equal(a.view(torch.uint8), a[:n].contiguous()[again].view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 9001, 100003])
def test_not_finite(vocab, dtype):
    """NaN and infinity make a row's numbers NaN, wherever they lie; its order stays."""
    say("not finite", vocab, dtype)
    x = logits(1, 9, vocab, dtype)
    x[0, vocab - 1] = float("nan")
    x[1, 0], x[1, vocab // 2] = INF, float("nan")
    x[2, 5] = x[2, vocab - 3] = INF
    x[3] = -INF
    x[4] = INF
    x[5] = float("nan")
    x[6, : vocab - 1] = -INF
    x[7, ::2] = -float("nan")
    t = tokens(3, 9, 2, vocab)
    got = ops().token_logprobs(x, t, top=8)
    check(x, t, 8, got)
    assert bool(torch.isnan(got.entropy[:6]).all()) and bool(torch.isfinite(got.entropy[[6, 8]]).all())
    assert got.entropy[6] == 0 and got.top_logprobs[6, 0] == 0


def test_tokens_outside():
    say("tokens outside")
    x = logits(1, 4, 500, F32)
    t = torch.tensor([[-1, 0, 499], [500, 3, 2**40], [-2**63, 2**63 - 1, 7], [2**32 + 5, -2**32, 4]], device="cuda")
    got = ops().token_logprobs(x, t)
    check(x, t, 0, got)
    assert torch.isnan(got.logprobs).sum() == 7


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [37, 4095, 33333])
def test_rows_anywhere(vocab, dtype):
    """Rows at every offset from a 16-byte address, inside NaN that must not be seen, and one row
    for all."""
    say("anywhere", vocab, dtype)
    x = logits(1, 5, vocab, dtype)
    t = tokens(2, 5, 2, vocab)
    want = ops().token_logprobs(x, t, top=6)
    for front, extra in ((1, 9), (3, 4), (7, 8), (2, 11)):
        whole = torch.full((5, vocab + extra), float("nan"), dtype=dtype, device="cuda")
        view = whole[:, front:front + vocab]
        view.copy_(x)
        got = ops().token_logprobs(view, t, top=6)
        check(x, t, 6, got)
        assert torch.equal(got.top_tokens, want.top_tokens)
    one = x[2:3].expand(5, vocab)
    check(one, t, 6, ops().token_logprobs(one, t, top=6))


def test_same_bits_again():
    """The order in which candidates are found changes nothing."""
    say("same bits")
    for rows, vocab in ((1, 248320), (40, 100000), (600, 5000)):
        x, t = logits(1, rows, vocab, BF), tokens(2, rows, 1, vocab)
        first = ops().token_logprobs(x, t, top=32)
        for _ in range(5):
            got = ops().token_logprobs(x, t, top=32)
            assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_far_rows():
    """Rows that start past 2^32 elements."""
    say("far rows")
    vocab, step = 3001, (1 << 31) + 5
    whole = torch.empty(2 * step + vocab, dtype=BF, device="cuda")
    view = whole.as_strided((3, vocab), (step, 1))
    view.copy_(logits(1, 3, vocab, BF))
    t = tokens(2, 3, 1, vocab)
    check(view, t, 5, ops().token_logprobs(view, t, top=5))


@pytest.mark.parametrize("rows,vocab,top", [(1, 100000, 5), (3, 248320, 32), (900, 3000, 2)])
def test_outputs_and_workspace_of_the_caller(rows, vocab, top):
    say("caller's", rows, vocab, top)
    o = ops()
    x, t = logits(1, rows, vocab, BF), tokens(2, rows, 1, vocab)[:, 0].contiguous()
    want = o.token_logprobs(x, t, top=top)
    assert want.logprobs.shape == (rows,)
    n = o.token_logprobs_workspace(rows, vocab, 1, top)
    around = torch.full((n + 512,), 255, dtype=torch.uint8, device="cuda")
    out = o.TokenLogprobs(torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
                          torch.empty(rows, top, dtype=torch.int64, device="cuda"), torch.empty(rows, top, device="cuda"))
    for _ in range(3):
        got = o.token_logprobs(x, t, top=top, out=out, workspace=around[256:256 + n])
        assert got.entropy is out.entropy and all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((around[:256] == 255).all()) and bool((around[256 + n:] == 255).all())
    if n:
        for bad in (around[256:256 + n - 1], around[264:264 + n]):
            with pytest.raises(o.CQ35Error, match="workspace"):
                o.token_logprobs(x, t, top=top, workspace=bad)


@pytest.mark.parametrize("rows,vocab", [(1, 248320), (500, 4000)])
def test_captured_and_on_another_stream(rows, vocab):
    say("captured", rows, vocab)
    o = ops()
    x, t = logits(1, rows, vocab, BF), tokens(2, rows, 1, vocab)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o.token_logprobs(x, t, top=9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = o.token_logprobs(x, t, top=9)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.copy_(logits(10 + i, rows, vocab, BF))
        t.copy_(tokens(20 + i, rows, 1, vocab))
        graph.replay()
        torch.cuda.synchronize()
        want = o.token_logprobs(x, t, top=9)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    side.wait_stream(torch.cuda.current_stream())
    other = o.token_logprobs(x, t, top=9, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_two_graphs_that_share_a_workspace():
    """Replayed one after the other, in any order."""
    say("shared workspace")
    o = ops()
    cases = [(2, 100000, 7), (1, 248320, 32)]
    work = torch.empty(max(o.token_logprobs_workspace(r, v, 1, k) for r, v, k in cases), dtype=torch.uint8, device="cuda")
    held = []
    side = torch.cuda.Stream()
    for rows, vocab, top in cases:
        x, t = logits(rows, rows, vocab, BF), tokens(2, rows, 1, vocab)
        n = o.token_logprobs_workspace(rows, vocab, 1, top)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = o.token_logprobs(x, t, top=top, workspace=work[:n])
        torch.cuda.current_stream().wait_stream(side)
        held.append((graph, got, x, t, top))
    for i in (0, 1, 1, 0, 1, 0, 0):
        graph, got, x, t, top = held[i]
        x.copy_(logits(30 + i, *x.shape, BF))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, o.token_logprobs(x, t, top=top)))


@pytest.mark.parametrize("given", [300, 1024])
def test_many_given_tokens(given):
    say("given", given)
    for rows, vocab in ((2, 70000), (600, 900)):
        x, t = logits(1, rows, vocab, F32), tokens(2, rows, given, vocab)
        check(x, t, 2, ops().token_logprobs(x, t, top=2))


def test_empty_and_refused():
    say("empty and refused")
    o = ops()
    x, t = logits(1, 4, 50, BF), tokens(2, 4, 1, 50)
    none = o.token_logprobs(x[:0], t[:0], top=3)
    assert none.top_tokens.shape == (0, 3) and none.entropy.shape == (0,)
    for call, text in [
        (lambda: o.token_logprobs(x.half(), t), "bfloat16"), (lambda: o.token_logprobs(x[0], t), "dimensions"),
        (lambda: o.token_logprobs(x.t(), t), "contiguous"), (lambda: o.token_logprobs(x, t.int()), "int64"),
        (lambda: o.token_logprobs(x, t[:3]), "tokens must be"), (lambda: o.token_logprobs(x, t.cpu()), "GPU"),
        (lambda: o.token_logprobs(x, t.view(4, 1, 1)), "dimensions"), (lambda: o.token_logprobs(x, t, top=33), "top"),
        (lambda: o.token_logprobs(x, t, top=-1), "top"), (lambda: o.token_logprobs(x, t.t().expand(4, 4)), "contiguous"),
        (lambda: o.token_logprobs(x, t, top=2, out=o.token_logprobs(x, t, top=1)), "out.top_tokens"),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(o.CQ35Error, match="alternatives"):
        o.token_logprobs(x[:, :5], t, top=6)
    with pytest.raises(o.CQ35Error, match="logits"):
        o.token_logprobs(x[:, :0], t)
    with pytest.raises(TypeError):
        o.token_logprobs(x, t, top=1.5)
    with pytest.raises(TypeError):
        o.token_logprobs(x, None)


def test_answer_of_a_head_in_8_bits():
    """The end of a round: final norm, vocabulary head, log probabilities of what was drawn."""
    say("head")
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(4)
    rows, hidden, vocab = 6, 512, 8192
    x = torch.empty(rows, hidden, device="cuda").normal_(generator=g).to(BF)
    head = o.quantize_rows(torch.empty(vocab, hidden, device="cuda").normal_(0, 0.1, generator=g).to(BF))
    n = o.norm_quantize(x, torch.ones(hidden, device="cuda"))
    for dtype in TYPES:
        out = o.int8_linear(n, head, dtype=dtype)
        assert torch.equal(out, ref.linear(n[:2], head, dtype))
        t = out.argmax(-1)
        got = o.token_logprobs(out, t, top=4)
        check(out, t[:, None], 4, got)
        assert torch.equal(got.logprobs, got.top_logprobs[:, 0])

"""Which keys paged attention reads, over the cases of paged_cases.py: every
tile of every split once, each row's last key its own, none of a page outside
the cache; and random cases in which every key weighs in."""
import numpy as np
import pytest

import test_gpu_paged as base
from paged_cases import LONG, SHAPES, TILE, VERY_LONG, Marked, random_case, starts
from test_gpu_paged import BF, KEYS, check_attention, i32, ops, run_attention, say

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

steered = base.steered  # both kernels


def on_device(s):
    return dict(s, k=s["k"].cuda(), v=s["v"].cuda())


@pytest.mark.parametrize("case", SHAPES)
@pytest.mark.parametrize("gate", [False, True])
def test_random(case, gate, steered):
    new, lengths, QH, KVH, HD, page = case
    say("random", new, lengths, QH, KVH, HD, page)
    s = on_device(random_case(sum(lengths) + HD, new, lengths, QH, KVH, HD, page, gate, qstd=2.0 if max(lengths) > 2000 else 1.0))
    check_attention(s, run_attention(s))
    check_attention(s, run_attention(s, max_rows=max(new), max_keys=max(lengths)))
    check_attention(s, run_attention(s, max_rows=1, max_keys=1))


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", LONG)
def test_random_long(new, length, QH, KVH, HD, page, steered):
    say("random, long", new, length, HD)
    s = on_device(random_case(length, [new, 1], [length, 40], QH, KVH, HD, page, qstd=2.0))
    for hints in (dict(max_keys=1), dict(max_keys=length), {}):
        check_attention(s, run_attention(s, max_rows=new, **hints))


@pytest.mark.parametrize("R,most_new,most,HD,QH,KVH", [(64, 3, 200, 64, 2, 1), (65, 40, 300, 128, 4, 2), (300, 2, 100, 64, 2, 2)])
def test_random_requests(R, most_new, most, HD, QH, KVH, steered):
    rng = np.random.default_rng(R)
    new = rng.integers(0, most_new + 1, R).tolist()
    lengths = [int(n + rng.integers(0, most)) for n in new]
    lengths[3] += 2000
    s = on_device(random_case(R, new, lengths, QH, KVH, HD, 16))
    check_attention(s, run_attention(s, max_rows=most_new, max_keys=max(lengths)))


def marked_calls(m):
    """The operator over a Marked request, for any marks; hints of every kind."""
    q = torch.zeros(m.new, m.QH, m.HD, dtype=BF, device="cuda")
    k = torch.randn(m.count, m.page, m.KVH, m.HD, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    rest = m.table.cuda(), starts([m.new]).cuda(), i32([m.length]).cuda()
    def call(marks):
        v = m.values(marks, "cuda")
        return [ops().paged_attention(q, k, v, *rest, max_rows=m.new, max_keys=x) for x in sorted({0, 1, m.length, KEYS[0]})]
    return call


def check_marked(m, call, kinds):
    for marks in kinds:
        want = m.shares(marks)[:, None]
        for got in call(marks):
            off = (got.cpu().double() - want).abs()
            bad = (off > want * m.TOLERANCE).nonzero()
            assert bad.numel() == 0, (bad[:4].tolist(), float(off.max()))


MARKED = LONG + [VERY_LONG, (300, 4500, 1, 1, 128, 16), (600, 900, 8, 2, 64, 32), (5, 33000, 2, 2, 128, 64), (260, 20000, 2, 1, 64, 128)]


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", MARKED)
def test_every_tile_counts_once(new, length, QH, KVH, HD, page, steered):
    say("tiles", new, length, HD)
    m = Marked(new, length, QH, KVH, HD, page, seed=length)
    check_marked(m, marked_calls(m), m.tiles())


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", MARKED + [(64, 64, 2, 1, 64, 16), (255, 255, 2, 2, 128, 16), (31, 63, 4, 1, 256, 32)])
def test_each_row_ends_with_its_own_key(new, length, QH, KVH, HD, page, steered):
    say("ends", new, length, HD)
    m = Marked(new, length, QH, KVH, HD, page, seed=length)
    check_marked(m, marked_calls(m), m.last_keys())


def far_apart(length):
    """Positions whose pages are taken away: the ends of splits, waves' and
    windows' tiles, and the last keys."""
    tiles = [0, 1, 7, 8, 31, 32, 33, 63, 64, 95, 96, 127, 128, 129, 255, 256, 383, 384, 512, 1094, 1100, 2200, 4000]
    return sorted({t * TILE + o for t in tiles for o in (0, 16) if t * TILE + o < length} | {length - 1, max(0, length - 40)})


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", MARKED)
def test_bad_pages_are_not_counted(new, length, QH, KVH, HD, page, steered):
    say("bad pages, marked", new, length, HD)
    m = Marked(new, length, QH, KVH, HD, page, seed=length + 1, bad=far_apart(length))
    check_marked(m, marked_calls(m), [*m.last_keys(), *list(m.tiles())[::8]])


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", MARKED)
def test_bad_pages_would_outweigh_the_rest(new, length, QH, KVH, HD, page, steered):
    """Every key scores -sqrt(head_dim) or less; a key of a bad page taken for
    zeros would score 0 and outweigh thousands. Values are ones: so are the
    results, or zeros where all pages seen are bad."""
    say("bad pages, low scores", new, length, HD)
    m = Marked(new, length, QH, KVH, HD, page, seed=length + 2, bad=far_apart(length))
    q = torch.ones(new, QH, HD, dtype=BF, device="cuda")
    k = torch.full((m.count, page, KVH, HD), -1.0, dtype=BF, device="cuda")
    v = torch.ones_like(k)
    any_seen = torch.stack([m.good[:length - new + i + 1].any() for i in range(new)]).double()
    for most in sorted({0, 1, length, KEYS[0]}):
        got = ops().paged_attention(q, k, v, m.table.cuda(), starts([new]).cuda(), i32([length]).cuda(), max_rows=new, max_keys=most)
        assert bool(((got.cpu().double() - any_seen[:, None, None]).abs() <= 2.0 ** -8 * any_seen[:, None, None]).all())

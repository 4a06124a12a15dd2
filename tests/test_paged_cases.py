"""What the device tests over paged_cases.py can see, by planting the mistake in
the reference: a lost tile, a lost split, a bad page that is counted, a row one
key off each move a result past its bound."""
import pytest

import paged_reference as ref
from paged_cases import LONG, SHAPES, TILE, VERY_LONG, Marked, random_case

torch = pytest.importorskip("torch")


def one_row(s, r, i):
    """Row i of request r as a request of its own."""
    b, e = int(s["row_start"][r]), int(s["row_start"][r + 1])
    length = int(s["lengths"][r]) - (e - b) + i + 1
    return dict(q=s["q"][b + i:b + i + 1], k=s["k"], v=s["v"], table=s["table"][r:r + 1].clone(), row_start=[0, 1],
                lengths=[length], scale=s["scale"])


def attend(s):
    return ref.attention(s["q"], s["k"], s["v"], s["table"], s["row_start"], s["lengths"], s["scale"])


@pytest.mark.parametrize("new,length,QH,KVH,HD,page", [c for c in LONG if c[1] <= 3000])
def test_a_lost_tile_shows(new, length, QH, KVH, HD, page):
    """In the random cases of up to 3000 keys; a tile's share shrinks with the
    keys, and the longer ones rest on the marked cases."""
    s = random_case(length, [new, 1], [length, 40], QH, KVH, HD, page, qstd=2.0)
    rows = [one_row(s, 0, i) for i in (0, new // 2, new - 1)]
    plain = [attend(row) for row in rows]
    tiles = rows[0]["lengths"][0] // TILE
    for t in sorted({0, 1, 7, 8, 31, 32, tiles // 2, 63, 64, tiles - 1} & set(range(tiles))):
        off = []
        for row, (want, tol) in zip(rows, plain):
            lost = dict(row, table=row["table"].clone())
            lost["table"][0, t * TILE // page:ref.ceil((t + 1) * TILE, page)] = -1
            off.append(float(((attend(lost)[0] - want).abs() / tol).max()))
        assert max(off) > 2, (t, off)


@pytest.mark.parametrize("case", SHAPES + [([n, 1], [x, 40], *rest) for n, x, *rest in LONG])
def test_no_key_outweighs_the_others(case):
    new, lengths, QH, KVH, HD, page = case
    s = random_case(sum(lengths) + HD, new, lengths, QH, KVH, HD, page, qstd=2.0 if max(lengths) > 2000 else 1.0)
    for r, n in enumerate(new):
        for i in {0, n - 1} if n else ():
            row = one_row(s, r, i)
            keys = row["lengths"][0]
            if keys < 64:
                continue
            j = torch.arange(keys)
            k = row["k"][row["table"][0, j // page].long(), j % page].double()
            for h in range(QH):
                p = torch.softmax(k[:, h // (QH // KVH)] @ row["q"][0, h].double() * row["scale"], 0)
                assert float(p.max()) < 0.5


@pytest.mark.parametrize("case", LONG + [VERY_LONG])
def test_marked_keys_show(case):
    new, length, QH, KVH, HD, page = case
    m = Marked(new, length, QH, KVH, HD, page, bad=[length // 2])
    j, last = torch.arange(length), length - new + torch.arange(new)
    seen = m.good & (j <= last[:, None])
    for marks in [next(iter(m.tiles())), *m.last_keys()]:
        want = m.shares(marks)
        assert float(want.max()) <= 1
        some = [t for t in (0, 1, 40, 4 * 40 + 3) if t * TILE < min(length, HD * TILE)]
        for what, other in [("tile %d" % t, seen & (j // TILE != t)) for t in some] + [
                ("one key more", m.good & (j <= last[:, None] + 1)), ("one less", m.good & (j < last[:, None]))]:
            got = m.shares(marks, other)
            off = (got - want).abs() > want * m.TOLERANCE
            tiled = int(marks[0]) == 0 and int((marks == 0).sum()) == TILE
            if what.startswith("tile"):
                assert not tiled or bool(off.any()), what
            elif not tiled and int(marks[-1]) == 0:  # the last keys
                # each row but the last gains the key behind its own; each loses its own
                rows = range(new - 1) if "more" in what else range(new)
                assert all(bool(off[i].any()) for i in rows if length - 1 - int(last[i]) < HD - 1), what

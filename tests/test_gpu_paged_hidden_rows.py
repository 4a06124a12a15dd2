"""Rows of paged attention that get zeros, beside values that are not finite:
rows that see no key because their request holds fewer tokens than it has rows,
and rows whose every score is -inf."""
import pytest

import test_gpu_paged as base
from test_gpu_paged import attention_case, check_attention, run_attention, say

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

steered = base.steered  # both kernels
NAN, INF = float("nan"), float("inf")


def rows_of(s, r, positions):
    """(pages, rows inside them) of a request's positions."""
    page = s["k"].shape[1]
    j = torch.as_tensor(positions)
    return s["table"][r, j // page].long().cuda(), (j % page).cuda()


@pytest.mark.parametrize("HD,QH,KVH", [(64, 8, 2), (128, 4, 1), (256, 8, 2), (256, 2, 2)])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_rows_that_see_nothing_beside_non_finite_values(HD, QH, KVH, value, steered):
    """More rows than tokens: the first rows see none of the keys that later
    rows of their tile see, whose values are not finite."""
    for new, length, gate in ((70, 30, False), (50, 45, True), (300, 270, True), (9, 2, False)):
        say("nothing seen beside", value, HD, new, length)
        s = attention_case(HD + new, [new, 3], [length, 40], QH, KVH, HD, 16, gate=gate)
        clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
        at = rows_of(s, 0, [length // 2, length - 1])
        s["v"][at] = value
        s["k"][at[0][1:], at[1][1:]] = NAN
        got = run_attention(s)
        hidden = new - length
        assert bool((got[:hidden] == 0).all())
        check_attention(clean, got, rows=list(range(hidden + length // 2)) + list(range(new, new + 3)))
        assert not bool(torch.isfinite(got[hidden + length // 2:new]).any())


@pytest.mark.parametrize("HD,QH,KVH,new,length,most", [
    (64, 8, 2, 3, 40, 0), (256, 8, 2, 60, 60, 0), (128, 4, 1, 300, 500, 0),
    (256, 4, 1, 40, 3000, 3000), (64, 2, 1, 1, 9000, 9000), (64, 1, 1, 300, 1200, 1200),  # split, and joined
])
@pytest.mark.parametrize("value", [NAN, INF])
def test_rows_whose_every_score_is_minus_infinity(HD, QH, KVH, new, length, most, value, steered):
    """Zeros whatever the values and the gate, joined or not; the other
    request's rows are what they are without it."""
    say("no score", HD, new, length, value)
    s = attention_case(HD + new, [new, 3], [length, 40], QH, KVH, HD, 16, gate=True)
    s["q"][:new, :, 0] = 1.0
    clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
    at = rows_of(s, 0, list(range(length)))
    k = s["k"][at]
    k[..., 0] = -INF
    s["k"][at] = k
    s["v"][rows_of(s, 0, [0, length // 3, length - 1])] = value
    s["gate"][:new:2] = value
    for hints in ({}, dict(max_rows=new, max_keys=most)) if most else ({},):
        got = run_attention(s, **hints)
        assert bool((got[:new] == 0).all())
        check_attention(clean, got, rows=slice(new, new + 3))


def test_first_keys_without_a_score(steered):
    """Only the rows that see nothing else get zeros; in the others a weight of
    0 meets what the value is, as in the formula."""
    HD, new, length, few = 128, 90, 90, 37
    s = attention_case(3, [new], [length], 4, 2, HD, 16)
    s["q"][:, :, 0] = 1.0
    at = rows_of(s, 0, list(range(few)))
    k = s["k"][at]
    k[..., 0] = -INF
    s["k"][at] = k
    v = s["v"][at]
    v[..., 5] = INF
    s["v"][at] = v
    got = run_attention(s)
    assert bool((got[:few] == 0).all()) and bool(torch.isnan(got[few:, :, 5]).all())
    rest = [c for c in range(HD) if c != 5]
    assert bool(torch.isfinite(got[few:][..., rest]).all())


def test_a_gate_that_is_not_finite(steered):
    """It reaches its own row alone, and not that of a row that sees no key."""
    HD, new, length = 64, 70, 60
    s = attention_case(5, [new], [length], 4, 2, HD, 16, gate=True)
    clean = dict(s, gate=s["gate"].clone())
    clean["gate"][65] = 0
    s["gate"][[3, 9, 65]] = NAN
    s["gate"][4], s["gate"][66] = INF, -INF
    clean["gate"][66], clean["gate"][4] = -INF, INF
    got = run_attention(s)
    assert bool((got[:10] == 0).all()) and bool(torch.isnan(got[65]).all()) and bool((got[66] == 0).all())
    clean["gate"][[3, 9]] = 0
    check_attention(clean, got, rows=[t for t in range(new) if t != 65])

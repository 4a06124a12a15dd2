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

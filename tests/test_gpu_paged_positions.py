"""Positions of several axes as callers hold them, and heads at the ends of the
number range, through cq35.paged_prepare."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import cache_tensors, check_prepare, i32, ops, prepare_case, say

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def call(s, k, v, T, **kw):
    qg, kv = s["qg"].cuda(), s["kv"].cuda()
    HD, KVH = kv.shape[2], kv.shape[1] // 2
    args = dict(positions=s["positions"].cuda(), pair_axis=s["axis"], slots=i32(np.arange(T)).cuda())
    args.update(kw)
    return ops().paged_prepare(qg[:, :, :HD], kv[:, :KVH], kv[:, KVH:], s["qw"].cuda(), s["kw"].cuda(), s["freq"].cuda(),
                               args.pop("positions"), args.pop("slots"), k, v, **args)


@pytest.mark.parametrize("kind", [np.int64, np.int32, np.uint8, "tensor", bytes, tuple])
def test_pair_axis_in_any_container(kind):
    say("pair_axis", kind)
    T, QH, KVH, HD = 9, 4, 2, 64
    s = prepare_case(4, T, QH, KVH, HD, 32, 3)
    k, v = cache_tensors(1, 16, KVH, HD)
    before = k.cpu().clone(), v.cpu().clone()
    axis = torch.tensor(s["axis"]) if kind == "tensor" else kind(s["axis"]) if kind in (bytes, tuple) else np.array(s["axis"], kind)
    check_prepare(s, call(s, k, v, T, pair_axis=axis), k, v, before, list(range(T)), 16)


@pytest.mark.parametrize("T,axes", [(1, 3), (2, 2), (33, 3), (700, 4)])
def test_one_row_of_positions_for_every_axis(T, axes):
    """Text beside images has one position on all axes: an expanded view of it
    gives what a copy for each axis gives."""
    say("expanded positions", T, axes)
    QH, KVH, HD = 4, 2, 128
    s = prepare_case(6, T, QH, KVH, HD, 64, axes)
    s["positions"] = s["positions"][:1].expand(axes, T).contiguous()
    page = ref.ceil(T, 16)
    k, v = cache_tensors(page, 16, KVH, HD)
    before = k.cpu().clone(), v.cpu().clone()
    out = call(s, k, v, T, positions=s["positions"][:1].cuda().expand(axes, T))
    check_prepare(s, out, k, v, before, list(range(T)), 16)


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("size", [1e30, -3e38])
def test_heads_whose_squares_pass_the_range(HD, size):
    """One channel's square passes F32: the head gives zeros, rotated or not;
    the other heads are what they are without it."""
    T, QH, KVH = 5, 4, 2
    s = prepare_case(11, T, QH, KVH, HD, 32, 1)
    huge = dict(s, qg=s["qg"].clone(), kv=s["kv"].clone())
    huge["qg"][1, 2, HD - 1] = size
    huge["qg"][4, 0, 3] = size
    huge["kv"][2, 1, 7] = size
    huge["kv"][3, KVH, 5] = size  # a value: copied as it is
    k, v = cache_tensors(1, 16, KVH, HD)
    say("huge heads", HD, size)
    out = call(huge, k, v, T, positions=s["positions"][0].cuda(), pair_axis=None).cpu()
    assert bool((out[1, 2] == 0).all()) and bool((out[4, 0] == 0).all()) and bool((k[0, 2, 1] == 0).all())
    assert torch.equal(v[0, :T].cpu(), huge["kv"][:, KVH:])
    k2, v2 = cache_tensors(1, 16, KVH, HD)
    plain = call(s, k2, v2, T, positions=s["positions"][0].cuda(), pair_axis=None).cpu()
    for t in range(T):
        for h in range(QH):
            assert (t, h) in ((1, 2), (4, 0)) or torch.equal(out[t, h], plain[t, h])
        for h in range(KVH):
            assert (t, h) == (2, 1) or torch.equal(k[0, t, h], k2[0, t, h])

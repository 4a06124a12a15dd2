"""Prompts whose matrix-core attention runs in one pass
(cq35_session_set_online_attention): within the gate of the reference's
matrix-core components against the exact path, single tokens' results and calls
without the component as they were, and the option's handling."""
import numpy as np
import pytest

import cq35
import cq35.config as cc
from cq35.model import Session

pytestmark = pytest.mark.gpu

ATT = Session.MATRIX_ATTENTION


def say(*a):
    print(*a, flush=True)


def f32(bits):
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32)


def rel_rms(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.sqrt(np.mean((a - b) ** 2) / np.mean(b ** 2)))


def prompts(cfg, sizes, seed=3):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, cfg["vocab"], n).tolist() for n in sizes]


@pytest.mark.parametrize("name", ["mini", "mini-moe"])
@pytest.mark.parametrize("sizes", [(300, 77), (2, 5, 40), (1100, 3), (33, 1500)])
def test_prompts_within_reference_gate(name, sizes):
    cfg = dict(cc.preset(name))
    say("one-pass attention", name, sizes)
    m = cq35.Model.synthetic(cfg, seed=5)
    exact, online = m.session(sum(sizes) + 7), m.session(sum(sizes) + 7)
    online.set_matrix_prefill(ATT)
    online.set_online_attention(True)
    for prompt in prompts(cfg, sizes):
        le, _ = exact.step_raw(prompt)
        lo, _ = online.step_raw(prompt)
        r = rel_rms(f32(lo), f32(le))
        say("  ", len(prompt), "rows: relative logit RMS %.4f" % r)
        assert np.all(np.isfinite(f32(lo))) and r <= 0.05
    r = rel_rms(f32(online.export_state(0)), f32(exact.export_state(0)))
    say("  state %.4f" % r)
    assert r <= 0.05


def test_differs_from_two_passes_by_rounding_alone():
    """The same prompt through both kernels: not the same bits (another order
    and rounding), within the gate of each other; off again, the two-pass
    kernel's bits."""
    cfg = dict(cc.preset("mini"))
    m = cq35.Model.synthetic(cfg, seed=6)
    prompt = prompts(cfg, [700])[0]
    out = {}
    for key, on in (("two", False), ("one", True), ("again", True), ("off", False)):
        s = m.session(800)
        s.set_matrix_prefill(ATT)
        s.set_online_attention(True)
        s.set_online_attention(on)
        out[key] = s.step_raw(prompt)[0]
    assert np.array_equal(out["two"], out["off"]) and np.array_equal(out["one"], out["again"])
    assert not np.array_equal(out["one"], out["two"])
    assert rel_rms(f32(out["one"]), f32(out["two"])) <= 0.05


def test_only_the_attention_component_is_affected():
    """Without CQ35_MATRIX_ATTENTION the option changes nothing, and single
    tokens after a prompt never."""
    cfg = dict(cc.preset("mini-moe"))
    m = cq35.Model.synthetic(cfg, seed=7)
    a, b = m.session(400), m.session(400)
    b.set_online_attention(True)
    prompt = prompts(cfg, [200])[0]
    (la, ta), (lb, tb) = a.step_raw(prompt), b.step_raw(prompt)
    assert ta == tb and np.array_equal(la, lb)
    for _ in range(3):
        (la, ta), (lb, tb) = a.step_raw([ta]), b.step_raw([tb])
        assert ta == tb and np.array_equal(la, lb)


def test_option_travels_and_is_checked():
    cfg = dict(cc.preset("mini"))
    m = cq35.Model.synthetic(cfg, seed=8)
    s = m.session(300)
    assert s.online_attention is False
    s.set_matrix_prefill(ATT)
    s.set_online_attention(True)
    assert s.online_attention is True
    first, second = prompts(cfg, [120, 50])
    s.step_raw(first)
    again = m.resume_checkpoint(s.into_checkpoint())
    assert again.online_attention is True
    other = m.session(300)
    other.set_matrix_prefill(ATT)
    other.set_online_attention(True)
    other.step_raw(first)
    assert np.array_equal(again.step_raw(second)[0], other.step_raw(second)[0])
    from cq35 import _lib
    assert _lib.load().cq35_session_set_online_attention(other._h, 2) == -1
    assert _lib.load().cq35_session_set_online_attention(None, 1) == -1


@pytest.mark.parametrize("held", [8900, 1500])
def test_long_context_chunk(held):
    """A chunk far into a context that is split over the device, and a long one
    (of the kernel for long chunks), with the other components: against the
    two-pass kernel."""
    cfg = dict(cc.preset("mini"))
    m = cq35.Model.synthetic(cfg, seed=9)
    ids = prompts(cfg, [9000])[0]
    out = []
    for on in (False, True):
        s = m.session(9100)
        s.set_matrix_prefill(ATT | Session.MATRIX_PROJECTIONS)
        s.set_online_attention(on)
        s.step_raw(ids[:held])
        out.append(f32(s.step_raw(ids[held:])[0]))
    r = rel_rms(out[1], out[0])
    say("long chunk: relative logit RMS %.4f" % r)
    assert r <= 0.05


@pytest.mark.parametrize("name,components,sizes", [("mini", ATT, [2065, 300]), ("mini", ATT | Session.MATRIX_PROJECTIONS, [40, 4100]),
                                                   ("mini-moe", ATT | Session.MATRIX_EXPERTS, [3, 2500])])
def test_chunk_rows_of_short_memory_change_no_bit(monkeypatch, name, components, sizes):
    """Chunks of 2048 rows and of 1024, as where memory is short: which of them
    a call gets follows from what else is allocated, its results must not. The
    layers behind the fourth, whose attention is compared, keep what every row
    of it left in their state."""
    cfg = dict(cc.preset(name), layers=8)
    m = cq35.Model.synthetic(cfg, seed=10)
    out = []
    for rows in (0, 1024):
        monkeypatch.setenv("CQ35_PREFILL_ROWS", str(rows))
        s = m.session(sum(sizes) + 5)
        s.set_matrix_prefill(components)
        s.set_online_attention(True)
        say("one-pass attention, chunk rows", name, rows)
        logits = [s.step_raw(p)[0] for p in prompts(cfg, sizes, seed=11)]
        out.append(logits + [s.export_state(0)])
    for a, b in zip(*out):
        assert np.array_equal(a, b)

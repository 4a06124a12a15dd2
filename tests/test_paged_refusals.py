"""The paged-cache operators on a machine without a GPU: every malformed
argument is refused before any device work, and the index arithmetic that the
kernels share with the host (paged_index.h) against a plain statement."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import paged_reference as ref
from cq35 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BASE = 1 << 20  # an address of the right alignment that is never read


def lib():
    return _lib.load()


def cache(**kw):
    c = dict(keys=BASE, values=2 * BASE, pages=10, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, row_stride=128,
             head_stride=64)
    c.update(kw)
    return _lib.PagedCache(*[c[n] for n, _ in _lib.PagedCache._fields_])


def heads(data=BASE, row=256, head=64):
    return _lib.Heads(data, row, head)


def refused(rc, code, text):
    assert rc == code, (rc, lib().cq35_last_error())
    assert text in lib().cq35_last_error().decode(), lib().cq35_last_error()


BAD_CACHES = [
    (dict(keys=None), -1, "null"), (dict(values=None), -1, "null"), (dict(head_dim=96), -4, "head_dim"),
    (dict(head_dim=0), -4, "head_dim"), (dict(kv_heads=0), -1, "heads"), (dict(kv_heads=-2), -1, "heads"),
    (dict(page_size=24), -4, "power of two"), (dict(page_size=8), -4, "power of two"), (dict(page_size=0), -4, "power of two"),
    (dict(page_size=1 << 17), -4, "power of two"), (dict(pages=0), -2, "pages"), (dict(pages=1 << 27), -2, "pages"),
    (dict(pages=-1), -2, "pages"), (dict(keys=BASE + 8), -1, "16-byte"), (dict(values=BASE + 2), -1, "16-byte"),
    (dict(row_stride=132), -1, "multiples of 8"), (dict(page_stride=-2048), -1, "multiples of 8"),
    (dict(row_stride=64), -1, "overlap"), (dict(row_stride=(1 << 26) + 8), -4, "apart"), (dict(page_stride=1024), -1, "overlap"), (dict(head_stride=32), -1, "overlap"),
    (dict(page_stride=0), -1, "overlap"), (dict(page_stride=1 << 62), -1, "overlap"),
]


def attention(c=None, q=None, gate=None, out=None, rows=3, q_heads=4, table=BASE, table_stride=5, requests=2, width=5,
              row_start=BASE, lengths=BASE, scale=0.125, max_rows=0, max_keys=0, workspace=BASE, size=1 << 40):
    c, q, out = c or cache(), q or heads(), out or heads()
    return lib().cq35_paged_attention(ctypes.byref(c), ctypes.byref(q), gate, ctypes.byref(out), rows, q_heads, table,
                                      table_stride, requests, width, row_start, lengths, scale, max_rows, max_keys,
                                      workspace, size, None)


@pytest.mark.parametrize("change,code,text", BAD_CACHES)
def test_cache_refusals(change, code, text):
    refused(attention(c=cache(**change)), code, text)
    refused(prepare(c=cache(**change)), code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(q_heads=3), -1, "query heads"), (dict(q_heads=0), -1, "query heads"), (dict(rows=-1), -2, "rows"),
    (dict(rows=1 << 31), -2, "rows"), (dict(requests=-1), -2, "requests"), (dict(requests=8193), -2, "requests"), (dict(rows=1 << 30), -2, "rows"),
    (dict(max_rows=-1), -2, "rows"),
    (dict(max_keys=-1), -2, "keys"), (dict(table=None), -1, "null"), (dict(row_start=None), -1, "null"),
    (dict(lengths=None), -1, "null"), (dict(width=0), -2, "tables"), (dict(width=1 << 28), -2, "tables"),
    (dict(width=(1 << 26) + 1), -2, "tables"), (dict(scale=3e38), -1, "scale"), (dict(rows=1 << 29, q_heads=2), -2, "rows"),
    (dict(table_stride=-1), -2, "tables"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
    (dict(q=heads(BASE + 4)), -1, "16-byte"), (dict(q=heads(None)), -1, "null"), (dict(q=heads(row=130)), -1, "multiples of 8"),
    (dict(q=heads(head=-64)), -1, "multiples of 8"), (dict(out=heads(row=128)), -1, "overlap"),
    (dict(out=heads(row=0)), -1, "overlap"), (dict(out=heads(head=0)), -1, "overlap"), (dict(out=heads(None)), -1, "null"),
    (dict(gate=ctypes.byref(heads(BASE + 6))), -1, "16-byte"),
])
def test_attention_refusals(change, code, text):
    refused(attention(**change), code, text)


def prepare(c=None, q=None, k=None, v=None, rows=3, q_heads=4, qw=BASE, kw=BASE, eps=1e-6, freq=BASE, rope=16, pos=BASE,
            stride=3, axes=1, pair_axis=None, slots=BASE, out=None):
    c, q, k, v, out = c or cache(), q or heads(), k or heads(), v or heads(), out or heads()
    return lib().cq35_paged_prepare(ctypes.byref(c), ctypes.byref(q), ctypes.byref(k), ctypes.byref(v), rows, q_heads, qw, kw,
                                    eps, freq, rope, pos, stride, axes, pair_axis, slots, ctypes.byref(out), None)


@pytest.mark.parametrize("change,code,text", [
    (dict(rows=-1), -2, "rows"), (dict(rows=(1 << 26) + 1), -2, "rows"), (dict(q_heads=5), -1, "query heads"), (dict(rope=8), -1, "rotary"), (dict(rope=24), -1, "rotary"),
    (dict(rope=80), -1, "rotary"), (dict(axes=0), -1, "axes"), (dict(axes=5), -1, "axes"), (dict(axes=3), -1, "each pair"),
    (dict(pair_axis=(ctypes.c_uint8 * 8)(0, 0, 0, 1)), -1, "pair 3"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(qw=None), -1, "null"), (dict(kw=None), -1, "null"), (dict(freq=None), -1, "null"), (dict(pos=None), -1, "null"),
    (dict(slots=None), -1, "null"), (dict(qw=BASE + 4), -1, "16-byte"), (dict(kw=BASE + 8), -1, "16-byte"),
    (dict(axes=2, stride=2, pair_axis=(ctypes.c_uint8 * 8)(0, 1)), -1, "axes overlap"), (dict(k=heads(BASE + 2)), -1, "16-byte"),
    (dict(v=heads(row=100)), -1, "multiples of 8"), (dict(out=heads(row=64)), -1, "overlap"),
])
def test_prepare_refusals(change, code, text):
    refused(prepare(**change), code, text)


@pytest.mark.parametrize("name", ["table", "cached", "lengths", "free_pages", "free_count", "row_start", "positions", "slots",
                                  "free_left", "status"])
def test_plan_refuses_null(name):
    refused(plan(**{name: None}), -1, "null")


def plan(table=BASE, stride=5, requests=2, width=5, cached=BASE, lengths=BASE, free_pages=BASE, pages=9, free_count=BASE,
         page=16, rows=7, row_start=BASE, positions=BASE, slots=BASE, free_left=BASE + 64, status=BASE):
    return lib().cq35_page_plan(table, stride, requests, width, cached, lengths, free_pages, pages, free_count, page, rows,
                                row_start, positions, slots, free_left, status, None)


@pytest.mark.parametrize("change,code,text", [
    (dict(requests=0), -2, "requests"), (dict(requests=8193), -2, "requests"), (dict(page=20), -4, "power of two"),
    (dict(pages=0), -2, "pages"), (dict(pages=1 << 27), -2, "pages"), (dict(width=0), -2, "tables"), (dict(rows=-1), -2, "rows"),
    (dict(rows=1 << 31), -2, "rows"), (dict(stride=4), -1, "overlap"), (dict(free_left=BASE), -1, "count left"),
])
def test_plan_refusals(change, code, text):
    refused(plan(**change), code, text)


def test_host_memory_is_refused():
    """Well-formed calls whose pointers are not device memory."""
    refused(attention(), -1, "not device memory")
    refused(prepare(), -1, "not device memory")
    refused(plan(), -1, "not device memory")


def test_empty_calls_do_nothing():
    assert attention(rows=0) == 0 and attention(requests=0) == 0 and prepare(rows=0) == 0


def test_python_refusals():
    """The torch binding refuses tensors of another type, place or shape."""
    torch = pytest.importorskip("torch")
    import cq35
    i = torch.zeros(2, dtype=torch.int32)
    q, c = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        cq35.paged_attention(q, c, c, i.view(1, 2), i, i[:1])
    with pytest.raises(ValueError, match="bfloat16"):
        cq35.paged_attention(q, c.float(), c, i.view(1, 2), i, i[:1])
    with pytest.raises(ValueError, match="dimensions"):
        cq35.page_plan(i, i, i, i, i, page_size=16, rows=1)
    with pytest.raises(TypeError, match="tensor"):
        cq35.page_plan([[0]], i, i, i, i, page_size=16, rows=1)
    assert cq35.PLAN_STATUS[0] == "ok"
    with pytest.raises(AttributeError):
        cq35.no_such_operator


SOURCE = r"""
#include "paged_index.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace cq35;
int main(int argc, char** argv) {
  // needs: cached length width shift ...; verdicts; requests of rows; slots
  char what;
  while (scanf(" %c", &what) == 1) {
    long long a, b, c, d, e, f, g;
    if (what == 'n') {
      scanf("%lld %lld %lld %lld", &a, &b, &c, &d);
      const PlanNeed n = plan_need(a, b, c, (int)d);
      printf("%lld %lld %lld %d\n", (long long)n.rows, (long long)n.take, (long long)n.give, (int)n.bad);
    } else if (what == 'v') {
      scanf("%lld %lld %lld %lld %lld %lld %lld", &a, &b, &c, &d, &e, &f, &g);
      const PlanVerdict v = plan_verdict(a != 0, b, c, d, e, f, g);
      printf("%d %lld\n", (int)v.code, (long long)v.missing);
    } else if (what == 's') {
      scanf("%lld %lld %lld %lld", &a, &b, &c, &d);
      printf("%d\n", (int)slot_of((int32_t)a, b, c, (int)d));
    } else if (what == 'c') {  // the cut of a launch: every (packed row, key tile) once, slots apart and within the bound
      CutRule c{};
      long long R;
      scanf("%d %d %d %d %d %d %d %d %d", &c.rows, &c.most_keys, &c.group, &c.kv_heads, &c.tile_rows, &c.target_shift,
             &c.min_tiles, &c.max_splits, &c.search);
      scanf("%lld", &R);
      std::vector<int32_t> start(R + 1), length(R);
      for (auto& x : start) scanf("%d", &x);
      for (auto& x : length) scanf("%d", &x);
      const int64_t tiles = most_tiles(c.rows, R, c.group, c.tile_rows);
      const int64_t items_bound = most_items(tiles, c.kv_heads, c.target_shift, c.max_splits) / c.kv_heads;
      c.slots = most_slots(tiles, c.kv_heads, c.target_shift, c.max_splits);
      int64_t pairs = 0, items = 0, parts = 0, tile_count = 0;
      for (long long r = 0; r < R; ++r) {
        const CutRequest q = cut_request(c, start[r], start[r + 1], length[r]);
        pairs += request_work(c, q);
      }
      const int32_t chunk = cut_chunk(c, pairs, [&](int32_t x) {
        int64_t n = 0;
        for (long long r = 0; r < R; ++r) {
          const CutRequest q = cut_request(c, start[r], start[r + 1], length[r]);
          n += (int64_t)q.tiles * cut_splits(c, q, x);
        }
        return n;
      });
      for (long long r = 0; r < R; ++r) {
        const CutRequest q = cut_request(c, start[r], start[r + 1], length[r]);
        const int32_t n = cut_splits(c, q, chunk), each = split_tiles(q, n);
        tile_count += q.tiles;
        int64_t covered = 0, want = 0;
        for (int32_t i = 0; i < q.tiles; ++i) {
          const int32_t seen = key_tiles_of(tile_keys(c, q, i));
          want += seen;
          for (int32_t s = 0; s < n; ++s) {
            const int32_t t0 = s * each, t1 = t0 + each < seen ? t0 + each : seen;
            if (t1 > t0) covered += t1 - t0;
          }
          if (seen > each && n == 1) return 2;  // parts without a slot
        }
        if (covered != want || (int64_t)n * each < q.key_tiles) return 3;
        items += (int64_t)q.tiles * n;
        parts += n > 1 ? (int64_t)q.tiles * n : 0;
      }
      if (tile_count > tiles) return 4;
      if (items > items_bound) return 5;
      if (parts * c.kv_heads > c.slots) return 6;
      printf("%lld %lld\n", (long long)items, (long long)parts);
    } else {
      scanf("%lld %lld", &a, &b);
      int32_t* s = (int32_t*)malloc(sizeof(int32_t) * a);
      for (long long i = 0; i < a; ++i) scanf("%d", &s[i]);
      printf("%d\n", request_of(s, (int)a, b));
      free(s);
    }
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def index_program(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_index")
    src, exe = d / "index.cpp", d / "index"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined,address", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "catena-models_amd", "csrc"), "-o", str(exe), str(src)], check=True)
    return str(exe)


def ask(exe, lines):
    p = subprocess.run([exe], input="\n".join(lines), capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stderr
    return [[int(x) for x in line.split()] for line in p.stdout.splitlines()]


def test_plan_arithmetic(index_program):
    cases = [(c, x, w, s) for c in (-1, 0, 1, 15, 16, 17, 31, 32, 1000) for x in (-5, 0, 1, 16, 17, 999, 2**31 - 1)
             for w, s in ((1, 4), (3, 4), (100, 4), (1 << 27, 4), (4, 8))]
    got = ask(index_program, ["n %d %d %d %d" % c for c in cases])
    for (c, x, w, s), g in zip(cases, got):
        h, t = ref.ceil(max(c, 0), 1 << s), ref.ceil(max(x, 0), 1 << s)
        bad = c < 0 or x < 0 or h > w or t > w
        assert g == ([0, 0, 0, 1] if bad else [max(x - c, 0), max(t - h, 0), max(h - t, 0), 0]), (c, x, w, s)


def test_plan_verdicts(index_program):
    # bad, free, pages, rows_total, take, give, rows -> code, missing
    cases = [((1, 5, 9, 0, 0, 0, 9), [3, 0]), ((0, -1, 9, 0, 0, 0, 9), [4, 0]), ((0, 5, 9, 0, 0, 5, 9), [4, 0]),
             ((0, 5, 9, 10, 0, 0, 9), [2, 1]), ((0, 5, 9, 3, 8, 2, 9), [1, 1]), ((0, 5, 9, 3, 7, 2, 9), [0, 0]),
             ((0, 0, 9, 0, 0, 0, 0), [0, 0])]
    assert ask(index_program, ["v " + " ".join(map(str, c)) for c, _ in cases]) == [w for _, w in cases]


def test_slots_of_bad_pages(index_program):
    cases = [(3, 10, 37, 4), (0, 10, 0, 4), (9, 10, 15, 4), (10, 10, 0, 4), (-1, 10, 5, 4), (2**31 - 1, 10, 5, 4),
             (-2**31, 10, 5, 4), (2**15 - 1, 2**15 - 1, 2**16 - 1, 16)]
    got = ask(index_program, ["s %d %d %d %d" % c for c in cases])
    assert [g[0] for g in got] == [(p << s) + (x & ((1 << s) - 1)) if 0 <= p < n else -1 for p, n, x, s in cases]


def test_request_of_row(index_program):
    rng = np.random.default_rng(1)
    lines, want = [], []
    for _ in range(200):
        new = rng.integers(0, 4, rng.integers(1, 20))
        starts = np.concatenate([[0], np.cumsum(new)[:-1]])
        for t in range(int(new.sum())):
            lines.append("r %d %d %s" % (len(starts), t, " ".join(map(str, starts))))
            want.append([int(np.searchsorted(np.cumsum(new), t, side="right"))])
    assert ask(index_program, lines) == want


def test_cut_covers_every_tile_once(index_program):
    """Any lengths: each row tile's key tiles are dealt to its splits once, and
    items and partial results stay within the bounds that size the launch and
    the workspace (checked in the program)."""
    rng = np.random.default_rng(3)
    lines = []
    for i in range(400):
        R = int(rng.choice([1, 2, 5, 40, 300]))
        group, kvh = int(rng.choice([1, 3, 8, 12])), int(rng.choice([1, 2, 8]))
        new = rng.integers(0, int(rng.choice([2, 9, 600])), R)
        length = new + rng.integers(0, int(rng.choice([1, 50, 40000])), R)
        if i % 7 == 0:
            length = rng.integers(-5, 100, R)  # rows that see nothing among them
        rows = int(new.sum()) + int(rng.integers(0, 4)) - (i % 5 == 0)
        if rows < 1:
            continue
        tile_rows = int(rng.choice([32, 256]))
        lines.append("c %d %d %d %d %d %d %d %d %d %d %s %s" % (
            rows, 1 << 16, group, kvh, tile_rows, int(rng.choice([0, 5, 9, 10])), int(rng.choice([1, 4, 16])),
            int(rng.choice([1, 2, 7, 1024])), int(R <= 64 and i % 2), R, " ".join(map(str, np.concatenate([[0], np.cumsum(new)]))),
            " ".join(map(str, length))))
    assert len(ask(index_program, lines)) == len(lines) > 300


@pytest.mark.parametrize("kind", ["list", "tuple", "bytes", "int64", "int32", "uint8", "tensor", "range"])
def test_pair_axis_in_any_container(kind):
    """The axes of the pairs as a user may hold them: their values count, not
    the bytes that hold them."""
    torch = pytest.importorskip("torch")
    from cq35 import paged
    want = [0, 1, 2, 1, 0, 2, 2, 1] if kind != "range" else [0, 1, 2]
    given = {"list": list, "tuple": tuple, "bytes": bytes, "int64": lambda x: np.array(x, np.int64),
             "int32": lambda x: np.array(x, np.int32), "uint8": lambda x: np.array(x, np.uint8), "tensor": torch.tensor,
             "range": lambda x: range(3)}[kind](want)
    assert list(paged._pair_axis(given, len(want), 3)) == want
    for bad, pairs, axes in ((given, len(want), 2), (given, len(want) + 1, 3), (given, 0, 3)):
        with pytest.raises(ValueError, match="pair_axis"):
            paged._pair_axis(bad, pairs, axes)


def test_pair_axis_refusals():
    pytest.importorskip("torch")
    from cq35 import paged
    for bad in ([0, -1], [0, 256], [0, 2**40], [0, 2**80], [0.0, 1.0], np.array([0.0, 1.0]), "01", [None, 0], 3):
        with pytest.raises((ValueError, TypeError), match="pair_axis"):
            paged._pair_axis(bad, 2, 2)


def test_positions_repeated_on_every_axis_are_no_overlap():
    refused(prepare(axes=2, stride=0, pair_axis=(ctypes.c_uint8 * 8)(0, 1)), -1, "not device memory")
    for stride in (1, 2, -3):
        refused(prepare(axes=2, stride=stride, pair_axis=(ctypes.c_uint8 * 8)(0, 1)), -1, "axes overlap")


def test_numbers_past_32_bits_are_refused():
    """Not taken modulo 2^32: a page size of 2^32 + 16 is not one of 16."""
    torch = pytest.importorskip("torch")
    import cq35
    i = torch.zeros(2, dtype=torch.int32)
    for x in (2**32 + 16, -2**32 + 16, 2**64 + 16):
        with pytest.raises(ValueError, match="page_size"):
            cq35.page_plan(i.view(1, 2), i[:1], i[:1], i, i[:1], page_size=x, rows=1)
    with pytest.raises(TypeError):
        cq35.page_plan(i.view(1, 2), i[:1], i[:1], i, i[:1], page_size=16.5, rows=1)
    for at, name in ((2, "q_heads"), (3, "kv_heads"), (4, "head_dim")):
        sizes = [40, 2, 8, 2, 256]
        sizes[at] += 2**32
        with pytest.raises(ValueError, match=name):
            cq35.paged_attention_workspace(*sizes)
    assert cq35.paged_attention_workspace(40, 2, 8, 2, 256, 40, 3000) > 0


def test_star_import_with_and_without_torch():
    """The package's public names come without torch too, the operators' then aside."""
    import sys
    path = os.path.join(ROOT, "catena-models_amd")
    for hide in ("", "sys.modules['torch'] = None; "):
        code = ("import sys; sys.path.insert(0, %r); %sfrom cq35 import *; import cq35; assert Model is cq35.Model; "
                "assert ('page_plan' in globals()) is %s; assert hasattr(cq35, '__all__') and 'page_plan' in dir(cq35)"
                % (path, hide, not hide))
        p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
        assert p.returncode == 0, p.stderr

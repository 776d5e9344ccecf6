"""What the paged cache refuses, and its host arithmetic: no GPU needed."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from nanokv_b200 import _lib, ops
from nanokv_b200.page_cache import PageCache, PageTable

SOURCES = Path(__file__).resolve().parent.parent / "nanokv_b200" / "csrc"


def struct(*, batch=2, row_pages=4, pages=8, page=64, kv_heads=2, head_dim=128, dtype=_lib.NKV_BF16, address=256, v=512):
    return _lib.PageCache(address, v, 256, 256, batch, row_pages, pages, page, kv_heads, head_dim, dtype)


def rows(heads, address=256):
    return _lib.Tokens(address, 1024, 512, 128, heads)


def status_of(name, *args):
    lib = _lib.library()
    return getattr(lib, name)(*args), lib.nkv_last_error().decode()


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=96), "head width"), (dict(dtype=_lib.NKV_F32), "bf16 or fp16"), (dict(pages=0), "pages"), (dict(page=48), "48 tokens"),
    (dict(page=256), "256 tokens"), (dict(kv_heads=0), "kv_heads"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"),
    (dict(address=264), "aligned"), (dict(address=None), "missing"), (dict(pages=2 ** 24, kv_heads=64), "pages"),
    (dict(row_pages=2 ** 25), "entries"), (dict(row_pages=0), "entries")])
def test_caches_that_are_refused(change, word):
    caches = (_lib.PageCache * 1)(struct(**change))
    for name, args in (("nkv_page_append", (struct(**change), rows(2), rows(2), None, None, 1, None, None, 256, None)),
                       ("nkv_page_attend", (struct(**change), rows(2), 1, None, None, 0, 1, 1.0, 256, 256, 256, None, 0, None)),
                       ("nkv_page_keep", (caches, 1, 256, 1, None, 256, None))):
        status, text = status_of(name, *args)
        assert status in (_lib.NKV_ERR_INVALID, _lib.NKV_ERR_UNSUPPORTED) and word in text, (name, text)


def test_calls_that_are_refused():
    turn = _lib.Rotation(256, 256, 8, 32, 0)
    two = (_lib.PageCache * 2)(struct(), struct(address=1024))          # values of both in one place
    other = (_lib.PageCache * 2)(struct(), struct(address=1024, v=2048, kv_heads=4))
    for name, args, word in (
            ("nkv_page_append", (struct(), rows(1), rows(2), None, None, 1, None, None, 256, None), "heads"),
            ("nkv_page_append", (struct(), rows(2), rows(2), None, None, -1, None, None, 256, None), "tokens"),
            ("nkv_page_append", (struct(), rows(2, None), rows(2), None, None, 1, None, None, 256, None), "missing"),
            ("nkv_page_append", (struct(), rows(2), rows(2), None, None, 1, None, None, None, None), "missing"),
            ("nkv_page_append", (struct(), rows(2), rows(2), rows(4), 256, 1, None, None, 256, None), "without a rotation"),
            ("nkv_page_append", (struct(), rows(2), rows(2), rows(4), 264, 1, None, turn, 256, None), "aligned"),
            ("nkv_page_append", (struct(), rows(2), rows(2), rows(4), None, 1, None, turn, 256, None), "missing"),
            ("nkv_page_append", (struct(), rows(2), rows(2), None, None, 1, None, _lib.Rotation(256, None, 8, 24, 0), 256, None), "multiple of 16"),
            ("nkv_page_append", (struct(), rows(2), rows(2), None, None, 1, None, _lib.Rotation(256, 256, 8, 256, 0), 256, None), "rotary_dim"),
            ("nkv_page_append", (struct(), rows(2), rows(2), None, None, 1, None, _lib.Rotation(None, 256, 8, 32, 0), 256, None), "arrays"),
            ("nkv_page_attend", (struct(), rows(3), 1, None, None, 0, 1, 1.0, 256, 256, 256, None, 0, None), "3 query heads"),
            ("nkv_page_attend", (struct(), rows(2), -1, None, None, 0, 1, 1.0, 256, 256, 256, None, 0, None), "tokens"),
            ("nkv_page_attend", (struct(), rows(2), 2 ** 29, None, None, 0, 1, 1.0, 256, 256, 256, None, 0, None), "tokens"),
            ("nkv_page_attend", (struct(), rows(2), 1, None, None, 0, 1, 1.0, 256, None, 256, None, 0, None), "missing"),
            ("nkv_page_attend", (struct(), rows(2), 1, None, None, 0, 1, 1.0, 264, 256, 256, None, 0, None), "aligned"),
            ("nkv_page_attend", (struct(), rows(2), 33, None, 256, 65, 1, 1.0, 256, 256, 256, None, 0, None), "masks of 66 words"),
            ("nkv_page_attend", (struct(), rows(2), 1, None, None, 0, 1, float("nan"), 256, 256, 256, None, 0, None), "finite"),
            ("nkv_page_keep", (two, 2, 256, 1, None, 256, None), "are one"),
            ("nkv_page_keep", (other, 2, 256, 1, None, 256, None), "share"),
            ("nkv_page_keep", (two, 1, None, 1, None, 256, None), "missing"),
            ("nkv_page_keep", (two, 1, 256, -1, None, 256, None), "tokens"),
            ("nkv_tree_mask", (256, 1, 4097, 256, 256, 256, None), "tokens=4097"),
            ("nkv_tree_mask", (None, 1, 4, 256, 256, 256, None), "missing")):
        status, text = status_of(name, *args)
        assert status in (_lib.NKV_ERR_INVALID, _lib.NKV_ERR_TOO_LARGE) and word in text, (name, text)
        with pytest.raises(ValueError):
            _lib.check(status)


def test_calls_without_work_do_nothing():
    assert status_of("nkv_page_append", struct(), rows(2), rows(2), None, None, 0, None, None, 256, None)[0] == 0
    assert status_of("nkv_page_attend", struct(batch=0), rows(2), 4, None, None, 0, 1, 1.0, None, None, None, None, 0, None)[0] == 0
    assert status_of("nkv_page_keep", None, 0, None, 4, None, None, None)[0] == 0
    assert status_of("nkv_tree_mask", None, 0, 4, None, None, None, None)[0] == 0


def test_there_is_no_cpu_path():
    table, lengths = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        PageTable.over(table, lengths, pages=8, page=64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.tree_mask(torch.zeros(4, dtype=torch.int32))


@pytest.mark.parametrize("args,word", [((0, 64), "positive"), ((1, 0), "positive")])
def test_tables_that_are_refused(args, word):
    with pytest.raises(ValueError, match=word):
        PageTable(*args, pages=4)
    with pytest.raises(ValueError, match="48"):
        PageTable(1, 64, pages=4, page=48)
    for table, lengths in ((torch.zeros(2, 4), torch.zeros(2, dtype=torch.int32)), (torch.zeros(2, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)),
                           (torch.zeros(2, 0, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="int32"):
            PageTable.over(table, lengths, pages=8, page=64)


# ------------------------------------------------------------------ pages dealt out, on a table of the host's
class HostTable(PageTable):
    """The host's part of a table: the arrays lie in host memory."""

    def __init__(self, batch, capacity, pages, page):
        self.table = torch.full((batch, -(-capacity // page)), -1, dtype=torch.int32)
        self.lengths = torch.zeros(batch, dtype=torch.int32)
        self.batch, self.pages, self.page, self.device = batch, pages, page, torch.device("cpu")
        self._held, self._free = [[] for _ in range(batch)], list(range(pages - 1, -1, -1))


@pytest.fixture
def on_host(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)


def test_pages_are_dealt_out_and_given_back(on_host):
    table = HostTable(3, 100, 10, 16)
    table.reserve([1, 16, 17])
    assert table.free == 6
    held = table.table.clone()
    assert [(row >= 0).sum().item() for row in held] == [1, 1, 2]
    assert len(set(held[held >= 0].tolist())) == 4
    table.reserve([0, 33, 5])                       # what is held stays
    assert table.free == 4 and torch.equal(table.table[2], held[2]) and table.table[1, 0] == held[1, 0]
    with pytest.raises(RuntimeError, match="are free"):
        table.reserve([100, 0, 0])
    assert table.free == 4
    table.lengths[1] = 30
    table.release(1)
    assert table.free == 7 and table.lengths[1] == 0 and (table.table[1] == -1).all()
    table.reserve([100, 0, 0])
    rows = table.table[table.table >= 0].tolist()
    assert len(rows) == len(set(rows)) == 9


@pytest.mark.parametrize("tokens,error", [([1, 2], ValueError), ([-1, 0, 0], ValueError), ([113, 0, 0], ValueError), ([1.5, 0, 0], TypeError)])
def test_reservations_that_are_refused(on_host, tokens, error):
    table = HostTable(3, 100, 10, 16)
    with pytest.raises(error):
        table.reserve(tokens)
    assert table.free == 10 and (table.table == -1).all()


def test_tables_over_arrays_deal_out_nothing():
    table = HostTable(3, 100, 10, 16)
    table._free = table._held = None
    for call in (lambda: table.free, lambda: table.reserve([1, 1, 1]), lambda: table.release(0)):
        with pytest.raises(RuntimeError, match="dealt out by the caller"):
            call()
    with pytest.raises(ValueError, match="sequences 0"):
        HostTable(3, 100, 10, 16).release(3)


@pytest.mark.parametrize("shape,dtype,word", [((10, 2, 32, 64), torch.bfloat16, "k_pages"), ((9, 2, 16, 64), torch.bfloat16, "k_pages"),
                                              ((10, 2, 16, 96), torch.bfloat16, "wide"), ((10, 2, 16, 64), torch.float32, "bf16 or fp16")])
def test_pages_that_are_refused(shape, dtype, word):
    with pytest.raises(ValueError, match=word):
        PageCache.over(HostTable(3, 100, 10, 16), torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype))


def test_values_that_are_not_as_the_keys():
    k = torch.zeros(10, 2, 16, 64, dtype=torch.bfloat16)
    for v in (k.half(), k[:, :1], k.transpose(0, 1)):
        with pytest.raises(ValueError, match="v_pages"):
            PageCache.over(HostTable(3, 100, 10, 16), k, v)


# ------------------------------------------------------------------ what kernels take from memory, and how work is dealt out
PROGRAM = """
#include "nkv_page_plan.h"
#include <vector>
using namespace nkv::page;
extern "C" int extent(int length, int count, int tokens, int room, int* out) {
  bool bad; const Extent e = extent_in(length, count, tokens, room, bad);
  out[0] = e.length; out[1] = e.count; out[2] = e.there; return bad;
}
extern "C" uint32_t sight(int kind, int length, int there, int count, int t, int first, const uint32_t* words, int n) {
  return sight_bits(kind, Extent{length, count, there}, t, first, [&](int w) { return w >= 0 && w < n ? words[w] : 0u; });
}
extern "C" int before(int kind, int length, int there, int count, int t) { return sees_all_before(kind, Extent{length, count, there}, t); }
// pieces as [run, b, h, unit, tile0, nt, whole]; the number of them
extern "C" int pieces(int kind, int group, int tokens, int unit, int heads, int n, const int* lengths, const int* counts, int runs, int* out) {
  const int rows = group * tokens;
  const Shape s{kind, group, rows, unit, (rows + unit - 1) / unit, heads};
  std::vector<Extent> e; std::vector<uint32_t> start(1, 0);
  for (int b = 0; b < n; ++b) {
    bool bad; e.push_back(extent_in(lengths[b], counts[b], tokens, 1 << 30, bad));
    uint32_t cost = 0;
    for (int u = 0; u < s.units; ++u) cost += cost_of(tiles_seen(s, e[b], u * unit, unit));
    start.push_back(start.back() + cost * heads);
  }
  Plan p{start.data(), e.data(), n, 0, 0};
  p.deal(runs);
  int found = 0;
  for (int r = 0; r < runs; ++r) {
    Walk w(p, s, r);
    Piece piece;
    while (w.next(p, s, piece)) {
      int* const at = out + 7 * found++;
      at[0] = r; at[1] = piece.b; at[2] = piece.h; at[3] = piece.unit; at[4] = piece.tile0; at[5] = piece.nt; at[6] = piece.whole;
    }
  }
  return found;
}
// the same pieces by the tours of `blocks` thread blocks, `rounds` runs each
extern "C" int toured(int kind, int group, int tokens, int unit, int heads, int n, const int* lengths, const int* counts, int blocks, int rounds, int* out) {
  const int rows = group * tokens;
  const Shape s{kind, group, rows, unit, (rows + unit - 1) / unit, heads};
  std::vector<Extent> e; std::vector<uint32_t> start(1, 0);
  for (int b = 0; b < n; ++b) {
    bool bad; e.push_back(extent_in(lengths[b], counts[b], tokens, 1 << 30, bad));
    uint32_t cost = 0;
    for (int u = 0; u < s.units; ++u) cost += cost_of(tiles_seen(s, e[b], u * unit, unit));
    start.push_back(start.back() + cost * heads);
  }
  Plan p{start.data(), e.data(), n, 0, 0};
  p.deal(blocks * rounds);
  int found = 0;
  for (int block = 0; block < blocks; ++block) {
    Tour t(p, s, block, blocks, rounds);
    Piece piece;
    while (t.next(p, s, piece)) {
      int* const at = out + 8 * found++;
      at[0] = t.run; at[1] = piece.b; at[2] = piece.h; at[3] = piece.unit; at[4] = piece.tile0; at[5] = piece.nt; at[6] = piece.whole;
      at[7] = t.last_run(p);
    }
  }
  return found;
}
extern "C" int rounds(uint64_t bytes, uint32_t places, int blocks, int least, int most) { return rounds_of(bytes, places, blocks, least, most); }
extern "C" int tiles(int kind, int group, int tokens, int unit, int length, int count, int u) {
  bool bad; const Extent e = extent_in(length, count, tokens, 1 << 30, bad);
  const int rows = group * tokens;
  return tiles_seen(Shape{kind, group, rows, unit, (rows + unit - 1) / unit, 1}, e, u * unit, unit);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{SOURCES}", "-o", str(folder / "plan.so"),
                    str(folder / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(folder / "plan.so"))
    lib.sight.restype = ctypes.c_uint32
    return lib


@pytest.mark.parametrize("length", [-2 ** 31, -1, 0, 5, 63, 64, 65, 2 ** 31 - 1])
@pytest.mark.parametrize("count", [-2 ** 31, -1, 0, 1, 4, 5, 2 ** 31 - 1])
def test_extents_stay_within_the_table(plan, length, count):
    out = (ctypes.c_int * 3)()
    bad = plan.extent(length, count, 4, 64, out)
    n, c, there = out
    assert 0 <= n <= 64 and 0 <= c <= 4 and 0 <= there <= c and n + there <= 64
    assert bad == (not (0 <= length <= 64 and 0 <= count <= 4 and length + count <= 64))
    if not bad:
        assert [n, c, there] == [length, count, count]


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_sight_bits_token_by_token(plan, kind):
    import random
    rng = random.Random(kind)
    for _ in range(400):
        tokens = rng.choice([1, 5, 31, 32, 33, 64, 70])
        length, count = rng.choice([0, 1, 31, 32, 100]), rng.randint(1, tokens)
        there, t = rng.randint(0, count), rng.randrange(count)
        mask = rng.getrandbits(tokens)
        n = -(-tokens // 32)
        words = (ctypes.c_uint32 * n)(*[(mask >> 32 * w) & 0xFFFFFFFF for w in range(n)])
        first = rng.randint(0, length + count + 40)
        got = plan.sight(kind, length, there, count, t, first, words, n)
        for i in range(32):
            j = first + i - length
            pending = 0 <= j < there and (kind == 0 or (kind == 1 and j <= t) or (kind == 2 and mask >> j & 1))
            assert (got >> i & 1) == (j < 0 or pending), (length, there, t, first, i)
        clear = plan.before(kind, length, there, count, t)
        assert all(plan.sight(kind, length, there, count, t, x, words, n) & 1 for x in range(max(0, clear - 3), clear))


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("unit", [128, 256])
def test_pieces_cover_every_tile_once(plan, kind, unit):
    import random
    rng = random.Random(unit + kind)
    for _ in range(60):
        n, heads, runs = rng.randint(1, 9), rng.randint(1, 4), rng.choice([1, 2, 7, 148])
        group = rng.choice([1, 3, 8])
        tokens = rng.randint(1, 128 // group) if unit == 128 else rng.randint(129 // group + 1, 1000)
        lengths = [rng.choice([0, 0, 1, 127, 128, 129, 1000, 5000]) for _ in range(n)]
        counts = [rng.choice([0, 1, tokens, tokens, rng.randint(0, tokens)]) for _ in range(n)]
        out = (ctypes.c_int * 70000)()
        array = ctypes.c_int * n
        found = plan.pieces(kind, group, tokens, unit, heads, n, array(*lengths), array(*counts), runs, out)
        assert found < 10000
        seen, places = {}, set()
        for i in range(found):
            run, b, h, u, tile0, nt, whole = out[7 * i:7 * i + 7]
            assert nt > 0 and tile0 >= 0
            for t in range(tile0, tile0 + nt):
                assert (b, h, u, t) not in seen
                seen[b, h, u, t] = run
            if not whole:      # two places a run: a piece that starts with its unit, and one that does not
                assert (run, tile0 == 0) not in places
                places.add((run, tile0 == 0))
        units = -(-group * tokens // unit)
        want = {(b, h, u, t) for b in range(n) for h in range(heads) for u in range(units)
                for t in range(plan.tiles(kind, group, tokens, unit, lengths[b], counts[b], u))}
        assert set(seen) == want


def test_counts_that_advance(on_host):
    table = HostTable(2, 64, 8, 16)
    table.advance(3)
    table.advance(torch.tensor([1, 0], dtype=torch.int32))
    assert table.lengths.tolist() == [4, 3]
    for counts in (-1, torch.tensor([1, 0]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(ValueError, match="counts"):
            table.advance(counts)
    with pytest.raises(TypeError):
        table.advance(1.5)
    assert table.lengths.tolist() == [4, 3]


@pytest.mark.parametrize("rounds", [1, 2, 3])
def test_tours_have_the_pieces_of_all_runs(plan, rounds):
    import random
    rng = random.Random(rounds)
    for _ in range(40):
        n, heads, blocks, group = rng.randint(1, 5), rng.randint(1, 4), rng.choice([1, 3, 20]), rng.choice([1, 3])
        tokens = rng.randint(200, 900)
        lengths = [rng.choice([0, 1, 128, 1000, 5000]) for _ in range(n)]
        counts = [rng.choice([0, 1, tokens, tokens]) for _ in range(n)]
        array = ctypes.c_int * n
        runs, tours = (ctypes.c_int * 70000)(), (ctypes.c_int * 70000)()
        a = plan.pieces(1, group, tokens, 256, heads, n, array(*lengths), array(*counts), blocks * rounds, runs)
        b = plan.toured(1, group, tokens, 256, heads, n, array(*lengths), array(*counts), blocks, rounds, tours)
        pieces = [tuple(runs[7 * i:7 * i + 7]) for i in range(a)]
        toured = [tuple(tours[8 * i:8 * i + 7]) for i in range(b)]
        assert sorted(pieces) == sorted(toured)
        by_unit = {}
        for run, sequence, h, u, *_ in pieces:
            by_unit.setdefault((sequence, h, u), []).append(run)
        for i in range(b):
            run, sequence, h, u, tile0, nt, whole, last = tours[8 * i:8 * i + 8]
            assert last == max(by_unit[sequence, h, u]) and by_unit[sequence, h, u] == list(range(min(by_unit[sequence, h, u]), last + 1))


def test_rounds_are_as_few_as_fit(plan):
    plan.rounds.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    fits = 64 << 20
    assert plan.rounds(fits, 10 ** 6, 148, 64, 3) == 1 and plan.rounds(fits + 1, 10 ** 6, 148, 64, 3) == 2
    assert plan.rounds(100 * fits, 10 ** 6, 148, 64, 3) == 3 and plan.rounds(100 * fits, 10 ** 6, 148, 64, 1) == 1
    assert plan.rounds(100 * fits, 148 * 127, 148, 64, 3) == 1 and plan.rounds(100 * fits, 148 * 128, 148, 64, 3) == 2

"""CPU: the index arithmetic of the paged-cache kernels (``csrc/paged_index.h``), compiled by the host compiler.

Divisions, the clamps that hold whatever device memory says, and the cut of a batch into row tiles and key chunks: every
row and key of every sequence in exactly one share, no share past the grid, no partial tile past the workspace.
"""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "qwen3.5-35b-dflash_amd" / "csrc"
SOURCE = """
#include "paged_index.h"
using namespace dflash;
extern "C" {
uint32_t quotient(uint32_t x, uint32_t d) { return divide(x, fast_div(d)); }
void span(int start, int end, int length, int T, int capacity, int* out) {
  const SeqSpan s = seq_span(start, end, length, T, capacity);
  out[0] = s.start; out[1] = s.tokens; out[2] = s.keys;
}
int tiles(int tokens, int group, int rows) { return seq_tiles(tokens, group, rows); }
int units(int keys, int unit) { return seq_units(keys, unit); }
int chunk(int64_t total, int kv, int slots, int least) { return chunk_units(total, kv, 1.0 / slots, least); }
int chunks(int units, int c) { return tile_chunks(units, c); }
int chunk_last(int k0, int c, int unit, int n) { return chunk_end(k0, c, unit, n); }
int visible(int keys, int tokens, int i, int causal) { return visible_keys(keys, tokens, i, causal); }
int64_t tile_bound(int64_t T, int64_t B, int64_t group, int64_t rows) { return max_tiles(T, B, group, rows); }
int64_t chunk_bound(int64_t tiles, int64_t kv, int64_t slots) { return max_chunks(tiles, kv, slots); }
int64_t partial_bound(int64_t tiles, int64_t kv, int64_t slots, int always) { return max_partial_tiles(tiles, kv, slots, always); }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("paged_index")
    source, library = folder / "probe.cpp", folder / "probe.so"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(source), "-o",
                    str(library)], check=True)
    lib = ctypes.CDLL(str(library))
    i64, i32 = ctypes.c_int64, ctypes.c_int
    lib.quotient.argtypes, lib.quotient.restype = [ctypes.c_uint32] * 2, ctypes.c_uint32
    lib.chunk.argtypes = [i64, i32, i32, i32]
    for name, n in (("tile_bound", 4), ("chunk_bound", 3)):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [i64] * n, i64
    lib.partial_bound.argtypes, lib.partial_bound.restype = [i64, i64, i64, i32], i64
    return lib


def test_division(index):
    rng = random.Random(1)
    for d in [1, 2, 3, 4, 5, 6, 7, 8, 63, 64, 65, 1000, 4097, (1 << 26) - 1, 1 << 26]:
        for x in [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, (1 << 27) - 1, (1 << 31) - 1,
                  *(rng.randrange(1 << 31) for _ in range(200))]:
            assert index.quotient(x, d) == x // d, (x, d)


@pytest.mark.parametrize("start,end,length,want", [
    (0, 5, 9, (0, 5, 9)), (-3, 5, 9, (0, 5, 9)), (4, 2, 9, (4, 0, 9)), (4, 99, 9, (4, 6, 9)), (99, 120, 9, (10, 0, 9)),
    (0, 5, -1, (0, 5, 0)), (0, 5, 1 << 30, (0, 5, 64)), (-(1 << 31), (1 << 31) - 1, -(1 << 31), (0, 10, 0))])
def test_spans_stay_inside(index, start, end, length, want):
    """Starts and lengths that are no such thing leave tokens in [0, 10) and keys in [0, 64]."""
    out = (ctypes.c_int * 3)()
    index.span(start, end, length, 10, 64, out)
    assert tuple(out) == want


def test_visible_keys(index):
    assert [index.visible(5, 3, i, 1) for i in range(3)] == [3, 4, 5]
    assert [index.visible(2, 4, i, 1) for i in range(4)] == [0, 0, 1, 2]      # a block longer than its sequence
    assert [index.visible(2, 4, i, 0) for i in range(4)] == [2, 2, 2, 2]
    assert index.visible(0, 1, 0, 1) == 0


def _shares(index, spans, group, kv, rows, unit, slots, least, always):
    """The kernels' numbering: (sequence, tile, first key, end, partial tile or -1) per share, in order."""
    total = sum(index.tiles(t, group, rows) * index.units(n, unit) for t, n in spans)
    c = index.chunk(total, kv, slots, least)
    out, held = [], 0
    for b, (t, n) in enumerate(spans):
        tiles, chunks = index.tiles(t, group, rows), index.chunks(index.units(n, unit), c)
        kept = chunks > 1 or always
        for i in range(tiles * chunks):
            k = i % chunks
            out.append((b, i // chunks, k * c * unit, min((k + 1) * c * unit, n), held + i if kept else -1))
        held += tiles * chunks if kept else 0
    return out, held


@pytest.mark.parametrize("always", [0, 1])
@pytest.mark.parametrize("rows,unit,least", [(16, 128, 1), (128, 64, 4), (128, 128, 2)])
def test_shares_cover_every_row_and_key_once(index, rows, unit, least, always):
    rng = random.Random(rows + unit + always)
    for trial in range(120):
        count = rng.choice((1, 2, 7, 64, 65, 200))
        spans = [(rng.choice((0, 1, 1, 3, 16, rng.randrange(300))), rng.choice((0, 1, unit, unit + 1, rng.randrange(9000))))
                 for _ in range(count)]
        group, kv = rng.choice((1, 3, 8)), rng.choice((1, 2, 8))
        slots = rng.choice((256, 512, 304))
        tokens, shares_held = sum(t for t, _ in spans), None
        shares, shares_held = _shares(index, spans, group, kv, rows, unit, slots, least, always)
        tiles = index.tile_bound(tokens, count, group, rows)
        assert len(shares) <= index.chunk_bound(tiles, kv, slots)
        assert shares_held * kv <= index.partial_bound(tiles, kv, slots, always)
        seen = {}
        for b, tile, k0, k1, _ in shares:
            seen.setdefault((b, tile), []).append((k0, k1))
        for b, (t, n) in enumerate(spans):
            for tile in range(-(-t * group // rows)):
                parts = [(a, z) for a, z in seen.pop((b, tile)) if z > a]
                assert parts == sorted(parts) and (parts or n == 0)
                assert n == 0 or (parts[0][0] == 0 and parts[-1][1] == n)
                assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
        assert not seen
        partial = [s[4] for s in shares if s[4] >= 0]
        assert partial == list(range(len(partial)))


def test_chunks_are_long_enough_at_any_size(index):
    """c slots >= total kv, which the bounds above rest on, also where the product is rounded; and no chunk much longer."""
    rng = random.Random(3)
    for _ in range(20000):
        total, kv = rng.randrange(1, 1 << rng.randrange(1, 45)), rng.choice((1, 2, 3, 8, 31))
        slots = rng.choice((1, 7, 256, 304, 512, 1024))
        c = index.chunk(total, kv, slots, 1)
        assert c > 1000000000 or total * kv <= c * slots <= total * kv + slots, (total, kv, slots, c)


def test_a_chunk_ends_at_the_last_key_at_any_size(index):
    for c in (1, 7, 1 << 23, 1 << 25, 1 << 26, 1_000_000_001):
        for unit in (64, 128):
            for k0, n in ((0, 1), (0, 1 << 30), (unit, 5), ((1 << 30) - unit, 1 << 30), (0, 0)):
                assert index.chunk_last(k0, c, unit, n) == min(k0 + c * unit, n)


def test_a_row_tile_too_few_is_seen(index):
    """The cover check above fails for a cut that drops the ragged last tile."""
    shares, _ = _shares(index, [(3, 40)], 8, 2, 16, 128, 512, 1, 0)
    assert {s[1] for s in shares} == {0, 1} and {s[1] for s in shares if s[1] < 3 * 8 // 16} == {0}

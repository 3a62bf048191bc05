"""CPU: the cut of a shared prefix and its sequences' own keys into one launch (``csrc/paged_index.h``), compiled by the host compiler.

However the places that run at once are divided between the two sides, every row and key of both is in exactly one share,
all shares lie inside the grid and their partial results inside the workspace.  The share lists are checked by one
function, which is itself checked to find a list that lacks a share, holds one twice or cuts one short.
"""
import ctypes
import random
import shutil
import subprocess

import pytest

import test_paged_index as single

SOURCE = single.SOURCE.rstrip().removesuffix("}") + """
float for_own(double own, int tiles, double front, int kv, int slots, float unit, float start) {
  return own_places(own, tiles, front, kv, slots, unit, start);
}
int front_c(double units, int kv, int slots, float own, int least) { return front_chunk(units, kv, slots, own, least); }
int own_c(double units, int kv, float own, int least) { return own_chunk(units, kv, own, least); }
}
"""
SMALL, LARGE = (16, 128, 1), (128, 64, 4)       # rows a tile, keys a unit, units a chunk at least
# own side, prefix side, cost of an own unit and of an own tile's start: the three kernels' choices, and some others
KINDS = [(SMALL, SMALL, 1.0, 2.0), (SMALL, LARGE, 3.0, 4.5), (LARGE, LARGE, 1.0, 8.0), (SMALL, LARGE, 0.3, 0.0), (LARGE, LARGE, 7.0, 90.0)]


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    folder = tmp_path_factory.mktemp("paged_pair_index")
    source, library = folder / "probe.cpp", folder / "probe.so"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{single.CSRC}", str(source), "-o",
                    str(library)], check=True)
    lib = ctypes.CDLL(str(library))
    i64, i32, f32, f64 = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_double
    lib.for_own.argtypes, lib.for_own.restype = [f64, i32, f64, i32, i32, f32, f32], f32
    lib.front_c.argtypes, lib.own_c.argtypes = [f64, i32, i32, f32, i32], [f64, i32, f32, i32]
    for name, n in (("tile_bound", 4), ("chunk_bound", 3)):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [i64] * n, i64
    lib.partial_bound.argtypes, lib.partial_bound.restype = [i64, i64, i64, i32], i64
    return lib


def shares_of(index, spans, group, kind, c):
    """(sequence, tile, first key, end) of every share in order, chunks of c units."""
    rows, unit, _ = kind
    out = []
    for b, (t, n) in enumerate(spans):
        chunks = index.chunks(index.units(n, unit), c)
        for i in range(index.tiles(t, group, rows) * chunks):
            k = i % chunks
            out.append((b, i // chunks, min(k * c * unit, n), min((k + 1) * c * unit, n)))
    return out


def check_cover(shares, spans, group, rows):
    """Every row tile of every sequence once, each over all its keys without a gap or an overlap; one share where there are no keys."""
    seen = {}
    for b, tile, k0, k1 in shares:
        seen.setdefault((b, tile), []).append((k0, k1))
    for b, (t, n) in enumerate(spans):
        for tile in range(-(-t * group // rows)):
            parts = seen.pop((b, tile), None)
            assert parts is not None, ("no share", b, tile)
            assert parts[0][0] == 0 and parts[-1][1] == n, (b, tile, parts)
            assert all(x[1] == y[0] for x, y in zip(parts, parts[1:])), (b, tile, parts)
            assert n or len(parts) == 1, (b, tile, parts)
    assert not seen, seen


def total(index, spans, group, kind):
    tiles = [index.tiles(t, group, kind[0]) for t, _ in spans]
    return sum(tiles), float(sum(n * index.units(s[1], kind[1]) for n, s in zip(tiles, spans)))


@pytest.mark.parametrize("own,front,unit_cost,start_cost", KINDS)
def test_both_sides_fit_the_grid_and_the_workspace(index, own, front, unit_cost, start_cost):
    rng = random.Random(own[0] + front[0])
    for trial in range(250):
        count = rng.choice((1, 1, 2, 7, 64, 65, 200))
        longest = rng.choice((0, 1, 40, 900, 9000))
        spans = [(rng.choice((0, 1, 1, 1, 3, 16, rng.randrange(300))), rng.choice((0, 1, own[1], own[1] + 1, rng.randrange(longest + 1))))
                 for _ in range(count)]
        group, kv, slots = rng.choice((1, 3, 8, 20)), rng.choice((1, 2, 3, 8)), rng.choice((256, 512, 304))
        tokens = sum(t for t, _ in spans) + rng.choice((0, 0, 5))          # tokens in no sequence too: the prefix has rows for them
        prefix = [(tokens, rng.choice((0, 1, 63, 64, 65, 1000, rng.randrange(40_000))))]
        own_tiles, own_units = total(index, spans, group, own)
        front_tiles, front_units = total(index, prefix, group, front)
        places = index.for_own(own_units, own_tiles, front_units, kv, slots, unit_cost, start_cost)
        assert 1.0 <= places <= slots - 1
        c0 = index.front_c(front_units, kv, slots, places, front[2])
        c1 = index.own_c(own_units, kv, places, own[2])
        first, second = shares_of(index, prefix, group, front, c0), shares_of(index, spans, group, own, c1)
        check_cover(first, prefix, group, front[0])
        check_cover(second, spans, group, own[0])
        bound = index.tile_bound(tokens, count, group, own[0])
        assert len(first) + len(second) <= index.chunk_bound(bound + front_tiles, kv, slots), (spans, prefix, group, kv, slots)
        assert len(first) * kv <= index.partial_bound(front_tiles, kv, slots, 1)
        assert len(second) * kv <= index.partial_bound(bound, kv, slots, 1)


def test_places_are_divided_whatever_the_work_is(index):
    """Counts that overflowed, from starts that are no such thing, leave each side a place at least, and the prefix inside its bound."""
    wild = (0.0, 1.0, -1.0, 1e18, -1e18, float("inf"), float("nan"))
    for own in wild:
        for tiles in (0, 1, -5, (1 << 31) - 1, -(1 << 31)):
            for front in (0.0, 1.0, 1e6, 2.0 ** 40):
                places = index.for_own(own, tiles, front, 1, 512, 3.0, 4.5)
                assert 1.0 <= places <= 511.0, (own, tiles, front, places)
                c = index.front_c(front, 2, 512, places, 4)
                assert c > 1_000_000_000 or c * 512 >= front * 2, (own, tiles, front, c)


def test_a_cut_with_a_fault_is_seen(index):
    spans, group = [(3, 400), (0, 9), (17, 0), (40, 1000)], 8
    for kind in (SMALL, LARGE):
        shares = shares_of(index, spans, group, kind, 2)
        check_cover(shares, spans, group, kind[0])
        faults = [shares[:i] + shares[i + 1:] for i in range(len(shares))]                  # one share too few
        faults += [shares + [shares[i]] for i in (0, len(shares) - 1)]                        # one twice
        faults += [shares[:i] + [(*shares[i][:3], shares[i][3] - 1)] + shares[i + 1:] for i in range(len(shares)) if shares[i][3]]
        faults += [[s for s in shares if s[1] < -(-spans[s[0]][0] * group // kind[0]) - 1]]     # the ragged last tiles
        for fault in faults:
            with pytest.raises(AssertionError):
                check_cover(fault, spans, group, kind[0])

"""Every tile of a grouped product, walked on the CPU through the functions that deal them (csrc/grouped_tiles.h): with ordered
offsets each value of the output is one block's, with any offsets every tile lies in the rows there are and every block ends."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

from tests.grouped_util import CUT, NARROW, WIDE

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r"""
#include <cstdint>
#include <cstddef>
#include <vector>
#include "grouped_tiles.h"
using namespace brx;

static long taken;
// the runs as tall_table makes them: entry E the rows behind the last, E + 1 their end
struct Table {
    std::vector<int> first, tiles;
    Table(const int* offsets, int E, int P, int bm) : first(E + 2), tiles(E + 2) {
        int n = 0;
        for (int e = 0; e <= E; ++e) {
            const RowRun r = run_between(e ? offsets[e] : 0, e < E ? offsets[e + 1] : P, P);
            if (r.first < 0 || r.end < r.first || r.end > P) n = -(1 << 30);
            first[e] = r.first;
            tiles[e] = n;
            n += run_tiles(r, bm);
            if (e == E) first[E + 1] = r.end;
        }
        tiles[E + 1] = n;
    }
    int of(int mt, int E) const {
        int e = 0;
        for (int i = 0; i <= E; ++i)
            if (tiles[i] <= mt) e = i;
        return e;
    }
};

extern "C" {
long walk_taken() { return taken; }
int form(int P, int E, int N, int across) { return row_form(P, E, N, across != 0); }
void rounds(int tiles, int* out) {
    const Rounds r = rounds_of(tiles, kChipCus);
    out[0] = r.rounds; out[1] = r.last; out[2] = r.cut;
}
int count_row_tiles(const int* offsets, int E, int P, int bm) { return Table(offsets, E, P, bm).tiles[E + 1]; }
long most_row_tiles(int P, int E, int bm) { return row_tiles(P, E, bm); }

// Mistakes of the persistent kernel of a product of rows. `ordered`: each row's columns are to be taken once, for its expert.
long walk_rows(const int* offsets, int E, int P, int N, int ordered) {
    long bad = 0;
    taken = 0;
    const Table t(offsets, E, P, kTall);
    const int ntiles = (N + kTall - 1) / kTall, mtiles = t.tiles[E + 1], per = kChipCus / kChipXcds;
    if (mtiles < 0) return 1;
    const Rounds r = rounds_of(mtiles * ntiles, kChipCus);
    std::vector<uint8_t> seen((std::size_t)P * ntiles);
    for (int xcd = 0; xcd < kChipXcds; ++xcd)
        for (int place = 0; place < per; ++place)
            for (int round = 0;; ++round) {
                const Dealt d = deal(r, round, xcd, place, per);
                if (!d.rows) break;
                if (round > r.rounds) return ++bad;
                const RowColumn rc = row_column(d.tile, mtiles, ntiles);
                const int e = t.of(rc.mt, E), lo = t.first[e], hi = t.first[e + 1] > lo ? t.first[e + 1] : lo;
                const int m0 = lo + (rc.mt - t.tiles[e]) * kTall + d.part * d.rows, rows = min_of(hi - m0, d.rows);
                if (rc.mt >= mtiles || rc.nt >= ntiles || rc.nt < 0) ++bad;
                if (rows <= 0) {
                    if (round < r.rounds || !d.part) ++bad;     // only a part of a cut tile may be empty
                    break;
                }
                if (m0 < 0 || m0 + rows > P) return ++bad;
                ++taken;
                if (!ordered) continue;
                for (int m = m0; m < m0 + rows; ++m) {
                    bad += seen[(std::size_t)m * ntiles + rc.nt]++ != 0;
                    bad += e < E ? m < (e ? offsets[e] : 0) || m >= offsets[e + 1] : m < offsets[E];
                }
            }
    if (ordered)
        for (uint8_t v : seen) bad += v != 1;
    return bad;
}

// ... of the product over the runs: each tile of each expert's matrix once, whatever the offsets.
long walk_runs(int E, int K, int N) {
    long bad = 0;
    const int mtiles = (K + kTall - 1) / kTall, ntiles = (N + kTall - 1) / kTall, per = kChipCus / kChipXcds;
    const Rounds r = rounds_of(E * mtiles * ntiles, kChipCus);
    std::vector<uint8_t> seen((std::size_t)E * K * ntiles);
    for (int xcd = 0; xcd < kChipXcds; ++xcd)
        for (int place = 0; place < per; ++place)
            for (int round = 0;; ++round) {
                const Dealt d = deal(r, round, xcd, place, per);
                if (!d.rows) break;
                if (round > r.rounds) return ++bad;
                const int u = d.tile / ntiles, nt = d.tile - u * ntiles, e = u / mtiles, m0 = u % mtiles * kTall + d.part * d.rows;
                const int rows = min_of(K - m0, d.rows);
                if (e >= E) return ++bad;
                if (rows <= 0) {
                    if (round < r.rounds || !d.part) ++bad;
                    break;
                }
                for (int m = m0; m < m0 + rows; ++m) bad += seen[((std::size_t)e * K + m) * ntiles + nt]++ != 0;
            }
    for (uint8_t v : seen) bad += v != 1;
    return bad;
}
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    d = tmp_path_factory.mktemp("grouped_tiles")
    (d / "walk.cpp").write_text(SRC)
    so = str(d / "walk.so")
    r = subprocess.run([shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I",
                        os.path.join(ROOT, "bigrig_amd", "csrc"), str(d / "walk.cpp"), "-o", so],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    for f in ("walk_taken", "walk_rows", "walk_runs", "most_row_tiles"):
        getattr(lib, f).restype = C.c_long
    return lib


def offsets_of(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def ints(v):
    return (C.c_int * len(v))(*v)


def cases():
    rng = random.Random(1)
    yield [5000], 0
    yield [0, 0, 0], 4000
    yield [1] * 512, 0
    yield [256] * 40, 256
    for _ in range(40):
        E = rng.choice([1, 2, 7, 64, 200, 512])
        yield [rng.choice([0, 1, 63, 64, 65, 128, 255, 256, 257, rng.randint(0, 600)]) for _ in range(E)], rng.choice([0, 1, 300])


@pytest.mark.parametrize("N", [8, 256, 264, 2048, 5896, 8192])
def test_every_value_of_a_product_of_rows_is_one_blocks(walk, N):
    for counts, behind in cases():
        at = offsets_of(counts)
        P = at[-1] + behind
        assert walk.walk_rows(ints(at), len(counts), P, N, 1) == 0, (counts, behind)
        for bm in (16, 32, 64, 128, 256):      # a launch has blocks for every tile
            assert walk.count_row_tiles(ints(at), len(counts), P, bm) <= walk.most_row_tiles(P, len(counts), bm)


@pytest.mark.parametrize("E,K,N", [(1, 8, 8), (16, 72, 5896), (17, 5896, 72), (60, 712, 1000), (512, 264, 264), (9, 8192, 520)])
def test_every_value_of_a_product_over_the_runs_is_one_blocks(walk, E, K, N):
    assert walk.walk_runs(E, K, N) == 0


def test_any_offsets_stay_in_the_rows(walk):
    rng = random.Random(2)
    top, low = (1 << 31) - 1, -(1 << 31)
    P = 5000
    odd = [[0, 60, -5, 100, 1 << 30], [5, 10, 10, 20, 20], [0, 3000, 1000, 4000, 5000], [low, 0, 0, 0, 0], [top] * 5, [low] * 5,
           [0, P, 0, P, 0], [0, top, low, top, low], [0, 5001, 4999, 0, 7]]
    odd += [[rng.choice([low, -1, 0, rng.randint(0, P), P, P + 1, top]) for _ in range(65)] for _ in range(200)]
    for o in odd:
        for N in (8, 2048, 8192):
            assert walk.walk_rows(ints(o), len(o) - 1, P, N, 0) == 0, o


def test_tiles_of_any_offsets_are_counted_in_an_int(walk):
    # the largest call, each of 256 pairs of experts with every row
    E, P = 512, 1 << 23
    o = [0, P] * 256 + [0]
    assert walk.count_row_tiles(ints(o), E, P, 256) * (8192 // 256) < 1 << 30
    assert walk.most_row_tiles(P, E, 256) * (8192 // 256) < 1 << 21


def test_which_kernel(walk):
    thin, low, half, square, tall = range(5)
    for P, E, N, across, want in (
            (8, 128, 2048, 0, thin), (9, 128, 2048, 0, low), (8, 128, 2048, 1, low), (2048, 128, 1536, 0, low),
            (2049, 128, 1536, 0, half), (6144, 128, 1536, 0, half), (6145, 128, 1536, 0, square), (8192, 256, 4096, 0, half),
            (8192, 256, 4096, 1, tall), (32768, 128, 1536, 0, tall), (1000, 8, 2048, 0, square), (1000, 8, 1024, 0, half),
            (4000, 8, 2048, 0, square), (0, 4, 64, 1, low)):
        assert walk.form(P, E, N, across) == want, (P, E, N, across)


@pytest.mark.parametrize("name", CUT)
def test_calls_whose_last_round_is_cut(walk, name):
    # what the GPU tests of the cut rounds are meant to run
    counts, behind, rows, runs = CUT[name]
    at, E = offsets_of(counts), len(counts)
    P, out = at[-1] + behind, ints([0, 0, 0])
    columns = -(-WIDE // 256)
    for across in (0, 1):
        assert walk.form(P, E, WIDE, across) == 4
    walk.rounds(walk.count_row_tiles(ints(at), E, P, 256) * columns, out)
    assert tuple(out) == rows
    assert E * columns * (-(-NARROW // 256)) >= 256
    walk.rounds(E * columns, out)
    assert tuple(out) == runs
    assert walk.walk_rows(ints(at), E, P, WIDE, 1) == 0
    assert walk.walk_runs(E, WIDE, NARROW) == 0 and walk.walk_runs(E, NARROW, WIDE) == 0

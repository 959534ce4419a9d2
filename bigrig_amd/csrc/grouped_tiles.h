// Which tiles a grouped product has and which block takes which (k_grouped.hip): plain C++, so that a host program can walk
// them all. Offsets come from the device's memory and may be anything: what they name is clamped into the rows there are.
#pragma once

#include <cstdint>

namespace brx {

constexpr int kChipCus = 256, kChipXcds = 8;
constexpr int kTall = 256;            // rows and columns of a persistent kernel's tile
constexpr int kThinRows = 16;         // rows of a thin tile
constexpr int kThinMost = 8, kLowRun = 16, kHalfRun = 48;

constexpr int min_of(int a, int b) { return a < b ? a : b; }
constexpr int max_of(int a, int b) { return a > b ? a : b; }

// The rows [first, end) of a run between two offsets, of P rows. Offsets out of order make an empty run, or runs that overlap.
struct RowRun {
    int first, end;
};
constexpr RowRun run_between(int lo, int hi, int P) {
    const int first = min_of(max_of(lo, 0), P);
    return {first, min_of(max_of(hi, first), P)};
}
constexpr int run_tiles(const RowRun& r, int bm) { return (r.end - r.first + bm - 1) / bm; }

// Row tiles of bm rows that a call of ordered offsets can have: the whole ones, and one of each run that is not empty.
constexpr int64_t row_tiles(int P, int E, int bm) { return P / bm + min_of(E + 1, P); }

// The kernel of a product of rows (k_grouped.hip says why). `across`: the matrices are read across their rows (the rows'
// gradient); N: values of a row of the output.
enum RowForm { kFormThin, kFormLow, kFormHalf, kFormSquare, kFormTall };
constexpr RowForm row_form(int P, int E, int N, bool across) {
    const bool tall = (int64_t)(P / kTall) * ((N + kTall - 1) / kTall) >= kChipCus;
    return !across && P <= kThinMost                                             ? kFormThin
           : P <= kLowRun * E                                                    ? kFormLow
           : (P <= kHalfRun * E && !(across && tall)) ||
                   row_tiles(P, E, 128) * ((N + 127) / 128) < kChipCus           ? kFormHalf
           : !tall                                                               ? kFormSquare
                                                                                 : kFormTall;
}

// The tiles of a persistent kernel dealt to its blocks: whole rounds of one each, and a last round of `last`, each cut 2^cut
// times by its rows where the blocks suffice. (Of ordered offsets there are below 2^21, of any below 2^30: 513 runs of 2^15 row
// tiles by 32.)
struct Rounds {
    int rounds, last, cut;
};
constexpr Rounds rounds_of(int tiles, int blocks) {
    const int rounds = tiles / blocks, last = tiles - rounds * blocks;
    return {rounds, last, 4 * last <= blocks ? 2 : 2 * last <= blocks ? 1 : 0};
}

// What round `round` gives the block at `place` of `per` on XCD `xcd`: a tile, or the part of one of `rows` rows; rows 0: nothing,
// then or later.
struct Dealt {
    int tile, part, rows;
};
constexpr Dealt deal(const Rounds& r, int round, int xcd, int place, int per) {
    const int at = round * per * kChipXcds;
    if (round < r.rounds) return {at + xcd * per + place, 0, kTall};
    const int n = r.last << r.cut, share = (n + kChipXcds - 1) / kChipXcds, v = xcd * share + place;
    if (round > r.rounds || place >= share || v >= n) return {0, 0, 0};
    return {at + (v >> r.cut), v & ((1 << r.cut) - 1), kTall >> r.cut};
}

// Tile `at` of a product of rows: two row tiles by all columns after another, a last single one by all.
struct RowColumn {
    int mt, nt;
};
constexpr RowColumn row_column(int at, int mtiles, int ntiles) {
    const int two = at / (2 * ntiles), rem = at - two * (2 * ntiles);
    return 2 * two + 1 < mtiles ? RowColumn{2 * two + (rem & 1), rem >> 1} : RowColumn{2 * two, rem};
}

}  // namespace brx

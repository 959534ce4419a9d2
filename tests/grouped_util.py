"""Calls of grouped products whose persistent tiles end in a round that is cut: shared by the tests that run them and the one
that holds them to the rule (csrc/grouped_tiles.h)."""

NARROW, WIDE = 72, 5896       # widths of the matrices; the wide one has 24 tiles, the last of 8
_LONG = [0, 300, 513, 700, 0, 256, 1024, 511, 900]
# name: (runs' rows, rows behind the last run; of the products of rows over the wide width: whole rounds, tiles of the last, how
# often those are halved; of the product over the runs the same)
CUT = {
    "quarters": (_LONG + [500, 130, 193, 0, 65], 0, (2, 64, 2), (1, 80, 1)),
    "quarters-behind": (_LONG + [257, 129], 1, (2, 40, 2), (1, 8, 2)),
    "halves": (_LONG + [193, 129, 65, 0, 1, 193, 65], 0, (2, 88, 1), (1, 128, 1)),
    "halves-behind": (_LONG + [129, 0, 65, 193, 1, 129, 65, 0], 129, (2, 112, 1), (1, 152, 0)),
}

"""Attention over batches whose rows come in any order, twice or cut into runs of
every length, and at the row counts where its kernels change."""
import numpy as np
import pytest

import serving_catalog as sc
from oracle import blockscaled as bs
from test_norm_mx import note, stored
from test_serving import load
from test_serving_ranges import case_of, run


def ordered(case, order):
    """The case's rows in another order (a row may come twice)."""
    seq, pos, table, cache, qs, qv = case
    return seq[order], pos[order], table, cache, qs[order], qv[order]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["group4", "group3", "alone", "group20", "window", "usual", "far", "far_f16", "far_group20", "far_window", "wide_f16"])
def test_rows_in_any_order(gpu, name):
    """Rows mixed, reversed, interleaved, doubled, with rows that pad between
    them: each has its own answer."""
    c = sc.ATTEND[name]
    room, slots = c[5], c[4]
    rng = np.random.default_rng(len(name))
    low = 127 - bs.EMAX[c[8]]
    grp = load(f"pagedattn_{name}_rt")
    near = min(room, 1700)
    for i, parts in enumerate(([(0, 3, 20), (2, near - 9, 9)], [(1, near - 80, 80), (0, 0, 45), (2, 31, 40)])):
        case = case_of(rng, c, parts, lambda k: low - k % 3, pad=5)
        n = len(case[0])
        runs = np.argsort(np.arange(n) % 7, kind="stable")  # runs of one row that follow no other
        cut = np.concatenate([np.arange(s, min(s + 1 + s % 11, n)) for s in rng.permutation(np.arange(0, n, 5))])  # runs that overlap
        for what, order in (("mixed", rng.permutation(n)), ("reversed", np.arange(n)[::-1]), ("interleaved", runs), ("doubled", np.repeat(np.arange(n), 2)),
                            ("cut", cut)):
            note(f"{name} batch {i} {what}")
            run(grp, c, gpu, *ordered(case, order))


@pytest.mark.gpu
@pytest.mark.parametrize("name,counts", [("group4", (1, 63, 64, 65, 66)), ("alone", (79, 80, 81, 127, 129)), ("far_alone", (63, 64, 65, 128, 129)),
                                         ("far_group20", (8, 64, 65, 2047, 2048, 2049)), ("many", (1023, 1024, 1025, 1199, 1200, 1201))])
def test_row_counts_where_kernels_change(gpu, name, counts):
    c = sc.ATTEND[name]
    room, slots = c[5], c[4]
    rng = np.random.default_rng(len(name))
    low = 127 - bs.EMAX[c[8]]
    grp = load(f"pagedattn_{name}_rt")
    for rows in counts:
        note(f"{name} {rows} rows")
        long = min(rows, room - 3)
        parts, left, s = [(0, 2, long)], rows - long, 1
        while left:
            k = min(left, room - 7, 1 + 40 * s)
            parts.append((s, 5, k))
            left, s = left - k, s + 1
        assert s <= slots
        run(grp, c, gpu, *case_of(rng, c, parts, lambda k: low - k % 3))

"""Releases of sequences that gave pages up: entries of a table that are no pages (include/zq_paged.h) do not come back as
free ones."""
import numpy as np
import pytest
import torch

import paged_plain as P
from test_paged import dev, full_table

gpu = pytest.mark.gpu


def release(lens, keep, table, free, free_count, ps):
    """(free, free_left): as paged_plain.release, without the entries that are no pages."""
    cap, free, pages, back = table.shape[1] * ps, free.copy(), len(free), []
    for s in range(len(lens)):
        n = min(max(lens[s], 0), cap)
        back += [p for p in table[s, P.cdiv(min(max(keep[s], 0), n), ps):P.cdiv(n, ps)] if 0 <= p < pages]
    top = min(max(free_count, 0), pages)
    for i, p in enumerate(reversed(back)):
        if top + i < pages:
            free[top + i] = p
    return free, min(top + len(back), pages)


def test_the_plain_form_without_given_up_pages_is_the_other_one():
    rng = np.random.default_rng(1)
    lens, keep = rng.integers(0, 90, 12), rng.integers(-3, 60, 12)
    table, free, fc = full_table(rng, lens, 7, 16, 70)
    for a, b in zip(release(lens, keep, table, free, fc, 16), P.release(lens, keep, table, free, fc, 16)):
        assert np.array_equal(a, b)


NONE = (-1, -2 ** 31, 2 ** 31 - 1)


def give_up(rng, table, lens, ps, pages, how):
    """Entries that are no pages in a table, of those that its sequences have; how many there were."""
    gone = 0
    for s, n in enumerate(lens):
        have = min(P.cdiv(n, ps), table.shape[1])
        if how == "first":  # all but the last pages, as a window that moves on leaves them
            which = range(max(0, have - 2))
        elif how == "all":
            which = range(have)
        else:
            which = np.nonzero(rng.random(have) < how)[0]
        for j in which:
            table[s, j] = (*NONE, pages)[rng.integers(4)]
            gone += 1
    return gone


def check_release(zq, lens, keep, table, free, fc, ps, in_place=(False, True)):
    S, W = table.shape
    for same in in_place:
        t, f, c = dev(table), dev(free), dev([fc])
        h = zq.PageTables(t, f, S, W, len(free), ps)
        left = c if same else dev([-1])
        zq.page_tables_release_dev(h, dev(lens), dev(keep), c, left)
        want, n = release(lens, keep, table, free, fc, ps)
        assert int(left) == n, same
        assert np.array_equal(f.cpu().numpy()[:n], want[:n]), same
        assert np.array_equal(t.cpu().numpy(), table)


@gpu
@pytest.mark.parametrize("how", ["first", "all", 0.02, 0.5])
@pytest.mark.parametrize("S, ps, most", [(1, 16, 1), (1, 16, 64), (1, 16, 40000), (3, 32, 200), (5, 16, 17000), (100, 16, 300),
                                         (256, 16, 900), (257, 32, 100), (700, 16, 500), (1025, 16, 1600), (8192, 16, 17)])
def test_release_leaves_out_what_is_no_page(zq, S, ps, most, how):
    rng = np.random.default_rng(S + most)
    lens = rng.integers(0, most + 1, S)
    lens[0] = most
    keep = np.where(rng.random(S) < 0.6, 0, np.maximum(-1, lens - rng.integers(-3, 400, S)))
    if S == 1:
        keep[0] = 0
    W = P.cdiv(most, ps) + 1
    pages = sum(P.cdiv(n, ps) for n in lens) + 5
    table, free, fc = full_table(rng, lens, W, ps, pages)
    give_up(rng, table, lens, ps, pages, how)
    check_release(zq, lens, keep, table, free, fc, ps)


@gpu
def test_release_of_more_entries_than_the_pool_has_room_for(zq):
    """Many entries that are no pages and a few that are: these all find room; and more pages than there is room for."""
    rng = np.random.default_rng(4)
    pages, ps, W, S = 40, 16, 100, 3
    table = np.full((S, W), -1, np.int64)
    table[0, [0, 50, 99]], table[1, 98], table[2, :2] = [7, 8, 9], 10, [11, 12]
    free = np.full(pages, -5, np.int64)
    free[:34] = 13
    lens = [W * ps] * 3
    check_release(zq, lens, [0, 0, 0], table, free, 34, ps)
    check_release(zq, lens, [0, 0, 40], table, free, 39, ps)
    check_release(zq, lens, [0, 0, 0], table, free, 40, ps)
    table[:] = rng.integers(-40, 2 * pages, table.shape)
    check_release(zq, lens, [0, 17, 0], table, free, 5, ps)


@gpu
def test_a_release_as_long_as_can_be(zq):
    """300,000 entries of two sequences, every third of which is no page."""
    rng = np.random.default_rng(5)
    ps, W = 16, 200000
    lens = [W * ps, 100000 * ps]
    pages = 300000
    table, free, fc = full_table(rng, lens, W, ps, pages)
    table[rng.random(table.shape) < 1 / 3] = -1
    check_release(zq, lens, [0, 0], table, free, fc, ps)


@gpu
def test_pages_given_up_are_not_granted_again(zq):
    """A sequence whose window has moved on ends; another one takes the pages that it had, and every token has a slot."""
    rng = np.random.default_rng(6)
    ps, W, pages = 16, 12, 14
    lens = [160, 20]
    table, free, fc = full_table(rng, lens, W, ps, pages)
    given = [int(p) for p in table[0, :6]]
    table[0, :6] = -1
    free[fc:fc + 6] = given  # by the caller, as the pages were given up
    fc += 6
    t, f, c = dev(table), dev(free), dev([fc])
    h = zq.PageTables(t, f, 2, W, pages, ps)
    zq.page_tables_release_dev(h, dev(lens), dev([0, 20]), c, c)
    assert int(c) == pages - 2 and sorted(f.cpu().tolist()[:pages - 2] + [int(p) for p in table[1, :2]]) == list(range(pages))
    granted, start, slots = dev([0, 0]), dev([0] * 3), dev([0] * 300, torch.int64)
    zq.page_tables_step_dev(h, dev([0, 20]), dev([0, 10 * ps]), c, c, granted, start, slots, None, None, 300)
    assert int(granted[1]) == 10 * ps
    got = slots.cpu().numpy()[:10 * ps]
    assert (got >= 0).all() and len(set(got)) == 10 * ps

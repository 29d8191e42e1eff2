"""Attention over the paged KV cache (include/zq_paged.h) uses every row that a query sees once, with its own key and value.
Values are small whole numbers, and scores are all equal (queries of zeros) or one of two, so far apart that only the rows
whose key has a one in a head's place count: an output times the number of rows that count is then a whole number that a
row too few, too many or of another page changes.  Sequences share their pages, which keeps the caches small where a
workgroup has more than 4096 keys of a pair in a row."""
import math

import numpy as np
import pytest
import torch

import paged_plain as P
from test_paged import DEV, KINDS, dev

gpu = pytest.mark.gpu


class Whole:
    """One run of `rows` rows, of which every sequence has a part from its start."""

    def __init__(self, kind, KH, D, ps, rows, seed, extra=2):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.KH, self.D, self.ps, self.rows = kind, KH, D, ps, rows
        n = P.cdiv(rows, ps)
        self.pages = n + extra
        self.order = rng.permutation(self.pages)[:n]
        self.v = rng.integers(-8, 9, (rows, KH, D))
        self.k = rng.integers(0, 2, (rows, KH, D))

    def before(self, h, place):
        """(numbers of rows, sums of values [D]) of the first 0, 1, .. rows of kv head h whose keys have a one at `place`
        (None: of all rows)."""
        one = np.ones(self.rows, np.int64) if place is None else self.k[:, h, place]
        add = lambda x: np.concatenate([np.zeros_like(x[:1]), x.cumsum(0)])
        return add(one), add(one[:, None] * self.v[:, h])

    def upload(self, zq, seqs, width):
        KH, D, ps, n = self.KH, self.D, self.ps, len(self.order)
        at = torch.from_numpy(self.order).to(DEV)
        to = []
        for x in (self.k, self.v):  # what no sequence has is NaN
            rows = np.full((n * ps, KH, D), math.nan, np.float32)
            rows[:self.rows] = x
            pool = torch.full((self.pages, KH, ps, D), math.nan, dtype=P.TYPES[self.kind], device=DEV)
            pool[at] = torch.from_numpy(rows.reshape(n, ps, KH, D).transpose(0, 2, 1, 3).copy()).to(pool.dtype).to(DEV)
            to.append(pool)
        self.gk, self.gv = to
        self.gt = torch.full((seqs, width), -1, dtype=torch.int32, device=DEV)
        self.gt[:, :n] = at.int()
        self.cache = zq.KVPaged(self.gk, self.gv, self.pages, KH, D, ps)
        self.tables = zq.PageTables(self.gt, None, seqs, width, self.pages, ps)


def wrong(got, sums, rows):
    """Outputs [n][D] that are not sums [n][D] / rows [n].

    The rows that count have one weight; its products with whole numbers below 2^4, and the sums of fewer than 2^20 of
    them, are exact in fp32 in any order.  Others weigh e^-40 of that, 2^20 * 8 * e^-40 < 2^-34 in all.  The quotient and the
    product with it are off by 2^-23 of at most 8 rows: below 1/4 in all."""
    return ~(np.abs(got.astype(np.float64) * rows[:, None] - sums) < 0.25)


def test_a_lost_row_shows():
    """The check refuses outputs without one row, a page, a unit of keys, and with these rows twice."""
    x = Whole("f16", 1, 64, 16, 20011, seed=1)
    for place in (None, 3):
        rows, sums = x.before(0, place)
        for n in (300, 4097, 9000, 20011):
            assert not wrong((sums[n] / rows[n]).astype(np.float32)[None], sums[n], rows[n:n + 1]).any()
            for a, b in ((n - 1, n), (0, 16), (n - 128, n), (0, 1), (n // 2, n // 2 + 32)):
                count, lost = rows[b] - rows[a], sums[b] - sums[a]
                for y in ((sums[n] - lost) / (rows[n] - count), (sums[n] + lost) / (rows[n] + count)):
                    assert wrong(y.astype(np.float32)[None], sums[n], rows[n:n + 1]).any() or not count


def check(zq, x, G, lens, seq_of, width, seqs, select=None, runs=lambda n: [(0, n)]):
    """Queries with lens[i] rows before them, of sequences seq_of (None: one each); select [pages] for all of them, and the
    runs of rows (a, b) that a query with n rows sees then."""
    n, H = len(lens), x.KH * G
    x.upload(zq, seqs, width)
    need = zq.attention_paged_workspace_bytes(x.cache, x.tables, n, H)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=DEV)
    more = {}
    if select is not None:
        more = dict(select=dev(np.broadcast_to(select, (n, x.KH, len(select))).copy()), keep=len(select))
    sees = [np.array(runs(m + 1), np.int64).reshape(-1, 2) for m in lens]
    for keys in (False, True):
        q, out = torch.zeros(n, x.KH, G, x.D, device=DEV), torch.full((n, x.KH, G, x.D), math.nan, device=DEV)
        places = [(7 * g + 3) % x.D for g in range(G)]
        if keys:
            for g, place in enumerate(places):
                q[:, :, g, place] = 40.0
        zq.attention_paged_dev(x.cache, x.tables, q, out, n, H, dev(lens), 1.0, seq_of=None if seq_of is None else dev(seq_of),
                               workspace=ws, workspace_bytes=need, **more)
        got = out.cpu().numpy()
        for h in range(x.KH):
            every = x.before(h, None)
            for g in sorted({0, 1, 2, G - 1} & set(range(G))) if keys else range(G):
                rows, sums = x.before(h, places[g]) if keys else every
                r = np.array([(rows[y[:, 1]] - rows[y[:, 0]]).sum() for y in sees])
                t = np.stack([(sums[y[:, 1]] - sums[y[:, 0]]).sum(0) for y in sees])
                for i in np.nonzero(r == 0)[0]:  # none counts: all do
                    r[i] = max(sum(b - a for a, b in sees[i]), 1)
                    t[i] = sum((every[1][b] - every[1][a] for a, b in sees[i]), np.zeros(x.D, np.int64))
                bad = wrong(got[:, h, g], t, r)
                assert not bad.any(), (keys, h, g, [(i, lens[i] + 1) for i in np.nonzero(bad.any(1))[0][:8]])


EDGES = [4095, 4096, 4097, 4096 + 127, 4096 + 128, 4096 + 129, 4224 + 16, 4300]  # 4096 keys are what a workgroup has ahead


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_pairs_of_their_own(zq, kind):
    """512 pairs of a workgroup each with up to 4300 keys (1.1 MB of rows a pair)."""
    x = Whole(kind, 8, 64, 16, 4300, seed=1)
    lens = [EDGES[i % 8] - 1 if i % 3 else int(x.rng.integers(0, 4300)) for i in range(64)]
    check(zq, x, 3, lens, None, 270, 64)


@gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_long_pairs_of_selected_pages(zq, kind):
    """512 pairs of a workgroup each with up to 268 selected pages of longer sequences, in any order, holes among them."""
    x = Whole(kind, 8, 64, 16, 9000, seed=2)
    select = x.rng.permutation(P.cdiv(9000, 16))[:268]
    select[[5, 100, 266]] = [-1, 5000, 2 ** 30]

    def runs(n):
        pages = [int(p) * 16 for p in select[:min(268, P.cdiv(n, 16))] if 0 <= p < 5000]
        return [(p, min(p + 16, n)) for p in pages if p < n]
    lens = [8999] * 20 + [4095 + i for i in range(40)] + [99, 2000, 0, 4290]
    check(zq, x, 2, lens, None, 570, 64, select=select, runs=runs)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, KH, seqs", [(64, 2, 128), (128, 2, 128), (256, 1, 132)])
def test_long_shares(zq, kind, D, KH, seqs):
    """More than 4096 keys of a share of a workgroup, and of a pair of its own among the shares."""
    x = Whole(kind, KH, D, 32, 10500, seed=3)
    lens = [EDGES[i % 8] - 1 if i % 4 == 1 else 10499 if i % 4 else int(x.rng.integers(8500, 10500)) for i in range(seqs)]
    check(zq, x, 2, lens, None, 400, seqs)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G", [(64, 17), (128, 16)])
def test_long_shares_of_selected_pages(zq, kind, D, G):
    """300 pages of 64 selected, a pair or less a workgroup."""
    x = Whole(kind, 1, D, 64, 40000, seed=4)
    select = np.sort(x.rng.permutation(P.cdiv(40000, 64))[:300])
    select[-1] = P.cdiv(40000, 64) - 1

    def runs(n):
        return [(int(p) * 64, min(int(p) * 64 + 64, n)) for p in select[:min(300, P.cdiv(n, 64))] if p * 64 < n]
    lens = [39999 - 7 * (i % 5) if i % 9 else 3000 + i for i in range(200)]
    check(zq, x, G, lens, None, 700, 200, select=select, runs=runs)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, G, seqs, each, width", [
    (64, 8, 64, 2, 270),     # groups in one tile; 2-byte types: a workgroup of their own
    (64, 4, 100, 4, 820),    # one tile, shares
    (128, 8, 90, 2, 820), (256, 5, 100, 3, 820), (256, 8, 90, 4, 820),
    (64, 8, 100, 4, 820),    # two tiles
    (128, 4, 90, 8, 820), (128, 16, 100, 2, 820), (64, 1, 60, 41, 820)])
def test_long_groups(zq, kind, D, G, seqs, each, width):
    """Drafted tokens, which share a product, over more than 4096 keys of a workgroup, each of which sees a row more."""
    KH = 8 if width == 270 else 2
    rows = 4300 if width == 270 else 13000
    x = Whole(kind, KH, D, 16, rows, seed=5)
    seq_of, lens = [], []
    for s in range(seqs):
        last = EDGES[s % 8] if s % 12 == 0 or width == 270 else rows - 3 * (s % 50)
        seq_of += [s] * each
        lens += [last - each + i for i in range(each)]
    check(zq, x, G, lens, seq_of, width, seqs)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, KH, G, lens", [
    (128, 8, 4, [5000]), (64, 1, 8, [20011]), (128, 2, 3, [9000, 10, 4000]), (256, 1, 2, [6001, 6000]), (128, 2, 17, [3001, 5]),
    (64, 1, 40, [2000]), (64, 1, 33, [700, 3]), (128, 4, 1, [1, 0, 20000, 127, 128, 129])])
def test_shares_and_joins(zq, kind, D, KH, G, lens):
    """One unit of keys a workgroup, and as many partials of a pair."""
    x = Whole(kind, KH, D, 16, max(lens) + 1, seed=6)
    check(zq, x, G, lens, None, 1300, len(lens))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_prompts(zq, kind):
    """Two prompts of hundreds of tokens, from the first row and behind held ones, and tokens of others."""
    x = Whole(kind, 2, 128, 16, 3000, seed=7)
    seq_of = [0] * 500 + [2] * 700 + [1] + [3] * 5 + [0]
    lens = list(range(500)) + list(range(2300, 3000)) + [2999] + [15, 16, 17, 18, 19] + [1200]
    for width in (190, 3000):
        check(zq, x, 4, lens, seq_of, width, 4)

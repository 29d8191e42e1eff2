"""Softmax weights far below the largest one, in attention over the paged KV cache (include/zq_paged.h): a first row that
takes nearly all of the weight, and many equal rows behind it whose share has a known value."""
import math

import numpy as np
import pytest
import torch

import paged_plain as P
from test_paged import DEV, KINDS, dev

gpu = pytest.mark.gpu

U = 2.0 ** -24
GAPS = [3.0 + 0.9375 * h for h in range(16)]  # how far the equal rows' score is below the first one's, a head each: to 17.06


def share(x, n):
    """What n - 1 rows have of the weight, x below one other row."""
    low = (n - 1) * math.exp(-x)
    return low / (1 + low)


def bound(x, n, kind, depth):
    """How far an output may be off that is the equal rows' share, and one that is 1.

    With u = 2^-24, relative to the equal rows' weight: the score (log2 units, x log2(e)) is off by the rounding of
    scale * log2(e), of the product and of the running maximum, half a step u each of at most 1.443 x, which moves a
    weight by ln 2 times that: 3 x u; the argument of the exponential (at most 1.443 x + 14) is rounded, another
    (x + 10) u, the exponential itself is off by 2 u.  Sums are of `depth` additions one after the other, of the numerator
    and the denominator: 2 depth u.  Quotient and rescalings: 8 u.  An fp16 cache's weights have 22 bits, 2^-22, or are
    multiples of 2^-38 of the largest, which is off by half of that: n 2^-39 in all, in the numerator alone."""
    s = share(x, n)
    own = (4 * x + 12 + 8 + 2 * depth) * U
    held = 2.0 ** -22 * s + n * 2.0 ** -39 * (1 - s) if kind == "f16" else 0.0
    largest = (2 * depth + 8 + 2) * U + (2.0 ** -22 + n * 2.0 ** -39 if kind == "f16" else 0.0)
    return s * own + held, largest


def test_the_bound_rejects_weights_of_few_bits():
    """Weights 2^6 of the largest in two fp16 parts, the second a multiple of 2^-24: the bound of an fp16 cache refuses
    them at some of the gaps, in both lengths that the tests use."""
    for n, depth in ((8190, 150), (1200, 912)):
        off = []
        for x in GAPS:
            w = np.float32(math.exp(-x) * 64)
            hi = np.float16(w)
            held = (float(hi) + float(np.float16(w - np.float32(hi)))) / 64
            got = (n - 1) * held / (1 + (n - 1) * math.exp(-x))
            off.append(abs(got - share(x, n)) > bound(x, n, "f16", depth)[0])
        assert sum(off) >= 3, (n, off)
        fine = []
        for x in GAPS:  # 2^14 of the largest
            w = np.float32(math.exp(-x) * 16384)
            hi = np.float16(w)
            held = (float(hi) + float(np.float16(w - np.float32(hi)))) / 16384
            fine.append(abs((n - 1) * held / (1 + (n - 1) * math.exp(-x)) - share(x, n)) <= bound(x, n, "f16", depth)[0])
        assert all(fine)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("queries", [1, 3, 9])
@pytest.mark.parametrize("n, spare, depth", [(8190, 3000, 150), (1200, 2, 912)], ids=["shares", "pairs"])
def test_many_rows_far_below_the_first(zq, kind, queries, n, spare, depth):
    """Values of 0 in the first row and 1 in the others (the first 32 elements), and of 1 in all rows.

    depth: with shares, a unit of 128 keys (fp32: 64) is a workgroup's, 32 keys a wave in three products at most, four waves
    are joined and then up to 130 partials by four waves, 96 + 4 + 33 + 4 and what rounds up; a workgroup of its own has
    304 keys a wave in three products."""
    D, ps, G = 64, 16, 16 if queries == 1 else 4
    pages = P.cdiv(n, ps)
    k = torch.zeros(pages * ps, D)
    v = torch.ones(pages * ps, D)
    k[0, 0] = 1
    v[0, :32] = 0
    k[n:], v[n:] = math.nan, math.nan
    order = np.random.default_rng(n).permutation(pages)
    pool = [torch.empty(pages, 1, ps, D, dtype=P.TYPES[kind]) for _ in range(2)]
    for x, to in zip((k, v), pool):
        to[torch.from_numpy(order), 0] = x.reshape(pages, ps, D).to(to.dtype)
    gk, gv = (x.to(DEV) for x in pool)
    gt = dev(np.concatenate([order, np.full(spare, -1)])[None])
    cache = zq.KVPaged(gk, gv, pages, 1, D, ps)
    tables = zq.PageTables(gt, None, 1, pages + spare, pages, ps)
    for first in range(0, 16, G):
        gaps = GAPS[first:first + G]
        q = torch.zeros(queries, G, D, device=DEV)
        q[:, :, 0] = torch.tensor(gaps)
        out = torch.full_like(q, math.nan)
        lens = list(range(n - queries, n))
        need = zq.attention_paged_workspace_bytes(cache, tables, queries, G)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        zq.attention_paged_dev(cache, tables, q, out, queries, G, dev(lens), 1.0,
                               seq_of=None if queries == 1 else dev([0] * queries), workspace=ws, workspace_bytes=need)
        got = out.cpu().double().numpy()
        for i, rows in enumerate(lens):
            for h, x in enumerate(gaps):
                low, all_ = bound(x, rows + 1, kind, depth)
                want = share(x, rows + 1)
                assert np.abs(got[i, h, :32] - want).max() <= low, (i, x, np.abs(got[i, h, :32] - want).max() / want)
                assert np.abs(got[i, h, 32:] - 1).max() <= all_, (i, x, np.abs(got[i, h, 32:] - 1).max())


@gpu
@pytest.mark.parametrize("queries", [1, 9])
def test_values_and_keys_below_the_least_normal_number(zq, queries):
    """An fp16 cache's rows are exact there too: values of 2^-24 .. 2^-21, and keys that make two scores of 0 and of 12 with
    queries of 3 * 2^24."""
    D, ps, G, n = 64, 16, 4, 700
    rng = np.random.default_rng(3)
    pages = P.cdiv(n, ps)
    v = rng.integers(-8, 9, (n, D))
    one = rng.integers(0, 2, n)
    k = np.zeros((pages * ps, D))
    k[:n, 5] = 4 * 2.0 ** -24 * one
    held = np.full((pages * ps, D), math.nan)
    held[:n] = v * 2.0 ** -24
    pool = [torch.from_numpy(x.reshape(pages, 1, ps, D)).half().to(DEV) for x in (k, held)]
    cache = zq.KVPaged(*pool, pages, 1, D, ps)
    tables = zq.PageTables(dev(np.arange(pages)[None]), None, 1, pages, pages, ps)
    q = torch.zeros(queries, G, D, device=DEV)
    q[:, :, 5] = 3 * 2.0 ** 24
    out = torch.full_like(q, math.nan)
    lens = list(range(n - queries, n))
    need = zq.attention_paged_workspace_bytes(cache, tables, queries, G)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    zq.attention_paged_dev(cache, tables, q, out, queries, G, dev(lens), 1.0, seq_of=None if queries == 1 else dev([0] * queries),
                           workspace=ws, workspace_bytes=need)
    got = out.cpu().double().numpy()
    for i, r in enumerate(lens):
        w = np.where(one[:r + 1] == 1, 1.0, math.exp(-12.0))
        want, size = (w[:, None] * v[:r + 1]).sum(0) / w.sum(), (w[:, None] * np.abs(v[:r + 1])).sum(0) / w.sum()
        # (the scores' rounding, 4 * 12 + 12 units, and sums of at most 3 * 700 / 4 additions, in values and weights)
        assert (np.abs(got[i] * 2.0 ** 24 - want) <= 2 * (60 + 525) * U * size + 2.0 ** -22 * size).all(), i

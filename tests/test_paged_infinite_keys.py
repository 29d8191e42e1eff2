"""Infinite keys in attention over the paged KV cache (include/zq_paged.h): a score of +infinity or NaN gives outputs that are
no numbers; one of -infinity may, or the row has no weight; other queries and heads see nothing of it."""
import math

import numpy as np
import pytest

import paged_plain as P
from test_paged import KINDS, Pool, queries, run_attention, spare  # noqa: F401 (spare is a fixture)

gpu = pytest.mark.gpu
ROW = 37  # of sequence 0, kv head 1


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_key(zq, kind, drafted, sign, spare):  # noqa: F811
    pool = Pool(zq, kind, [90, 60], 2, 64, 16, seed=30, spare_width=spare)
    seq_of, lens = ([0, 0, 0, 1], [36, 37, 89, 59]) if drafted else (None, [89, 59])
    q = queries(pool.rng, len(lens), 6, 64)
    q[:, :, 5] = np.abs(q[:, :, 5]) + 0.1
    q[:, 4, 5] = 0.5  # exact in every type
    want = np.empty((len(lens), 6, 64))
    tol = np.empty_like(want)
    for i, n in enumerate(lens):
        s = seq_of[i] if drafted else i
        for h in range(6):
            k, v = pool.rows(s, h // 3, n + 1)
            if s == 0 and h >= 3 and n >= ROW:  # without the row
                k, v = np.delete(k, ROW, 0), np.delete(v, ROW, 0)
            want[i, h], tol[i, h] = P.attention(q[i, h], k, v, 0.125, kind == "f16")
    pool.k[pool.table[0, ROW // 16], 1, ROW % 16, 5] = sign * math.inf
    pool.upload(zq)
    got = run_attention(zq, pool, q, lens, 0.125, seq_of=seq_of)
    for i, n in enumerate(lens):
        s = seq_of[i] if drafted else i
        for h in range(6):
            near = (np.abs(got[i, h] - want[i, h]) <= tol[i, h]).all()
            if s == 0 and h >= 3 and n >= ROW:
                none = not np.isfinite(got[i, h]).any()
                assert none or (sign < 0 and near), (i, h)
            else:
                assert near, (i, h)

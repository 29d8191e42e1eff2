"""Plain implementations in 64 bits, on the CPU, of the paged KV cache's operators (include/zq_paged.h), written from
their definitions, one sequence, token and head at a time."""
import math

import numpy as np
import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def cdiv(a, b):
    return -(-a // b)


def step(lens, counts, table, free, free_count, ps, pages, tokens):
    """(granted, start, slots, positions, seq_of, table, free_left)."""
    W = table.shape[1]
    table, stack = table.copy(), list(free[:max(0, min(free_count, pages))])
    top = len(stack)
    granted, start, slots, pos, seq = [], [0], [], [], []
    want_p = want_t = 0
    for s in range(len(lens)):
        n, c, got = min(max(lens[s], 0), W * ps), max(counts[s], 0), 0
        if n + c <= W * ps:
            want_t += c
            want_p += cdiv(n + c, ps) - cdiv(n, ps)
            if want_p <= top and want_t <= tokens:
                got = c
        for p in range(n, n + got):
            if p % ps == 0:
                table[s, p // ps] = stack.pop()
            page = int(table[s, p // ps])
            slots.append(page * ps + p % ps if 0 <= page < pages else -1)
            pos.append(p)
            seq.append(s)
        granted.append(got)
        start.append(start[-1] + got)
    pad = [-1] * (tokens - len(slots))
    return granted, start, slots + pad, pos + pad, seq + pad, table, len(stack)


def release(lens, keep, table, free, free_count, ps):
    """(free, free_left)."""
    cap, free, back = table.shape[1] * ps, free.copy(), []
    for s in range(len(lens)):
        n = min(max(lens[s], 0), cap)
        back += list(table[s, cdiv(min(max(keep[s], 0), n), ps):cdiv(n, ps)])
    for i, p in enumerate(reversed(back)):
        if free_count + i < len(free):
            free[free_count + i] = p
    return free, min(free_count + len(back), len(free))


def exponent(a):
    """The least e in -50 .. 50 with a <= 127 * 2^e (50 if there is none, -50 for 0)."""
    if a == 0:
        return -50
    if math.isinf(a):
        return 50
    e = math.frexp(a)[1] - 8
    while a > 127.0 * 2.0 ** e:
        e += 1
    return max(-50, min(50, e))


def bounds(rows):
    """(least [D], greatest [D], e) of a page's held rows [r][D], float64."""
    with np.errstate(invalid="ignore"):
        lo = np.fmin.reduce(rows, 0)
        hi = np.fmax.reduce(rows, 0)
    lo, hi = np.where(np.isnan(lo), 0.0, lo), np.where(np.isnan(hi), 0.0, hi)
    e = exponent(float(np.maximum(np.abs(lo), np.abs(hi)).max()))
    return (np.clip(np.floor(lo / 2.0 ** e), -127, 127).astype(np.int64),
            np.clip(np.ceil(hi / 2.0 ** e), -127, 127).astype(np.int64), e)


def seen(i, lens, counts, seq_of, seqs, cap, full):
    """(sequence or None, rows) of query i."""
    s = int(seq_of[i]) if seq_of is not None else i
    c = int(counts[i]) if counts is not None else 1
    if not 0 <= s < seqs or c <= 0:
        return None, 0
    n = min(max(int(lens[i]), 0), cap)
    return s, min(n + (0 if full else c), cap)


def scores(q, codes, exps):
    """Scores [n] of pages with bounds codes [n][2][D] and exps [n] for the heads q [G][D]."""
    best = np.full(len(exps), -np.inf)
    for row in q.astype(np.float64):
        a = np.abs(row)
        eq = exponent(float(np.fmax.reduce(a)) if not np.isnan(a).all() else 0.0)
        c = np.where(np.isnan(row), 0, np.clip(np.rint(row / 2.0 ** eq), -127, 127))
        best = np.maximum(best, np.maximum(c * codes[:, 0], c * codes[:, 1]).sum(-1) * 2.0 ** (eq + exps.astype(np.float64)))
    return best


def select(score, n, keep, recent, first):
    """Places of the pages that stay, ascending, of scores [n]."""
    if n <= keep:
        return list(range(n))
    must = lambda p: p < first or p >= n - recent
    return sorted(sorted(range(n), key=lambda p: (not must(p), 0.0 if must(p) else -score[p], p))[:keep])


def attention(q, k, v, scale, f16):
    """(out [D], tolerance) of one head over rows k, v [n][D].

    Per output row, with u = 2^-24, A = max_p sum_d |scale q_d k_pd|:
      - a score is off by at most A (D u + 2 u + 2^-21): D - 1 additions and the products in fp32 of every query
        part, the rounding of scale * log2(e) and of the product with it, and for an fp16 cache a query held in
        two fp16 parts (2^-11 * 2^-11 = 2^-22, as much again where they are summed); elements far below the
        row's largest are held to 2^-39 of that; the running maximum in log2 units adds 2 A u;
      - a weight's exponential and its own parts add 2^-22 + 2^-22 (parts of fp16: multiples of 2^-24 where the
        largest weight is 2^6 or more: 2^-31 of it a row, which is below n u in all), the sums over n rows 2 n u, the
        quotient, rescalings and joins 40 u;
      - a relative error e of every weight moves the output by at most 2 e max |v|."""
    n, D = k.shape
    if not n:
        return np.zeros(q.shape[-1]), 0.0
    x = q.astype(np.float64) * scale
    a = (np.abs(x) * np.abs(k)).sum(-1).max() * ((D + 4) * U + 2.0 ** -21)
    if f16:
        a += np.abs(x).max() * np.abs(k).sum(-1).max() * 2.0 ** -39
    p = k @ x
    p = np.exp(p - p.max())
    p /= p.sum()
    return p @ v, 2 * (a + 2.0 ** -21 + (2 * n + 40) * U) * np.abs(v).max()

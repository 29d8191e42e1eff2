"""The paged KV cache (include/zq_paged.h): page tables, append with bounds, selection and attention against plain
implementations in 64 bits (tests/paged_plain.py), and their refusals.  Tables, slots, held rows, bounds and the pages
selected are compared bit for bit; attention within the bound of its arithmetic (paged_plain.attention)."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

import paged_plain as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
ids = lambda o: ",".join(f"{k}={v}" for k, v in o.items()) if isinstance(o, dict) else None


# ---- CPU: the interface and its refusals ------------------------------------------
def test_header_and_binding_agree():
    from zeninfer_amd import zq
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "zq_paged.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(zq_hip_[a-z0-9_]+)\s*\(", text))
    assert declared == set(zq.PAGED_SIGNATURES)
    assert all(hasattr(zq.lib(), n) for n in declared)


def tables_of(zq, **over):
    f = dict(table=1 << 20, free_pages=2 << 20, seqs=3, width=8, pages=40, page_size=16)
    f.update(over)
    return zq.PageTablesC(*[f[n] for n, _ in zq.PageTablesC._fields_])


def cache_of(zq, **over):
    f = dict(k=3 << 20, v=4 << 20, bounds=5 << 20, bounds_exp=6 << 20, pages=40, kv_heads=2, head_dim=64, page_size=16,
             type=zq.KV_F16)
    f.update(over)
    return zq.KVCachePaged(*[f[n] for n, _ in zq.KVCachePaged._fields_])


def call_all(zq, cache, tables, X=7 << 20, **over):
    """Statuses of the five calls with arguments that are right but for those given (made-up addresses)."""
    L = zq.lib()
    f = dict(lens=X, counts=X, free_count=X, free_left=X, granted=X, start=X, slots=X, tokens=5, q=X, out=X, queries=3,
             heads=4, stride=0, seq_of=None, qcounts=None, select=None, keep=0, flags=0, ws=X, bytes=1 << 40, k=X, v=X,
             astride=0, skeep=4, recent=1, first=1, sselect=X)
    f.update(over)
    c, t = ctypes.byref(cache), ctypes.byref(tables)
    return {
        "step": L.zq_hip_page_tables_step_dev(t, f["lens"], f["counts"], f["free_count"], f["free_left"], f["granted"],
                                              f["start"], f["slots"], None, None, f["tokens"], None),
        "release": L.zq_hip_page_tables_release_dev(t, f["lens"], f["counts"], f["free_count"], f["free_left"], None),
        "append": L.zq_hip_kv_paged_append_dev(c, f["k"], f["v"], f["tokens"], f["astride"], f["slots"], None),
        "attention": L.zq_hip_attention_paged_dev(c, t, f["q"], f["out"], f["queries"], f["heads"], f["stride"],
                                                  f["seq_of"], f["lens"], f["qcounts"], f["select"], f["keep"], 1.0,
                                                  f["flags"], f["ws"], f["bytes"], None),
        "select": L.zq_hip_page_select_dev(c, t, f["q"], f["sselect"], f["queries"], f["heads"], f["stride"], f["seq_of"],
                                           f["lens"], f["qcounts"], f["skeep"], f["recent"], f["first"], f["flags"],
                                           f["ws"], f["bytes"], None),
        "attention_bytes": L.zq_hip_attention_paged_workspace_bytes(c, t, f["queries"], f["heads"]),
        "select_bytes": L.zq_hip_page_select_workspace_bytes(c, t, f["queries"], f["heads"], f["skeep"]),
    }


CALLS = ("step", "release", "append", "attention", "select")


@pytest.mark.parametrize("over", [
    dict(table=None), dict(table=(1 << 20) + 2), dict(free_pages=(2 << 20) + 1), dict(seqs=0), dict(seqs=8193),
    dict(width=0), dict(width=(1 << 20) + 1), dict(pages=0), dict(pages=(1 << 24) + 1), dict(page_size=0),
    dict(page_size=8), dict(page_size=24), dict(page_size=512), dict(width=1 << 63), dict(seqs=1 << 63)], ids=ids)
def test_calls_refuse_bad_tables(over):
    from zeninfer_amd import zq
    r = call_all(zq, cache_of(zq, page_size=over.get("page_size", 16)), tables_of(zq, **over))
    for name in ("step", "release", "attention", "select"):
        assert r[name] == zq.ERR_ARG, name
    assert r["attention_bytes"] == r["select_bytes"] == 0


@pytest.mark.parametrize("over", [
    dict(k=None), dict(v=None), dict(k=(3 << 20) + 8), dict(v=(4 << 20) + 4), dict(bounds=(5 << 20) + 4), dict(bounds=None),
    dict(bounds_exp=None), dict(pages=0), dict(pages=(1 << 24) + 1), dict(kv_heads=0), dict(kv_heads=1025),
    dict(head_dim=0), dict(head_dim=96), dict(head_dim=32), dict(page_size=15), dict(page_size=512), dict(type=3),
    dict(type=-1)], ids=ids)
def test_calls_refuse_a_bad_cache(over):
    from zeninfer_amd import zq
    r = call_all(zq, cache_of(zq, **over), tables_of(zq))
    for name in ("append", "attention", "select"):
        assert r[name] == zq.ERR_ARG, name
    assert r["attention_bytes"] == r["select_bytes"] == 0


@pytest.mark.parametrize("over, refused", [
    (dict(lens=None), "step release attention select"), (dict(lens=(7 << 20) + 2), "step release attention select"),
    (dict(counts=None), "step release"), (dict(counts=(7 << 20) + 1), "step release"),
    (dict(free_count=None), "step release"), (dict(free_left=None), "step release"),
    (dict(free_left=(7 << 20) + 2), "step release"), (dict(granted=None), "step"), (dict(start=None), "step"),
    (dict(slots=None), "step append"), (dict(slots=(7 << 20) + 4), "step append"), (dict(tokens=0), "step append"),
    (dict(tokens=(1 << 24) + 1), "step append"), (dict(tokens=1 << 63), "step append"), (dict(k=None), "append"),
    (dict(v=None), "append"), (dict(k=(7 << 20) + 4), "append"), (dict(astride=124), "append"),
    (dict(astride=130), "append"), (dict(astride=(1 << 31) + 4), "append"), (dict(q=None), "attention select"),
    (dict(q=(7 << 20) + 8), "attention select"), (dict(out=None), "attention"), (dict(out=(7 << 20) + 4), "attention"),
    (dict(queries=0), "attention select"), (dict(queries=4), "attention select"),
    (dict(queries=8193, seq_of=7 << 20), "attention select"), (dict(heads=0), "attention select"),
    (dict(heads=3), "attention select"), (dict(heads=1026), "attention select"), (dict(stride=252), "attention select"),
    (dict(stride=258), "attention select"), (dict(seq_of=(7 << 20) + 2), "attention select"),
    (dict(qcounts=(7 << 20) + 2), "attention select"), (dict(flags=2), "attention select"),
    (dict(select=7 << 20), "attention"), (dict(select=7 << 20, keep=(1 << 20) + 1), "attention"),
    (dict(select=(7 << 20) + 2, keep=2), "attention"), (dict(ws=None), "attention select"),
    (dict(ws=(7 << 20) + 8), "attention select"), (dict(bytes=64), "attention select"), (dict(skeep=0), "select"),
    (dict(sselect=None), "select"), (dict(recent=4), "select"), (dict(first=4), "select"), (dict(recent=1 << 63), "select"),
    (dict(first=(1 << 64) - 1), "select"), (dict(skeep=(1 << 20) + 1), "select")], ids=ids)
def test_calls_refuse_bad_arguments(over, refused):
    from zeninfer_amd import zq
    r = call_all(zq, cache_of(zq), tables_of(zq), **over)
    for name in refused.split():
        assert r[name] == zq.ERR_ARG, name


def test_calls_refuse_tables_of_another_pool():
    from zeninfer_amd import zq
    for c, t in ((dict(pages=39), {}), (dict(page_size=32), {}), ({}, dict(page_size=32))):
        r = call_all(zq, cache_of(zq, **c), tables_of(zq, **t))
        assert r["attention"] == r["select"] == zq.ERR_ARG and r["attention_bytes"] == r["select_bytes"] == 0
    r = call_all(zq, cache_of(zq), tables_of(zq, free_pages=None))
    assert r["step"] == r["release"] == zq.ERR_ARG and r["attention_bytes"] > 0
    r = call_all(zq, cache_of(zq, bounds=None, bounds_exp=None), tables_of(zq))
    assert r["select"] == zq.ERR_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="answers without a GPU")
def test_calls_without_a_gpu():
    from zeninfer_amd import zq
    r = call_all(zq, cache_of(zq), tables_of(zq))
    assert all(r[name] == zq.ERR_NO_DEVICE for name in CALLS)


def test_wrappers_refuse_wrong_buffers(monkeypatch):
    from zeninfer_amd import zq
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype)
    half = dict(dtype=torch.float16)
    with pytest.raises(ValueError, match="table: needs int32"):
        zq.PageTables(z(3, 8, dtype=torch.int64), z(40), 3, 8, 40, 16)
    with pytest.raises(ValueError, match="free_pages: buffer holds"):
        zq.PageTables(z(3, 8), z(39), 3, 8, 40, 16)
    with pytest.raises(ValueError, match="below zero"):
        zq.PageTables(z(3, 8), z(40), -3, 8, 40, 16)
    t = zq.PageTables(z(3, 8), z(40), 3, 8, 40, 16)
    pool = lambda **kw: z(40, 2, 16, 64, **{"dtype": torch.float16, **kw})
    with pytest.raises(ValueError, match="KVPaged k: needs float32"):
        zq.KVPaged(pool(dtype=torch.int16), pool(), 40, 2, 64, 16)
    with pytest.raises(ValueError, match="not of the cache's type"):
        zq.KVPaged(pool(), pool(dtype=torch.bfloat16), 40, 2, 64, 16)
    with pytest.raises(ValueError, match="KVPaged v: buffer holds"):
        zq.KVPaged(pool(), pool()[:39], 40, 2, 64, 16)
    with pytest.raises(ValueError, match="no type"):
        zq.KVPaged(1 << 20, 2 << 20, 40, 2, 64, 16)
    with pytest.raises(ValueError, match="bounds: needs int8"):
        zq.KVPaged(pool(), pool(), 40, 2, 64, 16, bounds=z(40, 2, 2, 64), bounds_exp=z(40, 2, dtype=torch.int8))
    with pytest.raises(ValueError, match="bounds_exp: buffer holds"):
        zq.KVPaged(pool(), pool(), 40, 2, 64, 16, bounds=z(40, 2, 2, 64, dtype=torch.int8),
                   bounds_exp=z(39, 2, dtype=torch.int8))
    c = zq.KVPaged(pool(), pool(), 40, 2, 64, 16)
    i = z(3)
    with pytest.raises(ValueError, match="slots: needs int64"):
        zq.page_tables_step_dev(t, i, i, z(1), z(1), i, z(4), z(5), None, None, 5)
    with pytest.raises(ValueError, match="start: buffer holds"):
        zq.page_tables_step_dev(t, i, i, z(1), z(1), i, z(3), z(5, dtype=torch.int64), None, None, 5)
    with pytest.raises(ValueError, match="keep: needs int32"):
        zq.page_tables_release_dev(t, i, z(3, dtype=torch.int64), z(1), z(1))
    f = lambda *s: torch.zeros(*s)
    with pytest.raises(ValueError, match="append_dev k: buffer holds"):
        zq.kv_paged_append_dev(c, f(4, 2, 64), f(5, 2, 64), 5, z(5, dtype=torch.int64))
    with pytest.raises(ValueError, match="append_dev v: needs float32"):
        zq.kv_paged_append_dev(c, f(5, 2, 64), torch.zeros(5, 2, 64, **half), 5, z(5, dtype=torch.int64))
    with pytest.raises(ValueError, match="rows must be 200"):
        zq.kv_paged_append_dev(c, f(5, 300)[:, :128], f(5, 200)[:, :128], 5, z(5, dtype=torch.int64), stride=200)
    with pytest.raises(ValueError, match="q: buffer holds"):
        zq.attention_paged_dev(c, t, f(2, 4, 64), f(3, 4, 64), 3, 4, i, 1.0)
    with pytest.raises(ValueError, match="select: buffer holds"):
        zq.attention_paged_dev(c, t, f(3, 4, 64), f(3, 4, 64), 3, 4, i, 1.0, select=z(3, 2, 3), keep=4)
    with pytest.raises(ValueError, match="seq_of: needs int32"):
        zq.attention_paged_dev(c, t, f(3, 4, 64), f(3, 4, 64), 3, 4, i, 1.0, seq_of=z(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="below zero"):
        zq.page_select_dev(c, t, f(3, 4, 64), z(3, 2, 4), 3, 4, i, 4, recent=-1)
    with pytest.raises(ValueError, match="select: buffer holds"):
        zq.page_select_dev(c, t, f(3, 4, 64), z(3, 2, 3), 3, 4, i, 4)


def test_plain_exponent_and_bounds():
    for a, e in ((127.0, 0), (127.0000001, 1), (64.0, 0), (63.5, -1), (1e-30, -50), (1e30, 50), (math.inf, 50), (0.0, -50)):
        assert P.exponent(a) == e, a
    lo, hi, e = P.bounds(np.array([[1.0, -3.0, np.nan, np.nan], [2.5, 127.0, np.nan, 0.25]]))
    assert e == 0 and list(lo) == [1, -3, 0, 0] and list(hi) == [3, 127, 0, 1]


# ---- GPU ------------------------------------------------------------------------------
gpu = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(dtype).to(DEV)


def run_step(zq, lens, counts, table, free, free_count, ps, pages, tokens, in_place=False, extra=True, stream=None):
    S, W = table.shape
    t, f = dev(table), dev(free)
    h = zq.PageTables(t, f, S, W, pages, ps)
    fc, counts = dev([free_count]), dev(counts)
    left = fc if in_place else dev([-7])
    granted = counts if in_place else dev([-7] * S)
    start, slots = dev([-7] * (S + 1)), dev([-7] * tokens, torch.int64)
    pos, seq = (dev([-7] * tokens), dev([-7] * tokens)) if extra else (None, None)
    zq.page_tables_step_dev(h, dev(lens), counts, fc, left, granted, start, slots, pos, seq, tokens, stream=stream)
    torch.cuda.synchronize()
    out = [x.cpu().numpy() if x is not None else None for x in (granted, start, slots, pos, seq, t)]
    assert (f.cpu().numpy() == free).all()
    return out + [int(left)]


def check_step(zq, lens, counts, table, free, free_count, ps, pages, tokens, **kw):
    got = run_step(zq, lens, counts, table, free, free_count, ps, pages, tokens, **kw)
    want = P.step(lens, counts, table, free, free_count, ps, pages, tokens)
    for name, g, w in zip(("granted", "start", "slots", "positions", "seq_of", "table", "free_left"), got, want):
        if g is not None:
            assert np.array_equal(g, np.asarray(w)), name
    return want


def full_table(rng, lens, W, ps, pages):
    """A table whose sequences have the pages of their lengths, and the stack of the others."""
    order = rng.permutation(pages)
    table, at = np.full((len(lens), W), -1, np.int64), 0
    for s, n in enumerate(lens):
        c = min(P.cdiv(max(n, 0), ps), W)
        table[s, :c] = order[at:at + c]
        at += c
    free = np.full(pages, -5, np.int64)
    free[:pages - at] = order[at:]
    return table, free, pages - at


@gpu
@pytest.mark.parametrize("S, ps, most_len, most_new, spare, room", [
    (1, 16, 0, 1, 1.0, 1), (1, 16, 16, 1, 1.0, 3), (1, 256, 255, 2, 1.0, 2), (5, 16, 60, 40, 1.0, 1.0), (7, 32, 100, 64, 0.5, 1.2),
    (64, 64, 500, 3, 1.0, 0.6), (300, 16, 90, 20, 0.7, 1.0), (1025, 16, 40, 1, 1.0, 1.0), (2500, 32, 70, 9, 0.8, 1.1),
    (8192, 16, 20, 2, 0.9, 1.0)])
def test_step(zq, S, ps, most_len, most_new, spare, room):
    rng = np.random.default_rng(S + ps)
    lens = rng.integers(0, most_len + 1, S)
    counts = rng.integers(0, most_new + 1, S) if S > 1 else np.array([most_new])
    W = P.cdiv(most_len + most_new, ps)
    need = sum(P.cdiv(n + c, ps) for n, c in zip(lens, counts))
    held = sum(P.cdiv(n, ps) for n in lens)
    pages = held + max(1, int((need - held) * spare))
    table, free, fc = full_table(rng, lens, W, ps, pages)
    tokens = max(1, int(counts.sum() * room)) if isinstance(room, float) else room
    for kw in (dict(), dict(in_place=True, extra=False)):
        check_step(zq, lens, counts, table, free, fc, ps, pages, tokens, **kw)


@gpu
def test_step_edges(zq):
    """Lengths below zero and past the table, sequences that do not fit among those that do, a stack whose count or
    pages are wrong, entries that are no pages, counts near 2^31, nothing to do."""
    ps, W, pages = 16, 3, 20
    table = np.array([[0, 1, 2], [3, -1, -1], [-1, -1, -1], [99, 4, 5], [6, 7, 8]])
    free = np.array([9, 10, 40, 11, -1, 12] + [-1] * 14)
    for lens, counts, fc, tokens in [
            ([48, 5, -3, 20, 33], [1, 20, 7, 4, 2], 6, 64),      # the first is full, the fourth sits behind a bad entry
            ([47, 5, 0, 10, 33], [2, 20, 48, 4, 16], 6, 100),    # the first does not fit, those behind it do
            ([40, 16, 0, 30, 31], [8, 16, 17, 18, 17], 6, 59),   # rows run out
            ([40, 16, 0, 30, 31], [8, 16, 17, 18, 17], 2, 99),   # pages run out
            ([100, 16, 0, 30, 31], [0, 2 ** 31 - 1, -5, 2 ** 31 - 1, 1], 6, 9),
            ([1, 2, 3, 4, 5], [1, 1, 1, 1, 1], -4, 9), ([16, 2, 0, 4, 5], [1, 1, 1, 1, 1], 99, 9),
            ([1, 2, 3, 4, 5], [0, 0, 0, 0, 0], 6, 4)]:
        check_step(zq, lens, counts, table, free, fc, ps, pages, tokens)


@gpu
@pytest.mark.parametrize("S, ps, most", [(1, 16, 1), (1, 16, 64), (3, 32, 200), (100, 16, 300), (700, 16, 500), (8192, 16, 17)])
def test_release(zq, S, ps, most):
    rng = np.random.default_rng(S)
    lens = rng.integers(0, most + 1, S)
    lens[0] = most
    keep = np.where(rng.random(S) < 0.4, 0, np.maximum(-1, lens - rng.integers(-3, 40, S)))
    W = P.cdiv(most, ps) + 1
    pages = sum(P.cdiv(n, ps) for n in lens) + 5
    table, free, fc = full_table(rng, lens, W, ps, pages)
    for in_place in (False, True):
        t, f = dev(table), dev(free)
        h = zq.PageTables(t, f, S, W, pages, ps)
        c = dev([fc])
        left = c if in_place else dev([-1])
        zq.page_tables_release_dev(h, dev(lens), dev(keep), c, left)
        want, n = P.release(lens, keep, table, free, fc, ps)
        assert np.array_equal(f.cpu().numpy(), want) and int(left) == n and np.array_equal(t.cpu().numpy(), table)


@gpu
def test_release_of_more_than_the_pool_ends_at_its_end(zq):
    table = np.array([[0, 1, 2], [3, 4, 5]])
    free = np.array([7, 8, -1, -1, -1, -1, -1, -1, -1])
    f, left = dev(free), dev([-1])
    h = zq.PageTables(dev(table), f, 2, 3, 9, 16)
    zq.page_tables_release_dev(h, dev([48, 200]), dev([0, 0]), dev([5]), left)
    want, n = P.release([48, 200], [0, 0], table, free, 5, 16)
    assert np.array_equal(f.cpu().numpy(), want) and int(left) == n == 9


@gpu
def test_release_undoes_a_step(zq):
    rng = np.random.default_rng(5)
    lens, counts = rng.integers(0, 70, 40), rng.integers(0, 50, 40)
    table, free, fc = full_table(rng, lens, 8, 16, 400)
    t, f, c = dev(table), dev(free), dev([fc])
    h = zq.PageTables(t, f, 40, 8, 400, 16)
    granted, start = dev([0] * 40), dev([0] * 41)
    slots = dev([0] * 3000, torch.int64)
    zq.page_tables_step_dev(h, dev(lens), dev(counts), c, c, granted, start, slots, None, None, 3000)
    assert int(c) < fc and int(start[-1]) == counts.sum()
    zq.page_tables_release_dev(h, dev(lens) + granted, dev(lens), c, c)
    assert int(c) == fc and np.array_equal(f.cpu().numpy(), free)


class Pool:
    """A cache on the GPU and its rows on the host; everything that no sequence holds is NaN."""

    def __init__(self, zq, kind, lens, KH, D, ps, seed, extra_pages=3, bounds=True, spare_width=2, fill=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.kind, self.KH, self.D, self.ps, self.lens = kind, KH, D, ps, list(lens)
        counts = [P.cdiv(n, ps) for n in lens]
        self.S, self.pages, self.W = len(lens), sum(counts) + extra_pages, max(counts + [1]) + spare_width
        self.table, self.free, self.fc = full_table(rng, lens, self.W, ps, self.pages)
        self.k = torch.full((self.pages, KH, ps, D), math.nan, dtype=P.TYPES[kind])
        self.v = self.k.clone()
        wide = np.where(rng.random((KH, 1, D)) < 0.06, 5.0, 1.0) * fill
        for s, n in enumerate(lens):
            for j in range(counts[s]):
                r = min(ps, n - j * ps)
                x = torch.from_numpy(rng.standard_normal((2, KH, r, D)))
                self.k[self.table[s, j], :, :r] = (x[0] * torch.from_numpy(wide)).to(self.k.dtype)
                self.v[self.table[s, j], :, :r] = (x[1] * 0.7).to(self.v.dtype)
        self.codes = np.full((self.pages, KH, 2, D), 77, np.int64)
        self.exps = np.full((self.pages, KH), 99, np.int64)
        if bounds:
            for s, n in enumerate(lens):
                for j in range(counts[s]):
                    self.rebound(self.table[s, j], min(ps, n - j * ps))
        self.upload(zq)

    def rebound(self, page, rows):
        for h in range(self.KH):
            lo, hi, e = P.bounds(self.k[page, h, :rows].double().numpy())
            self.codes[page, h, 0], self.codes[page, h, 1], self.exps[page, h] = lo, hi, e

    def upload(self, zq):
        self.gk, self.gv = self.k.to(DEV), self.v.to(DEV)
        self.gb, self.ge = dev(self.codes, torch.int8), dev(self.exps, torch.int8)
        self.gt = dev(self.table)
        self.cache = zq.KVPaged(self.gk, self.gv, self.pages, self.KH, self.D, self.ps, bounds=self.gb, bounds_exp=self.ge)
        self.tables = zq.PageTables(self.gt, None, self.S, self.W, self.pages, self.ps)

    def rows(self, s, h, n, places=None):
        """Keys and values (float64) of the first n rows of sequence s that lie in the pages at `places`."""
        k, v = [], []
        for j in (range(P.cdiv(n, self.ps)) if places is None else places):
            page = int(self.table[s, j]) if 0 <= j < self.W else -1
            r = min(self.ps, n - j * self.ps)
            if j < 0 or r <= 0 or not 0 <= page < self.pages:
                continue
            k.append(self.k[page, h, :r].double().numpy())
            v.append(self.v[page, h, :r].double().numpy())
        return (np.concatenate(k), np.concatenate(v)) if k else (np.zeros((0, self.D)),) * 2

    def attend(self, q, lens, scale, counts=None, seq_of=None, select=None, full=False):
        """(out, tolerance) [n][H][D], NaN where nothing is written."""
        n, H, D = q.shape
        G = H // self.KH
        out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
        for i in range(n):
            s, rows = P.seen(i, lens, counts, seq_of, self.S, self.W * self.ps, full)
            if s is None:
                continue
            for h in range(H):
                places = None
                if select is not None:
                    places = list(select[i, h // G])[:min(select.shape[-1], P.cdiv(rows, self.ps))]
                k, v = self.rows(s, h // G, rows, places)
                out[i, h], tol[i, h] = P.attention(q[i, h], k, v, scale, self.kind == "f16")
        return out, tol

    def choose(self, q, lens, keep, recent, first, counts=None, seq_of=None, full=False, was=-9):
        n, H, D = q.shape
        G = H // self.KH
        out = np.full((n, self.KH, keep), was, np.int64)
        for i in range(n):
            s, rows = P.seen(i, lens, counts, seq_of, self.S, self.W * self.ps, full)
            if s is None:
                continue
            N = P.cdiv(rows, self.ps)
            page = self.table[s, :N]
            bad = (page < 0) | (page >= self.pages)
            for h in range(self.KH):
                sc = P.scores(q[i, h * G:(h + 1) * G], self.codes[np.where(bad, 0, page), h], self.exps[np.where(bad, 0, page), h])
                best = P.select(np.where(bad, -np.inf, sc), N, keep, recent, first)
                out[i, h] = best + [-1] * (keep - len(best))
        return out


def run_attention(zq, pool, q, lens, scale, counts=None, seq_of=None, select=None, full=False, stride=0, stream=None, was=math.nan):
    n, H, D = q.shape
    if stride:
        wide = torch.full((n, stride), math.nan, device=DEV)
        wide[:, :H * D] = torch.from_numpy(q).reshape(n, -1).float().to(DEV)
        gq = wide[:, :H * D]
    else:
        gq = torch.from_numpy(q).float().to(DEV)
    out = torch.full((n, H, D), was, device=DEV)
    need = zq.attention_paged_workspace_bytes(pool.cache, pool.tables, n, H)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)  # NaN, and a guard behind it
    opt = lambda x: None if x is None else dev(x)
    zq.attention_paged_dev(pool.cache, pool.tables, gq, out, n, H, dev(lens), scale, counts=opt(counts), seq_of=opt(seq_of),
                           select=opt(select), keep=0 if select is None else select.shape[-1], stride=stride,
                           flags=zq.ATTN_PAGED_FULL if full else 0, workspace=ws, workspace_bytes=need, stream=stream)
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all()
    return out.cpu().numpy()


def check_attention(zq, pool, q, lens, scale, **kw):
    got = run_attention(zq, pool, q, lens, scale, **kw)
    kw.pop("stride", None)
    want, tol = pool.attend(q, lens, scale, **kw)
    idle = np.isnan(want)
    assert (np.isnan(got) == idle).all(), "idle queries, or NaN"
    err = np.abs(got.astype(np.float64) - want)[~idle]
    assert (err <= tol[~idle]).all(), (err / np.maximum(tol[~idle], 1e-300)).max()
    return got


def queries(rng, n, H, D, size=1.0):
    return (rng.standard_normal((n, H, D)) * size).astype(np.float32)


KINDS = ("f16", "bf16", "f32")


@pytest.fixture(params=[2, 3000], ids=["pairs", "shares"])
def spare(request):
    """Entries of the tables that no sequence uses.  With few, a (query, kv head) pair has a workgroup of its own; with
    many, pairs are cut into shares and joined."""
    return request.param


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps, KH, G, lens", [
    (16, 2, 4, [1, 16, 17, 300]), (64, 1, 1, [63, 64, 65, 129]), (256, 3, 7, [500, 2]), (32, 2, 16, [33, 700, 31])])
def test_attention(zq, kind, D, ps, KH, G, lens, spare):
    pool = Pool(zq, kind, lens, KH, D, ps, seed=D + ps, spare_width=spare)
    held = [n - 1 for n in lens]
    check_attention(zq, pool, queries(pool.rng, len(lens), KH * G, D), held, 1 / math.sqrt(D))


@gpu
@pytest.mark.parametrize("kind, D, KH, G, lens", [
    ("f16", 128, 8, 4, [5000]), ("bf16", 64, 1, 8, [20011]), ("f32", 128, 2, 3, [9000, 10, 4000]),
    ("f16", 256, 1, 2, [6001, 6000]), ("bf16", 128, 2, 17, [3001, 5]), ("f16", 64, 1, 40, [2000]), ("f32", 64, 1, 33, [700, 3])])
def test_attention_split_over_workgroups(zq, kind, D, KH, G, lens):
    pool = Pool(zq, kind, lens, KH, D, 16, seed=G)
    a = check_attention(zq, pool, queries(pool.rng, len(lens), KH * G, D), [n - 1 for n in lens], 1 / math.sqrt(D))
    assert np.isfinite(a).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_lengths_counts_and_idle_queries(zq, kind):
    """Lengths below zero and past the table, counts of zero and below, sequences that are none; FULL with no rows."""
    pool = Pool(zq, kind, [40, 100, 200, 16, 0], 2, 64, 16, seed=3, spare_width=0)
    cap = pool.W * 16
    for s in (0, 1, 3, 4):  # what is behind a sequence is no page
        assert (pool.table[s, P.cdiv(pool.lens[s], 16):] == -1).all()
    n = 9
    q = queries(pool.rng, n, 6, 64)
    seq_of = [0, 1, 2, 3, 4, 2, -1, 5, 2]
    for lens, counts, full in (([39, 90, cap + 50, 10, -3, 0, 5, 5, 100], None, False),
                               ([30, 90, 10, 15, 0, -20, 5, 5, 100], [10, 10, 0, 1, -1, 3, 1, 1, 2 ** 31 - 1], False),
                               ([39, 0, cap + 50, 10, -3, -2, 5, 5, 100], None, True),
                               ([39, 0, cap, 10, 0, 0, 5, 5, 100], [1, 1, 0, 1, 1, 5, 1, 1, 1], True)):
        got = check_attention(zq, pool, q, lens, 0.125, counts=counts, seq_of=seq_of, full=full)
        if full:
            assert (got[1] == 0).all()


@gpu
@pytest.mark.parametrize("kind, G, n", [("f16", 4, 1500), ("bf16", 9, 1025), ("f32", 1, 3001), ("f16", 8, 8192)])
def test_attention_of_more_queries_than_a_workgroup_holds(zq, kind, G, n):
    pool = Pool(zq, kind, [90, 17, 200], 1, 64, 16, seed=n, spare_width=3000)
    seq_of = pool.rng.integers(-1, 3, n)
    if n != 1025:
        seq_of = np.sort(seq_of)
    lens = [int(pool.rng.integers(0, pool.lens[max(s, 0)])) for s in seq_of]
    check_attention(zq, pool, queries(pool.rng, n, G, 64), lens, 0.125, seq_of=seq_of)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_queries_that_share_a_sequence(zq, kind, spare):
    pool = Pool(zq, kind, [700, 33], 2, 128, 32, seed=4, spare_width=spare)
    seq_of = [0] * 37 + [1] * 33 + [-1] * 3
    lens = list(range(663, 700)) + list(range(33)) + [0] * 3
    check_attention(zq, pool, queries(pool.rng, len(lens), 8, 128), lens, 0.09, seq_of=seq_of)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_over_selected_pages(zq, kind, spare):
    """Any order, places twice, past the rows seen, none; fewer pages than keep."""
    pool = Pool(zq, kind, [333, 40, 500], 2, 64, 16, seed=6, spare_width=spare)
    K = 9
    select = np.full((3, 2, K), -1)
    select[0, 0] = [20, 3, 3, 0, 19, -1, 7, 1000, 5]
    select[0, 1] = [0, 1, 2, 3, 4, 5, 6, 7, 8]
    select[1, 0, :3] = [2, 0, 1]
    select[1, 1, :3] = [2, 2, -7]
    select[2, 0] = [31] * 9
    select[2, 1] = [-1] * 9  # nothing is seen: zeros
    got = check_attention(zq, pool, queries(pool.rng, 3, 6, 64), [332, 39, 499], 0.2, select=select)
    assert (got[2, 3:] == 0).all()
    check_attention(zq, pool, queries(pool.rng, 3, 6, 64), [332, 39, 499], 0.2, select=select[..., :1].copy())


@gpu
def test_attention_pages_that_were_given_up(zq, spare):
    pool = Pool(zq, "f16", [300, 64], 2, 128, 16, seed=8, spare_width=spare)
    pool.table[0, [0, 1, 2, 7]] = [-1, pool.pages, 2 ** 31 - 1, -2 ** 31]
    pool.table[1, :4] = -1
    pool.upload(zq)
    got = check_attention(zq, pool, queries(pool.rng, 2, 4, 128), [299, 63], 0.1)
    assert (got[1] == 0).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_strides_scales_and_peaks(zq, kind, spare):
    """Columns of a packed row; a negative scale, zero and one so large that one row takes all; rows far apart in size."""
    pool = Pool(zq, kind, [200, 77], 2, 64, 32, seed=9, spare_width=spare)
    q = queries(pool.rng, 2, 6, 64)
    for scale in (0.125, -0.3, 0.0, 30.0):
        check_attention(zq, pool, q, [199, 76], scale, stride=6 * 64 + 128)
    check_attention(zq, pool, q * np.float32(1e-30), [199, 76], 1.0)
    q[:, :, 0] *= 3e4
    check_attention(zq, pool, q, [199, 76], 1e-3)
    q[1] = 0
    check_attention(zq, pool, q, [199, 76], 1e-3)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_nan_and_infinity_reach_only_those_who_see_them(zq, kind, spare):
    pool = Pool(zq, kind, [100, 100], 2, 64, 16, seed=10, spare_width=spare)
    pool.k[pool.table[0, 3], 1, 5, 7] = math.nan      # row 53 of kv head 1
    pool.v[pool.table[1, 2], 0, 0, 9] = math.inf      # row 32 of kv head 0
    pool.upload(zq)
    q = queries(pool.rng, 6, 4, 64)
    q[5, 1, 3] = math.nan
    got = run_attention(zq, pool, q, [52, 53, 99, 31, 99, 20], 0.125, seq_of=[0, 0, 0, 1, 1, 1])
    bad = np.zeros((6, 4, 64), bool)
    bad[1:3, 2:] = True
    bad[4, :2, 9] = True
    bad[5, 1] = True
    assert (np.isfinite(got) == ~bad).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G, each", [(8, 8), (3, 23), (16, 5), (1, 50), (7, 9)])
def test_attention_of_many_drafted_tokens(zq, kind, D, G, each):
    """More queries a sequence than one tile of rows takes, and long tables: two tiles."""
    pool = Pool(zq, kind, [1500, 200, 77], 1, D, 16, seed=G, spare_width=3000)
    seq_of = np.repeat([0, 1, 2], each)
    lens = np.concatenate([np.arange(n - each, n) for n in pool.lens])
    check_attention(zq, pool, queries(pool.rng, 3 * each, G, D), lens, 0.1, seq_of=seq_of)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_a_value_that_is_no_number_reaches_only_the_drafted_tokens_that_see_it(zq, kind, D, value, spare):
    """Queries of one sequence share products; each of them sees one row more."""
    pool = Pool(zq, kind, [70], 2, D, 16, seed=13, spare_width=spare)
    pool.v[pool.table[0, 4], 1, 1, 9] = value      # row 65 of kv head 1
    pool.v[pool.table[0, 3], 0, 15, D - 1] = -value   # row 63 of kv head 0
    pool.upload(zq)
    lens = list(range(58, 70))
    got = run_attention(zq, pool, queries(pool.rng, 12, 6, D), lens, 0.125, seq_of=[0] * 12)
    bad = np.zeros((12, 6, D), bool)
    for i, n in enumerate(lens):
        bad[i, 3:, 9] = n >= 65
        bad[i, :3, D - 1] = n >= 63
    assert (np.isfinite(got) == ~bad).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 9, 16, 17])
def test_attention_of_drafted_tokens(zq, kind, D, G, spare):
    """Runs of queries of one sequence, of all lengths, in any order of lengths, idle ones among them."""
    pool = Pool(zq, kind, [400, 40, 17, 1], 2, D, 16, seed=G, spare_width=spare)
    seq_of = [0] * 21 + [1] * 3 + [2] + [0] + [3] + [1] * 9 + [-1] + [1] * 2
    lens = [int(pool.rng.integers(0, pool.lens[max(s, 0)])) for s in seq_of]
    counts = [int(pool.rng.integers(0, 3)) for _ in seq_of]
    for c in (None, counts):
        if c is not None:
            lens = [min(n, pool.lens[max(s, 0)] - x) for n, s, x in zip(lens, seq_of, c)]
        check_attention(zq, pool, queries(pool.rng, len(lens), 2 * G, D), lens, 0.125, seq_of=seq_of, counts=c)


@gpu
def test_attention_of_infinite_scores_and_a_spread_of_sizes(zq, spare):
    """Keys so large that the scores of the reference are past fp32's range in exp only: the largest takes all."""
    pool = Pool(zq, "bf16", [90], 1, 64, 16, seed=11, fill=1e4, spare_width=spare)
    check_attention(zq, pool, queries(pool.rng, 1, 3, 64, 100.0), [89], 1.0)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_attention_rows_past_4_gib(zq, kind):
    """A pool whose last pages lie past 32 bits of bytes and, with fp32, of elements."""
    KH, D, ps = 8, 256, 256
    es = 4 if kind == "f32" else 2
    pages = ((5 << 30) * (4 if kind == "f32" else 1)) // (KH * ps * D * es)
    table = np.array([[pages - 1, 0, pages // 2, pages - 2]])
    pool = Pool.__new__(Pool)
    pool.rng, pool.kind, pool.KH, pool.D, pool.ps, pool.S, pool.W, pool.pages = np.random.default_rng(1), kind, KH, D, ps, 1, 4, pages
    pool.table = table
    gk = torch.empty(pages, KH, ps, D, dtype=P.TYPES[kind], device=DEV)
    gv = torch.empty_like(gk)
    gt = dev(table)
    pool.cache = zq.KVPaged(gk, gv, pages, KH, D, ps)
    pool.tables = zq.PageTables(gt, None, 1, 4, pages, ps)
    new = [torch.from_numpy(pool.rng.standard_normal((4 * ps, KH, D)).astype(np.float32)) for _ in range(2)]
    slots = np.concatenate([table[0, j] * ps + np.arange(ps) for j in range(4)])
    zq.kv_paged_append_dev(pool.cache, new[0].to(DEV), new[1].to(DEV), 4 * ps, dev(slots, torch.int64))
    at = {int(p): j for j, p in enumerate(table[0])}
    held = [x.reshape(4, ps, KH, D).transpose(1, 2).to(gk.dtype) for x in new]
    for j, p in enumerate(table[0]):
        assert torch.equal(gk[p].cpu(), held[0][j]) and torch.equal(gv[p].cpu(), held[1][j])

    class View:  # the host's copy of the pages that are used
        def __init__(self, x):
            self.x = x

        def __getitem__(self, i):
            return self.x[(at[int(i[0])], *i[1:])]
    pool.k, pool.v = View(held[0]), View(held[1])
    check_attention(zq, pool, queries(pool.rng, 1, 2 * KH, D), [4 * ps - 10], 0.0625)
    del gk, gv
    torch.cuda.empty_cache()


# ---- append -----------------------------------------------------------------------
def check_append(zq, pool, slots, k, v, stride=0):
    """Appends rows k, v [T][KH][D] (fp32) and compares the whole pool and its bounds."""
    T = len(slots)
    k0, v0, c0, e0 = pool.k.clone(), pool.v.clone(), pool.codes.copy(), pool.exps.copy()
    last = {}
    for t, x in enumerate(slots):
        if 0 <= x < pool.pages * pool.ps:
            pool.k[x // pool.ps, :, x % pool.ps] = k[t].to(k0.dtype)
            pool.v[x // pool.ps, :, x % pool.ps] = v[t].to(v0.dtype)
            last[x // pool.ps] = x % pool.ps
    for p, r in last.items():
        pool.rebound(p, r + 1)
    gk, gv = k.to(DEV), v.to(DEV)
    if stride:
        wide = torch.full((T, stride), math.nan, device=DEV)
        W = pool.KH * pool.D
        wide[:, 4:4 + W], wide[:, 8 + W:8 + 2 * W] = gk.reshape(T, -1), gv.reshape(T, -1)
        gk, gv = wide[:, 4:4 + W], wide[:, 8 + W:8 + 2 * W]
    zq.kv_paged_append_dev(pool.cache, gk, gv, T, dev(slots, torch.int64), stride=stride)
    same = lambda a, b: torch.equal(torch.nan_to_num(a.float().cpu(), 12345.0), torch.nan_to_num(b.float(), 12345.0))
    assert same(pool.gk, pool.k) and same(pool.gv, pool.v)
    assert np.array_equal(pool.gb.cpu().numpy(), pool.codes) and np.array_equal(pool.ge.cpu().numpy(), pool.exps)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D, KH, ps", [(64, 1, 16), (64, 5, 256), (128, 8, 16), (128, 2, 64), (256, 3, 32)])
def test_append(zq, kind, D, KH, ps):
    """New tokens behind lengths on both sides of a page's end, prompts over several pages, rows that are no tokens."""
    lens, new = [0, 1, ps - 1, ps, 3 * ps - 2, 5], [1, 1, 1, 1, 5, 0]
    new += [2 * ps + 3, ps, 300]
    lens += [0, ps // 2, 7]
    pool = Pool(zq, kind, [a + b for a, b in zip(lens, new)], KH, D, ps, seed=D + KH)
    slots = []
    for s, (n, c) in enumerate(zip(lens, new)):
        slots += [int(pool.table[s, p // ps]) * ps + p % ps for p in range(n, n + c)]
        if s % 3 == 1:
            slots += [-1, pool.pages * ps, -2 ** 62]
    T = len(slots)
    k = torch.from_numpy(pool.rng.standard_normal((T, KH, D)).astype(np.float32)) * 3
    v = torch.from_numpy(pool.rng.standard_normal((T, KH, D)).astype(np.float32))
    check_append(zq, pool, slots, k, v)
    check_append(zq, pool, slots, v, k, stride=2 * KH * D + 24)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_append_values_at_the_ends(zq, kind):
    """Zeros, ties of the rounding, the largest and the smallest values, infinities and NaN; powers of two times 127."""
    pool = Pool(zq, kind, [16] * 8, 1, 64, 16, seed=2)
    T = 16 * 8
    k = torch.from_numpy(pool.rng.standard_normal((T, 1, 64)).astype(np.float32))
    k[0:16] = 0
    k[16:32] *= 1e-38
    k[32:48] *= 1e37
    k[48] = math.inf
    k[49, 0, :32] = -math.inf
    k[50:64, 0, 5] = math.nan
    k[64:80, 0, 7] = math.nan  # all of a page's
    k[80:96] = torch.where(torch.rand(16, 1, 64) < 0.5, 127.0, -127.0)
    k[96:112] = 127.0 * 2.0 ** -14
    k[112:] = 1 + 2.0 ** -9 * torch.arange(16.0)[:, None, None] + 2.0 ** -12 * torch.arange(64.0)
    slots = [int(pool.table[s, 0]) * 16 + r for s in range(8) for r in range(16)]
    check_append(zq, pool, slots, k, torch.flip(k, [0]))


@gpu
def test_append_without_bounds(zq):
    pool = Pool(zq, "f16", [20], 2, 64, 16, seed=1)
    cache = zq.KVPaged(pool.gk, pool.gv, pool.pages, 2, 64, 16)
    k = torch.randn(2, 2, 64, device=DEV)
    slots = [int(pool.table[0, 1]) * 16 + 4, int(pool.table[0, 1]) * 16 + 5]
    zq.kv_paged_append_dev(cache, k, k, 2, dev(slots, torch.int64))
    assert torch.equal(pool.gk[int(pool.table[0, 1]), :, 4:6].transpose(0, 1), k.half())
    assert np.array_equal(pool.gb.cpu().numpy(), pool.codes)


# ---- selection ---------------------------------------------------------------------
def run_select(zq, pool, q, lens, keep, recent, first, counts=None, seq_of=None, full=False, stride=0, stream=None):
    n, H, D = q.shape
    gq = torch.from_numpy(q).to(DEV)
    if stride:
        wide = torch.full((n, stride), math.nan, device=DEV)
        wide[:, :H * D] = gq.reshape(n, -1)
        gq = wide[:, :H * D]
    select = dev(np.full((n, pool.KH, keep), -9))
    need = zq.page_select_workspace_bytes(pool.cache, pool.tables, n, H, keep)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    opt = lambda x: None if x is None else dev(x)
    zq.page_select_dev(pool.cache, pool.tables, gq, select, n, H, dev(lens), keep, recent=recent, first=first,
                       counts=opt(counts), seq_of=opt(seq_of), stride=stride, flags=zq.ATTN_PAGED_FULL if full else 0,
                       workspace=ws, workspace_bytes=need, stream=stream)
    torch.cuda.synchronize()
    assert (ws[need:] == 255).all()
    return select.cpu().numpy()


def check_select(zq, pool, q, lens, keep, recent, first, **kw):
    got = run_select(zq, pool, q, lens, keep, recent, first, **kw)
    kw.pop("stride", None)
    want = pool.choose(q, lens, keep, recent, first, **kw)
    assert np.array_equal(got, want)
    return got


def scored(zq, n_pages, KH, D, ps, seed, like=None):
    """A pool whose bounds are made up (selection reads nothing else), of sequences of n_pages pages each."""
    pool = Pool.__new__(Pool)
    rng = pool.rng = np.random.default_rng(seed)
    pool.kind, pool.KH, pool.D, pool.ps, pool.S = "f16", KH, D, ps, len(n_pages)
    pool.pages, pool.W = sum(n_pages) + 2, max(n_pages) + 1
    pool.table, _, _ = full_table(rng, [n * ps for n in n_pages], pool.W, ps, pool.pages)
    c = rng.integers(-127, 128, (pool.pages, KH, 2, D)) if like is None else np.broadcast_to(like, (pool.pages, KH, 2, D))
    pool.codes = np.ascontiguousarray(np.sort(c, 2))
    pool.exps = rng.integers(-9, -6, (pool.pages, KH)) if like is None else np.full((pool.pages, KH), -7)
    pool.k = pool.v = torch.zeros(1)
    pool.gk = torch.zeros(16, dtype=torch.float16, device=DEV)
    pool.gb, pool.ge, pool.gt = dev(pool.codes, torch.int8), dev(pool.exps, torch.int8), dev(pool.table)
    pool.cache = zq.KVPaged(pool.gk.data_ptr(), pool.gk.data_ptr(), pool.pages, KH, D, ps, bounds=pool.gb, bounds_exp=pool.ge,
                            type=zq.KV_F16)
    pool.tables = zq.PageTables(pool.gt, None, pool.S, pool.W, pool.pages, ps)
    return pool


@gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("pages, KH, G, keep, recent, first", [
    ([1, 2, 9, 70], 2, 4, 8, 2, 1), ([300, 17, 1000, 16], 3, 7, 16, 0, 0), ([260], 1, 16, 100, 1, 4), ([65, 40], 2, 20, 1, 1, 0),
    ([50], 1, 1, 5, 2, 3), ([1024, 1025, 3], 1, 2, 1, 0, 0), ([513], 1, 3, 512, 4, 1)])
def test_select(zq, D, pages, KH, G, keep, recent, first):
    pool = scored(zq, pages, KH, D, 16, seed=D + keep)
    q = queries(pool.rng, len(pages), KH * G, D)
    check_select(zq, pool, q, [16 * n - 1 - 5 * (n % 2) for n in pages], keep, recent, first)


@gpu
@pytest.mark.parametrize("pages, keep", [(4097, 300), (8192, 256), (8193, 4000), (20000, 1000), (20000, 19999)])
def test_select_of_many_pages(zq, pages, keep):
    pool = scored(zq, [pages, 50], 1, 64, 16, seed=keep)
    check_select(zq, pool, queries(pool.rng, 2, 2, 64), [16 * pages - 1, 799], keep, 4, 1)


@gpu
def test_select_for_more_queries_than_a_workgroup_holds(zq):
    pool = scored(zq, [100, 40, 3], 2, 64, 16, seed=14)
    n = 1700
    seq_of = pool.rng.integers(-1, 4, n)
    check_select(zq, pool, queries(pool.rng, n, 2, 64), pool.rng.integers(-2, 1700, n), 9, 2, 1, seq_of=seq_of)


@gpu
def test_select_for_more_heads_and_queries_than_one_grid_dimension_takes(zq):
    """4200 * 1024 workgroups of 1024 threads are more than 2^32 threads."""
    n, KH = 4200, 1024
    pool = scored(zq, [2], KH, 64, 16, seed=3)
    lens = np.full(n, 15, np.int32)
    lens[7] = lens[-1] = 16  # these see the second page, which is the recent one
    q = torch.zeros(n, KH * 64, device=DEV)
    got = torch.full((n, KH, 1), 55, dtype=torch.int32, device=DEV)
    need = zq.page_select_workspace_bytes(pool.cache, pool.tables, n, KH, 1)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    zq.page_select_dev(pool.cache, pool.tables, q, got, n, KH, dev(lens), 1, recent=1,
                       seq_of=dev(np.zeros(n, np.int32)), workspace=ws, workspace_bytes=need)
    assert torch.equal(got[:, :, 0], dev(lens - 15)[:, None].expand(n, KH))


@gpu
def test_select_ties_go_to_the_lowest(zq):
    """All pages alike; a query of zeros; two values only."""
    pool = scored(zq, [500, 3000], 2, 64, 16, 1, like=np.stack([np.full(64, -3), np.full(64, 5)]))
    q = queries(pool.rng, 2, 4, 64)
    for keep, recent, first in ((7, 2, 1), (100, 0, 0), (499, 3, 3), (1, 0, 0)):
        check_select(zq, pool, q, [7999, 47999], keep, recent, first)
    pool = scored(zq, [500, 3000], 2, 64, 16, 2)
    check_select(zq, pool, q * 0, [7999, 47999], 60, 1, 2)
    pool.exps[:] = np.where(pool.rng.random(pool.exps.shape) < 0.5, -7, -8)
    pool.codes[:] = np.stack([np.full(64, -2), np.full(64, 2)])
    pool.gb.copy_(dev(pool.codes, torch.int8))
    pool.ge.copy_(dev(pool.exps, torch.int8))
    check_select(zq, pool, q, [7999, 47999], 200, 1, 2)


@gpu
def test_select_sizes_of_queries_and_bounds(zq):
    """Queries and bounds at the ends of the exponents, halves to be rounded, NaN and infinities in the queries."""
    pool = scored(zq, [400], 1, 128, 32, seed=3)
    pool.exps[:] = pool.rng.integers(-50, 51, pool.exps.shape)
    pool.ge.copy_(dev(pool.exps, torch.int8))
    for size in (1.0, 1e-20, 1e20, 1e38, 1e-40):
        check_select(zq, pool, queries(pool.rng, 1, 3, 128, 1.0) * np.float32(size), [12799], 50, 1, 1)
    q = (np.arange(3 * 128).reshape(1, 3, 128) - 200).astype(np.float32) / 2
    check_select(zq, pool, q, [12799], 50, 1, 1)
    q[0, 0, 3], q[0, 1, 5], q[0, 1, 6] = math.nan, math.inf, -math.inf
    check_select(zq, pool, q, [12799], 50, 1, 1)
    q[0, 2] = math.nan
    check_select(zq, pool, q, [12799], 50, 1, 1)


@gpu
def test_select_lengths_idle_queries_and_holes(zq):
    pool = scored(zq, [100, 200, 30], 2, 64, 16, seed=4)
    pool.table[0, [3, 50, 51, 99]] = [-1, pool.pages, -2 ** 31, 2 ** 31 - 1]
    pool.table[1, 10:195] = -1
    pool.gt.copy_(dev(pool.table))
    q = queries(pool.rng, 8, 6, 64)
    seq_of, lens = [0, 1, 2, -1, 3, 0, 1, 2], [1599, 3199, 479, 9, 9, 160, -5, 10 ** 6]
    check_select(zq, pool, q, lens, 20, 2, 1, seq_of=seq_of)
    check_select(zq, pool, q, lens, 20, 2, 1, seq_of=seq_of, counts=[1, 0, 1, 1, 1, 700, 2000, -1], stride=6 * 64 + 4)
    check_select(zq, pool, q, lens, 20, 2, 1, seq_of=seq_of, full=True)


@gpu
def test_bound_is_above_every_score(zq):
    """The score is no less than (the 8-bit query) . k of every row of the page."""
    pool = Pool(zq, "bf16", [333], 1, 128, 16, seed=12)
    q = queries(pool.rng, 1, 1, 128)[0]
    s = P.scores(q, pool.codes[pool.table[0, :21], 0], pool.exps[pool.table[0, :21], 0])
    eq = P.exponent(float(np.abs(q).max()))
    c = np.rint(q[0].astype(np.float64) / 2.0 ** eq) * 2.0 ** eq
    for j in range(21):
        r = min(16, 333 - 16 * j)
        assert (pool.k[pool.table[0, j], 0, :r].double().numpy() @ c).max() <= s[j]


# ---- as they are used ---------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_equal_calls_give_equal_bits(zq, kind, spare):
    pool = Pool(zq, kind, [3000, 100, 1], 2, 128, 16, seed=20, spare_width=spare)
    q = queries(pool.rng, 3, 8, 128)
    a = [run_attention(zq, pool, q, [2999, 99, 0], 0.1) for _ in range(4)]
    assert all(np.array_equal(a[0], x) for x in a[1:])


class Server:
    """Sequences that come, grow and go: the four calls as a program makes them, beside the plain ones."""

    def __init__(self, zq, kind, KH, G, D, ps, S, W, pages, room, keep, seed):
        self.zq, self.rng, self.keep = zq, np.random.default_rng(seed), keep
        pool = self.pool = Pool.__new__(Pool)
        pool.kind, pool.KH, pool.D, pool.ps, pool.S, pool.W, pool.pages = kind, KH, D, ps, S, W, pages
        pool.k = torch.full((pages, KH, ps, D), math.nan, dtype=P.TYPES[kind])
        pool.v = pool.k.clone()
        pool.codes, pool.exps = np.full((pages, KH, 2, D), 77, np.int64), np.full((pages, KH), 9, np.int64)
        pool.table = np.full((S, W), -1, np.int64)
        pool.upload(zq)
        self.free, self.fc = self.rng.permutation(pages), pages
        self.gfree, self.gfc = dev(self.free), dev([pages])
        pool.tables = zq.PageTables(pool.gt, self.gfree, S, W, pages, ps)
        self.lens, self.room, self.H = [0] * S, room, KH * G
        z = lambda n, dtype=torch.int32: torch.zeros(n, dtype=dtype, device=DEV)
        self.g = dict(lens=z(S), counts=z(S), granted=z(S), start=z(S + 1), slots=z(room, torch.int64), pos=z(room), seq=z(room),
                      k=torch.zeros(room, KH, D, device=DEV), v=torch.zeros(room, KH, D, device=DEV),
                      q=torch.zeros(room, self.H, D, device=DEV), select=z(room * KH * keep),
                      out=torch.zeros(room, self.H, D, device=DEV), sparse=torch.zeros(room, self.H, D, device=DEV), go=z(S))
        need = max(zq.attention_paged_workspace_bytes(pool.cache, pool.tables, room, self.H),
                   zq.page_select_workspace_bytes(pool.cache, pool.tables, room, self.H, keep))
        self.ws, self.need = torch.zeros(need, dtype=torch.uint8, device=DEV), need

    def enqueue(self, stream=None):
        zq, p, g, n = self.zq, self.pool, self.g, self.room
        zq.page_tables_release_dev(p.tables, g["lens"], g["go"], self.gfc, self.gfc, stream=stream)
        g["lens"].copy_(torch.minimum(g["lens"], g["go"]))
        zq.page_tables_step_dev(p.tables, g["lens"], g["counts"], self.gfc, self.gfc, g["granted"], g["start"], g["slots"],
                                g["pos"], g["seq"], n, stream=stream)
        zq.kv_paged_append_dev(p.cache, g["k"], g["v"], n, g["slots"], stream=stream)
        w = dict(seq_of=g["seq"], workspace=self.ws, workspace_bytes=self.need, stream=stream)
        zq.attention_paged_dev(p.cache, p.tables, g["q"], g["out"], n, self.H, g["pos"], 0.1, **w)
        zq.page_select_dev(p.cache, p.tables, g["q"], g["select"], n, self.H, g["pos"], self.keep, recent=1, first=1, **w)
        zq.attention_paged_dev(p.cache, p.tables, g["q"], g["sparse"], n, self.H, g["pos"], 0.1, select=g["select"],
                               keep=self.keep, **w)
        g["lens"].add_(g["granted"])

    def inputs(self, counts, go):
        g, p = self.g, self.pool
        for name in ("k", "v", "q"):
            x = torch.from_numpy(self.rng.standard_normal(g[name].shape).astype(np.float32))
            g[name].copy_(x)
            setattr(self, name, x)
        g["counts"].copy_(dev(counts))
        g["go"].copy_(dev(go))
        g["out"].fill_(math.nan)
        g["sparse"].fill_(math.nan)
        self.counts, self.go = list(counts), list(go)

    def check(self):
        g, p, ps = self.g, self.pool, self.pool.ps
        torch.cuda.synchronize()
        self.free, self.fc = P.release(self.lens, self.go, p.table, self.free, self.fc, ps)
        self.lens = [min(a, max(b, 0)) for a, b in zip(self.lens, self.go)]
        granted, start, slots, pos, seq, p.table, self.fc = P.step(self.lens, self.counts, p.table, self.free, self.fc, ps,
                                                                   p.pages, self.room)
        for name, want in (("granted", granted), ("start", start), ("slots", slots), ("pos", pos), ("seq", seq)):
            assert np.array_equal(g[name].cpu().numpy(), want), name
        assert int(self.gfc) == self.fc and np.array_equal(p.gt.cpu().numpy(), p.table)
        last = {}
        for t, x in enumerate(slots):
            if x >= 0:
                p.k[x // ps, :, x % ps], p.v[x // ps, :, x % ps] = self.k[t].to(p.k.dtype), self.v[t].to(p.v.dtype)
                last[x // ps] = x % ps
        for page, r in last.items():
            p.rebound(page, r + 1)
        assert np.array_equal(p.gb.cpu().numpy(), p.codes)
        q = self.q.numpy()
        select = p.choose(q, pos, self.keep, 1, 1, seq_of=seq)
        rows = [i for i, s in enumerate(seq) if s >= 0]
        got = g["select"].reshape(self.room, p.KH, self.keep).cpu().numpy()
        assert np.array_equal(got[rows], select[rows])
        for name, sel in (("out", None), ("sparse", select)):
            want, tol = p.attend(q, pos, 0.1, seq_of=seq, select=sel)
            y = g[name].cpu().numpy()
            assert (np.isnan(y) == np.isnan(want)).all(), name
            assert (np.abs(y - want)[rows] <= tol[rows]).all(), name
        self.lens = [a + b for a, b in zip(self.lens, granted)]


STEPS = [  # new tokens; what stays of each sequence before them (past its length: all)
    ([20, 1, 0, 33, 5], [99] * 5), ([1, 1, 1, 1, 1], [99] * 5), ([1, 40, 1, 0, 1], [99] * 5), ([1, 1, 1, 1, 1], [0, 99, 99, 20, 4]),
    ([30, 1, 1, 1, 1], [99] * 5), ([9, 9, 9, 9, 9], [99, 0, 99, 99, 0]), ([60, 60, 0, 1, 0], [99] * 5)]


@gpu
@pytest.mark.parametrize("kind, KH, G, D", [("f16", 2, 4, 64), ("bf16", 1, 3, 128), ("f32", 2, 1, 64)])
def test_a_server_of_sequences(zq, kind, KH, G, D):
    s = Server(zq, kind, KH, G, D, 16, 5, 8, 16, 70, 3, seed=G)
    for counts, go in STEPS:
        s.inputs(counts, go)
        s.enqueue()
        s.check()


@gpu
def test_a_captured_step_replays_while_sequences_grow(zq):
    s = Server(zq, "f16", 2, 2, 64, 16, 5, 8, 16, 70, 3, seed=7)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    s.inputs([0] * 5, [99] * 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.enqueue(stream)
    for counts, go in STEPS:
        s.inputs(counts, go)
        torch.cuda.synchronize()
        graph.replay()
        s.check()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_captured_calls_of_wide_heads_replay(zq, kind):
    """Workgroups of more than 64 KB of LDS; a replay after other work, with other queries and lengths."""
    pool = Pool(zq, kind, [700, 90, 5], 1, 256, 32, seed=21, spare_width=3000)
    n, H = 3, 16
    need = max(zq.attention_paged_workspace_bytes(pool.cache, pool.tables, n, H),
               zq.page_select_workspace_bytes(pool.cache, pool.tables, n, H, 4))
    ws = torch.zeros(need, dtype=torch.uint8, device=DEV)
    q, out, lens = torch.zeros(n, H, 256, device=DEV), torch.zeros(n, H, 256, device=DEV), dev([0] * n)
    select, sparse = dev(np.zeros((n, 1, 4))), torch.zeros(n, H, 256, device=DEV)
    w = dict(workspace=ws, workspace_bytes=need)

    def enqueue(stream):
        zq.attention_paged_dev(pool.cache, pool.tables, q, out, n, H, lens, 0.06, stream=stream, **w)
        zq.page_select_dev(pool.cache, pool.tables, q, select, n, H, lens, 4, recent=1, first=1, stream=stream, **w)
        zq.attention_paged_dev(pool.cache, pool.tables, q, sparse, n, H, lens, 0.06, select=select, keep=4, stream=stream, **w)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        enqueue(stream)
    for ls in ([699, 89, 4], [3, 60, 0], [512, 33, 2]):
        x = queries(pool.rng, n, H, 256)
        q.copy_(torch.from_numpy(x))
        lens.copy_(dev(ls))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        picked = pool.choose(x, ls, 4, 1, 1)
        assert np.array_equal(select.cpu().numpy(), picked)
        for got, sel in ((out, None), (sparse, picked)):
            want, tol = pool.attend(x, ls, 0.06, select=sel)
            assert (np.abs(got.cpu().numpy() - want) <= tol).all()
        eager = [t.clone() for t in (out, sparse)]
        enqueue(None)
        torch.cuda.synchronize()
        assert torch.equal(eager[0], out) and torch.equal(eager[1], sparse)


@gpu
def test_two_calls_at_once(zq):
    """Two streams read one cache, with a workspace each."""
    pool = Pool(zq, "bf16", [4000, 300, 2500], 2, 128, 16, seed=22)
    x = [queries(pool.rng, 3, 8, 128) for _ in range(2)]
    lens = [[3999, 299, 2499], [3000, 10, 2400]]
    alone = [run_attention(zq, pool, q, n, 0.1) for q, n in zip(x, lens)]
    need = zq.attention_paged_workspace_bytes(pool.cache, pool.tables, 3, 8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [torch.zeros(need, dtype=torch.uint8, device=DEV) for _ in range(2)]
    q = [torch.from_numpy(a).to(DEV) for a in x]
    gl = [dev(n) for n in lens]
    out = [[torch.zeros(3, 8, 128, device=DEV) for _ in range(2)] for _ in range(10)]
    torch.cuda.synchronize()
    for o in out:
        for i in range(2):
            zq.attention_paged_dev(pool.cache, pool.tables, q[i], o[i], 3, 8, gl[i], 0.1, workspace=ws[i], workspace_bytes=need,
                                   stream=streams[i])
    torch.cuda.synchronize()
    for o in out:
        for i in range(2):
            assert np.array_equal(o[i].cpu().numpy(), alone[i])


@gpu
def test_on_another_stream(zq):
    s = Server(zq, "bf16", 2, 2, 128, 16, 5, 8, 16, 70, 3, seed=8)
    stream = torch.cuda.Stream()
    for counts, go in STEPS[:4]:
        s.inputs(counts, go)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            s.enqueue(stream)
        torch.cuda.current_stream().wait_stream(stream)
        s.check()

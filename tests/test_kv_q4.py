"""The 4-bit KV cache (include/zq_kv.h): append, read, attention and eviction
against plain implementations in 64 bits, and their refusals.

What the cache holds, and which rows an eviction keeps, is compared bit for
bit.  The attention's tolerance is a bound of its arithmetic, per output row:
with u = 2^-24, A = max_p sum_d |scale q_d k_pd| and n visible rows,
  - a score is off by at most A (D u + 2 u + 2^-21): D - 1 additions and the
    products in fp32 of either query part, the rounding of q * scale and of
    scale * log2(e), and a query held in two fp16 parts (each rounding half a
    step: 2^-11 * 2^-11 = 2^-22, and as much again where the parts are summed);
    the running maximum in log2 units adds 2 A u;
  - a weight's exponential and its own two parts add 2^-22 + 2^-22, the sums of
    products over n rows n u, the sum of the weights n u, the quotient and the
    rescalings (at most 16 of them, and the merges) 40 u;
  - a relative error e of every weight moves the output by at most 2 e max |v|.
A weight is also a multiple of 2^-24 where the largest so far is 2^6 at least, off
by up to 2^-31 of it, which over n rows is below the n u above.  The accumulated weights take the same relative error each, and the sum over
their R queries adds R u."""
import ctypes
import math
import os
import re

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24


# ---- plain implementations, on the CPU in 64 bits -----------------------------
def q4_scale(m):
    """fp16(bf16(m / -8)) within +-4096, as float64 (m: float64 array)."""
    f, e = np.frexp(m / -8.0)
    d = np.clip(np.ldexp(np.rint(f * 256.0), e - 8), -4096.0, 4096.0)
    return np.where(np.abs(d) < 2.0 ** -14, np.rint(d * 2.0 ** 24) * 2.0 ** -24, d)


def q4_rows(x):
    """(codes uint8 [..., D/2], scales float64 [..., D/32]) of finite rows x [..., D]."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    at = np.argmax(np.abs(b), -1)  # the first of equals
    d = q4_scale(np.take_along_axis(b, at[..., None], -1)[..., 0])
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(d[..., None] == 0, 0.0, np.clip(np.rint(b / d[..., None]), -8, 7))
    c = (c + 8).astype(np.uint8)
    return (c[..., :16] | c[..., 16:] << 4).reshape(*x.shape[:-1], -1), np.where(d == 0, 0.0, d)


def q4_values(codes, d):
    """float64 rows [..., D] of codes [..., D/2] and scales [..., D/32]."""
    b = codes.reshape(*codes.shape[:-1], -1, 16)
    c = np.concatenate([b & 15, b >> 4], -1).astype(np.float64) - 8
    return (c * d[..., None]).reshape(*codes.shape[:-1], -1)


class Plain:
    """A cache as lists of rows: per (sequence, kv head) values, weight and pos, with the operators on them."""

    def __init__(self, S, KH, D, C):
        self.S, self.KH, self.D, self.C = S, KH, D, C
        self.k = np.zeros((S, KH, C, D))
        self.v = np.zeros((S, KH, C, D))
        self.weight = np.zeros((S, KH, C))
        self.pos = np.zeros((S, KH, C), np.int64)

    def append(self, k, v, lens, counts, first_pos=None):
        """k, v [S][T][KH][D]."""
        for s in range(self.S):
            for t in range(min(counts[s], k.shape[1])):
                slot = lens[s] + t
                if lens[s] < 0 or slot >= self.C:
                    continue
                for h in range(self.KH):
                    kx, vx = k[s, t, h], v[s, t, h]
                    if np.isfinite(kx).all() and np.isfinite(vx).all():
                        self.k[s, h, slot] = q4_values(*q4_rows(kx))
                        self.v[s, h, slot] = q4_values(*q4_rows(vx))
                    else:
                        self.k[s, h, slot], self.v[s, h, slot] = np.nan, 0
                    self.weight[s, h, slot] = 0
                    self.pos[s, h, slot] = (first_pos[s] if first_pos is not None else lens[s]) + t

    def attention(self, q, lens, counts, scale, full=False, weights=None):
        """(out, tolerance) [S][T][H][D], NaN where nothing is written; weights: None, "set" or "add"."""
        S, T, H, D = q.shape
        G = H // self.KH
        out, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
        drawn, drawn_tol = np.zeros_like(self.weight), np.zeros_like(self.weight)
        for s in range(S):
            live = max(0, min(counts[s], T))
            for t in range(live):
                n = min(self.C, max(lens[s], 0) + (0 if full else t + 1))
                for h in range(H):
                    x = q[s, t, h].astype(np.float64) * scale
                    k, v = self.k[s, h // G, :n], self.v[s, h // G, :n]
                    if n == 0:
                        out[s, t, h], tol[s, t, h] = 0, 0
                        continue
                    a = (np.abs(x) * np.abs(k)).sum(-1)
                    p = k @ x
                    p = np.exp(p - p.max())
                    p /= p.sum()
                    e = 2 * (a.max() * ((D + 4) * U + 2.0 ** -21) + 2.0 ** -21 + (2 * n + 40) * U)
                    out[s, t, h], tol[s, t, h] = p @ v, e * np.abs(v).max()
                    drawn[s, h // G, :n] += p
                    drawn_tol[s, h // G, :n] += e * p
            if weights and live:
                n = min(self.C, max(lens[s], 0) + (0 if full else live))
                w = drawn[s, :, :n] + (self.weight[s, :, :n] if weights == "add" else 0)
                drawn_tol[s, :, :n] += (live * G + 1) * U * w
                self.weight[s, :, :n] = w
        return out, tol, drawn_tol

    def evict(self, lens, keep, recent, first, next_pos=None, to=None):
        to = to or self
        for s in range(self.S):
            n = min(max(lens[s], 0), self.C)
            K = min(n, keep)
            newest = (next_pos[s] if next_pos is not None else n) - recent
            for h in range(self.KH):
                p, w = self.pos[s, h, :n], self.weight[s, h, :n]
                held = (p >= 0) & ((p >= newest) | (p < first))
                rank = sorted(range(n), key=lambda i: (not held[i], 0.0 if held[i] else (math.inf if np.isnan(w[i]) else -w[i]),
                                                       not held[i] and np.isnan(w[i]), i))
                stay = sorted(rank[:K])
                up = [i for i in stay if i >= K]
                own = set(stay)
                frm = [i if i in own else up.pop(0) for i in range(K)]
                for name in ("k", "v", "weight", "pos"):
                    rows = getattr(self, name)[s, h, frm].copy()
                    getattr(to, name)[s, h, :K] = rows
                if to is self and n > K:
                    self.weight[s, h, K:n], self.pos[s, h, K:n] = -np.inf, -1


# ---- CPU ------------------------------------------------------------------------
def test_plain_quantiser_takes_the_nearest_code():
    r = np.random.default_rng(1)
    x = r.standard_normal((200, 64)) * np.exp(r.uniform(-8, 8, (200, 1)))
    codes, d = q4_rows(x.astype(np.float32).astype(np.float64))
    v = q4_values(codes, d)
    x = x.astype(np.float32).astype(np.float64)
    levels = (np.arange(16) - 8) * np.repeat(d, 32, -1)[..., None]
    best = np.abs(x[..., None] - levels).min(-1)
    assert (np.abs(x - v) <= best).all()
    # codes end at 7 on the side away from the largest element, so |x| there up to 8 scales is one step off, and the
    # scale's own rounding (half a step of 8 bits, of 8 scales) comes on top
    assert (np.abs(x - v) <= np.repeat(np.abs(d), 32, -1) * (1 + 8 * 2.0 ** -8)).all()


def test_header_and_binding_agree():
    from zeninfer_amd import zq
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "zq_kv.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(zq_[a-z0-9_]+)\s*\(", text))
    assert declared == set(zq.KV_SIGNATURES)
    assert all(hasattr(zq.lib(), n) for n in declared)


def test_layout():
    from zeninfer_amd import zq
    assert zq.kv_q4_bytes(8, 128, 4096) == 2 * 8 * 4096 * (64 + 8)
    assert zq.kv_q4_bytes(8, 96, 4096) == zq.kv_q4_bytes(8, 128, 4095) == zq.kv_q4_bytes(0, 128, 64) == 0
    assert zq.kv_q4_bytes(1, 64, (1 << 24) + 32) == 0


def handle(zq, **over):
    """A cache of made-up addresses: for calls that are refused before they use them."""
    f = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, weight=5 << 20, pos=6 << 20, seqs=2, kv_heads=2,
             head_dim=64, capacity=64)
    f.update(over)
    return zq.KVCacheQ4(*[f[n] for n, _ in zq.KVCacheQ4._fields_])


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=(1 << 20) + 4),
              dict(v_scale=(1 << 20) + 8), dict(pos=(1 << 20) + 2), dict(seqs=0), dict(kv_heads=0), dict(head_dim=96),
              dict(head_dim=32), dict(head_dim=0), dict(capacity=0), dict(capacity=48), dict(capacity=(1 << 24) + 32),
              dict(seqs=1 << 21), dict(seqs=1 << 19, kv_heads=4), dict(seqs=1 << 63, kv_heads=2)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=lambda o: ",".join(f"{k}={v}" for k, v in o.items()))
def test_calls_refuse_a_bad_cache(over):
    from zeninfer_amd import zq
    L, c = zq.lib(), ctypes.byref(handle(zq, **over))
    p = 7 << 20
    assert L.zq_hip_kv_q4_append_dev(c, p, p, 1, 0, p, None, None, None) == zq.ERR_ARG
    assert L.zq_hip_kv_q4_read_dev(c, p, p, 1, p, None, None) == zq.ERR_ARG
    assert L.zq_hip_attention_q4_dev(c, p, p, 1, 4, 0, p, None, 1.0, 0, p, 1 << 30, None) == zq.ERR_ARG
    assert L.zq_hip_attention_q4_workspace_bytes(c, 1, 4, 2) == 0
    assert L.zq_hip_kv_q4_evict_dev(c, None, p, 16, 4, 4, None, p, 1 << 30, None) == zq.ERR_ARG
    assert L.zq_hip_kv_q4_evict_workspace_bytes(c, 16) == 0


def test_calls_refuse_bad_arguments():
    from zeninfer_amd import zq
    L, p = zq.lib(), 7 << 20
    h = handle(zq)
    c = ctypes.byref(h)
    bare = ctypes.byref(handle(zq, weight=None, pos=None))
    app = lambda k=p, v=p, tokens=1, stride=0, lens=p, counts=None, first=None: L.zq_hip_kv_q4_append_dev(
        c, k, v, tokens, stride, lens, counts, first, None)
    for bad in (dict(k=None), dict(v=None), dict(lens=None), dict(k=p + 4), dict(v=p + 8), dict(lens=p + 2),
                dict(counts=p + 1), dict(first=p + 2), dict(tokens=0), dict(tokens=1 << 26), dict(tokens=1 << 63),
                dict(stride=127), dict(stride=124), dict(stride=130), dict(stride=1 << 40)):
        assert app(**bad) == zq.ERR_ARG, bad
    read = lambda k=p, v=p, tokens=1, first=p, counts=None: L.zq_hip_kv_q4_read_dev(c, k, v, tokens, first, counts, None)
    for bad in (dict(k=None, v=None), dict(k=p + 4), dict(v=p + 4), dict(tokens=0), dict(first=None), dict(first=p + 1),
                dict(counts=p + 3), dict(tokens=1 << 40)):
        assert read(**bad) == zq.ERR_ARG, bad

    def attn(cache=c, q=p, out=p, tokens=1, heads=4, stride=0, lens=p, counts=None, flags=0, ws=p, nbytes=1 << 40):
        return L.zq_hip_attention_q4_dev(cache, q, out, tokens, heads, stride, lens, counts, 1.0, flags, ws, nbytes, None)
    need = L.zq_hip_attention_q4_workspace_bytes(c, 3, 4, 2)
    assert need > 0
    for bad in (dict(q=None), dict(out=None), dict(q=p + 4), dict(out=p + 8), dict(lens=None), dict(lens=p + 2),
                dict(counts=p + 1), dict(tokens=0), dict(tokens=1 << 40), dict(heads=0), dict(heads=3),
                dict(heads=1 << 21), dict(stride=252), dict(stride=258), dict(flags=8), dict(flags=4), dict(flags=5),
                dict(flags=-1), dict(flags=2, cache=bare), dict(flags=2, tokens=3, ws=None),
                dict(flags=2, tokens=3, nbytes=need - 1), dict(flags=2, tokens=3, ws=p + 8)):
        assert attn(**bad) == zq.ERR_ARG, bad
    for bad in ((1, 0, 0), (0, 4, 0), (1, 3, 0)):
        assert L.zq_hip_attention_q4_workspace_bytes(c, *bad) == 0

    def evict(cache=c, dst=None, lens=p, keep=16, recent=4, first=4, nxt=None, ws=p, nbytes=1 << 30):
        return L.zq_hip_kv_q4_evict_dev(cache, dst, lens, keep, recent, first, nxt, ws, nbytes, None)
    other = dict(k=8 << 20, v=9 << 20, k_scale=10 << 20, v_scale=11 << 20, weight=12 << 20, pos=13 << 20)
    d = lambda **o: ctypes.byref(handle(zq, **{**other, **o}))
    need = L.zq_hip_kv_q4_evict_workspace_bytes(c, 16)
    assert need == 4 * 3 * 16 * 4 and L.zq_hip_kv_q4_evict_workspace_bytes(c, 0) == 0
    for bad in (dict(cache=bare), dict(lens=None), dict(lens=p + 2), dict(nxt=p + 1), dict(keep=0), dict(recent=17, first=0),
                dict(recent=13), dict(recent=0, first=17), dict(recent=1 << 63, first=1 << 63), dict(ws=None),
                dict(ws=p + 4), dict(nbytes=need - 1), dict(dst=d(weight=None)), dict(dst=d(pos=None)), dict(dst=d(seqs=1)),
                dict(dst=d(kv_heads=1)), dict(dst=d(head_dim=128)), dict(dst=d(capacity=32), keep=33),
                dict(dst=d(v=2 << 20)), dict(dst=d(k_scale=3 << 20)), dict(dst=d(v_scale=4 << 20)),
                dict(dst=d(weight=5 << 20)), dict(dst=d(pos=6 << 20)), dict(dst=d(k=1 << 20)),
                dict(dst=ctypes.byref(handle(zq, capacity=32)))):
        assert evict(**bad) == zq.ERR_ARG, bad


def test_wrappers_refuse_host_and_short_tensors(monkeypatch):
    from zeninfer_amd import zq
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    with pytest.raises(ValueError, match="KVQ4 k: tensor must be on the GPU"):
        zq.KVQ4(torch.zeros(4096, dtype=torch.uint8), 1 << 20, 1 << 20, 1 << 20, 1, 2, 64, 64)
    c = zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, 1, 2, 64, 64, weight=5 << 20, pos=6 << 20)
    with pytest.raises(ValueError, match="attention_q4_dev lens: tensor must be on the GPU"):
        zq.attention_q4_dev(c, 1 << 20, 1 << 20, 1, 4, i32(1), 1.0)
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    u8 = lambda n: torch.zeros(n, dtype=torch.uint8)
    with pytest.raises(ValueError, match="KVQ4 v: buffer holds"):
        zq.KVQ4(u8(2 * 64 * 32), u8(2 * 64 * 32 - 1), u8(512), u8(512), 1, 2, 64, 64)
    with pytest.raises(ValueError, match="KVQ4 k_scale: buffer holds"):
        zq.KVQ4(u8(2 * 64 * 32), u8(2 * 64 * 32), u8(511), u8(512), 1, 2, 64, 64)
    with pytest.raises(ValueError, match="KVQ4 pos: buffer holds"):
        zq.KVQ4(u8(2 * 64 * 32), u8(2 * 64 * 32), u8(512), u8(512), 1, 2, 64, 64, pos=i32(127))
    f = torch.zeros
    with pytest.raises(ValueError, match="kv_q4_append_dev v: buffer holds"):
        zq.kv_q4_append_dev(c, f(3, 128), f(3, 128)[:2], 3, i32(1))
    with pytest.raises(ValueError, match="kv_q4_append_dev k: rows must be"):
        zq.kv_q4_append_dev(c, f(3, 300)[:, :128], f(3, 300)[:, :128], 3, i32(1), stride=256)
    with pytest.raises(ValueError, match="kv_q4_append_dev k: buffer holds"):
        zq.kv_q4_append_dev(c, f(3, 256)[:, 132:], f(3, 256)[:, 128:], 3, i32(1), stride=256)
    with pytest.raises(ValueError, match="kv_q4_read_dev k: buffer holds"):
        zq.kv_q4_read_dev(c, f(3, 127), None, 3, i32(1))
    with pytest.raises(ValueError, match="attention_q4_dev out: buffer holds"):
        zq.attention_q4_dev(c, f(2, 256), f(2, 255), 2, 4, i32(1), 1.0)
    with pytest.raises(ValueError, match="attention_q4_dev counts: buffer holds"):
        zq.attention_q4_dev(c, f(2, 256), f(2, 256), 2, 4, i32(1), 1.0, counts=i32(0))
    with pytest.raises(ValueError, match="attention_q4_dev workspace: buffer holds"):
        zq.attention_q4_dev(c, f(2, 256), f(2, 256), 2, 4, i32(1), 1.0, workspace=u8(15), workspace_bytes=16)
    with pytest.raises(ValueError, match="kv_q4_evict_dev next_pos: buffer holds"):
        zq.kv_q4_evict_dev(c, i32(1), 16, 4, 4, next_pos=i32(0), workspace=u8(1 << 12), workspace_bytes=1 << 12)


def test_wrappers_refuse_lengths_of_other_types(monkeypatch):
    """torch's default integer has 64 bits: its buffer is long enough and would be read as other lengths."""
    from zeninfer_amd import zq
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    c = zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, 1, 2, 64, 64, weight=5 << 20, pos=6 << 20)
    p, wrong, right = 7 << 20, torch.zeros(4, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    for bad in (wrong, torch.zeros(4), torch.zeros(8, dtype=torch.int16)):
        for call in (lambda: zq.kv_q4_append_dev(c, p, p, 1, bad), lambda: zq.kv_q4_append_dev(c, p, p, 1, right, counts=bad),
                     lambda: zq.kv_q4_append_dev(c, p, p, 1, right, first_pos=bad),
                     lambda: zq.kv_q4_read_dev(c, p, p, 1, bad), lambda: zq.kv_q4_read_dev(c, p, p, 1, right, counts=bad),
                     lambda: zq.attention_q4_dev(c, p, p, 1, 4, bad, 1.0),
                     lambda: zq.attention_q4_dev(c, p, p, 1, 4, right, 1.0, counts=bad),
                     lambda: zq.kv_q4_evict_dev(c, bad, 16, 4, 4), lambda: zq.kv_q4_evict_dev(c, right, 16, 4, 4, next_pos=bad)):
            with pytest.raises(ValueError, match="needs int32"):
                call()


def test_calls_refuse_launches_past_32_bits():
    """A launch has fewer than 2^32 threads: 256 for 4 to 16 rows of an append, for 64 kept rows of an eviction, which
    must not stop between its two launches."""
    from zeninfer_amd import zq
    L, p = zq.lib(), 7 << 20
    c = ctypes.byref(handle(zq, kv_heads=64, seqs=1, capacity=1 << 24))
    assert L.zq_hip_kv_q4_evict_dev(c, None, p, 1 << 24, 4, 4, None, p, 1 << 62, None) == zq.ERR_ARG
    assert L.zq_hip_kv_q4_append_dev(c, p, p, (1 << 19) + 1, 0, p, None, None, None) == zq.ERR_ARG
    assert L.zq_hip_kv_q4_read_dev(c, p, p, (1 << 19) + 1, p, None, None) == zq.ERR_ARG
    assert L.zq_hip_attention_q4_dev(c, p, p, 1 << 19, 128, 0, p, None, 1.0, 0, p, 1 << 62, None) == zq.ERR_ARG
    assert L.zq_hip_attention_q4_workspace_bytes(c, 1 << 19, 128, 0) == 0


# ---- GPU ------------------------------------------------------------------------
class Dev:
    """A cache on the GPU beside its plain counterpart.  Everything past what is appended starts as garbage: codes of
    all ones, scales and weights NaN."""

    def __init__(self, zq, S, KH, D, C, weight=True):
        self.zq, self.S, self.KH, self.D, self.C = zq, S, KH, D, C
        cuda = dict(device="cuda")
        self.k = torch.full((S, KH, C, D // 2), 0xff, dtype=torch.uint8, **cuda)
        self.v = torch.full((S, KH, C, D // 2), 0xff, dtype=torch.uint8, **cuda)
        self.ks = torch.full((S, KH, D // 32, C), math.nan, dtype=torch.float16, **cuda)
        self.vs = torch.full((S, KH, D // 32, C), math.nan, dtype=torch.float16, **cuda)
        self.weight = torch.full((S, KH, C), math.nan, **cuda) if weight else None
        self.pos = torch.full((S, KH, C), -7, dtype=torch.int32, **cuda) if weight else None
        self.c = zq.KVQ4(self.k, self.v, self.ks, self.vs, S, KH, D, C, weight=self.weight, pos=self.pos)
        self.plain = Plain(S, KH, D, C)

    def ints(self, x):
        return None if x is None else torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")

    def append(self, k, v, lens, counts=None, first_pos=None, stride=0, stream=None):
        S, T = k.shape[:2]
        if stride:
            buf = torch.full((S, T, 2 * stride), math.nan, device="cuda")
            kd, vd = buf[..., :self.KH * self.D], buf[..., stride:stride + self.KH * self.D]
            kd.copy_(torch.from_numpy(k.reshape(S, T, -1)))
            vd.copy_(torch.from_numpy(v.reshape(S, T, -1)))
            stride = 2 * stride
        else:
            kd, vd = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
        self.zq.kv_q4_append_dev(self.c, kd, vd, T, self.ints(lens), counts=self.ints(counts),
                                 first_pos=self.ints(first_pos), stride=stride, stream=stream)
        torch.cuda.synchronize()
        self.plain.append(k, v, lens, counts if counts is not None else [T] * S, first_pos)

    def attention(self, q, lens, scale, counts=None, full=False, weights=None, stride=0):
        zq = self.zq
        S, T, H, D = q.shape
        flags = (zq.ATTN_Q4_FULL if full else 0) | {None: 0, "set": zq.ATTN_Q4_WEIGHTS,
                                                    "add": zq.ATTN_Q4_WEIGHTS | zq.ATTN_Q4_ADD}[weights]
        n = zq.attention_q4_workspace_bytes(self.c, T, H, flags)
        ws = torch.full((n + 64,), 0xff, dtype=torch.uint8, device="cuda")
        if stride:
            qd = torch.full((S, T, stride), math.nan, device="cuda")[..., :H * D]
            qd.copy_(torch.from_numpy(q.reshape(S, T, -1)))
        else:
            qd = torch.from_numpy(q).cuda()
        out = torch.full((S, T, H, D), 123.25, device="cuda")
        zq.attention_q4_dev(self.c, qd, out, T, H, self.ints(lens), scale, counts=self.ints(counts), stride=stride,
                            flags=flags, workspace=ws[:n] if n else None, workspace_bytes=n)
        torch.cuda.synchronize()
        assert (ws[n:] == 0xff).all(), "written behind the workspace"
        want, tol, wtol = self.plain.attention(q, lens, counts if counts is not None else [T] * S, float(np.float32(scale)),
                                               full, weights)
        return out.cpu().numpy().astype(np.float64), want, tol, wtol

    def check_attention(self, q, lens, scale, counts=None, full=False, weights=None, stride=0):
        before = self.weight.cpu().numpy().copy() if self.weight is not None else None
        S, T = q.shape[:2]
        out, want, tol, wtol = self.attention(q, lens, scale, counts, full, weights, stride)
        for s in range(S):
            live = T if counts is None else max(0, min(counts[s], T))
            assert (out[s, live:] == 123.25).all(), f"sequence {s}: rows behind the live ones were written"
            o, w, t = out[s, :live], want[s, :live], tol[s, :live]
            assert (np.isnan(o) == np.isnan(w)).all(), f"sequence {s}: NaN in other places"
            ok = ~np.isnan(w)
            bad = np.abs(o - w)[ok] > t[ok]
            assert not bad.any(), f"sequence {s}: {bad.sum()} off, worst {np.abs(o - w)[ok].max()} (tolerance {t[ok].min()})"
        if self.weight is not None:
            got = self.weight.cpu().numpy().astype(np.float64)
            for s in range(S):
                live = T if counts is None else max(0, min(counts[s], T))
                n = min(self.C, max(lens[s], 0) + (0 if full else live)) if weights and live else 0
                assert np.array_equal(got[s, :, n:], before[s, :, n:], equal_nan=True), "weights of unseen rows changed"
                w = self.plain.weight[s, :, :n]
                ok = ~np.isnan(w)
                assert (np.isnan(got[s, :, :n]) == ~ok).all()
                assert (np.abs(got[s, :, :n] - w)[ok] <= wtol[s, :, :n][ok] + 1e-30).all(), (
                    f"sequence {s}: weights off by {np.abs(got[s, :, :n] - w)[ok].max()}")

    def fill(self, lens, seed):
        """Rows below lens from a seed, in one append."""
        r = np.random.default_rng(seed)
        n = max(1, max(lens))
        wide = np.where(r.random(self.D) < 0.06, 5.0, 1.0)
        k = (r.standard_normal((self.S, n, self.KH, self.D)) * wide).astype(np.float32)
        v = (r.standard_normal((self.S, n, self.KH, self.D)) * 0.7).astype(np.float32)
        self.append(k, v, [0] * self.S, counts=lens)

    def rows_equal(self, lens):
        """The rows below lens, read back, against the plain ones, bit for bit (as values)."""
        n = max(1, max(lens))
        out = [torch.full((self.S, n, self.KH, self.D), 77.5, device="cuda") for _ in range(2)]
        self.zq.kv_q4_read_dev(self.c, out[0], out[1], n, self.ints([0] * self.S), counts=self.ints(lens))
        torch.cuda.synchronize()
        for name, y in zip(("k", "v"), out):
            y = y.cpu().numpy()
            for s in range(self.S):
                want = getattr(self.plain, name)[s, :, :lens[s]].transpose(1, 0, 2)
                assert np.array_equal(y[s, :lens[s]].astype(np.float64), want, equal_nan=True), (name, s)
                assert (y[s, lens[s]:] == 77.5).all()
        if self.pos is not None:
            for s in range(self.S):
                assert np.array_equal(self.pos[s, :, :lens[s]].cpu().numpy(), self.plain.pos[s, :, :lens[s]])


def tokens(r, S, T, KH, D, scale=1.0):
    return (r.standard_normal((S, T, KH, D)) * scale).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("S,T,KH,stride", [(1, 1, 1, 0), (3, 5, 2, 0), (2, 33, 3, 4), (5, 1, 8, 12)])
def test_append_and_read(zq, D, S, T, KH, stride):
    r = np.random.default_rng(D + T)
    d = Dev(zq, S, KH, D, 64)
    lens = [(7 * s) % 40 for s in range(S)]
    d.fill(lens, 5)
    k, v = tokens(r, S, T, KH, D), tokens(r, S, T, KH, D, 30.0)
    counts = [max(0, T - s) for s in range(S)]
    d.append(k, v, lens, counts=counts, first_pos=[100 * s + 3 for s in range(S)],
             stride=KH * D + stride if stride else 0)
    now = [min(64, lens[s] + counts[s]) for s in range(S)]
    d.rows_equal(now)
    for s in range(S):  # behind the new rows all is as it was
        assert (d.k[s, :, now[s]:] == 0xff).all() and d.ks[s, :, :, now[s]:].isnan().all()
        assert (d.pos[s, :, now[s]:] == -7).all() and d.weight[s, :, now[s]:].isnan().all()
        assert (d.weight[s, :, :now[s]] == 0).all()
    # the scales as they lie, and a cache without weight and pos
    b = Dev(zq, S, KH, D, 64, weight=False)
    b.append(k, v, lens)
    for s in range(S):
        n = lens[s] + counts[s]
        assert torch.equal(b.ks[s, :, :, lens[s]:n], d.ks[s, :, :, lens[s]:n])


@pytest.mark.gpu
def test_append_special_values(zq):
    D, KH = 64, 1
    r = np.random.default_rng(3)
    rows = []
    base = r.standard_normal(D).astype(np.float32)
    rows.append(np.zeros(D))
    rows.append(np.full(D, -0.0))
    for f in (1e-9, 3e-8, 1e-6, 1e-4, 1e4, 4e4, 1e6, 3e38):  # fp16's smallest steps, its range, fp32's range
        rows.append(base / np.abs(base).max() * f)
    x = np.tile(np.array([1.0, -1.0]), D // 2)  # equal magnitudes: the first one's sign
    rows += [x, -x, np.roll(x * (np.arange(D) % 5 == 1), 1)]
    for d in (0.25, 0.3125, 255 / 256, 129 * 2.0 ** -20):  # quotients on halves, and the next float on either side
        half = (np.arange(32) % 16 - 8 + 0.5) * d
        half[0] = -8 * d
        h32 = half.astype(np.float32)
        rows += [np.concatenate([h32, np.nextafter(h32, np.float32(np.inf))]),
                 np.concatenate([-h32, np.nextafter(h32, np.float32(-np.inf))])]
    for bad in (np.nan, np.inf, -np.inf):
        y = base.copy()
        y[5] = bad
        rows.append(y)
    k = np.array(rows, np.float32)[None, :, None]
    v = np.roll(k, 2, 1)  # values that are odd where the key is not, and the reverse
    dv = Dev(zq, 1, KH, D, 64)
    dv.append(k, v, [0])
    dv.rows_equal([len(rows)])


@pytest.mark.gpu
def test_append_stops_at_the_capacity(zq):
    r = np.random.default_rng(4)
    d = Dev(zq, 4, 2, 64, 32)
    lens = [30, 32, 0, 31]
    d.fill(lens, 9)
    before = [t.clone() for t in (d.k, d.v)]
    d.append(tokens(r, 4, 40, 2, 64), tokens(r, 4, 40, 2, 64), lens, counts=[40, 40, 40, -3])
    d.rows_equal([32, 32, 32, 31])
    for a, b in zip((d.k, d.v), before):
        assert torch.equal(a[1], b[1]) and torch.equal(a[3], b[3]) and torch.equal(a[0, :, :30], b[0, :, :30])
    # lengths that no cache has: nothing is written or read
    d.append(tokens(r, 4, 2, 2, 64), tokens(r, 4, 2, 2, 64), [-1, 33, 2 ** 31 - 1, -2 ** 31], counts=[2] * 4)
    d.rows_equal([32, 32, 32, 31])
    y = torch.full((4, 3, 2, 64), 5.5, device="cuda")
    zq.kv_q4_read_dev(d.c, y, None, 3, d.ints([-1, 32, 2 ** 31 - 1, 30]), counts=d.ints([3, 3, 3, 1]))
    torch.cuda.synchronize()
    assert (y[:3] == 5.5).all() and (y[3, 1:] == 5.5).all() and (y[3, 0] != 5.5).any()


SHAPES = [  # S, KH, G, D, C, lens, T
    (1, 1, 1, 64, 32, [0], 1),
    (1, 2, 4, 128, 32, [31], 1),
    (2, 1, 3, 256, 64, [33, 5], 1),
    (4, 2, 7, 64, 160, [0, 1, 100, 150], 5),
    (3, 2, 4, 128, 352, [300, 17, 31], 9),
    (2, 3, 1, 128, 128, [40, 63], 40),
    (1, 1, 20, 64, 224, [140], 3),
    (2, 2, 2, 256, 192, [96, 129], 33),
    (1, 2, 4, 128, 224, [0], 200),
    (1, 2, 8, 64, 416, [130], 270),
    (8, 4, 2, 256, 128, [0, 88, 13, 32, 64, 1, 80, 47], 40),  # many row tiles: the 128-row kernel at its widest
    (1, 1, 100, 64, 96, [60], 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [None, "set", "add"])
@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("S,KH,G,D,C,lens,T", SHAPES)
def test_attention(zq, S, KH, G, D, C, lens, T, full, weights):
    r = np.random.default_rng(S * 1000 + T)
    d = Dev(zq, S, KH, D, C)
    d.fill(lens, 11)
    if not full:
        d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D, 0.7), lens)
    if weights == "add":
        w = r.random((S, KH, C)).astype(np.float32)
        d.weight.copy_(torch.from_numpy(w))
        d.plain.weight[:] = w
    q = tokens(r, S, T, KH * G, D, 1.4)
    d.check_attention(q, lens, 1 / math.sqrt(D), full=full, weights=weights, stride=KH * G * D + 8 if T % 2 else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("D,T", [(64, 1), (128, 6), (128, 130), (256, 70)])
def test_attention_of_a_padded_batch(zq, D, T):
    """Idle sequences and short ones: their outputs, and nothing behind them, are written."""
    r = np.random.default_rng(T)
    S, KH, G = 6, 2, 4
    lens, counts = [0, 50, 64, 3, 0, 77], [T, 0, max(1, T // 2), T, 0, T + 5]
    d = Dev(zq, S, KH, D, 256)
    d.fill(lens, 2)
    d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D), lens, counts=[min(c, T) for c in counts])
    d.check_attention(tokens(r, S, T, KH * G, D), lens, 0.1, counts=counts, weights="set")
    d.check_attention(tokens(r, S, T, KH * G, D), lens, 0.1, counts=counts, full=True, weights="add")


@pytest.mark.gpu
@pytest.mark.parametrize("T,G", [(4, 4), (40, 4)])
def test_attention_nan_and_infinity_stay_where_they_are_seen(zq, T, G):
    """A new token with a NaN or an infinity turns the queries NaN that see it, not those before it; a query with one
    turns its own output NaN only; rows past the length are garbage already (Dev)."""
    r = np.random.default_rng(8)
    D, KH, S = 64, 2, 2
    lens = [45, 0]
    d = Dev(zq, S, KH, D, 128)
    d.fill(lens, 3)
    k, v = tokens(r, S, T, KH, D), tokens(r, S, T, KH, D)
    k[0, T // 2, 0, 7] = np.nan
    v[1, T - 1, 1, 9] = np.inf
    d.append(k, v, lens)
    q = tokens(r, S, T, KH * G, D)
    d.check_attention(q, lens, 0.125, weights="set")
    q[0, 1, 2, 3] = np.nan
    out, want, tol, _ = d.attention(q, lens, 0.125)
    assert np.isnan(out[0, 1, 2]).all()
    out[0, 1, 2] = want[0, 1, 2] = np.nan
    assert (np.isnan(out) == np.isnan(want)).all()
    ok = ~np.isnan(want)
    assert (np.abs(out - want)[ok] <= tol[ok]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 50])
def test_attention_far_scores(zq, T):
    """Scores that rise and fall by hundreds along the cache (the running maximum moves and weights vanish), queries of
    very small and very large magnitude, a negative and a zero scale."""
    r = np.random.default_rng(6)
    D, KH, G, n = 128, 1, 4, 700
    d = Dev(zq, 1, KH, D, 768)
    k = tokens(r, 1, n, KH, D, 0.05)
    k[0, :, 0] += np.sin(np.arange(n) / 40.0)[:, None] * 2
    d.append(k, tokens(r, 1, n, KH, D), [0])
    d.append(tokens(r, 1, T, KH, D), tokens(r, 1, T, KH, D), [n])
    q = tokens(r, 1, T, KH * G, D, 0.2) + 1.5
    q[:, :, 1] *= 1e-12
    q[:, :, 2] *= 30
    for scale in (1.0, -1.0, 0.0, 0.01):
        d.check_attention(q.astype(np.float32), [n], scale, weights="set")


@pytest.mark.gpu
@pytest.mark.parametrize("D,T,G", [(64, 1, 8), (128, 2, 4), (256, 1, 1), (64, 20, 8), (128, 12, 4),
                                     (128, 40, 4), (256, 70, 1), (256, 30, 2)])
def test_attention_of_a_long_cache(zq, D, T, G):
    """Keys split over many workgroups, and the capacity far above the length."""
    r = np.random.default_rng(D)
    n = 5003
    d = Dev(zq, 1, 1, D, 40000)
    d.fill([n], 1)
    d.append(tokens(r, 1, T, 1, D), tokens(r, 1, T, 1, D), [n])
    d.check_attention(tokens(r, 1, T, G, D, 1.5), [n], 1 / math.sqrt(D), weights="set")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
def test_many_rows_over_split_keys(zq, D):
    """Enough rows and heads for the 128-row kernel, and keys split over its workgroups, with lengths that leave some
    of the splits without keys."""
    r = np.random.default_rng(D)
    S, KH, G, T = 2, 8, 2, 70
    lens = [1400, 300]
    d = Dev(zq, S, KH, D, 2048)
    d.fill(lens, 7)
    d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D), lens)
    d.check_attention(tokens(r, S, T, KH * G, D, 1.3), lens, 1 / math.sqrt(D))
    d.check_attention(tokens(r, S, T, KH * G, D, 1.3), lens, 1 / math.sqrt(D), counts=[33, T], full=True, weights="set")


@pytest.mark.gpu
@pytest.mark.parametrize("D,T,G", [(64, 1, 4), (128, 9, 4), (64, 70, 2), (128, 70, 2), (256, 70, 2)])
def test_equal_calls_give_equal_bits(zq, D, T, G):
    """No result depends on the order in which waves or workgroups come to it."""
    r = np.random.default_rng(D + T)
    S, KH = 3, 8
    lens = [900, 410, 0]
    d = Dev(zq, S, KH, D, 1024)
    d.fill(lens, 11)
    d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D), lens)
    q = torch.from_numpy(tokens(r, S, T, KH * G, D, 1.4)).cuda()
    n = zq.attention_q4_workspace_bytes(d.c, T, KH * G, zq.ATTN_Q4_WEIGHTS)
    got = []
    for i in range(8):
        ws = torch.full((n,), 0xff if i % 2 else 0, dtype=torch.uint8, device="cuda")
        out = torch.full((S, T, KH * G, D), math.nan, device="cuda")
        zq.attention_q4_dev(d.c, q, out, T, KH * G, d.ints(lens), 0.1, flags=zq.ATTN_Q4_WEIGHTS, workspace=ws,
                            workspace_bytes=n)
        torch.cuda.synchronize()
        assert not out.isnan().any()
        got.append((out, d.weight.clone()))
    for out, w in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(w.view(torch.int32), got[0][1].view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_lengths_that_no_cache_has(zq, T):
    """Negative lengths count as 0 and those past the capacity as the capacity; counts below 0 as 0."""
    r = np.random.default_rng(T)
    S, KH, G, D, C = 6, 2, 4, 64, 96
    d = Dev(zq, S, KH, D, C)
    d.fill([C] * S, 3)
    lens = [-1, -2 ** 31, C, C + 1, 2 ** 31 - 1, C - 1]
    for counts in (None, [T, T, T, T, T, -5]):
        q = tokens(r, S, T, KH * G, D)
        d.check_attention(q, lens, 0.2, counts=counts, weights="set")
        d.check_attention(q, lens, 0.2, counts=counts, full=True, weights="add")


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_random_calls(zq, seed):
    """Shapes, lengths, idle sequences, strides and flags drawn at random, an append, an attention and an eviction each."""
    r = np.random.default_rng(1000 + seed)
    D = int(r.choice([64, 128, 256]))
    S, KH, G = int(r.integers(1, 6)), int(r.integers(1, 5)), int(r.integers(1, 9))
    T = int(r.choice([1, 1, 2, 5, 17, 60]))
    C = 32 * int(r.integers(1 + T // 32 + 1, 16))
    lens = [int(r.integers(0, C - T + 1)) for _ in range(S)]
    counts = [int(r.integers(0, T + 1)) if r.random() < 0.5 else T for _ in range(S)]
    d = Dev(zq, S, KH, D, C)
    d.fill(lens, seed)
    d.weight.nan_to_num_(0.0)
    d.plain.weight[:] = 0
    at = [int(r.integers(C, 5000)) for _ in range(S)]
    d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D, 0.6), lens, counts=counts, first_pos=at,
             stride=KH * D + 4 if r.random() < 0.5 else 0)
    full = bool(r.random() < 0.3)
    weights = [None, "set", "add"][int(r.integers(3))]
    d.check_attention(tokens(r, S, T, KH * G, D, 1.5), lens, float(r.uniform(0.02, 0.3)), counts=counts, full=full,
                      weights=weights, stride=KH * G * D + 16 if r.random() < 0.5 else 0)
    now = [n + c for n, c in zip(lens, counts)]
    d.rows_equal(now)
    d.plain.weight[:] = d.weight.cpu().numpy()
    keep = int(r.integers(1, C + 10))
    recent = int(r.integers(0, keep + 1))
    first = int(r.integers(0, keep - recent + 1))
    nxt = [a + c for a, c in zip(at, counts)]
    n = zq.kv_q4_evict_workspace_bytes(d.c, keep)
    zq.kv_q4_evict_dev(d.c, d.ints(now), keep, recent, first, next_pos=d.ints(nxt),
                       workspace=torch.empty(n, dtype=torch.uint8, device="cuda"), workspace_bytes=n)
    torch.cuda.synchronize()
    d.plain.evict(now, keep, recent, first, nxt)
    d.rows_equal([min(x, keep) for x in now])


@pytest.mark.gpu
def test_offsets_past_32_bits(zq):
    """Codes of more than 8 GiB: the last slots of the last head.  All other rows are zero (scores 0, values 0), so
    the softmax has a closed form."""
    KH, D, C = 8, 128, 1 << 24
    cuda = dict(device="cuda")
    k, v = (torch.full((1, KH, C, D // 2), 0x88, dtype=torch.uint8, **cuda) for _ in range(2))
    ks, vs = (torch.zeros((1, KH, D // 32, C), dtype=torch.float16, **cuda) for _ in range(2))
    w, pos = torch.zeros((1, KH, C), **cuda), torch.arange(C, dtype=torch.int32, **cuda).expand(1, KH, C).contiguous()
    c = zq.KVQ4(k, v, ks, vs, 1, KH, D, C, weight=w, pos=pos)
    lens = torch.tensor([C - 2], dtype=torch.int32, **cuda)
    r = np.random.default_rng(1)
    x = torch.from_numpy(tokens(r, 1, 2, KH, D)).cuda()
    zq.kv_q4_append_dev(c, x, x, 2, lens)
    back = torch.empty_like(x)
    zq.kv_q4_read_dev(c, None, back, 2, lens)
    q = 3 * back[:, 1:].repeat_interleave(2, 2).contiguous()  # heads in the kv heads' order
    n = zq.attention_q4_workspace_bytes(c, 1, 2 * KH, zq.ATTN_Q4_WEIGHTS)
    ws = torch.empty(n, dtype=torch.uint8, **cuda)
    out = torch.empty(1, 1, 2 * KH, D, **cuda)
    full = torch.tensor([C], dtype=torch.int32, **cuda)
    zq.attention_q4_dev(c, q, out, 1, 2 * KH, full, 0.05, flags=zq.ATTN_Q4_FULL | zq.ATTN_Q4_WEIGHTS, workspace=ws,
                        workspace_bytes=n)
    torch.cuda.synchronize()
    b, qd = back.double(), q.double()[0, 0]
    for h in range(2 * KH):
        s = (b[0, :, h // 2] @ qd[h]) * float(np.float32(0.05))
        e = torch.exp(s)
        p = e / (e.sum() + (C - 2))
        want = p @ b[0, :, h // 2]
        # a lane sums about 2^24 / (96 workgroups * 4 waves * 4 key groups) = 2^13.4 weights one after the other, 2^-10.6
        # at most; a weight is a multiple of 2^-24 where the largest is 2^6 at least, so each of the two rows that are
        # not zero is off by up to 2^-31 of the largest
        assert torch.allclose(out[0, 0, h].double(), want, rtol=1e-3, atol=2 * 2.0 ** -31 * b.abs().max().item()), h
    assert abs(w[0, 3].double().sum().item() - 2) < 2e-3
    # evict down to 64: the last row drew the most, the one before it more than the zero rows where that is so; the
    # others are equal, and the lowest slots stay
    drew = [w[0, h, C - 2].item() > w[0, h, 0].item() for h in range(KH)]
    m = zq.kv_q4_evict_workspace_bytes(c, 64)
    zq.kv_q4_evict_dev(c, full, 64, 0, 0, workspace=torch.empty(m, dtype=torch.uint8, **cuda), workspace_bytes=m)
    first = torch.tensor([62], dtype=torch.int32, **cuda)
    again = torch.empty_like(x)
    zq.kv_q4_read_dev(c, None, again, 2, first)
    torch.cuda.synchronize()
    assert any(drew) and not all(drew)
    for h in range(KH):
        assert pos[0, h, 62:64].tolist() == [C - 2 if drew[h] else 62, C - 1], h
        assert torch.equal(again[0, 1, h], back[0, 1, h])
        assert torch.equal(again[0, 0, h], back[0, 0, h]) if drew[h] else (again[0, 0, h] == 0).all()
    assert (pos[0, :, 64:] == -1).all()


def random_cache(zq, r, S, KH, D, C, lens):
    d = Dev(zq, S, KH, D, C)
    d.fill(lens, int(r.integers(1 << 30)))
    w = r.exponential(size=(S, KH, C)).astype(np.float32) ** 3
    w[r.random(w.shape) < 0.2] = 0.0
    w[r.random(w.shape) < 0.1] = 1.5
    w[r.random(w.shape) < 0.02] = -0.0
    pos = np.argsort(r.random((S, KH, C)), -1) * 3
    d.weight.copy_(torch.from_numpy(w))
    d.pos.copy_(torch.from_numpy(pos.astype(np.int32)))
    d.plain.weight[:], d.plain.pos[:] = w, pos
    return d


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("D,C,lens,keep,recent,first", [
    (64, 96, [90, 0, 1, 33], 32, 8, 4), (64, 96, [90, 31, 32, 33], 1, 0, 0), (128, 128, [128, 100], 100, 100, 0),
    (128, 2112, [2100, 1025, 1024], 1000, 300, 16), (256, 96, [96, 64], 95, 0, 95), (64, 5024, [5000], 4999, 2000, 4),
    (64, 9024, [9001, 2], 64, 10, 10), (128, 64, [64, 50], 500, 100, 4),
    (64, 12032, [2048, 2049, 8192, 8193], 2000, 100, 4), (64, 26016, [26000, 16385], 7000, 100, 4)])
def test_evict(zq, D, C, lens, keep, recent, first, in_place):
    r = np.random.default_rng(keep + C)
    S, KH = len(lens), 3
    d = random_cache(zq, r, S, KH, D, C, lens)
    if C == 96 and keep == 32:  # what no attention gives, but a caller's own weights may hold
        for x in (d.weight, d.plain.weight):
            x[0, 0, 5], x[0, 0, 60], x[0, 1, 3], x[0, 1, 70] = math.nan, math.nan, math.inf, -math.inf
    next_pos = [3 * C] * S
    to = d if in_place else Dev(zq, S, KH, D, -(-min(keep, C) // 32) * 32)
    n = zq.kv_q4_evict_workspace_bytes(d.c, keep)
    ws = torch.full((n + 64,), 0xff, dtype=torch.uint8, device="cuda")
    args = (d.c, d.ints(lens), keep, recent, first)
    opts = dict(next_pos=d.ints(next_pos), dst=None if in_place else to.c, workspace=ws[:n], workspace_bytes=n)
    was = [t.clone() for t in (d.k, d.v, d.ks, d.vs, d.weight, d.pos)]
    zq.kv_q4_evict_dev(*args, **opts)
    torch.cuda.synchronize()
    assert (ws[n:] == 0xff).all()
    kept = [min(x, keep) for x in lens]
    d.plain.evict(lens, keep, recent, first, next_pos, to=None if in_place else to.plain)

    def check():
        to.rows_equal(kept)
        got, want = to.weight.cpu().numpy(), to.plain.weight
        for s in range(S):
            assert np.array_equal(got[s, :, :kept[s]], want[s, :, :kept[s]].astype(np.float32), equal_nan=True)
            if in_place:
                assert (got[s, :, kept[s]:lens[s]] == -np.inf).all() and (to.pos[s, :, kept[s]:lens[s]] == -1).all()
    check()
    if in_place:
        for s in range(S):
            assert torch.equal(was[5][s, :, lens[s]:], d.pos[s, :, lens[s]:])
        zq.kv_q4_evict_dev(*args, **opts)  # the emptied slots are the lowest: a second time changes nothing
        torch.cuda.synchronize()
        check()
    else:
        for a, b in zip(was, (d.k, d.v, d.ks, d.vs, d.weight, d.pos)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), "the source changed"
        for s in range(S):
            assert (to.k[s, :, kept[s]:] == 0xff).all() and (to.pos[s, :, kept[s]:] == -7).all()


@pytest.mark.gpu
def test_a_cache_in_use(zq):
    """Prompt, decode with accumulated weights, eviction, decode behind it, a drafted run of tokens: the operators
    one after the other, beside the plain cache."""
    r = np.random.default_rng(12)
    S, KH, G, D, C = 3, 2, 4, 64, 192
    d = Dev(zq, S, KH, D, C)
    scale = 1 / math.sqrt(D)
    lens, at = [0, 0, 0], [0, 0, 0]

    def step(T, counts, weights):
        k, v, q = tokens(r, S, T, KH, D), tokens(r, S, T, KH, D), tokens(r, S, T, KH * G, D, 1.3)
        d.append(k, v, lens, counts=counts, first_pos=at)
        d.check_attention(q, lens, scale, counts=counts, weights=weights)
        d.plain.weight[:] = d.weight.cpu().numpy()  # the device's own sums: ranks are compared exactly
        for s in range(S):
            lens[s] += counts[s]
            at[s] += counts[s]

    step(120, [120, 70, 99], "add")
    for i in range(4):
        step(1, [1, 1, i % 2], "add")
    keep = 64
    n = zq.kv_q4_evict_workspace_bytes(d.c, keep)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    for round_ in range(2):
        zq.kv_q4_evict_dev(d.c, d.ints(lens), keep, 16, 4, next_pos=d.ints(at), workspace=ws, workspace_bytes=n)
        torch.cuda.synchronize()
        d.plain.evict(lens, keep, 16, 4, at)
        for s in range(S):
            lens[s] = min(lens[s], keep)
        d.rows_equal(lens)
        for i in range(3):
            step(1, [1, 1, 1], "add")
        step(6, [6, 3, 0], "add")


@pytest.mark.gpu
def test_graph_replays_follow_the_lengths(zq):
    """append + attention + weights + eviction captured once; replays read lens, counts and positions on the device and
    equal the eager calls bit for bit, with eager work between them."""
    r = np.random.default_rng(2)
    S, KH, G, D, C, keep = 2, 2, 4, 128, 512, 480
    eager, graph = Dev(zq, S, KH, D, C), Dev(zq, S, KH, D, C)
    lens0 = [400, 77]
    for d in (eager, graph):
        d.fill(lens0, 4)
        d.weight.nan_to_num_(0.0)
    k, v, q = (torch.zeros(S, 1, h, D, device="cuda") for h in (KH, KH, KH * G))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lens, counts, nxt = i32(lens0), i32([1, 1]), i32([1000, 1000])
    flags = zq.ATTN_Q4_WEIGHTS | zq.ATTN_Q4_ADD
    n = zq.attention_q4_workspace_bytes(eager.c, 1, KH * G, flags)
    m = zq.kv_q4_evict_workspace_bytes(eager.c, keep)

    def run(d, ws, out, stream):
        zq.kv_q4_append_dev(d.c, k, v, 1, lens, counts=counts, first_pos=nxt, stream=stream)
        zq.attention_q4_dev(d.c, q, out, 1, KH * G, lens, 0.09, counts=counts, flags=flags, workspace=ws[:n],
                            workspace_bytes=n, stream=stream)
        zq.kv_q4_evict_dev(d.c, lens, keep, 32, 4, next_pos=nxt, workspace=ws[n:], workspace_bytes=m, stream=stream)

    n = -(-n // 16) * 16
    wa, wb = (torch.empty(n + m, dtype=torch.uint8, device="cuda") for _ in range(2))
    oa, ob = torch.zeros(S, 1, KH * G, D, device="cuda"), torch.zeros(S, 1, KH * G, D, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        run(graph, wb, ob, torch.cuda.current_stream())
    for step in range(5):
        for x in (k, v, q):
            x.copy_(torch.from_numpy(r.standard_normal(tuple(x.shape)).astype(np.float32)))
        counts.copy_(i32([1, step % 2]))
        torch.cuda.synchronize()
        run(eager, wa, oa, None)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa, ob)
        for a, b in ((eager.k, graph.k), (eager.vs, graph.vs), (eager.weight, graph.weight), (eager.pos, graph.pos)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), step
        lens += counts
        nxt += 1
        lens.clamp_(max=keep)


@pytest.mark.gpu
def test_two_streams_at_once(zq):
    """Two caches on two streams, each with its own workspace: the results of one after the other."""
    KH, G, D, C, n = 2, 4, 128, 2048, 1900
    ds = [Dev(zq, 1, KH, D, C) for _ in range(2)]
    r = np.random.default_rng(5)
    q = [torch.from_numpy(tokens(r, 1, 4, KH * G, D)).cuda() for _ in ds]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for i, d in enumerate(ds):
        d.fill([n + 4], i)
    need = zq.attention_q4_workspace_bytes(ds[0].c, 4, KH * G, zq.ATTN_Q4_WEIGHTS)
    outs = [[torch.zeros(1, 4, KH * G, D, device="cuda") for _ in range(6)] for _ in ds]
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    for j in range(6):
        for i, d in enumerate(ds):
            zq.attention_q4_dev(d.c, q[i], outs[i][j], 4, KH * G, lens, 0.1, flags=zq.ATTN_Q4_WEIGHTS, workspace=ws[i],
                                workspace_bytes=need, stream=streams[i])
    torch.cuda.synchronize()
    for i, d in enumerate(ds):
        one = torch.zeros(1, 4, KH * G, D, device="cuda")
        zq.attention_q4_dev(d.c, q[i], one, 4, KH * G, lens, 0.1, workspace=ws[i], workspace_bytes=need)
        torch.cuda.synchronize()
        assert all(torch.equal(o, one) for o in outs[i])


@pytest.mark.gpu
def test_host_addresses_are_refused(zq):
    """Raw addresses of host memory are found before a kernel gets them."""
    buf = np.zeros(1 << 16, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    c = zq.KVQ4(p, p + 8192, p + 16384, p + 20480, 1, 1, 64, 64)
    x = torch.zeros(64, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(zq.ZQError, match="status -1"):
        zq.kv_q4_append_dev(c, x, x, 1, lens)


@pytest.mark.gpu
def test_evict_refuses_a_host_destination(zq):
    """The rows' new cache must lie on the cache's device, as the cache itself."""
    d = Dev(zq, 1, 1, 64, 64)
    d.fill([40], 1)
    buf = np.zeros(1 << 16, np.uint8)
    p = (buf.ctypes.data + 255) // 256 * 256
    dst = zq.KVQ4(p, p + 4096, p + 8192, p + 12288, 1, 1, 64, 64, weight=p + 16384, pos=p + 20480)
    n = zq.kv_q4_evict_workspace_bytes(d.c, 16)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    with pytest.raises(zq.ZQError, match="status -1"):
        zq.kv_q4_evict_dev(d.c, d.ints([40]), 16, 4, 4, dst=dst, workspace=ws, workspace_bytes=n)
    torch.cuda.synchronize()
    assert not buf.any()


@pytest.mark.gpu
@pytest.mark.parametrize("to_other", [False, True])
def test_graph_replays_evict_what_the_replay_finds(zq, to_other):
    """A captured append, attention with weights and eviction, replayed while the lengths rise past `keep`: every replay
    drops the rows that the rule says, of the weights that the replay before has left, and equals the eager calls."""
    r = np.random.default_rng(21)
    S, KH, G, D, C, keep, recent, first, T = 3, 2, 4, 64, 512, 300, 32, 4, 5
    lens0, at0 = [298, 77, 299], [298, 77, 299]
    eager, graph = Dev(zq, S, KH, D, C), Dev(zq, S, KH, D, C)
    for d in (eager, graph):
        d.fill(lens0, 4)
    other = [Dev(zq, S, KH, D, 320) for _ in range(2)]
    k, v, q = (torch.zeros(S, T, h, D, device="cuda") for h in (KH, KH, KH * G))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    lens, counts, at = i32(lens0), i32([T] * S), i32(at0)
    held, nxt = i32([0] * S), i32([0] * S)
    flags = zq.ATTN_Q4_WEIGHTS | zq.ATTN_Q4_ADD
    n = -(-zq.attention_q4_workspace_bytes(eager.c, T, KH * G, flags) // 16) * 16
    m = zq.kv_q4_evict_workspace_bytes(eager.c, keep)

    def step_of(d, ws, out, stream):
        zq.kv_q4_append_dev(d.c, k, v, T, lens, counts=counts, first_pos=at, stream=stream)
        zq.attention_q4_dev(d.c, q, out, T, KH * G, lens, 0.11, counts=counts, flags=flags, workspace=ws[:n],
                            workspace_bytes=n, stream=stream)

    def evict(d, to, ws, stream):
        zq.kv_q4_evict_dev(d.c, held, keep, recent, first, next_pos=nxt, dst=to.c if to_other else None, workspace=ws[n:],
                           workspace_bytes=m, stream=stream)

    wa, wb = (torch.full((n + m,), 0xff, dtype=torch.uint8, device="cuda") for _ in range(2))
    oa, ob = (torch.zeros(S, T, KH * G, D, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        step_of(graph, wb, ob, torch.cuda.current_stream())
        evict(graph, other[1], wb, torch.cuda.current_stream())
    now, pos, dropped = list(lens0), list(at0), 0
    for step in range(4):
        for x in (k, v, q):
            x.copy_(torch.from_numpy(r.standard_normal(tuple(x.shape)).astype(np.float32) * 1.3))
        new = [T, step % 3, T - step]
        after, end = [a + b for a, b in zip(now, new)], [a + b for a, b in zip(pos, new)]
        for t, x in ((lens, now), (counts, new), (at, pos), (held, after), (nxt, end)):
            t.copy_(i32(x))
        torch.cuda.synchronize()
        plain = eager.plain
        plain.append(k.cpu().numpy(), v.cpu().numpy(), now, new, pos)
        step_of(eager, wa, oa, None)
        torch.cuda.synchronize()
        plain.weight[:] = eager.weight.cpu().numpy()  # the device's own sums: ranks are compared exactly
        evict(eager, other[0], wa, None)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa, ob)
        for a, b in ((eager, graph), other):
            for x in ("k", "v", "ks", "vs", "weight", "pos"):
                assert torch.equal(getattr(a, x).view(torch.uint8), getattr(b, x).view(torch.uint8)), (step, x)
        to = other[0] if to_other else eager
        plain.evict(after, keep, recent, first, end, to=to.plain if to_other else None)
        kept = [min(x, keep) for x in after]
        to.rows_equal(kept)
        for s in range(S):
            assert np.array_equal(to.weight[s, :, :kept[s]].cpu().numpy(), to.plain.weight[s, :, :kept[s]].astype(np.float32))
            assert to_other or (eager.pos[s, :, kept[s]:after[s]] == -1).all()
        dropped += sum(after) - sum(kept)
        now, pos = after if to_other else kept, end
    assert dropped >= 16


@pytest.mark.gpu
def test_two_streams_at_once_draw_the_same_weights(zq):
    """Two caches on two streams, each with its own workspace: outputs and accumulated weights of one after the other."""
    KH, G, D, C, n, T = 2, 4, 128, 2048, 1900, 4
    flags = zq.ATTN_Q4_WEIGHTS | zq.ATTN_Q4_ADD
    r = np.random.default_rng(5)
    ds, alone = ([Dev(zq, 1, KH, D, C) for _ in range(2)] for _ in range(2))
    for i in range(2):
        for d in (ds[i], alone[i]):
            d.fill([n + T], i)
    q = [torch.from_numpy(tokens(r, 1, T, KH * G, D)).cuda() for _ in ds]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    need = zq.attention_q4_workspace_bytes(ds[0].c, T, KH * G, flags)
    outs = [[torch.zeros(1, T, KH * G, D, device="cuda") for _ in range(6)] for _ in ds]
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    call = lambda d, i, out, stream: zq.attention_q4_dev(d.c, q[i], out, T, KH * G, lens, 0.1, flags=flags, workspace=ws[i],
                                                         workspace_bytes=need, stream=stream)
    torch.cuda.synchronize()
    for j in range(6):
        for i, d in enumerate(ds):
            call(d, i, outs[i][j], streams[i])
    torch.cuda.synchronize()
    for i, d in enumerate(alone):
        for j in range(6):
            one = torch.zeros(1, T, KH * G, D, device="cuda")
            call(d, i, one, None)
            torch.cuda.synchronize()
            assert torch.equal(outs[i][j], one)
        assert torch.equal(ds[i].weight.view(torch.int32), d.weight.view(torch.int32))
        # every head's weights of a query sum to 1: sums of n fp32 terms, 6 calls' T * G of them a kv head
        total = d.weight[0, :, :n + T].double().sum(-1)
        assert ((total - 6 * T * G).abs() <= 6 * T * G * (n + T) * 2 * U).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,T,G", [(64, 1, 4), (64, 512, 4), (128, 512, 4), (256, 2048, 2), (256, 3, 3)])
def test_equal_rows_of_a_long_cache(zq, D, T, G):
    """zq_kv.h's bound where sums round the same way again and again: one row, and 300,002 others that are equal.
    A lane's running sum takes 8 additions of a pair of weights for 32 (D = 256) or 64 keys, its outputs 4 rounded
    products: 12 / 32 n at most, and the products' own sums, the two halves of a weight, the merges and the quotient are
    within 128 roundings.  A score here is one product: 2^-21 of itself, and as much for the exponential."""
    n, KH = 300003, 8 if T > 1 else 2
    C = -(-n // 32) * 32
    cuda = dict(device="cuda")
    k, v = (torch.empty((1, KH, C, D // 2), dtype=torch.uint8, **cuda) for _ in range(2))
    ks, vs = (torch.empty((1, KH, D // 32, C), dtype=torch.float16, **cuda) for _ in range(2))
    w = torch.zeros((1, KH, C), **cuda)
    c = zq.KVQ4(k, v, ks, vs, 1, KH, D, C, weight=w)
    r = np.random.default_rng(D)
    new_k = torch.zeros(1, 2, KH, D, **cuda)
    new_k[0, 0, :, 0], new_k[0, 1, :, 0] = 1.0, 0.3
    new_v = torch.from_numpy((r.random((1, 2, KH, D)) + 1).astype(np.float32)).cuda()
    zero = torch.zeros(1, dtype=torch.int32, **cuda)
    zq.kv_q4_append_dev(c, new_k, new_v, 2, zero)
    hk, hv = torch.empty_like(new_k), torch.empty_like(new_v)
    zq.kv_q4_read_dev(c, hk, hv, 2, zero)
    for t in (k, v):
        t[:, :, 2:] = t[:, :, 1:2]
    for t in (ks, vs):
        t[..., 2:] = t[..., 1:2]
    q = torch.zeros(1, T, KH * G, D, **cuda)
    q[..., 0] = torch.from_numpy(r.uniform(0.5, 3, (1, T, KH * G)).astype(np.float32)).cuda()
    flags = zq.ATTN_Q4_FULL | zq.ATTN_Q4_WEIGHTS
    need = zq.attention_q4_workspace_bytes(c, T, KH * G, flags)
    ws, out = torch.empty(need, dtype=torch.uint8, **cuda), torch.empty_like(q)
    zq.attention_q4_dev(c, q, out, T, KH * G, torch.tensor([n], dtype=torch.int32, **cuda), 1.0, flags=flags, workspace=ws,
                        workspace_bytes=need)
    torch.cuda.synchronize()
    s = q[0, :, :, 0].double()[..., None] * hk[0, :, :, 0].double().T.repeat_interleave(G, 0)[None]  # [T][H][2 rows]
    e = torch.exp(s - s.amax(-1, keepdim=True)) * torch.tensor([1.0, n - 1.0], dtype=torch.float64, **cuda)
    p = e / e.sum(-1, keepdim=True)
    vv = hv[0].double().repeat_interleave(G, 1)  # [2][H][D]
    want = p[..., :1] * vv[0] + p[..., 1:] * vv[1]
    tol = (n / 2 + 128) * U + 2 * (s.abs().max().item() + 1) * 2.0 ** -21
    assert ((out[0].double() - want).abs().max() <= tol * vv.abs().max()).item()
    drawn = p.sum(0).reshape(KH, G, 2).sum(1)  # of row 0, and of the others together
    for i, at in ((0, 0), (1, 1), (1, n - 1)):
        each = drawn[:, i] / (1 if i == 0 else n - 1)
        assert ((w[0, :, at].double() - each).abs() <= (tol + T * G * U) * each).all()

"""GPU tier: the decoder on the 4-bit KV cache (zq_model_set_kv_cache) against a
forward pass in 64 bits that attends over the rows the device holds.

A row's values are the rounding of keys and values that the device computes in
fp32, so a value next to a border between two codes may fall on either side:
the rows are read back (zq_kv.h), each value compared with the 64-bit key or
value it stands for (one step of its block's scale at most: half a step of the
code, a whole one where the code ends at 7, and eight half steps of the scale's
8 bits), and the 64-bit forward goes on from them.  Logits then meet the bar of
the fp32 decoder, 1e-4 + 1e-4 * max|logit|."""
import ctypes
import math
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def build(zq, heads=8, kv_heads=2, head_dim=64, layers=2, max_positions=256, graph=True, rope_dim=0, fmt=0):
    from zeninfer_amd.model import Model
    os.environ["ZQ_MODEL_GRAPH"] = "1" if graph else "0"
    try:
        m = Model.synthetic(embedding=heads * head_dim, layers=layers, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                            ffn=1024, vocab=640, context=4096, max_positions=max_positions, rope_base=10000.0,
                            rms_epsilon=1e-5, eos_token=639, rope_dim=rope_dim, weight_format=fmt)
    finally:
        os.environ.pop("ZQ_MODEL_GRAPH", None)
    m.set_prefill_mode(1)
    return m


class Forward:
    """The decoder in 64 bits; keys and values come from the device's cache."""

    def __init__(self, zq, m):
        import torch
        from zeninfer_amd import model as M
        self.zq, self.m, self.c = zq, m, m.config

        def dense(layer, which):
            p, rows, cols, fmt = m.weight(layer, which)
            y = torch.empty(rows, cols, device="cuda")
            zq.dequantize_dev(fmt, p, y, rows, cols)
            torch.cuda.synchronize()
            return y.cpu().numpy().astype(np.float64)
        self.embed, self.out = dense(M.GLOBAL, M.W_EMBED), dense(M.GLOBAL, M.W_OUTPUT)
        self.layers = [[dense(l, w) for w in (M.W_Q, M.W_K, M.W_V, M.W_O, M.W_GATE, M.W_UP, M.W_DOWN)]
                       for l in range(self.c["layers"])]

    def rows(self, layer):
        """(k, v [KH][n][D], scales of both, pos [KH][n]) that the device holds."""
        import torch
        cache, n, _ = self.m.kv_cache(layer)
        KH, D, C = cache.kv_heads, cache.head_dim, cache.capacity
        k, v = (torch.empty(1, n, KH, D, device="cuda") for _ in range(2))
        first = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.zq.kv_q4_read_dev(cache, k, v, n, first)
        torch.cuda.synchronize()

        def host(addr, dtype, count):
            t = np.empty(count, dtype)
            hip = ctypes.CDLL("libamdhip64.so")
            assert hip.hipMemcpy(t.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(addr), ctypes.c_size_t(t.nbytes), 2) == 0
            return t
        ks = host(cache.c.k_scale, np.float16, KH * D // 32 * C).reshape(KH, D // 32, C)[..., :n]
        vs = host(cache.c.v_scale, np.float16, KH * D // 32 * C).reshape(KH, D // 32, C)[..., :n]
        pos = host(cache.c.pos, np.int32, KH * C).reshape(KH, C)[:, :n]
        f = lambda t: t[0].permute(1, 0, 2).cpu().numpy().astype(np.float64)
        return f(k), f(v), ks.astype(np.float64), vs.astype(np.float64), pos

    def rope(self, x, pos):
        """Adjacent pairs; the table's angles are fp32, as the host builds them (powf: another float's power may be a
        last place off, which at position 2000 turns an angle by 2000 * 2^-24)."""
        r = self.c["rope_dim"] or self.c["head_dim"]
        powf = ctypes.CDLL("libm.so.6").powf
        powf.restype, powf.argtypes = ctypes.c_float, [ctypes.c_float, ctypes.c_float]
        e = np.float32(-2.0) * np.arange(r // 2, dtype=np.float32) / np.float32(r)
        f = np.array([powf(self.c["rope_base"] or 10000.0, float(i)) for i in e], np.float32)
        a = np.asarray(pos, np.float32)[:, None] * f[None]
        cs, sn = np.cos(a).astype(np.float64)[:, None], np.sin(a).astype(np.float64)[:, None]
        y = x.copy()
        p, q = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = p * cs - q * sn, p * sn + q * cs
        return y

    def step(self, tokens, pos):
        """Logits of the last of `tokens` (the newest rows of the cache, at positions pos ...), and checks the rows."""
        c = self.c
        H, KH, D = c["heads"], c["kv_heads"], c["head_dim"]
        T = len(tokens)
        rms = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5)
        x = self.embed[np.asarray(tokens)]
        at = np.arange(pos, pos + T)
        for l, (wq, wk, wv, wo, wg, wu, wd) in enumerate(self.layers):
            h = rms(x)
            q = self.rope((h @ wq.T).reshape(T, H, D), at)
            k = self.rope((h @ wk.T).reshape(T, KH, D), at)
            v = (h @ wv.T).reshape(T, KH, D)
            K, V, ks, vs, kpos = self.rows(l)
            n = K.shape[1]
            assert (kpos[:, n - T:] == at).all()
            for held, new, s in ((K, k, ks), (V, v, vs)):
                step = np.repeat(np.abs(s[:, :, n - T:]).transpose(0, 2, 1), 32, -1)
                off = np.abs(held[:, n - T:] - new.transpose(1, 0, 2))
                assert (off <= step * (1 + 8 * 2.0 ** -8) + 1e-5 * np.abs(new).max()).all(), (l, off.max())
            y = np.empty((T, H, D))
            for t in range(T):
                m = n - T + t + 1
                for i in range(H):
                    s = K[i * KH // H, :m] @ q[t, i] / math.sqrt(D)
                    p = np.exp(s - s.max())
                    y[t, i] = (p / p.sum()) @ V[i * KH // H, :m]
            x = x + y.reshape(T, H * D) @ wo.T
            h = rms(x)
            g = h @ wg.T
            x = x + (g / (1 + np.exp(-g)) * (h @ wu.T)) @ wd.T
        return rms(x[-1]) @ self.out.T


def close(got, want):
    assert np.abs(got - want).max() <= 1e-4 + 1e-4 * np.abs(want).max(), (np.abs(got - want).max(), np.abs(want).max())


@pytest.mark.parametrize("heads,kv_heads,head_dim,rope_dim,fmt", [(8, 2, 64, 0, 0), (4, 4, 128, 0, 0), (7, 1, 64, 32, 0),
                                                                  (2, 1, 256, 0, 0), (8, 2, 64, 0, 12), (8, 4, 64, 62, 14)])
def test_prefill_and_decode(zq, heads, kv_heads, head_dim, rope_dim, fmt):
    """Every decode form (fused GEMV prologues, residual-norm K-quants, plain) and the prefill, packed q|k|v or not."""
    from zeninfer_amd.model import KV_Q4
    if fmt and heads * head_dim % 256:
        pytest.skip("super-block formats take widths of 256")
    m = build(zq, heads, kv_heads, head_dim, rope_dim=rope_dim, fmt=fmt)
    fp32 = m.memory()["kv_cache"]
    m.set_kv_cache(KV_Q4)
    assert m.memory()["kv_cache"] < fp32 / 6  # 4.5 of 32 bits, and weight and pos
    f = Forward(zq, m)
    r = np.random.default_rng(1)
    for n in (1, 37, 150):
        prompt = r.integers(0, 640, n).tolist()
        tok, lg = m.prefill(prompt)
        close(lg, f.step(prompt, 0))
        for i in range(3):
            new, lg = m.decode(tok)
            close(lg, f.step([tok], n + i))
            tok = new
        assert m.kv_cache(0)[1:] == (n + 3, n + 3)
    m.close()


def test_graph_equals_eager_and_forms_switch(zq):
    from zeninfer_amd import zq as Z
    from zeninfer_amd.model import KV_F32, KV_Q4
    prompt = list(range(3, 60))
    seqs = []
    for graph in (True, False):
        m = build(zq, graph=graph)
        base, _, _ = m.generate(prompt, 12)
        m.set_kv_cache(KV_Q4)
        with pytest.raises(Z.ZQError):
            m.set_kv_cache(KV_Q4, 16, 10, 7)
        with pytest.raises(Z.ZQError):
            m.set_kv_cache(KV_F32, 16)
        with pytest.raises(Z.ZQError):
            m.set_kv_cache(2)
        tok, lg = m.prefill(prompt)
        out = [lg]
        for _ in range(10):
            tok, lg = m.decode(tok)
            out.append(lg)
        seqs.append(out)
        m.set_kv_cache(KV_F32)
        assert m.kv_cache(0) == (None, 0, 0)
        again, _, _ = m.generate(prompt, 12)
        assert again == base, "the fp32 cache's results changed"
        m.close()
    for a, b in zip(*seqs):
        assert np.array_equal(a, b)


def test_capacity_without_eviction(zq):
    from zeninfer_amd import zq as Z
    from zeninfer_amd.model import KV_Q4
    m = build(zq, max_positions=70)
    m.set_kv_cache(KV_Q4, 20, 5, 2)  # 20 + a prefill pass is more than 70: every position has room
    m.prefill(list(range(60)))
    for t in range(10):
        m.decode(t)
    assert m.kv_cache(1)[1:] == (70, 70)
    with pytest.raises(Z.ZQError):
        m.decode(1)
    m.close()


def test_eviction_keeps_the_rule(zq):
    """A prompt of two passes over a cache of 200 + 1024 rows: what the second pass finds is the first pass's rows,
    evicted by its weights; then decode runs past the capacity and evicts again."""
    import torch
    from tests.test_kv_q4 import Plain
    from zeninfer_amd.model import KV_Q4
    keep, recent, first = 200, 60, 4
    r = np.random.default_rng(4)
    prompt = r.integers(0, 640, 1500).tolist()
    m = build(zq, max_positions=2600)
    m.set_kv_cache(KV_Q4, keep, recent, first)
    f = Forward(zq, m)
    m.prefill(prompt[:1024])
    want = []
    for l in range(2):
        cache, n, at = m.kv_cache(l)
        assert (n, at) == (1024, 1024)
        K, V, _, _, pos = f.rows(l)
        w = np.empty(cache.kv_heads * cache.capacity, np.float32)
        hip = ctypes.CDLL("libamdhip64.so")
        assert hip.hipMemcpy(w.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(cache.c.weight), ctypes.c_size_t(w.nbytes), 2) == 0
        w = w.reshape(cache.kv_heads, -1)[:, :n]
        # every query's heads add 1 to their kv head's rows (fp32 sums of up to 4096 weights)
        assert np.allclose(w.astype(np.float64).sum(-1), 1024 * 4, rtol=4096 * 2.0 ** -24)
        p = Plain(1, cache.kv_heads, cache.head_dim, n)
        p.k[0], p.v[0], p.weight[0], p.pos[0] = K, V, w, pos
        p.evict([n], keep, recent, first, [1024])
        want.append(p)
    tok, lg = m.prefill(prompt)
    assert m.kv_cache(0)[1:] == (keep + 476, 1500)
    for l in range(2):
        K, V, _, _, pos = f.rows(l)
        assert np.array_equal(pos[:, :keep], want[l].pos[0, :, :keep])
        assert np.array_equal(K[:, :keep], want[l].k[0, :, :keep]) and np.array_equal(V[:, :keep], want[l].v[0, :, :keep])
        assert (pos[:, keep:] == np.arange(1024, 1500)).all()
    close(lg, f.step(prompt[1024:], 1024))
    room = m.kv_cache(0)[0].capacity - 676  # steps until it is full: the next one evicts
    assert room >= 1024 - 476
    for i in range(room + 12):
        new, lg = m.decode(tok, logits=i >= room - 3)
        if i >= room - 3:
            close(lg, f.step([tok], 1500 + i))
        tok = new
    _, n, at = m.kv_cache(0)
    assert at == 1500 + room + 12 and n == keep + 12
    for l in range(2):
        pos = f.rows(l)[4]
        for h in range(pos.shape[0]):
            # the rows that were protected at the eviction, and those since
            kept = pos[h].tolist()
            assert set(range(1500 + room - recent, at)) <= set(kept) and set(range(first)) <= set(kept)
            assert len(set(kept)) == n
    m.close()


def test_switching_back_frees_what_the_4_bit_form_took(zq):
    """An fp32 model is charged for no 4-bit workspace, however often the form changes, and the memory is given back."""
    import torch
    from zeninfer_amd.model import KV_F32, KV_Q4
    m = build(zq)
    start = m.memory()
    m.set_kv_cache(KV_F32)
    assert m.memory() == start
    free = []
    for i in range(3):
        m.set_kv_cache(KV_Q4, 64, 8, 4)
        four = m.memory()
        assert four["activations"] > start["activations"] and four["kv_cache"] < start["kv_cache"]
        m.set_kv_cache(KV_Q4)
        m.prefill(list(range(20)))
        m.set_kv_cache(KV_F32)
        assert m.memory() == start
        with pytest.raises(zq.ZQError):
            m.set_kv_cache(KV_F32, 16)
        m.prefill(list(range(20)))
        free.append(torch.cuda.mem_get_info()[0])
    assert free[2] >= free[0]
    m.close()


def test_a_bound_that_is_never_reached_is_none(zq):
    """Rows and a prefill pass (1024 tokens) together reach max_positions: the cache of rows == 0, without weights; one
    row fewer and they are drawn."""
    from zeninfer_amd.model import KV_Q4
    hip = ctypes.CDLL("libamdhip64.so")
    for max_positions, rows, bounded in ((1100, 76, False), (1100, 75, True)):
        m = build(zq, max_positions=max_positions)
        m.set_kv_cache(KV_Q4)
        whole = m.memory()
        m.set_kv_cache(KV_Q4, rows, 5, 2)
        assert (m.memory() == whole) == (not bounded)
        m.prefill(list(range(60)))
        m.decode(3)
        cache, n, _ = m.kv_cache(1)
        w = np.empty(cache.kv_heads * cache.capacity, np.float32)
        assert hip.hipMemcpy(w.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(cache.c.weight), ctypes.c_size_t(w.nbytes), 2) == 0
        w = w.reshape(cache.kv_heads, -1)[:, :n]
        # 61 queries of 4 heads a kv head, whose weights each sum to 1
        assert np.allclose(w.astype(np.float64).sum(-1), 61 * 4 if bounded else 0, rtol=61 * 4 * 2.0 ** -22)
        m.close()

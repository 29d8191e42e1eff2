"""The 4-bit KV cache's attention reads nothing outside the cache's arrays.

CPU: every address that the 128-row kernel's threads stage (zq_attn_q4_at.hpp, the
kernel's own index functions, built for the host), for every step that a capacity
has.  GPU: arrays of their exact size inside larger ones, which hold NaN scales and
codes of all ones behind them, give the results of a cache by itself."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "zq_attn_q4_at.hpp"
#include <stddef.h>
using namespace zq;
// Steps of one (sequence, kv head) of `capacity` rows: 0 where every byte lies in its arrays (and a scale in its
// own plane) and every key below the capacity is read at its own place, else 1 + the first bad key of a step.
template <int D>
static long check(uint32_t capacity) {
    const size_t row = D / 2, planes = D / 32;
    for (uint32_t key0 = 0; key0 < capacity; key0 += StageShape<D>::TK)
        for (uint32_t e = 0; e < uint32_t(StageShape<D>::kTasks); ++e) {
            {
                const StageAt a = stage_k_at<D>(capacity, key0, e);
                const uint32_t key = key0 + e / (D / 32), b = e % (D / 32);
                const size_t code = key0 * row + a.codes, scale = key0 * size_t(2) + a.scales;
                if (code + 16 > capacity * row || scale + 2 > planes * capacity * 2 || scale / 2 / capacity != b) return 1 + key;
                if (key < capacity && (code != key * row + b * 16 || scale != (size_t(b) * capacity + key) * 2)) return 1 + key;
            }
            {
                const StageAt a = stage_v_at<D>(capacity, key0, e);
                const StageV t = stage_v_task<D>(e);
                const uint32_t key = key0 + 8 * t.o, b = t.ch / 8;
                const size_t code = key0 * row + a.codes, scale = key0 * size_t(2) + a.scales;
                if (code + 7 * row + 2 > capacity * row || scale + 16 > planes * capacity * 2 || scale / 2 / capacity != b ||
                    (scale / 2 + 7) / capacity != b || scale % 16) return 1 + key;
                if (key < capacity && (code != key * row + 2 * t.ch || scale != (size_t(b) * capacity + key) * 2)) return 1 + key;
            }
        }
    return 0;
}
extern "C" long check_stage(int D, uint32_t capacity) {
    return D == 64 ? check<64>(capacity) : D == 128 ? check<128>(capacity) : check<256>(capacity);
}
"""


@pytest.fixture(scope="module")
def check_stage(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("stage")
    (tmp / "stage.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "zeninfer_amd", "csrc"), "-o", str(tmp / "stage.so"), str(tmp / "stage.cpp")],
                   check=True)
    f = ctypes.CDLL(str(tmp / "stage.so")).check_stage
    f.restype, f.argtypes = ctypes.c_long, [ctypes.c_int, ctypes.c_uint32]
    return f


def views():
    """(name, view of a [2][8][512] buffer's rows of 128 floats, seqs, tokens, row stride, whether rows are in place)."""
    buf = torch.arange(2 * 8 * 512, dtype=torch.float32).reshape(2, 8, 512)
    flat = buf.reshape(16, 512)
    return [
        ("all tokens", buf[:, :, 128:256], 2, 8, 512, True),
        ("flattened", flat[:, 128:256], 2, 8, 512, True),
        ("heads apart", buf[:, :, 128:256].unflatten(-1, (2, 64)), 2, 8, 512, True),
        ("heads apart, flattened", flat[:, 128:256].unflatten(-1, (2, 64)), 2, 8, 512, True),
        ("one sequence", buf[1:, :3, :128], 1, 3, 512, True),
        ("one sequence without its dimension", buf[1, :3, 64:192], 1, 3, 512, True),
        ("one token", buf[:1, 4:5, :128], 1, 1, 512, True),
        ("more rows than asked", flat[:, :128], 2, 3, 512, True),
        ("wider rows than asked", buf[:, :, 128:300], 2, 8, 512, True),
        ("a token of each sequence", buf[:, 5, :128], 2, 1, 8 * 512, True),
        ("a token of each sequence, dimension kept", buf[:, 5:6, :128], 2, 1, 8 * 512, True),
        ("a row", flat[3:4, 128:256], 1, 1, 512, True),
        ("tokens before a batch of one", flat[:6, None, 128:256], 1, 6, 512, True),
        ("tokens before a batch of one, heads apart", flat[:6, 128:256].unflatten(-1, (2, 64))[:, None], 1, 6, 512, True),
        ("some tokens of each sequence", buf[:, :3, :128], 2, 3, 512, False),
        ("sequences in place, tokens not asked for", buf[:, :, :128], 2, 3, 512, False),
        ("a token of each sequence, by the tokens' stride", buf[:, 5, :128], 2, 1, 512, False),
        ("every other token", buf[:, ::2, :128], 2, 4, 512, False),
        ("another stride", buf[:, :, :128], 2, 8, 256, False),
        ("too few columns", flat[:4, 128:252], 1, 4, 512, False),
        ("every other column", flat[:4, ::4], 1, 4, 512, False),
        ("heads apart that are not adjacent", flat[:4].unflatten(-1, (4, 128))[:, ::2, :64], 1, 4, 512, False),
        ("sequences and tokens exchanged", buf.transpose(0, 1)[:, :, :128], 8, 2, 512, False),
        ("too few rows", flat[:4, :128], 1, 6, 512, False),
        ("one row", flat[3, ::4], 1, 1, 512, False),
    ]


@pytest.mark.parametrize("name,view,seqs,tokens,stride,right", views(), ids=lambda x: x if isinstance(x, str) else "")
def test_strided_views_are_the_rows_that_the_kernels_read(monkeypatch, name, view, seqs, tokens, stride, right):
    """What a view passes as is what the kernels read: row (s, t) at (s * tokens + t) * stride of its address."""
    from zeninfer_amd import zq
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    call = lambda: zq._need_rows(view, seqs, tokens, stride, 128, "rows", 0)
    if not right:
        with pytest.raises(ValueError, match="rows: (rows must be|buffer holds)"):
            call()
        return
    assert call() == view.data_ptr()
    read = torch.as_strided(view, (seqs, tokens, 128), (tokens * stride, stride, 1), view.storage_offset())
    rows = view.flatten(-2) if view.shape[-1] == 64 else view
    if rows.dim() == 2 or rows.shape[1] < tokens:
        rows = rows.reshape(-1, rows.shape[-1])[:seqs * tokens].unflatten(0, (seqs, tokens))
    assert torch.equal(read, rows[:seqs, :tokens, :128])


def test_wrappers_refuse_other_types(monkeypatch):
    """Buffers of other types are long enough, and would be read as other values."""
    from zeninfer_amd import zq
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    c = zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, 1, 2, 64, 64, weight=5 << 20, pos=6 << 20)
    p, lens = 7 << 20, torch.zeros(1, dtype=torch.int32)
    for dtype in (torch.float64, torch.float16, torch.bfloat16, torch.int32, torch.int64, torch.complex64):
        x = torch.zeros(4096, dtype=dtype)
        wide = torch.zeros(4, 512, dtype=dtype)[:, :256]
        for call in (lambda: zq.kv_q4_append_dev(c, x, p, 1, lens), lambda: zq.kv_q4_append_dev(c, p, x, 1, lens),
                     lambda: zq.kv_q4_append_dev(c, wide, p, 4, lens, stride=512), lambda: zq.kv_q4_read_dev(c, x, p, 1, lens),
                     lambda: zq.kv_q4_read_dev(c, None, x, 1, lens), lambda: zq.attention_q4_dev(c, x, p, 1, 4, lens, 1.0),
                     lambda: zq.attention_q4_dev(c, wide, p, 4, 4, lens, 1.0, stride=512),
                     lambda: zq.attention_q4_dev(c, p, x, 1, 4, lens, 1.0)):
            with pytest.raises(ValueError, match="needs float32, got torch"):
                call()
    z = lambda n, dtype: torch.zeros(n, dtype=dtype)
    right = dict(k=torch.uint8, v=torch.uint8, k_scale=torch.float16, v_scale=torch.float16, weight=torch.float32,
                 pos=torch.int32)
    wrong = dict(k=(torch.float16, torch.float32), v=(torch.bfloat16, torch.float32), k_scale=(torch.bfloat16, torch.float32),
                 v_scale=(torch.bfloat16, torch.float64), weight=(torch.float64, torch.float16, torch.int32),
                 pos=(torch.int64, torch.float32, torch.int16))
    for name, types in wrong.items():
        for dtype in types:
            with pytest.raises(ValueError, match=f"KVQ4 {name}: needs "):
                zq.KVQ4(seqs=1, kv_heads=2, head_dim=64, capacity=64, **{n: z(8192, dtype if n == name else t) for n, t in right.items()})
    # the types they have, their bits, and their bytes: what is too short is what is left to refuse
    for over in ({}, {n: torch.uint8 for n in right}, dict(k_scale=torch.int16, v_scale=torch.uint8)):
        with pytest.raises(ValueError, match="KVQ4 k: buffer holds"):
            zq.KVQ4(seqs=1, kv_heads=2, head_dim=64, capacity=64, **{n: z(8, over.get(n, t)) for n, t in right.items()})
    for x in (z(8, torch.float32), z(8, torch.uint8)):
        with pytest.raises(ValueError, match="k: buffer holds"):
            zq.kv_q4_append_dev(c, x, p, 1, lens)


def test_wrappers_refuse_what_is_no_tensor():
    """Arrays of the host and lists are refused as such, for every buffer."""
    from zeninfer_amd import zq
    c = zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, 1, 2, 64, 64, weight=5 << 20, pos=6 << 20)
    p = 7 << 20
    for bad in (np.zeros(4096, np.float32), np.zeros(4096, np.int32), [0.0] * 4096):
        for call in (lambda: zq.kv_q4_append_dev(c, bad, p, 1, p), lambda: zq.kv_q4_append_dev(c, p, bad, 1, p, stride=256),
                     lambda: zq.kv_q4_append_dev(c, p, p, 1, bad), lambda: zq.kv_q4_read_dev(c, bad, None, 1, p),
                     lambda: zq.attention_q4_dev(c, bad, p, 1, 4, p, 1.0), lambda: zq.attention_q4_dev(c, p, bad, 1, 4, p, 1.0),
                     lambda: zq.attention_q4_dev(c, p, p, 1, 4, p, 1.0, counts=bad),
                     lambda: zq.kv_q4_evict_dev(c, bad, 16, 4, 4), lambda: zq.KVQ4(p, p, bad, p, 1, 2, 64, 64)):
            with pytest.raises(ValueError, match="tensor must be on the GPU"):
                call()


def test_wrappers_refuse_sizes_below_zero(monkeypatch):
    """A size_t takes -1 as the largest number: any workspace would be long enough, and everything would be kept."""
    from zeninfer_amd import zq
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)
    c = zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, 1, 2, 64, 64, weight=5 << 20, pos=6 << 20)
    p, lens, ws = 7 << 20, torch.zeros(1, dtype=torch.int32), torch.zeros(16, dtype=torch.uint8)
    for w in (ws, p):
        with pytest.raises(ValueError, match="attention_q4_dev workspace: a size below zero"):
            zq.attention_q4_dev(c, p, p, 1, 4, lens, 1.0, flags=zq.ATTN_Q4_WEIGHTS, workspace=w, workspace_bytes=-1)
        with pytest.raises(ValueError, match="kv_q4_evict_dev workspace: a size below zero"):
            zq.kv_q4_evict_dev(c, lens, 16, 4, 4, workspace=w, workspace_bytes=-16)
    for bad in ((-1, 4, 4), (16, -1, 4), (16, 4, -1)):
        with pytest.raises(ValueError, match="a number of rows below zero"):
            zq.kv_q4_evict_dev(c, lens, *bad, workspace=ws, workspace_bytes=16)
    for bad in (dict(seqs=-1), dict(kv_heads=-2), dict(capacity=-64)):
        with pytest.raises(ValueError, match="KVQ4 k: a size below zero"):
            zq.KVQ4(1 << 20, 2 << 20, 3 << 20, 4 << 20, **{**dict(seqs=1, kv_heads=2, head_dim=64, capacity=64), **bad})
    for tokens in (-1, -3):
        with pytest.raises(ValueError, match="a size below zero"):
            zq.kv_q4_append_dev(c, p, p, tokens, lens)
        with pytest.raises(ValueError, match="a size below zero"):
            zq.kv_q4_read_dev(c, p, p, tokens, lens)
        with pytest.raises(ValueError, match="a size below zero"):
            zq.attention_q4_dev(c, p, p, tokens, 4, lens, 1.0)


def test_evict_refuses_a_destination_that_meets_the_cache():
    """An array of the destination inside any array of the cache, of whatever role, or ending in it: its rows would be
    overwritten while they are read.  Next to each other they may lie (that call gets as far as the device)."""
    from tests.test_kv_q4 import handle
    from zeninfer_amd import zq
    L, p, need = zq.lib(), 7 << 20, 1 << 20
    c = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20, weight=5 << 20, pos=6 << 20)
    size = dict(k=2 * 2 * 64 * 32, v=2 * 2 * 64 * 32, k_scale=2 * 2 * 64 * 4, v_scale=2 * 2 * 64 * 4, weight=2 * 2 * 64 * 4,
                pos=2 * 2 * 64 * 4)  # of the cache; half of it with 32 slots
    far = {n: a + (16 << 20) for n, a in c.items()}
    evict = lambda d: L.zq_hip_kv_q4_evict_dev(ctypes.byref(handle(zq)), ctypes.byref(handle(zq, capacity=32, **d)), p, 16, 4,
                                               4, None, p, need, None)
    for mine, a in c.items():
        for theirs in far:
            for at in (a, a + 16, a + size[mine] - 16, a - size[theirs] // 2 + 16):
                assert evict({**far, theirs: at}) == zq.ERR_ARG, (mine, theirs, at - a)
    if not torch.cuda.is_available():
        for mine, a in c.items():
            for theirs in far:
                for at in (a + size[mine], a - size[theirs] // 2):
                    assert evict({**far, theirs: at}) == zq.ERR_NO_DEVICE, (mine, theirs, at - a)


class FakeLibrary:
    """The decoder's entry points that Model.kv_cache meets, over made-up addresses."""

    def __init__(self, zq):
        self.zq, self.freed, self.status = zq, 0, zq.OK

    def zq_model_kv_cache(self, h, layer, cache, rows, positions):
        c = cache._obj
        c.k, c.v, c.k_scale, c.v_scale, c.weight, c.pos = [(i + 1) << 20 for i in range(6)]
        c.seqs, c.kv_heads, c.head_dim, c.capacity = 1, 2, 64, 64
        return self.zq.OK

    def zq_model_set_kv_cache(self, h, form, rows, recent, first):
        return self.status

    def zq_model_free(self, h):
        self.freed += 1


def test_a_models_cache_ends_with_its_arrays(monkeypatch):
    """The handle of a model's cache keeps the model alive, and is refused once the model has freed the arrays."""
    import gc
    from zeninfer_amd import model, zq
    fake = FakeLibrary(zq)
    with monkeypatch.context() as mp:
        mp.setattr(zq, "lib", lambda: fake)
        m = model.Model(1, zq.ModelConfig())
    lens = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(zq, "_check_device", lambda t, what: None)

    def uses(c):
        own = zq.KVQ4(*[i << 20 for i in range(11, 15)], 1, 2, 64, 64, weight=15 << 20, pos=16 << 20)
        return [lambda: zq.kv_q4_append_dev(c, 1 << 24, 1 << 24, 1, lens), lambda: zq.kv_q4_read_dev(c, 1 << 24, None, 1, lens),
                lambda: zq.attention_q4_dev(c, 1 << 24, 1 << 24, 1, 4, lens, 1.0),
                lambda: zq.attention_q4_workspace_bytes(c, 1, 4), lambda: zq.kv_q4_evict_workspace_bytes(c, 4),
                lambda: zq.kv_q4_evict_dev(c, lens, 4, 1, 1), lambda: zq.kv_q4_evict_dev(own, lens, 4, 1, 1, dst=c)]

    def refused(c):
        for use in uses(c):
            with pytest.raises(ValueError, match="has freed this 4-bit cache"):
                use()
    c = m.kv_cache(0)[0]
    assert isinstance(c, zq.KVQ4) and zq.kv_q4_evict_workspace_bytes(c, 4) == 2 * 3 * 4 * 4
    fake.status = zq.ERR_OOM  # the model keeps the cache it had
    with pytest.raises(zq.ZQError):
        m.set_kv_cache(model.KV_Q4)
    assert zq.kv_q4_evict_workspace_bytes(c, 4)
    fake.status = zq.OK
    m.set_kv_cache(model.KV_Q4)
    refused(c)
    c = m.kv_cache(1)[0]
    assert zq.attention_q4_workspace_bytes(c, 1, 4, zq.ATTN_Q4_WEIGHTS)
    del m
    gc.collect()
    assert fake.freed == 0 and zq.kv_q4_evict_workspace_bytes(c, 4)
    c._model.close()
    assert fake.freed == 1
    refused(c)


def test_a_models_row_budget_is_not_below_zero(monkeypatch):
    """A uint32_t takes -1 as 4,294,967,295: a cache without a bound."""
    from zeninfer_amd import model, zq
    with monkeypatch.context() as mp:
        mp.setattr(zq, "lib", lambda: FakeLibrary(zq))
        m = model.Model(1, zq.ModelConfig())
    for bad in (dict(rows=-1), dict(rows=64, recent=-1), dict(rows=64, first=-4)):
        with pytest.raises(ValueError, match="a number of rows below zero"):
            m.set_kv_cache(model.KV_Q4, **bad)
    m.set_kv_cache(model.KV_Q4, 64, 8, 4)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_staged_keys_lie_in_the_arrays(check_stage, D):
    bad = {C: check_stage(D, C) for C in [*range(32, 2049, 32), 40000, 65504, 99968]}
    assert not {C: n - 1 for C, n in bad.items() if n}


def inside(t):
    """A copy of t in a larger array: 64 KiB of ones before and behind it (codes of all ones, NaN scales and weights)."""
    pad = 1 << 16
    raw = t.contiguous().view(torch.uint8).flatten()
    buf = torch.full((raw.numel() + 2 * pad,), 0xff, dtype=torch.uint8, device="cuda")
    buf[pad:pad + raw.numel()] = raw
    return buf, buf[pad:pad + raw.numel()].view(t.dtype).view(t.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [None, "set"])
@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("S,KH,G,D,C,lens,T", [
    (4, 8, 4, 128, 96, [56, 1, 40, 50], 40), (2, 8, 8, 64, 416, [386, 200], 30), (1, 8, 4, 128, 224, [24], 200),
    (1, 1, 8, 64, 32, [2], 30), (4, 4, 4, 256, 160, [120, 3, 90, 60], 40), (3, 2, 4, 128, 160, [159, 0, 70], 1)])
def test_rows_behind_the_arrays_are_nothing_to_it(zq, S, KH, G, D, C, lens, T, full, weights):
    from tests.test_kv_q4 import Dev, tokens
    r = np.random.default_rng(C + T)
    d = Dev(zq, S, KH, D, C)
    d.fill(lens, 3)
    if not full:
        d.append(tokens(r, S, T, KH, D), tokens(r, S, T, KH, D, 0.7), lens)
    if full:  # every slot but the last sequence's is seen
        d.fill([C] * S, 4)
        lens = [C] * (S - 1) + lens[-1:] if S > 1 else [C]
    bufs = []
    for name in ("k", "v", "ks", "vs", "weight", "pos"):
        buf, view = inside(getattr(d, name))
        setattr(d, name, view)
        bufs.append(buf)
    d.c = zq.KVQ4(d.k, d.v, d.ks, d.vs, S, KH, D, C, weight=d.weight, pos=d.pos)
    d.check_attention(tokens(r, S, T, KH * G, D, 1.4), lens, 1 / math.sqrt(D), full=full, weights=weights)
    for b in bufs:
        assert (b[:1 << 16] == 0xff).all() and (b[-(1 << 16):] == 0xff).all()

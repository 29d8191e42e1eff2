"""The operators of the 4-bit KV cache, in their plain form and as calls of the framework.

A cache row is one token of one kv head, held as Q4_0 values: blocks of 32 with an fp16 scale d (of 8 significant
bits), value = (code - 8) * d, byte j of a block's 16 = elements j (low nibble) and j + 16.  The arrays of a cache of
S sequences, KH kv heads, head dimension D and C slots are

    k, v              [S][KH][C][D / 2]    uint8
    k_scale, v_scale  [S][KH][D / 32][C]   fp16
    weight            [S][KH][C]           fp32, the attention weight each row has drawn so far
    pos               [S][KH][C]           int32, the position of the row's token

Operators (``op`` of a case):
  append     k and v of new tokens are quantised into slots lens.. of every sequence, and read back as fp32
  attention  softmax(scale q.k) v over the rows, causal among the new tokens, with the rows' weights on request
  evict      the rows with the most accumulated weight, the newest and the first ones are kept, in a smaller cache
"""
import math

import torch

own = False

#: what one pass may cost at most in a drawn case: (query, key) pairs times head dimension, and rows of a cache
MOST_PAIRS, MOST_ROWS = 1024 * 8192 * 32 * 128, 32 * 8192 * 8 * 128


# ---- cases -------------------------------------------------------------------
def listed():
    attn = {"op": "attention", "seqs": 1, "kv_heads": 8, "group": 4, "head_dim": 128, "tokens": 1, "ragged": False,
            "full": False, "weights": False}
    return [
        # one prefill pass of the decoder writes its tokens behind a prompt's first part
        {"name": "append_prompt", "op": "append", "seqs": 1, "kv_heads": 8, "head_dim": 128, "rows": 512, "tokens": 1024,
         "ragged": False},
        # a decode step of a batch, some sequences idle: latency
        {"name": "append_step", "op": "append", "seqs": 32, "kv_heads": 8, "head_dim": 64, "rows": 1501, "tokens": 1,
         "ragged": True},
        # decode of a single chat at the length of the decoder's benchmark: latency
        {**attn, "name": "decode_short", "rows": 600},
        # decode at the decoder's longest context
        {**attn, "name": "decode_long", "rows": 24001},
        # decode of a full server: many sequences of all lengths
        {**attn, "name": "decode_batch", "seqs": 64, "rows": 8190, "ragged": True},
        # several drafted tokens a sequence in one pass, an odd group of heads
        {**attn, "name": "draft_batch", "seqs": 16, "kv_heads": 4, "group": 7, "head_dim": 64, "rows": 3001, "tokens": 6,
         "ragged": True},
        # decode that keeps the rows' weights for a later eviction
        {**attn, "name": "decode_weights", "seqs": 16, "rows": 4097, "weights": True},
        # a whole prompt at once
        {**attn, "name": "prompt", "rows": 0, "tokens": 2048},
        # the last pass over a long prompt, whose weights say what is evicted after it
        {**attn, "name": "chunk_weights", "rows": 7168, "tokens": 1024, "weights": True},
        # wide heads without groups, padded prompts, every query sees the held rows only
        {**attn, "name": "wide_full", "seqs": 4, "kv_heads": 4, "group": 1, "head_dim": 256, "rows": 1777, "tokens": 333,
         "ragged": True, "full": True},
        # after a long prompt: all layers of a decoder (as sequences) down to a quarter
        {"name": "evict_prompt", "op": "evict", "seqs": 16, "kv_heads": 8, "head_dim": 128, "rows": 8192, "keep": 2048,
         "recent": 256, "first": 4},
        # a short cache that is full, one sequence: latency
        {"name": "evict_step", "op": "evict", "seqs": 1, "kv_heads": 8, "head_dim": 64, "rows": 1153, "keep": 1024,
         "recent": 128, "first": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "evict"])
    c = {"op": op, "head_dim": rng.choice([64, 128, 128, 256]), "kv_heads": rng.choice([1, 2, 4, 5, 8, 8])}
    per_row = c["kv_heads"] * c["head_dim"]
    if op == "append":
        c["seqs"] = _log(rng, 1, 64)
        c["tokens"] = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
        c["rows"] = _log(rng, 1, 4000) - 1
        c["ragged"] = rng.random() < 0.5
        while c["seqs"] * (c["rows"] + c["tokens"]) * per_row > MOST_ROWS // 8:
            c["seqs"] = 1 if c["seqs"] < 4 else c["seqs"] // 2
            c["tokens"] = max(1, c["tokens"] // 2)
        return c
    if op == "evict":
        c["seqs"] = _log(rng, 1, 32)
        c["rows"] = _log(rng, 100, 16384)
        while c["seqs"] * c["rows"] * per_row > 16 * 8192 * 8 * 128:
            c["seqs"] = max(1, c["seqs"] // 2)
            c["rows"] = max(100, c["rows"] * 3 // 4)
        c["keep"] = max(8, int(c["rows"] * rng.uniform(0.1, 1.05)))
        c["recent"] = int(c["keep"] * rng.uniform(0, 0.7))
        c["first"] = rng.choice([0, 4, 4, 16]) if c["keep"] >= 64 else 0
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 4, 7, 8])
    kind = rng.choice(["decode", "decode", "draft", "prompt"])
    c["seqs"] = _log(rng, 1, 64) if kind != "prompt" else _log(rng, 1, 8)
    c["tokens"] = 1 if kind == "decode" else _log(rng, 2, 16) if kind == "draft" else _log(rng, 17, 2048)
    c["rows"] = _log(rng, 1, 24000) if kind != "prompt" else _log(rng, 1, 8000) - 1
    c["ragged"] = c["seqs"] > 1 and rng.random() < 0.6
    c["full"] = c["rows"] > 0 and rng.random() < 0.2
    c["weights"] = rng.random() < 0.3
    while (c["seqs"] * (c["rows"] + c["tokens"]) * c["tokens"] * c["group"] * per_row > MOST_PAIRS // 2
           or c["seqs"] * (c["rows"] + c["tokens"]) * per_row > MOST_ROWS):
        if c["seqs"] > 1 and rng.random() < 0.6:
            c["seqs"] = c["seqs"] * 2 // 3
        elif c["tokens"] > c["rows"]:
            c["tokens"] = max(1, c["tokens"] * 2 // 3)
        else:
            c["rows"] = max(1, c["rows"] * 2 // 3)
    return c


def lengths(case):
    """Rows held and new tokens of every sequence: all alike, or of all lengths with idle sequences among them."""
    S, rows, tokens = case["seqs"], case["rows"], case.get("tokens", 0)
    if not case.get("ragged"):
        return [rows] * S, [tokens] * S
    lens = [rows - rows * s // S for s in range(S)]
    lens[-1] = min(lens[-1], 1)  # a sequence at its start
    counts = [0 if s % 5 == 3 else tokens - (tokens - 1) * s // (2 * S) for s in range(S)]
    return lens, counts


def seen(case):
    """Pairs of a query token and a row that it sees, and rows that any query sees, over the sequences."""
    pairs = rows = 0
    for n, t in zip(*lengths(case)):
        if t:
            pairs += n * t + (0 if case["full"] else t * (t + 1) // 2)
            rows += n + (0 if case["full"] else t)
    return pairs, rows


def row_bytes(case):
    return case["head_dim"] // 2 + case["head_dim"] // 16


def work(case):
    D, KH, S = case["head_dim"], case["kv_heads"], case["seqs"]
    if case["op"] == "append":
        n = sum(lengths(case)[1])  # k and v read, their rows written, read back and written as fp32
        return {"bytes": n * KH * (16 * D + 4 * row_bytes(case)), "flops": n * KH * D * 8}
    if case["op"] == "evict":
        n = S * KH * min(case["rows"], case["keep"])  # every weight and position read; kept rows copied, read back and written
        return {"bytes": S * KH * case["rows"] * 8 + n * (8 + 6 * row_bytes(case) + 8 * D), "flops": S * KH * case["rows"]}
    pairs, rows = seen(case)
    n = sum(lengths(case)[1]) * KH * case["group"]
    w = case["weights"]
    return {"bytes": rows * KH * (2 * row_bytes(case) + (4 if w else 0)) + n * D * 8,
            "flops": pairs * KH * case["group"] * 4 * D}


# ---- inputs ------------------------------------------------------------------
def quantised(x):
    """Codes [..., D / 2] and scales [..., D / 32] of rows x [..., D]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs()
    at = torch.where(a == a.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = (b.gather(-1, at) / -8).to(torch.bfloat16).float().clamp(-4096, 4096).half()
    e = torch.where(d == 0, torch.ones_like(d), d)
    c = (torch.where(d == 0, torch.zeros_like(b), b).double() / e.double()).round().clamp(-8, 7).add(8).to(torch.uint8)
    return (c[..., :16] | c[..., 16:] << 4).flatten(-2), d[..., 0]


def slots(case):
    need = case["rows"] + (0 if case.get("full") else case.get("tokens", 0))
    return max(32, -(-need // 32) * 32)


def prepare(case, seed):
    S, KH, D, C = case["seqs"], case["kv_heads"], case["head_dim"], slots(case)
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    # keys have a few wide channels, values do not
    wide = torch.where(torch.rand(KH, 1, D, generator=g, device=dev) < 0.04, 6.0, 1.0) * (normal(KH, 1, D).abs() + 0.3)
    lens, counts = lengths(case)
    st = {"case": dict(case), "C": C}
    i32 = dict(dtype=torch.int32, device=dev)
    for name, scale in (("k", wide), ("v", torch.full((), 0.6, device=dev))):
        codes = torch.empty(S, KH, C, D // 2, dtype=torch.uint8, device=dev)
        d = torch.empty(S, KH, D // 32, C, dtype=torch.float16, device=dev)
        if case["op"] == "append":
            codes.zero_()
            d.zero_()
        else:
            for s in range(S):
                codes[s], ds = quantised(normal(KH, C, D) * scale)
                d[s] = ds.transpose(1, 2)
        st[name], st[name + "_scale"] = codes, d
    st["lens"], st["counts"] = torch.tensor(lens, **i32), torch.tensor(counts, **i32)
    st["weight"] = torch.zeros(S, KH, C, device=dev)
    st["pos"] = torch.arange(C, **i32).expand(S, KH, C).contiguous()
    if case["op"] == "append":
        T = case["tokens"]
        st["new_k"] = normal(S, T, KH, D) * wide[:, 0]
        st["new_v"] = normal(S, T, KH, D) * 0.6
        st["k_out"], st["v_out"] = torch.zeros(S, T, KH, D, device=dev), torch.zeros(S, T, KH, D, device=dev)
    elif case["op"] == "attention":
        T, H = case["tokens"], KH * case["group"]
        st["q"] = normal(S, T, H, D) * 1.3
        st["out"] = torch.zeros(S, T, H, D, device=dev)
        st["scale"] = 1.0 / math.sqrt(D)
    else:
        # what rows draw over time is spread widely, and some drew nothing; slots are in no order after earlier evictions
        u = torch.rand(S, KH, C, generator=g, device=dev)
        st["weight"] = torch.where(u < 0.05, torch.zeros_like(u), -torch.log(u) ** 3)
        st["pos"][..., :case["rows"]] = torch.rand(S, KH, case["rows"], generator=g, device=dev).argsort(-1).int() * 2
        st["next_pos"] = torch.full((S,), 2 * case["rows"], **i32)
        K = min(case["rows"], case["keep"])
        Cd = -(-case["keep"] // 32) * 32
        st["Cd"], st["first_row"], st["kept"] = Cd, torch.zeros(S, **i32), torch.full((S,), K, **i32)
        st["to"] = {"k": torch.zeros(S, KH, Cd, D // 2, dtype=torch.uint8, device=dev),
                    "v": torch.zeros(S, KH, Cd, D // 2, dtype=torch.uint8, device=dev),
                    "k_scale": torch.zeros(S, KH, D // 32, Cd, dtype=torch.float16, device=dev),
                    "v_scale": torch.zeros(S, KH, D // 32, Cd, dtype=torch.float16, device=dev),
                    "weight": torch.zeros(S, KH, Cd, device=dev), "pos": torch.zeros(S, KH, Cd, **i32)}
        st["k_out"], st["v_out"] = torch.zeros(S, K, KH, D, device=dev), torch.zeros(S, K, KH, D, device=dev)
    return st


# ---- the plain form ------------------------------------------------------------
def values(codes, d):
    """fp32 rows [..., C, D] of codes [..., C, D / 2] and scales [..., D / 32, C]."""
    b = codes.reshape(*codes.shape[:-1], -1, 16)
    c = torch.cat([b & 15, b >> 4], -1).float() - 8
    return (c * d.transpose(-1, -2).unsqueeze(-1).float()).flatten(-2)


def plain_append(st):
    case = st["case"]
    S, KH, T, D = case["seqs"], case["kv_heads"], case["tokens"], case["head_dim"]
    t = torch.arange(T, device=st["lens"].device)
    s, t = torch.nonzero(t < st["counts"][:, None], as_tuple=True)
    slot = st["lens"].long()[s] + t
    out = []
    for name in ("k", "v"):
        codes, d = quantised(st["new_" + name][s, t])
        st[name][s, :, slot] = codes
        st[name + "_scale"][s, :, :, slot] = d
        rows = values(st[name][s, :, slot].unsqueeze(-2), st[name + "_scale"][s, :, :, slot].unsqueeze(-1)).squeeze(-2)
        y = torch.zeros(S, T, KH, D, device=rows.device)
        y[s, t] = rows
        out.append(y)
    return {"k": out[0], "v": out[1]}


def plain_attention(st):
    case = st["case"]
    S, KH, G, T, D, C = case["seqs"], case["kv_heads"], case["group"], case["tokens"], case["head_dim"], st["C"]
    dev = st["q"].device
    t = torch.arange(T, device=dev)
    live = t < st["counts"][:, None]
    sees = st["lens"][:, None] + (0 if case["full"] else 1 + t)
    ok = (torch.arange(C, device=dev) < sees[..., None]) & live[..., None]  # [S][T][C]
    k, v = values(st["k"], st["k_scale"]), values(st["v"], st["v_scale"])
    v = torch.where(ok.any(1)[:, None, :, None], v, 0.0)
    q = st["q"].reshape(S, T, KH, G, D).permute(0, 2, 3, 1, 4).reshape(S, KH, G * T, D)
    x = torch.matmul(q * st["scale"], k.transpose(-1, -2)).reshape(S, KH, G, T, C)
    x = torch.where(ok[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.reshape(S, KH, G * T, C), v).reshape(S, KH, G, T, D)
    o = o.permute(0, 3, 1, 2, 4).reshape(S, T, KH * G, D)
    return {"out": o, "weight": p.sum((2, 3))} if case["weights"] else {"out": o}


def plain_evict(st):
    case = st["case"]
    n, K, KH, S = case["rows"], min(case["rows"], case["keep"]), case["kv_heads"], case["seqs"]
    w, pos = st["weight"][..., :n], st["pos"][..., :n]
    held = (pos >= st["next_pos"][:, None, None] - case["recent"]) | (pos < case["first"])
    order = torch.sort(torch.where(held, math.inf, w), dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros_like(w, dtype=torch.bool).scatter(-1, order[..., :K], True)
    # holes below K in order, then the chosen rows from K on in order: both are as many
    slot = torch.arange(n, device=w.device).expand_as(w)
    up = torch.where(chosen & (slot >= K), slot, n + slot).sort(-1).values
    hole = (~chosen).long().cumsum(-1)[..., :K] - 1
    frm = torch.where(chosen[..., :K], slot[..., :K], up.gather(-1, hole.clamp_min(0)))
    rows = {}
    for name in ("k", "v"):
        x = values(st[name][..., :n, :], st[name + "_scale"][..., :n])
        rows[name] = x.gather(2, frm.unsqueeze(-1).expand(-1, -1, -1, x.shape[-1])).transpose(1, 2).contiguous()
    return {**rows, "weight": w.gather(-1, frm), "pos": pos.gather(-1, frm)}


# ---- the framework's calls -------------------------------------------------------
def cache_of(zq, st, arrays, C):
    case = st["case"]
    return zq.KVQ4(arrays["k"], arrays["v"], arrays["k_scale"], arrays["v_scale"], case["seqs"], case["kv_heads"],
                   case["head_dim"], C, weight=arrays["weight"], pos=arrays["pos"])


def own_run(st):
    from zeninfer_amd import zq
    case = st["case"]
    op = case["op"]
    if "cache" not in st:  # the handles that a program keeps beside its buffers
        st["cache"] = cache_of(zq, st, st, st["C"])
        if op == "attention":
            flags = (zq.ATTN_Q4_FULL if case["full"] else 0) | (zq.ATTN_Q4_WEIGHTS if case["weights"] else 0)
            need = zq.attention_q4_workspace_bytes(st["cache"], case["tokens"], case["kv_heads"] * case["group"], flags)
            st["flags"], st["need"] = flags, need
        if op == "evict":
            st["dst"] = cache_of(zq, st, st["to"], st["Cd"])
            st["need"] = zq.kv_q4_evict_workspace_bytes(st["cache"], case["keep"])
        if "need" in st:
            st["workspace"] = torch.empty(max(st["need"], 16), dtype=torch.uint8, device=st["lens"].device)
    if op == "append":
        zq.kv_q4_append_dev(st["cache"], st["new_k"], st["new_v"], case["tokens"], st["lens"], counts=st["counts"])
        zq.kv_q4_read_dev(st["cache"], st["k_out"], st["v_out"], case["tokens"], st["lens"], counts=st["counts"])
        return {"k": st["k_out"], "v": st["v_out"]}
    if op == "attention":
        zq.attention_q4_dev(st["cache"], st["q"], st["out"], case["tokens"], case["kv_heads"] * case["group"], st["lens"],
                            st["scale"], counts=st["counts"], flags=st["flags"], workspace=st["workspace"],
                            workspace_bytes=st["need"])
        return {"out": st["out"], "weight": st["weight"]} if case["weights"] else {"out": st["out"]}
    K = min(case["rows"], case["keep"])
    zq.kv_q4_evict_dev(st["cache"], st["lens"], case["keep"], case["recent"], case["first"], next_pos=st["next_pos"],
                       dst=st["dst"], workspace=st["workspace"], workspace_bytes=st["need"])
    zq.kv_q4_read_dev(st["dst"], st["k_out"], st["v_out"], K, st["first_row"], counts=st["kept"])
    return {"k": st["k_out"], "v": st["v_out"], "weight": st["to"]["weight"][..., :K], "pos": st["to"]["pos"][..., :K]}


def run(state):
    if own:
        return own_run(state)
    return {"append": plain_append, "attention": plain_attention, "evict": plain_evict}[state["case"]["op"]](state)


# ---- the definition in 64 bits -----------------------------------------------------
def exact_rows(codes, d):
    """codes [C][D / 2], d [D / 32][C] -> [C][D], element by element of the definition."""
    C, half = codes.shape
    j = torch.arange(2 * half, device=codes.device)
    byte = (j // 32) * 16 + j % 16
    nibble = (codes.long()[:, byte] >> (4 * ((j % 32) // 16))) % 16
    return (nibble.double() - 8) * d.double()[j // 32].T


def exact_quantised(x):
    """The values that rows x [..., D] are held as."""
    b = x.double().unflatten(-1, (-1, 32))
    largest = (b.abs() == b.abs().amax(-1, keepdim=True)).double() * torch.arange(32, 0, -1, device=x.device)
    m, e = torch.frexp(b.gather(-1, largest.argmax(-1, keepdim=True))[..., 0] / -8)
    d = torch.ldexp(torch.round(m * 256), e - 8).clamp(-4096, 4096)
    d = torch.where(d.abs() < 2.0 ** -14, torch.round(d * 2.0 ** 24) * 2.0 ** -24, d)[..., None]
    c = torch.round(b / torch.where(d == 0, 1.0, d)).clamp(-8, 7)
    return torch.where(d == 0, 0.0, c * d).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    lens, counts = lengths(case)
    S, KH, D = case["seqs"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        out = {}
        for name in ("k", "v"):
            out[name] = exact_quantised(st["new_" + name])
            for s in range(S):
                out[name][s, counts[s]:] = 0
        return out
    if case["op"] == "evict":
        n, K = case["rows"], min(case["rows"], case["keep"])
        w, pos = st["weight"].double().cpu()[..., :n], st["pos"].cpu()[..., :n]
        out = {"k": torch.zeros(S, K, KH, D, dtype=torch.float64), "v": torch.zeros(S, K, KH, D, dtype=torch.float64),
               "weight": torch.zeros(S, KH, K, dtype=torch.float64), "pos": None}
        for s in range(S):
            for h in range(KH):
                p = pos[s, h].tolist()
                x = w[s, h].tolist()
                free = [p[i] < 2 * n - case["recent"] and p[i] >= case["first"] for i in range(n)]
                best = sorted(range(n), key=lambda i: (free[i], -x[i] if free[i] else 0, i))[:K]
                kept = set(best)
                above = iter(sorted(i for i in best if i >= K))
                frm = torch.tensor([i if i in kept else next(above) for i in range(K)])
                for name in ("k", "v"):
                    rows = exact_rows(st[name][s, h, :n], st[name + "_scale"][s, h, :, :n])
                    out[name][s, :, h] = rows.cpu()[frm]
                out["weight"][s, h] = w[s, h][frm]
        return out
    T, G, C = case["tokens"], case["group"], st["C"]
    out = torch.zeros(S, T, KH * G, D, dtype=torch.float64, device=st["q"].device)
    weight = torch.zeros(S, KH, C, dtype=torch.float64, device=out.device)
    for s in range(S):
        n, t = lens[s], counts[s]
        L = n if case["full"] else n + t
        if not t or not L:
            continue
        mask = torch.arange(L, device=out.device)[None] > (L - 1 if case["full"] else n + torch.arange(t, device=out.device)[:, None])
        for h in range(KH):
            k = exact_rows(st["k"][s, h, :L], st["k_scale"][s, h, :, :L])
            v = exact_rows(st["v"][s, h, :L], st["v_scale"][s, h, :, :L])
            for i in range(h * G, h * G + G):
                x = (st["q"][s, :t, i].double() @ k.T) * st["scale"]
                x = x.masked_fill(mask, -math.inf)
                p = torch.softmax(x, -1)
                out[s, :t, i] = p @ v
                weight[s, h, :L] += p.sum(0)
    return {"out": out, "weight": weight} if case["weights"] else {"out": out}

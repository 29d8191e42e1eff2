"""The operators of the paged KV cache, in their plain form and as calls of the framework.

The cache is a pool of pages that all sequences share; a page holds page_size consecutive tokens of one sequence:

    k, v         [pages][kv_heads][page_size][head_dim]   fp32, fp16 or bf16
    bounds       [pages][kv_heads][2][head_dim]           int8: least and greatest key of the page's rows, element by
                                                          element, in steps of 2^e, rounded outwards
    bounds_exp   [pages][kv_heads]                        int8: e, the least in -50 .. 50 with max |k| <= 127 * 2^e
    table        [seqs][width]                            int32: the page of a sequence's j-th page_size tokens
    free_pages   [pages]                                  int32: a stack of the pages that are free

Operators (``op`` of a case):
  tables     room for new tokens: pages from the stack, slots, positions and sequences of the packed tokens; or pages given back
  append     packed rows of keys and values into their slots, and the bounds of the pages that they go to
  attention  softmax(scale q.k) v of single query tokens over a sequence's rows
  sparse     the same over the pages with the largest bound on q.k
"""
import math
import random

import torch

own = False

#: what one pass may cost at most in a drawn case: rows read by the queries times kv heads times head dimension
MOST_READ = 4 * 131072 * 8 * 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -------------------------------------------------------------------
def listed():
    attn = {"op": "attention", "type": "f16", "seqs": 1, "queries": 1, "kv_heads": 8, "group": 4, "head_dim": 128,
            "page_size": 16, "ragged": False}
    sparse = {"op": "sparse", "type": "bf16", "kv_heads": 8, "group": 4, "head_dim": 128, "first": 1, "recent": 4}
    return [
        # a decode step of a full server, a token each: latency
        {"name": "step_decode", "op": "tables", "kind": "step", "seqs": 256, "page_size": 16, "held": 4001, "new": 1,
         "prompts": 0, "pool": 1.5},
        # a step that takes prompts in beside the decoding sequences, and runs out of pages before the last of them
        {"name": "step_prompts", "op": "tables", "kind": "step", "seqs": 600, "page_size": 16, "held": 6000, "new": 4099,
         "prompts": 64, "pool": 0.8},
        # half the sequences of a server end, the others give back what drafted tokens had taken
        {"name": "release", "op": "tables", "kind": "release", "seqs": 512, "page_size": 32, "held": 8191, "new": 0,
         "prompts": 256, "pool": 1.2},
        # keys and values of a decode step, bounds kept: latency
        {"name": "append_step", "op": "append", "type": "f16", "seqs": 64, "kv_heads": 8, "head_dim": 128, "page_size": 16,
         "held": 1501, "new": 1, "prompts": 0, "bounds": True},
        # a step with prompts in it, of uneven lengths
        {"name": "append_prompts", "op": "append", "type": "bf16", "seqs": 24, "kv_heads": 8, "head_dim": 128,
         "page_size": 32, "held": 777, "new": 2049, "prompts": 5, "bounds": True},
        # decode of a single chat: latency
        {**attn, "name": "decode_short", "rows": 600},
        # decode at the end of a very long document
        {**attn, "name": "decode_long", "type": "bf16", "page_size": 64, "rows": 131071},
        # decode of a full server: sequences of all lengths
        {**attn, "name": "decode_batch", "seqs": 64, "rows": 8190, "ragged": True},
        # drafted tokens, several query rows a sequence, an odd group of heads
        {**attn, "name": "decode_draft", "type": "bf16", "seqs": 16, "queries": 5, "kv_heads": 4, "group": 7, "head_dim": 64,
         "rows": 3001, "ragged": True},
        # the decoder's own fp32 rows, wide heads without groups
        {**attn, "name": "decode_wide", "type": "f32", "seqs": 5, "kv_heads": 4, "group": 1, "head_dim": 256, "page_size": 128,
         "rows": 20011, "ragged": True},
        # a few very long documents at once, 4096 rows of each attended to
        {**sparse, "name": "sparse_long", "seqs": 4, "page_size": 16, "rows": 131072, "keep": 256, "ragged": False},
        # a server of long chats
        {**sparse, "name": "sparse_batch", "type": "f16", "seqs": 32, "page_size": 32, "rows": 30011, "keep": 64,
         "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attention", "attention", "attention", "sparse"])
    c = {"op": op, "page_size": rng.choice([16, 16, 32, 64, 128, 256])}
    if op == "tables":
        c["kind"] = rng.choice(["step", "step", "release"])
        c["seqs"] = _log(rng, 1, 700)
        c["held"] = _log(rng, 1, 9000)
        c["prompts"] = rng.choice([0, rng.randint(0, c["seqs"]), min(c["seqs"], 16)])
        c["new"] = 0 if c["kind"] == "release" else 1 if not c["prompts"] else _log(rng, 1, 4200)
        while c["prompts"] * c["new"] > 64 * 4099:
            c["prompts"] //= 2
        c["pool"] = rng.choice([0.6, 1.0, 1.5])
        return c
    c["type"] = rng.choice(["f16", "bf16", "f32"])
    c["head_dim"] = rng.choice([64, 128, 128, 256])
    c["kv_heads"] = rng.choice([1, 2, 4, 5, 8, 8])
    if op == "append":
        c["seqs"] = _log(rng, 1, 300)
        c["held"] = _log(rng, 1, 3500)
        c["prompts"] = rng.choice([0, min(c["seqs"], _log(rng, 1, 12))])
        c["new"] = _log(rng, 1, 2500) if c["prompts"] else 1
        c["bounds"] = rng.random() < 0.6
        return c
    c["group"] = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    c["seqs"] = _log(rng, 1, 128)
    c["ragged"] = c["seqs"] > 1 and rng.random() < 0.6
    if op == "attention":
        c["queries"] = rng.choice([1, 1, 1, _log(rng, 2, 8)])
        c["rows"] = _log(rng, 1, 140000)
    else:
        c["rows"] = _log(rng, 200, 140000)
    while c["seqs"] * c.get("queries", 1) * c["rows"] * c["kv_heads"] * c["head_dim"] > MOST_READ:
        if c["seqs"] > 1 and rng.random() < 0.5:
            c["seqs"] = c["seqs"] * 2 // 3
        else:
            c["rows"] = max(1, c["rows"] * 2 // 3)
    if op == "sparse":
        pages = -(-c["rows"] // c["page_size"])
        c["keep"] = max(1, min(512, int(pages * rng.choice([0.03, 0.1, 0.3, 1.2]))))
        c["first"] = rng.choice([0, 1]) if c["keep"] > 2 else 0
        c["recent"] = min(rng.choice([0, 1, 2, 4]), c["keep"] - c["first"])
    return c


def cdiv(a, b):
    return -(-a // b)


def lengths(case):
    """Rows that the sequences hold, of all lengths where they are ragged, one of them at its start."""
    S, rows = case["seqs"], case["rows"]
    if not case["ragged"]:
        return [rows] * S
    lens = [rows - rows * s // S for s in range(S)]
    lens[-1] = 1
    return lens


def step_lengths(case, seed):
    """Tokens held and new of every sequence: prompts start behind nothing, or behind a part that is held already; the
    others bring a token each, some none.  The same numbers for every seed, in another order."""
    S, P = case["seqs"], case["prompts"]
    held = [case["held"] * (s + 1) // S for s in range(S)]
    new = [min(case["new"], 1)] * S
    for s in range(S):
        if case["op"] == "tables" and s % 9 == 7:
            new[s] = 0
        if s < P:
            new[s] = case["new"] - case["new"] * s // (2 * P)
            held[s] = 0 if s % 3 else case["held"] // 3
    order = list(range(S))
    random.Random(seed).shuffle(order)
    return [held[i] for i in order], [new[i] for i in order]


def kept_lengths(case, seed):
    """Tokens held and tokens that stay: 0 where a sequence ends, a few fewer where drafted ones go."""
    S, P = case["seqs"], case["prompts"]
    held = [case["held"] * (s + 1) // S for s in range(S)]
    keep = [0 if s % 2 and s // 2 < P else max(0, held[s] - s % 6) for s in range(S)]
    order = list(range(S))
    random.Random(seed).shuffle(order)
    return [held[i] for i in order], [keep[i] for i in order]


def work(case):
    ps, op = case["page_size"], case["op"]
    if op == "tables":
        S = case["seqs"]
        if case["kind"] == "release":
            held, keep = kept_lengths(case, 0)
            n = sum(cdiv(h, ps) - cdiv(k, ps) for h, k in zip(held, keep))
            return {"bytes": 8 * S + 8 * n, "flops": 8 * S + n}
        held, new = step_lengths(case, 0)
        n = sum(cdiv(h + c, ps) - cdiv(h, ps) for h, c in zip(held, new))
        return {"bytes": 16 * S + 16 * sum(new) + 8 * n * min(1.0, case["pool"]), "flops": 12 * S + 8 * sum(new)}
    KH, D = case["kv_heads"], case["head_dim"]
    es = 4 if case["type"] == "f32" else 2
    if op == "append":
        held, new = step_lengths(case, 0)
        n = sum(new)
        b = {"bytes": n * (8 + KH * D * (8 + 2 * es)), "flops": 2 * n * KH * D}
        if case["bounds"]:  # the rows held before in pages that get new ones, and the bounds
            pages = sum(cdiv(h + c, ps) - h // ps for h, c in zip(held, new) if c)
            b["bytes"] += KH * (sum(h % ps for h, c in zip(held, new) if c) * D * es + pages * (2 * D + 1))
            b["flops"] += 4 * KH * D * n
        return b
    G = case["group"]
    if op == "attention":
        Q = case["queries"]
        rows = sum(n + Q - 1 for n in lengths(case))
        pairs = sum(Q * n + Q * (Q - 1) // 2 for n in lengths(case))
        return {"bytes": rows * KH * 2 * D * es + case["seqs"] * Q * KH * G * D * 8, "flops": pairs * KH * G * 4 * D}
    pages = sum(cdiv(n, ps) for n in lengths(case))
    rows = sum(min(n, case["keep"] * ps) for n in lengths(case))
    picked = sum(min(cdiv(n, ps), case["keep"]) for n in lengths(case))
    return {"bytes": pages * KH * (2 * D + 1) + rows * KH * 2 * D * es + picked * KH * 4 + case["seqs"] * KH * G * D * 8,
            "flops": pages * KH * G * 4 * D + rows * KH * G * 4 * D}


# ---- inputs ------------------------------------------------------------------
def pow2(e):
    """2^e in fp32, from its bits, for whole e in -126 .. 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def page_bounds(k, rows):
    """int8 bounds [N][KH][2][D] and exponents [N][KH] of pages k [N][KH][ps][D] that hold their first rows [N] rows."""
    there = (torch.arange(k.shape[2], device=k.device) < rows[:, None])[:, None, :, None]
    x = k.float()
    lo = torch.where(there, x, math.inf).amin(2)
    hi = torch.where(there, x, -math.inf).amax(2)
    a = torch.maximum(lo.abs(), hi.abs()).amax(-1)
    f, e = torch.frexp(a)
    e = torch.where(f <= 127 / 128, e - 7, e - 6).clamp(-50, 50)
    e = torch.where(a == 0, -50, e)
    unit = pow2(-e)[..., None]
    codes = torch.stack([(lo * unit).floor(), (hi * unit).ceil()], 2).clamp(-127, 127)
    return codes.to(torch.int8), e.to(torch.int8)


def prepare_tables(case, seed, dev):
    ps, S = case["page_size"], case["seqs"]
    held, other = (kept_lengths if case["kind"] == "release" else step_lengths)(case, seed)
    used = sum(cdiv(h, ps) for h in held)
    fresh = (sum(h and cdiv(h, ps) for h in held) if case["kind"] == "release"
             else sum(cdiv(h + c, ps) - cdiv(h, ps) for h, c in zip(held, other)))
    spare = max(1, int(fresh * case["pool"]))
    pages = used + (spare if case["kind"] == "step" else max(1, spare // 8))
    width = cdiv(case["held"] + case["new"] + 1, ps) + 1
    g = torch.Generator(device=dev).manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=dev)
    ids = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((S, width), -1, **i32)
    lens = torch.tensor(held, **i32)
    live = torch.arange(width, device=dev) < ((lens + ps - 1) // ps)[:, None]
    table[live] = ids[:used]
    free = torch.full((pages,), -1, **i32)
    free[:pages - used] = ids[used:]
    # room for the step's tokens, and for some more that are not there
    tokens = sum(other) + 7 if case["kind"] == "step" else 0
    st = {"table": table, "free": free, "free_count": torch.tensor([pages - used], **i32), "lens": lens,
          "counts": torch.tensor(other, **i32), "pages": pages, "width": width, "tokens": tokens,
          "free_left": torch.zeros(1, **i32)}
    if case["kind"] == "step":
        st.update(granted=torch.zeros(S, **i32), start=torch.zeros(S + 1, **i32), positions=torch.zeros(tokens, **i32),
                  slots=torch.zeros(tokens, dtype=torch.int64, device=dev), seq_of=torch.zeros(tokens, **i32))
    return st


def pool_of(case, pages, g, dev):
    """Rows of keys with a few wide channels, and of values, in every page."""
    KH, D, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    wide = torch.where(torch.rand(KH, 1, D, generator=g, device=dev) < 0.04, 6.0, 1.0) * (
        torch.randn(KH, 1, D, generator=g, device=dev).abs() + 0.3)
    out = []
    for scale in (wide, 0.6):
        x = torch.empty(pages, KH, ps, D, dtype=TYPES[case["type"]], device=dev)
        for i in range(0, pages, 4096):
            n = min(4096, pages - i)
            x[i:i + n] = torch.randn(n, KH, ps, D, generator=g, device=dev) * scale
        out.append(x)
    return out[0], out[1], wide


def prepare_cache(case, seed, dev):
    KH, D, ps = case["kv_heads"], case["head_dim"], case["page_size"]
    g = torch.Generator(device=dev).manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] == "append":
        held, new = step_lengths(case, seed)
        total = [h + c for h, c in zip(held, new)]
    else:
        held, new = lengths(case), None
        total = [n + case.get("queries", 1) - 1 for n in held]
    counts = [cdiv(t, ps) for t in total]
    used = sum(counts)
    pages = used + 3
    width = max(counts) + 2
    ids = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((case["seqs"], width), -1, **i32)
    live = torch.arange(width, device=dev) < torch.tensor(counts, **i32)[:, None]
    table[live] = ids[:used]
    k, v, wide = pool_of(case, pages, g, dev)
    # rows behind a sequence's last one, and pages that are free, hold anything
    rows = torch.zeros(pages, dtype=torch.int64, device=dev)
    there = torch.tensor(held if case["op"] == "append" else total, **i32)[:, None] - torch.arange(width, device=dev) * ps
    rows[table[live].long()] = there[live].clamp(0, ps).long()
    junk = torch.arange(ps, device=dev) >= rows[:, None]
    for x in (k, v):
        x.masked_fill_(junk[:, None, :, None], math.nan)
    st = {"k": k, "v": v, "table": table, "pages": pages, "width": width}
    if case["op"] == "append":
        slots = []
        for s in range(case["seqs"]):
            at = torch.arange(held[s], total[s], device=dev)
            slots.append(table[s, at // ps].long() * ps + at % ps)
        slots.append(torch.full((5,), -1, dtype=torch.int64, device=dev))  # rows of the buffer that are no tokens
        st["slots"] = torch.cat(slots)
        T = st["tokens"] = st["slots"].numel()
        st["new_k"] = torch.randn(T, KH, D, generator=g, device=dev) * wide[:, 0]
        st["new_v"] = torch.randn(T, KH, D, generator=g, device=dev) * 0.6
        if case["bounds"]:
            st["bounds"], st["bounds_exp"] = page_bounds(k, rows.clamp_min(1))
            empty = rows == 0
            st["bounds"][empty], st["bounds_exp"][empty] = 0, 0
        return st
    Q, H = case.get("queries", 1), KH * case["group"]
    n = st["queries"] = case["seqs"] * Q
    s = torch.arange(n, device=dev) // Q
    st["lens"] = (torch.tensor(held, **i32)[s] - 1 + torch.arange(n, **i32) % Q).contiguous()  # held before the query's token
    st["seq_of"] = s.int() if Q > 1 else None
    # a query looks for a few rows of its sequence
    at = (torch.rand(n, generator=g, device=dev) * (st["lens"] + 1)).long().clamp_max(st["lens"].max().long())
    at = torch.minimum(at, st["lens"].long())
    near = k[table[s, at // ps].long(), :, at % ps].float() / wide[:, 0]
    st["q"] = (torch.randn(n, KH, case["group"], D, generator=g, device=dev) + 0.4 * near[:, :, None]).reshape(n, H, D)
    st["out"] = torch.zeros(n, H, D, device=dev)
    st["scale"] = 1.0 / math.sqrt(D)
    if case["op"] == "sparse":
        st["bounds"], st["bounds_exp"] = page_bounds(k, rows.clamp_min(1))
        st["select"] = torch.zeros(n, KH, case["keep"], **i32)
    return st


def prepare(case, seed):
    dev = torch.device("cuda")
    st = (prepare_tables if case["op"] == "tables" else prepare_cache)(case, seed, dev)
    st["case"] = dict(case)
    if own:
        own_handles(st)
    return st


# ---- the plain form ------------------------------------------------------------
def plain_step(st):
    ps, cap, T, pages = st["case"]["page_size"], st["width"] * st["case"]["page_size"], st["tokens"], st["pages"]
    n = st["lens"].long().clamp(0, cap)
    c = st["counts"].long().clamp_min(0)
    fits = n + c <= cap
    c = torch.where(fits, c, 0)
    old = (n + ps - 1) // ps
    need = (n + c + ps - 1) // ps - old
    P, C = need.cumsum(0), c.cumsum(0)
    fc = st["free_count"].long().clamp(0, pages)
    ok = fits & (P <= fc) & (C <= T)
    granted = torch.where(ok, c, 0)
    end = granted.cumsum(0)
    start = torch.cat([torch.zeros_like(end[:1]), end])
    r = torch.arange(T, device=n.device)
    s = torch.searchsorted(end, r, right=True)
    there = s < n.numel()
    s = s.clamp_max(n.numel() - 1)
    pos = n[s] + r - start[s]
    at = (pos // ps).clamp_max(st["width"] - 1)
    new = st["free"][(fc - 1 - (P - need)[s] - at + old[s]).clamp(0, pages - 1)].long()
    page = torch.where(at < old[s], st["table"][s, at].long(), new)
    rows = torch.nonzero(there & (pos % ps == 0))[:, 0]
    st["table"][s[rows], at[rows]] = page[rows].int()
    valid = there & (page >= 0) & (page < pages)
    left = fc - torch.where(ok, need, 0).sum()
    return {"granted": granted.int(), "start": start.int(), "slots": torch.where(valid, page * ps + pos % ps, -1),
            "positions": torch.where(there, pos, -1).int(), "seq_of": torch.where(there, s, -1).int(),
            "table": st["table"], "free_left": left.int()}


def plain_release(st):
    ps = st["case"]["page_size"]
    n = st["lens"].long().clamp(0, st["width"] * ps)
    k = torch.minimum(st["counts"].long().clamp_min(0), n)
    j = torch.arange(st["width"], device=n.device)
    pages = st["table"][(j >= ((k + ps - 1) // ps)[:, None]) & (j < ((n + ps - 1) // ps)[:, None])]
    fc = st["free_count"].long()
    at = fc + torch.arange(pages.numel() - 1, -1, -1, device=n.device)
    st["free"][at] = pages
    return {"free": st["free"], "free_left": (fc + pages.numel()).int()}


def plain_append(st):
    case = st["case"]
    ps, pages = case["page_size"], st["pages"]
    rows = torch.nonzero((st["slots"] >= 0) & (st["slots"] < pages * ps))[:, 0]
    slot = st["slots"][rows]
    page, at = slot // ps, slot % ps
    for name in ("k", "v"):
        st[name][page, :, at] = st["new_" + name][rows].to(st[name].dtype)
    out = {"k": st["k"], "v": st["v"]}
    if case["bounds"]:
        filled = torch.zeros(pages, dtype=torch.int64, device=slot.device).scatter_reduce(0, page, at + 1, "amax")
        p = torch.nonzero(filled)[:, 0]
        st["bounds"][p], st["bounds_exp"][p] = page_bounds(st["k"][p], filled[p])
        out.update(bounds=st["bounds"], bounds_exp=st["bounds_exp"])
    return out


def plain_rows(st, picked=None):
    """Keys and values [n][KH][L][D] in fp32, zeros where a query sees no row, and which rows it sees [n][KH][L].
    picked [n][KH][K]: the pages that a query sees, -1 where there is none."""
    case = st["case"]
    ps, KH = case["page_size"], case["kv_heads"]
    dev = st["q"].device
    sees = st["lens"].long() + 1
    table = st["table"].long() if st["seq_of"] is None else st["table"].long()[st["seq_of"].long()]
    if picked is None:
        picked = torch.arange(st["width"], device=dev).expand(sees.numel(), KH, -1)
    picked = picked.long()
    row = picked[..., None] * ps + torch.arange(ps, device=dev)
    ok = (picked >= 0)[..., None] & (row < sees[:, None, None, None])
    page = table.gather(1, picked.clamp_min(0).flatten(1)).view_as(picked).clamp_min(0)
    head = torch.arange(KH, device=dev)[:, None]
    out = []
    for name in ("k", "v"):
        x = st[name][page, head].float()  # [n][KH][K][ps][D]
        x.masked_fill_(~ok[..., None], 0.0)
        out.append(x.flatten(2, 3))
    return out[0], out[1], ok.flatten(2)


def plain_attention(st, picked=None):
    case = st["case"]
    n, KH, G, D = st["queries"], case["kv_heads"], case["group"], case["head_dim"]
    k, v, ok = plain_rows(st, picked)
    q = st["q"].reshape(n, KH, G, D) * st["scale"]
    x = torch.matmul(q, k.transpose(-1, -2))
    x = torch.where(ok[:, :, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p, v).reshape(n, KH * G, D)


def plain_select(st):
    case = st["case"]
    ps, KH, G, D, K = case["page_size"], case["kv_heads"], case["group"], case["head_dim"], case["keep"]
    q = st["q"].reshape(-1, KH, G, D)
    f, e = torch.frexp(q.abs().amax(-1))
    eq = torch.where(f == 0, -50, torch.where(f <= 127 / 128, e - 7, e - 6).clamp(-50, 50))
    qc = (q * pow2(-eq)[..., None]).round().clamp(-127, 127)
    pages = (st["lens"].long() + ps) // ps  # of lens + 1 rows
    j = torch.arange(st["width"], device=q.device)
    t = st["table"].long().clamp_min(0)
    b = st["bounds"][t].float()  # [n][W][KH][2][D]
    # whole numbers below 2^23: sums in fp32 are exact in any order
    s = torch.matmul(b[..., 1, :].transpose(1, 2), qc.clamp_min(0).transpose(-1, -2))
    s = s + torch.matmul(b[..., 0, :].transpose(1, 2), qc.clamp_max(0).transpose(-1, -2))  # [n][KH][W][G]
    s = s * pow2(eq)[:, :, None]
    s = s.amax(-1) * pow2(st["bounds_exp"][t]).transpose(1, 2)
    must = (j < case["first"]) | (j >= pages[:, None] - case["recent"])
    s = torch.where(must[:, None], math.inf, s)
    s = torch.where((j < pages[:, None])[:, None], s, -math.inf)
    order = torch.sort(s, dim=-1, descending=True, stable=True).indices
    if K > st["width"]:
        order = torch.nn.functional.pad(order, (0, K - st["width"]), value=st["width"])
    there = torch.arange(K, device=q.device) < pages[:, None].clamp_max(K)
    best = torch.where(there[:, None], order[..., :K], 1 << 30).sort(-1).values
    return torch.where(best == 1 << 30, -1, best).int()


def plain_sparse(st):
    picked = plain_select(st)
    return {"select": picked, "out": plain_attention(st, picked)}


# ---- the framework's calls -------------------------------------------------------
def own_handles(st):
    """The handles and workspaces that a program keeps beside its buffers."""
    from zeninfer_amd import zq
    case = st["case"]
    ps = case["page_size"]
    if case["op"] == "tables":
        st["tables"] = zq.PageTables(st["table"], st["free"], case["seqs"], st["width"], st["pages"], ps)
        return
    st["cache"] = zq.KVPaged(st["k"], st["v"], st["pages"], case["kv_heads"], case["head_dim"], ps,
                             bounds=st.get("bounds"), bounds_exp=st.get("bounds_exp"))
    if case["op"] == "append":
        return
    st["tables"] = zq.PageTables(st["table"], None, case["seqs"], st["width"], st["pages"], ps)
    n, H = st["queries"], case["kv_heads"] * case["group"]
    need = zq.attention_paged_workspace_bytes(st["cache"], st["tables"], n, H)
    if case["op"] == "sparse":
        need = max(need, zq.page_select_workspace_bytes(st["cache"], st["tables"], n, H, case["keep"]))
    st["workspace"], st["need"] = torch.empty(max(need, 16), dtype=torch.uint8, device=st["q"].device), need


def own_run(st):
    from zeninfer_amd import zq
    case = st["case"]
    op = case["op"]
    if op == "tables":
        if case["kind"] == "release":
            zq.page_tables_release_dev(st["tables"], st["lens"], st["counts"], st["free_count"], st["free_left"])
            return {"free": st["free"], "free_left": st["free_left"]}
        zq.page_tables_step_dev(st["tables"], st["lens"], st["counts"], st["free_count"], st["free_left"], st["granted"],
                                st["start"], st["slots"], st["positions"], st["seq_of"], st["tokens"])
        return {name: st[name] for name in ("granted", "start", "slots", "positions", "seq_of", "table", "free_left")}
    if op == "append":
        zq.kv_paged_append_dev(st["cache"], st["new_k"], st["new_v"], st["tokens"], st["slots"])
        return {name: st[name] for name in ("k", "v", "bounds", "bounds_exp") if name in st}
    n, H = st["queries"], case["kv_heads"] * case["group"]
    if op == "attention":
        zq.attention_paged_dev(st["cache"], st["tables"], st["q"], st["out"], n, H, st["lens"], st["scale"],
                               seq_of=st["seq_of"], workspace=st["workspace"], workspace_bytes=st["need"])
        return {"out": st["out"]}
    zq.page_select_dev(st["cache"], st["tables"], st["q"], st["select"], n, H, st["lens"], case["keep"],
                       recent=case["recent"], first=case["first"], workspace=st["workspace"], workspace_bytes=st["need"])
    zq.attention_paged_dev(st["cache"], st["tables"], st["q"], st["out"], n, H, st["lens"], st["scale"],
                           select=st["select"], keep=case["keep"], workspace=st["workspace"], workspace_bytes=st["need"])
    return {"select": st["select"], "out": st["out"]}


def run(state):
    if own:
        return own_run(state)
    case = state["case"]
    if case["op"] == "tables":
        return plain_release(state) if case["kind"] == "release" else plain_step(state)
    if case["op"] == "append":
        return plain_append(state)
    return plain_sparse(state) if case["op"] == "sparse" else {"out": plain_attention(state)}


# ---- the definition in 64 bits -----------------------------------------------------
def exact_step(st):
    case = st["case"]
    ps, W, T = case["page_size"], st["width"], st["tokens"]
    lens, counts, table = st["lens"].tolist(), st["counts"].tolist(), st["table"].cpu().clone()
    stack = st["free"].tolist()[:int(st["free_count"])]
    granted, start, slots, positions, seq_of = [], [0], [], [], []
    want_pages = want_tokens = 0
    for s, (n, c) in enumerate(zip(lens, counts)):
        got = 0
        if n + c <= W * ps:
            want_tokens += c
            want_pages += math.ceil((n + c) / ps) - math.ceil(n / ps)
            if want_pages <= int(st["free_count"]) and want_tokens <= T:
                got = c
        for p in range(n, n + got):
            if p % ps == 0:
                table[s, p // ps] = stack.pop()
            slots.append(int(table[s, p // ps]) * ps + p % ps)
            positions.append(p)
            seq_of.append(s)
        granted.append(got)
        start.append(start[-1] + got)
    pad = [-1] * (T - len(slots))
    ints = {"granted": granted, "start": start, "slots": slots + pad, "positions": positions + pad, "seq_of": seq_of + pad,
            "free_left": [len(stack)]}
    out = {name: torch.tensor(x) for name, x in ints.items()}
    return {**out, "table": table}


def exact_release(st):
    ps = st["case"]["page_size"]
    free, n = st["free"].cpu().clone(), int(st["free_count"])
    table = st["table"].tolist()
    back = []
    for s, (held, keep) in enumerate(zip(st["lens"].tolist(), st["counts"].tolist())):
        back += table[s][math.ceil(min(keep, held) / ps):math.ceil(held / ps)]
    free[n:n + len(back)] = torch.tensor(back[::-1], dtype=torch.int32)
    return {"free": free, "free_left": torch.tensor([n + len(back)])}


def rounded(x, kind):
    """The nearest value of the type to each of x (fp64), ties to even."""
    bits, least = {"f32": (24, -149), "f16": (11, -24), "bf16": (8, -133)}[kind]
    e = torch.frexp(x)[1] - bits
    unit = ((e.clamp_min(least).long() + 1023) << 52).view(torch.float64)
    return torch.round(x / unit) * unit


def exact_append(st):
    case = st["case"]
    ps, KH, D = case["page_size"], case["kv_heads"], case["head_dim"]
    out = {"k": st["k"].double(), "v": st["v"].double()}
    slots = st["slots"].tolist()
    rows = torch.tensor([r for r, x in enumerate(slots) if x >= 0], device=st["k"].device)
    slot = st["slots"][rows]
    for name in ("k", "v"):
        flat = out[name].transpose(1, 2).reshape(-1, KH, D)  # a row for every slot
        flat[slot] = rounded(st["new_" + name][rows].double(), case["type"])
        out[name] = flat.reshape(-1, ps, KH, D).transpose(1, 2).contiguous()
    if case["bounds"]:
        codes, exps = st["bounds"].cpu().clone().long(), st["bounds_exp"].cpu().clone().long()
        last = {}
        for x in slots:
            if x >= 0:
                last[x // ps] = max(last.get(x // ps, 0), x % ps)
        for p, at in last.items():
            x = out["k"][p, :, :at + 1].cpu()
            lo, hi = x.min(1).values, x.max(1).values
            a = torch.maximum(lo.abs(), hi.abs()).max(-1).values
            e = torch.tensor([max(-50, min(50, math.ceil(math.log2(y / 127) - 1e-12))) if y else -50 for y in a.tolist()])
            # the logarithm may be off next to a power of two
            e = torch.where(a > 127 * 2.0 ** e, e + 1, e)
            e = torch.where((e > -50) & (a <= 127 * 2.0 ** (e - 1)), e - 1, e)
            step = (2.0 ** e.double())[:, None]
            codes[p] = torch.stack([torch.floor(lo / step), torch.ceil(hi / step)], 1).long()
            exps[p] = e
        out.update(bounds=codes, bounds_exp=exps)
    return out


def exact_select(st, i, h, table):
    """The pages that query i sees of kv head h."""
    case = st["case"]
    G, ps, K = case["group"], case["page_size"], case["keep"]
    n = math.ceil((int(st["lens"][i]) + 1) / ps)
    page = table[i, :n].long()
    b = st["bounds"][page, h].double()
    e = st["bounds_exp"][page, h].double()
    best = torch.full((n,), -math.inf, dtype=torch.float64, device=b.device)
    for q in st["q"][i, h * G:(h + 1) * G].double():
        a = float(q.abs().max())
        eq = -50
        while eq < 50 and a > 127 * 2.0 ** eq:
            eq += 1
        c = torch.round(q / 2.0 ** eq).clamp(-127, 127)
        best = torch.maximum(best, torch.maximum(c * b[:, 0], c * b[:, 1]).sum(-1) * 2.0 ** eq * 2.0 ** e)
    score = best.tolist()
    must = [p < case["first"] or p >= n - case["recent"] for p in range(n)]
    order = sorted(range(n), key=lambda p: (not must[p], 0.0 if must[p] else -score[p], p))
    return sorted(order[:K])


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tables":
        return exact_release(st) if case["kind"] == "release" else exact_step(st)
    if case["op"] == "append":
        return exact_append(st)
    KH, G, D, ps = case["kv_heads"], case["group"], case["head_dim"], case["page_size"]
    sparse = case["op"] == "sparse"
    if st["queries"] * KH > 2000 or (sparse and KH * sum(cdiv(n, ps) for n in lengths(case)) > 600000):
        return None
    dev = st["q"].device
    out = torch.zeros(st["queries"], KH * G, D, dtype=torch.float64, device=dev)
    select = torch.full((st["queries"], KH, case.get("keep", 1)), -1)
    seq = st["seq_of"].tolist() if st["seq_of"] is not None else list(range(st["queries"]))
    table = st["table"][torch.tensor(seq, device=dev)]
    for i, n in enumerate(st["lens"].tolist()):
        for h in range(KH):
            which = list(range(math.ceil((n + 1) / ps)))
            if sparse:
                which = exact_select(st, i, h, table)
                select[i, h, :len(which)] = torch.tensor(which)
            row = (torch.tensor(which, device=dev)[:, None] * ps + torch.arange(ps, device=dev)).flatten()
            page = table[i, torch.tensor(which, device=dev)].long()
            k = st["k"][page, h].reshape(-1, D)[row <= n].double()
            v = st["v"][page, h].reshape(-1, D)[row <= n].double()
            q = st["q"][i, h * G:(h + 1) * G].double()
            out[i, h * G:(h + 1) * G] = torch.softmax((q @ k.T) * st["scale"], -1) @ v
    return {"select": select, "out": out} if sparse else {"out": out}

"""The dense paged-cache operators as cases to be measured: attention of the newest tokens over a paged
key-value cache (with a tanh cap, a distance bias, a window with sinks, document starts, and the attention
weights accumulated per cached key), eviction from that cache by the accumulated weights, and the append of a
step's rows.  ``run`` computes them in plain torch operations, or with ``own`` set through the package."""

from __future__ import annotations

import math

import torch

own = False

D = 128  # the framework's head dimension

_ATTEND = {
    "op": "attend", "dtype": "bf16", "requests": 1, "idle": 0, "kv_heads": 8, "group": 4, "tokens": 1, "shortest": 1024,
    "longest": 1024, "block": 16, "layout": "rows", "cap": 0.0, "alibi": False, "window": 0, "sinks": 0,
    "documents": False, "positions": False, "mass": False,
}
_EVICT = {
    "op": "evict", "dtype": "bf16", "requests": 1, "idle": 0, "kv_heads": 8, "shortest": 4352, "longest": 4352, "block": 16,
    "layout": "rows", "budget": 4096, "sinks": 4, "recent": 128,
}
_APPEND = {
    "op": "append", "dtype": "bf16", "requests": 1, "idle": 0, "kv_heads": 8, "tokens": 1, "shortest": 1000, "longest": 1000,
    "block": 16, "layout": "rows",
}


def listed():
    return [
        # a chat's first answers: one short request of the Llama-3-8B shape, where the launch and its chain count
        dict(_ATTEND, name="one request of 1K"),
        # the headline decode shape, dense: 2.1 GB of cache for one token of four requests
        dict(_ATTEND, name="batch 4, 128K", requests=4, shortest=131072, longest=131072),
        # a serving batch of mixed lengths with one idle row, scores capped as some models train them
        dict(_ATTEND, name="batch 16, 8K to 64K, capped", requests=16, idle=1, shortest=8192, longest=65536, layout="heads", cap=50.0),
        # one KV head of a 70B shape sharded over eight GPUs, G = 8, the longest contexts
        dict(_ATTEND, name="one KV head, G 8, 256K", requests=8, kv_heads=1, group=8, shortest=262144, longest=262144, layout="heads"),
        # a distance-bias model in fp32 with odd sizes; documents packed in one sequence
        dict(_ATTEND, name="fp32, distance bias, odd", dtype="fp32", requests=3, kv_heads=5, group=3, shortest=1001, longest=9001,
             block=13, alibi=True, documents=True),
        # a speculative step of four tokens through a sliding-window layer that keeps its first tokens
        dict(_ATTEND, name="speculative, window, fp16", dtype="fp16", requests=8, tokens=4, shortest=2500, longest=16384, window=4096, sinks=4),
        # the prompt's last step before an eviction: weights of every key accumulated
        dict(_ATTEND, name="weights over 32K", requests=4, shortest=32768, longest=32768, mass=True),
        # steady state of an evicting server: 64 requests of about 2K kept keys each, out of order
        dict(_ATTEND, name="evicted caches, weights", requests=64, shortest=2048, longest=2304, layout="heads", positions=True, mass=True),
        # one request back under its budget after 256 tokens
        dict(_EVICT, name="evict 256 of 4352"),
        # prompts of 128K down to 16K
        dict(_EVICT, name="evict 128K to 16K, batch 4", requests=4, shortest=131072, longest=131072, budget=16384),
        # a step's rows of one request, and of a full batch
        dict(_APPEND, name="append one token"),
        dict(_APPEND, name="append, 256 requests of 4", requests=256, tokens=4, shortest=100, longest=1000, layout="heads"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "evict", "append"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    block = rng.choice([1, 7, 13, 16, 16, 32, 48, 64, 128])
    layout = rng.choice(["rows", "heads"])
    heads = rng.choice([1, 2, 3, 5, 8])
    requests = _log_int(rng, 1, 64)
    idle = rng.choice([0, 0, 1]) if requests > 1 else 0
    if op == "append":
        return dict(_APPEND, dtype=dtype, requests=requests, idle=idle, kv_heads=heads, tokens=rng.randint(1, 8),
                    shortest=0 if rng.random() < 0.2 else rng.randint(1, 500), longest=rng.randint(500, 2000), block=block, layout=layout)
    # at most 1 GiB of 16-bit keys and values (2 GiB in fp32): 2^21 rows of one KV head
    longest = _log_int(rng, 1, min(200000, (1 << 21) // (requests * heads)))
    shortest = rng.randint(1, longest)
    if op == "evict":
        budget = _log_int(rng, 1, max(longest, 1))
        sinks = rng.randint(0, min(4, budget))
        return dict(_EVICT, dtype=dtype, requests=requests, idle=idle, kv_heads=heads, shortest=shortest, longest=longest, block=block,
                    layout=layout, budget=budget, sinks=sinks, recent=rng.randint(0, min(256, budget - sinks)))
    group = rng.randint(1, 8)
    tokens = rng.choice([1, 1, 1, rng.randint(2, 8)])
    positions = rng.random() < 0.25
    window = _log_int(rng, 1, 8192) if rng.random() < 0.3 else 0
    return dict(_ATTEND, dtype=dtype, requests=requests, idle=idle, kv_heads=heads, group=group, tokens=tokens, shortest=shortest,
                longest=longest, block=block, layout=layout, cap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3,
                window=window, sinks=rng.choice([0, 4]) if window else 0, documents=rng.random() < 0.2, positions=positions,
                mass=positions or rng.random() < 0.2)


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lens(case):
    """Request lengths spread evenly over the case's range, in mixed order; the first ``idle`` rows are padding."""
    n, lo, hi = case["requests"], case["shortest"], case["longest"]
    lens = [lo + (hi - lo) * ((r * 7 + 3) % n) // max(n - 1, 1) if n > 1 else hi for r in range(n)]
    return [0] * case["idle"] + lens[case["idle"]:]


def _firsts(case):
    """First token of each request's last document: every other request holds an earlier document."""
    return [n // 3 if r % 2 == 0 else 0 for r, n in enumerate(_lens(case))]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    e = _TYPES[case["dtype"]]
    B, H, bs = case["requests"], case["kv_heads"], case["block"]
    lens = _lens(case)
    room = max(max(lens) + (case["tokens"] if case["op"] == "append" else 0), 1)
    per = -(-room // bs)
    blocks = B * per + 3
    shape = (2, blocks, bs, H, D) if case["layout"] == "rows" else (blocks, H, bs, 2 * D)
    kv = torch.randn(shape, dtype=e, device="cuda", generator=g)
    keys = kv[0] if case["layout"] == "rows" else kv[..., :D]
    loud = torch.randperm(D, device="cuda", generator=g)[:4]
    keys[..., loud] = keys[..., loud] * 4  # outlier channels, as keys have them
    table = torch.randperm(blocks, device="cuda", generator=g)[: B * per].view(B, per).to(torch.int32)
    st = {"case": dict(case), "kv": kv, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    slots = per * bs
    if case["op"] == "attend":
        G, T = case["group"], case["tokens"]
        q = torch.randn(B, T, H, G, D, device="cuda", generator=g)
        at = (torch.rand(B, device="cuda", generator=g) * st["lens"]).long()  # a key each query has something to do with
        near = _rows(case, kv)[0][table.gather(1, (at // bs).view(B, 1)).long().view(B), at % bs]
        st["q"] = (q + 0.1 * near.float().view(B, 1, H, 1, D)).reshape(B, T, H * G, D).to(e)
        st["out"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty(B, T, H * G, dtype=torch.float32, device="cuda")
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, H * G + 1, device="cuda") / (H * G)).float() if case["alibi"] else None
        st["first"] = torch.tensor(_firsts(case), dtype=torch.int32, device="cuda") if case["documents"] else None
        st["pos"] = st["qpos"] = st["mass"] = None
        if case["positions"]:
            # every third token of the sequence is still there, in no order
            order = torch.rand(B, H, slots, device="cuda", generator=g)
            order[torch.arange(slots, device="cuda").expand(B, H, slots) >= st["lens"].view(B, 1, 1)] = 2.0
            rank = order.argsort(2).argsort(2)
            st["pos"] = (3 * rank + torch.randint(0, 3, rank.shape, device="cuda", generator=g)).to(torch.int32)
            st["qpos"] = 3 * st["lens"] + T
        if case["mass"]:
            st["mass"] = torch.rand(B, H, slots, device="cuda", generator=g)
    elif case["op"] == "evict":
        # weights spread over decades as attention leaves them; a fifth have underflowed to nothing
        mass = torch.exp(2.0 * torch.randn(B, H, slots, device="cuda", generator=g))
        mass[torch.rand(B, H, slots, device="cuda", generator=g) < 0.2] = 0.0
        st["mass"], st["pos"] = mass, torch.arange(slots, dtype=torch.int32, device="cuda").repeat(B, H, 1)
        st["qpos"] = st["lens"] - 1
        st["new_mass"], st["new_pos"], st["new_lens"] = mass.clone(), st["pos"].clone(), st["lens"].clone()
        st["source"] = torch.empty(B, H, case["budget"], dtype=torch.int32, device="cuda")
    else:
        T = case["tokens"]
        st["k"] = torch.randn(B, T, H, D, device="cuda", generator=g).to(e)
        st["v"] = torch.randn(B, T, H, D, device="cuda", generator=g).to(e)
        st["pos"] = torch.arange(slots, dtype=torch.int32, device="cuda").repeat(B, H, 1)
        st["mass"] = torch.rand(B, H, slots, device="cuda", generator=g)
        st["qpos"] = 3 * st["lens"] + T
        st["new_lens"] = torch.empty_like(st["lens"])
    if own:
        from pqhsa_release_b200 import PagedAttention

        c = case
        st["attn"] = PagedAttention(
            num_query_heads=H * c.get("group", 1), num_kv_heads=H, max_requests=B, token_capacity=slots, dtype=e, device="cuda",
            max_query_len=c.get("tokens", 1), softcap=c.get("cap", 0.0), alibi_slopes=st.get("slopes"), window=c.get("window", 0),
            sink_tokens=c.get("sinks", 0))
        st["attn"].bind_kv_paged(kv, table)
    return st


def _rows(case, kv):
    """Views (keys, values) [blocks, block, heads, D] of either page layout."""
    if case["layout"] == "rows":
        return kv[0], kv[1]
    return kv[..., :D].transpose(1, 2), kv[..., D:].transpose(1, 2)


def run(st):
    op = st["case"]["op"]
    if op == "attend":
        return _own_attend(st) if own else _plain_attend(st)
    if op == "evict":
        return _own_evict(st) if own else _plain_evict(st)
    return _own_append(st) if own else _plain_append(st)


def _own_attend(st):
    st["attn"].forward(st["q"], st["lens"], out=st["out"], lse=st["lse"], first_key=st["first"], key_pos=st["pos"],
                       query_pos=st["qpos"], mass=st["mass"])
    return _attend_outputs(st, st["out"], st["lse"])


def _own_evict(st):
    c = st["case"]
    st["attn"].evict(st["lens"], mass=st["mass"], key_pos=st["pos"], query_pos=st["qpos"], budget=c["budget"], recent=c["recent"],
                     new_lens=st["new_lens"], new_mass=st["new_mass"], new_pos=st["new_pos"], source=st["source"])
    return _evict_outputs(st)


def _own_append(st):
    st["attn"].append(st["k"], st["v"], st["lens"], new_lens=st["new_lens"], key_pos=st["pos"], query_pos=st["qpos"], mass=st["mass"])
    return _append_outputs(st)


def _attend_outputs(st, out, lse):
    r = {"out": out, "lse": lse}
    if st["mass"] is not None:
        r["mass"] = st["mass"]
    return r


def _evict_outputs(st):
    return {"kv": st["kv"], "lens": st["new_lens"], "mass": st["new_mass"], "pos": st["new_pos"], "source": st["source"]}


def _append_outputs(st):
    return {"kv": st["kv"], "lens": st["new_lens"], "mass": st["mass"], "pos": st["pos"]}


# ---- plain forms: every request padded to the longest, 32 bits throughout ------------------------------------


def _plain_attend(st):
    c = st["case"]
    B, H, G, T = c["requests"], c["kv_heads"], c["group"], c["tokens"]
    k, v = _rows(c, st["kv"])
    N = st["table"].shape[1] * c["block"]
    table = st["table"].long()
    k = k[table].reshape(B, N, H, D).permute(0, 2, 1, 3).float()
    v = v[table].reshape(B, N, H, D).permute(0, 2, 1, 3).float()
    q = st["q"].view(B, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, T * G, D).float()
    s = (torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(D))).view(B, H, T, G, N)
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    slot = torch.arange(N, device=s.device)
    pos = (st["pos"].long() if c["positions"] else slot.expand(B, H, N)).view(B, H, 1, 1, N)
    last = st["qpos"].long() if c["positions"] else st["lens"].long() - 1
    at = (last.view(B, 1) - (T - 1) + torch.arange(T, device=s.device)).view(B, 1, T, 1, 1)
    first = (st["first"].long() if c["documents"] else torch.zeros_like(last)).view(B, 1, 1, 1, 1)
    if c["alibi"]:
        s = s - st["slopes"].view(1, H, 1, G, 1) * (at - pos).float()
    seen = (slot < st["lens"].view(B, 1)).view(B, 1, 1, 1, N) & (pos >= first) & (pos <= at)
    if c["window"]:
        seen = seen & ((at - pos < c["window"]) | (pos - first < c["sinks"]))
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(s - top), 0.0)
    total = w.sum(-1, keepdim=True)
    v = torch.where(seen.amax((2, 3)).expand(B, H, N)[..., None], v, 0.0)
    w = torch.where(total > 0, w / total, 0.0)
    out = torch.matmul(w.reshape(B, H, T * G, N), v).view(B, H, T, G, D).permute(0, 2, 1, 3, 4)
    st["out"].copy_(out.reshape(B, T, H * G, D))
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    st["lse"].copy_(lse.view(B, H, T, G).permute(0, 2, 1, 3).reshape(B, T, H * G))
    if c["mass"]:
        st["mass"] += w.sum((2, 3))
    return _attend_outputs(st, st["out"], st["lse"])


def _plain_evict(st):
    c = st["case"]
    B, H, K, bs = c["requests"], c["kv_heads"], c["budget"], c["block"]
    N = st["mass"].shape[2]
    slot = torch.arange(N, device="cuda").expand(B, H, N)
    n = st["lens"].long().view(B, 1, 1)
    pos = st["pos"].long()
    safe = (pos < c["sinks"]) | (pos > st["qpos"].long().view(B, 1, 1) - c["recent"])
    key = torch.where(torch.isnan(st["mass"]), -math.inf, st["mass"])
    key = torch.where(safe, math.inf, key)
    # slots behind the request's end come last whatever their key: sort by it first, then stably by being there
    order = torch.sort(key, dim=2, descending=True, stable=True).indices
    order = order.gather(2, torch.sort((order < n).int(), dim=2, descending=True, stable=True).indices)
    rank = torch.empty_like(order).scatter_(2, order, slot)
    keep = (rank < K) & (slot < n)
    K1 = min(K, N)
    end = torch.clamp(n, max=K)
    hole = (slot < end) & ~keep
    late = (slot >= K) & keep
    at = torch.where(late, late.cumsum(2) - 1, N)
    moved = torch.zeros(B, H, N + 1, dtype=torch.long, device="cuda").scatter_(2, at, slot)
    source = torch.where(hole, moved.gather(2, torch.clamp(hole.cumsum(2) - 1, min=0)), slot)
    st["source"].fill_(-1)
    st["source"][..., :K1] = torch.where(slot < end, source, -1)[..., :K1].int()
    st["new_lens"].copy_(torch.minimum(st["lens"], torch.full_like(st["lens"], K)))
    head = slot[..., :K1] < end
    new_mass = torch.where(head, st["mass"].gather(2, source[..., :K1]), st["new_mass"][..., :K1])
    new_pos = torch.where(head, st["pos"].gather(2, source[..., :K1]), st["new_pos"][..., :K1])
    st["new_mass"][..., :K1], st["new_pos"][..., :K1] = new_mass, new_pos
    to, fro = slot[..., :K1], source[..., :K1]
    fro = torch.where(head, fro, to)
    table = st["table"].long().view(B, 1, -1).expand(B, H, -1)
    heads = torch.arange(H, device="cuda").view(1, H, 1).expand(B, H, K1)
    tb, fb = table.gather(2, to // bs), table.gather(2, fro // bs)
    k, v = _rows(c, st["kv"])
    k[tb, to % bs, heads] = k[fb, fro % bs, heads]
    v[tb, to % bs, heads] = v[fb, fro % bs, heads]
    return _evict_outputs(st)


def _plain_append(st):
    c = st["case"]
    B, H, T, bs = c["requests"], c["kv_heads"], c["tokens"], c["block"]
    step = torch.arange(T, device="cuda")
    slot = st["lens"].long().view(B, 1) + step
    blk = st["table"].long().gather(1, slot // bs)
    k, v = _rows(c, st["kv"])
    k[blk, slot % bs] = st["k"]
    v[blk, slot % bs] = st["v"]
    at = slot.view(B, 1, T).expand(B, H, T)
    st["pos"].scatter_(2, at, (st["qpos"].view(B, 1, 1) - (T - 1) + step.int()).expand(B, H, T).contiguous())
    st["mass"].scatter_(2, at, torch.zeros(B, H, T, device="cuda"))
    torch.add(st["lens"], T, out=st["new_lens"])
    return _append_outputs(st)


# ---- from the definitions, in 64 bits, one request and head at a time ----------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "evict": _exact_evict, "append": _exact_append}[case["op"]](case, st)


def _slots(case, st, r, lo, hi):
    """Page and row of the slots lo .. hi of request r."""
    i = torch.arange(lo, hi, device="cuda")
    return st["table"][r].long()[i // case["block"]], i % case["block"]


def _exact_attend(case, st):
    B, H, G, T = case["requests"], case["kv_heads"], case["group"], case["tokens"]
    k, v = _rows(case, st["kv"])
    out = torch.zeros(B, T, H * G, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, T, H * G), -math.inf, dtype=torch.float64, device="cuda")
    mass = st["mass"].double() if case["mass"] else None
    for r, n in enumerate(_lens(case)):
        if n == 0:
            continue
        blk, row = _slots(case, st, r, 0, n)
        f = _firsts(case)[r] if case["documents"] else 0
        for h in range(H):
            kk, vv = k[blk, row, h].double(), v[blk, row, h].double()
            pos = st["pos"][r, h, :n].long() if case["positions"] else torch.arange(n, device="cuda")
            for t in range(T):
                p = (int(st["qpos"][r]) if case["positions"] else n - 1) - (T - 1 - t)
                ok = (pos >= f) & (pos <= p)
                if case["window"]:
                    ok &= (p - pos < case["window"]) | (pos - f < case["sinks"])
                at = ok.nonzero().view(-1)
                if at.numel() == 0:
                    continue
                rows = slice(h * G, (h + 1) * G)
                s = st["q"][r, t, rows].double() @ kk[at].T / math.sqrt(D)
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if case["alibi"]:
                    s = s - st["slopes"][rows].double().view(G, 1) * (p - pos[at]).double()
                z = torch.logsumexp(s, 1)
                w = torch.exp(s - z.view(G, 1))
                out[r, t, rows], lse[r, t, rows] = w @ vv[at], z
                if mass is not None:
                    mass[r, h, at] += w.sum(0)
    res = {"out": out, "lse": lse}
    if mass is not None:
        res["mass"] = mass
    return res


def _exact_evict(case, st):
    H, K = case["kv_heads"], case["budget"]
    k, v = _rows(case, st["kv"])
    mass, pos = st["mass"].double(), st["pos"].clone()
    new_mass, new_pos, source = mass.clone(), pos.clone(), torch.full_like(st["source"], -1)
    for r, n in enumerate(_lens(case)):
        blk, row = _slots(case, st, r, 0, n)
        last = n - 1
        for h in range(H):
            m, p = mass[r, h, :n].clone(), pos[r, h, :n]
            m[(p < case["sinks"]) | (p > last - case["recent"])] = math.inf
            kept = torch.sort(-m, stable=True).indices[:K].sort().values
            end = min(n, K)
            src = torch.arange(end, device="cuda")
            stay = torch.zeros(max(n, 1), dtype=torch.bool, device="cuda")
            stay[kept] = True
            src[(~stay[:end]).nonzero().view(-1)] = kept[kept >= K]
            source[r, h, :end] = src.int()
            new_mass[r, h, :end], new_pos[r, h, :end] = mass[r, h, src], pos[r, h, src]
            k[blk[:end], row[:end], h] = k[blk[src], row[src], h]
            v[blk[:end], row[:end], h] = v[blk[src], row[src], h]
    return {"kv": st["kv"].double(), "lens": torch.clamp(st["lens"], max=K), "mass": new_mass, "pos": new_pos, "source": source}


def _exact_append(case, st):
    k, v = _rows(case, st["kv"])
    T = case["tokens"]
    for r, n in enumerate(_lens(case)):
        blk, row = _slots(case, st, r, n, n + T)
        for j in range(T):
            k[blk[j], row[j]], v[blk[j], row[j]] = st["k"][r, j], st["v"][r, j]
            st["pos"][r, :, n + j] = st["qpos"][r] - (T - 1) + j
            st["mass"][r, :, n + j] = 0.0
    return {"kv": st["kv"].double(), "lens": st["lens"] + T, "mass": st["mass"].double(), "pos": st["pos"]}


# ---- what one pass cannot do without -------------------------------------------------------------------------


def _seen(case, n, r):
    """(keys any query token of the request sees, (token, key) pairs), taken without stored positions."""
    T, W = case["tokens"], case["window"]
    f = _firsts(case)[r] if case["documents"] else 0
    if case["positions"]:
        # positions 3 i + 0..2 up to 3 (n - 1) + 2, query tokens at 3 n + 1 and on: a window of W positions holds W / 3 keys
        keys = n - -(-f // 3)
        if W:
            keys = min(keys, max(0, (W - T) // 3) + (case["sinks"] + 2) // 3)
        return max(keys, 0), max(keys, 0) * T
    pairs, least = 0, n
    for t in range(T):
        p = n - T + t
        lo = max(f, p - W + 1) if W else f
        sinks = min(f + case["sinks"], lo) - f if W else 0
        pairs += max(0, p - lo + 1) + (max(0, min(sinks, p - f + 1)) if p >= f else 0)
        least = min(least, max(lo, 0))
    sinks = max(0, min(f + case["sinks"], least) - f) if W else 0
    return max(0, n - least) + sinks, pairs


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    H = case["kv_heads"]
    lens = _lens(case)
    if case["op"] == "append":
        rows = case["requests"] * case["tokens"] * H
        return {"bytes": rows * (4 * D * e + 8) + 12 * case["requests"], "flops": 0}
    if case["op"] == "evict":
        total = 12 * case["requests"]
        for n in lens:
            if n <= case["budget"]:
                total += H * n * 12
                continue
            K, safe = case["budget"], min(case["sinks"] + case["recent"], case["budget"])
            late = min(case["recent"], n - K) + (K - safe) * max(0, n - K - case["recent"]) / max(1, n - safe)
            total += H * (8 * n + 12 * K + late * 4 * D * e)
        return {"bytes": total, "flops": 0}
    G, T = case["group"], case["tokens"]
    total = flops = 0
    for r, n in enumerate(lens):
        keys, pairs = _seen(case, n, r)
        total += H * keys * (2 * D * e + (8 if case["mass"] else 0) + (4 if case["positions"] else 0))
        total += T * H * G * (2 * D * e + 4)
        flops += 4 * D * pairs * H * G
    return {"bytes": total, "flops": flops}

"""Timed cases of the long-context cache in 8 bits: norms on the way in, quantised writes, reading back,
attention over the codes.

The paged cache of ``retrieve_amd.kv`` holds keys and values in 16 bits. Half the bytes hold twice the
tokens and halve what a decode step reads: a block's keys of one head are int8 codes with one scale once
the block is full, its values the same; a sequence's last, open block stays in 16 bits until then. Models
that norm each head's queries and keys do it right before the rotation. The cases are single calls:

- ``append``: the 16-bit cache's append with those norms;
- ``write``: the append to the 8-bit cache (``append_int8``);
- ``read``: tokens read back in 16 bits (``read_int8``);
- ``attend``: softmax attention over chosen blocks of the 8-bit cache (``block_attention_int8``).

Where ``own`` is false each is computed from elementary torch operations in 32 bits (the norms' sums in
64: a key next to a code's border moves by a whole code).
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# --- the cases --------------------------------------------------------------------------------


def listed():
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 64}
    mha = {"heads": 14, "kv_heads": 14, "dim": 64, "page": 16}
    return [
        # one user's next token, queries and keys normed: launch latency
        {"name": "append_norm_b1", "op": "append", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 1000, "high": 1000, "rot": 128, "interleaved": False, "norm": True},
        # ragged prompts
        {"name": "append_norm_9k", "op": "append", "dtype": "bf16", **gqa, "seqs": 3, "new": 9001,
         "low": 0, "high": 61, "rot": 128, "interleaved": False, "norm": True},
        # one user's next token into the 8-bit cache
        {"name": "write_b1", "op": "write", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 1000, "high": 1000, "rot": 128, "interleaved": False, "norm": True},
        # a large decode batch of short ragged contexts, small pages, half of each head rotated
        {"name": "write_b203", "op": "write", "dtype": "fp16", **mha, "seqs": 203, "new": 203,
         "low": 3, "high": 300, "rot": 32, "interleaved": True, "norm": False},
        # ragged prompts, normed
        {"name": "write_9k", "op": "write", "dtype": "bf16", **gqa, "seqs": 3, "new": 9001,
         "low": 0, "high": 61, "rot": 128, "interleaved": False, "norm": True},
        # many prompts, wide heads and pages
        {"name": "write_16k_d256", "op": "write", "dtype": "fp16", "heads": 16, "kv_heads": 8,
         "dim": 256, "page": 128, "seqs": 8, "new": 16384, "low": 0, "high": 120, "rot": 256,
         "interleaved": True, "norm": False},
        # a few short contexts back in 16 bits
        {"name": "read_b7", "op": "read", "dtype": "fp16", **mha, "seqs": 7, "new": 2003,
         "low": 0, "high": 40},
        # long contexts handed to a layer that wants 16 bits
        {"name": "read_131k", "op": "read", "dtype": "bf16", **gqa, "seqs": 4, "new": 131001,
         "low": 0, "high": 5000},
        # one user's next token over few blocks
        {"name": "attend_b1", "op": "attend", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 30001, "high": 30001, "count": 32},
        # many small blocks, no shared heads
        {"name": "attend_b48_p16", "op": "attend", "dtype": "fp16", **mha, "seqs": 48, "new": 48,
         "low": 100, "high": 12000, "count": 96},
        # a serving batch over long ragged contexts: the cache's bytes
        {"name": "attend_b64", "op": "attend", "dtype": "bf16", **gqa, "seqs": 64, "new": 64,
         "low": 2000, "high": 40000, "count": 64},
        # chunks of two prompts, neighbouring tokens' choices alike
        {"name": "attend_prompt_2k", "op": "attend", "dtype": "bf16", **gqa, "seqs": 2, "new": 2053,
         "low": 3000, "high": 14000, "count": 16},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """Ragged lengths: the listed cases hold the round ones."""
    c = _any(rng)
    for x in ("low", "high", "new"):
        c[x] += int(c[x] > 0 and c[x] % 1024 == 0)
    return c


def _any(rng):
    small = (64, 96, 128, 128, 192, 256)
    heads, kv, dims = rng.choice([(32, 8, (128, 128, 256)), (20, 20, small), (28, 4, small),
                                  (18, 6, small), (10, 2, small), (8, 1, small), (40, 10, small),
                                  (5, 5, small)])
    c = {"op": rng.choice(["append", "write", "write", "read", "attend", "attend"]),
         "dtype": rng.choice(["bf16", "fp16"]), "heads": heads, "kv_heads": kv,
         "dim": rng.choice(dims), "page": rng.choice([16, 32, 64, 64, 128])}
    prompt = rng.random() < 0.4
    d = c["dim"]
    if c["op"] in ("append", "write"):
        c["seqs"] = _spread(rng, 1, 8) if prompt else _spread(rng, 1, 256)
        most = max(c["seqs"], min(16384, 9001 * 48 * 128 // ((heads + 2 * kv) * d)))
        c["new"] = _spread(rng, c["seqs"], most) if prompt else c["seqs"]
        c["low"] = 0 if rng.random() < 0.3 else _spread(rng, 1, 100)
        c["high"] = c["low"] + rng.randrange(0, 200)
        c["rot"] = rng.choice([d, d, d // 2, 32, 20])
        c["interleaved"] = rng.random() < 0.5
        c["norm"] = c["op"] == "append" or rng.random() < 0.5
    elif c["op"] == "read":
        c["seqs"] = _spread(rng, 1, 16)
        c["new"] = _spread(rng, c["seqs"], 131001 * 1024 // (kv * d))
        c["low"] = 0 if rng.random() < 0.5 else _spread(rng, 1, 300)
        c["high"] = c["low"] + rng.randrange(0, 1000)
    else:
        c["count"] = rng.choice([4, 16, 32, 64, 96])
        keys = c["count"] * c["page"]
        if prompt:
            c["seqs"] = _spread(rng, 1, 3)
            most = 2053 * 1024 * 128 // (keys * d * max(kv / 8, heads / 32))
            c["new"] = _spread(rng, max(c["seqs"], 2), max(c["seqs"], 2, min(2053, int(most))))
            c["low"] = 0 if rng.random() < 0.2 else _spread(rng, 1, 8000)
            c["high"] = c["low"] + rng.randrange(0, 6000)
        else:
            most = 64 * 8 * 4096 * 128 // (kv * keys * d)
            c["seqs"] = c["new"] = _spread(rng, 1, max(1, min(64, most)))
            c["low"] = _spread(rng, 1, 4000)
            c["high"] = c["low"] + rng.randrange(0, 20000)
    return c


# --- what a case holds, from its plain values ----------------------------------------------------


def sequences(case):
    """(tokens already in the cache, new tokens) of each sequence: spread over the case's range, the
    first at its upper end, and shares of the new tokens that differ by up to a factor of two. A read
    takes the ``new`` tokens behind the first ones."""
    n = case["seqs"]
    part = [(i * 0.6180339887) % 1.0 for i in range(n)]
    had = [case["high"] - round((case["high"] - case["low"]) * x) for x in part]
    weight = [1.0 + x for x in part]
    spare = case["new"] - n
    extra = [int(spare * w / sum(weight)) for w in weight]
    extra[-1] += spare - sum(extra)
    return [(h, 1 + e) for h, e in zip(had, extra)]


def _tokens(case):
    """Positions and sequence numbers of the packed tokens, on the host."""
    pos, seq = [], []
    for i, (had, new) in enumerate(sequences(case)):
        pos += range(had, had + new)
        seq += [i] * new
    return pos, seq


def work(case):
    h, kv, d, page, t = (case[x] for x in ("heads", "kv_heads", "dim", "page", "new"))
    meta = 8 * t
    if case["op"] in ("append", "write"):
        full = before = still = 0
        for had, new in sequences(case):
            n = (had + new) // page - had // page
            full += n
            before += had % page if n else 0
            still += (had + new) % page if n else new
        moved = 2 * t * h * d * 2 + 2 * t * kv * d * 2 + t * case["rot"] * 4 + meta
        bounds = full * kv * (2 * d + 4)
        flops = t * (h + kv) * (3 * case["rot"] + 4 * d * case["norm"]) + 2 * full * kv * page * d
        if case["op"] == "append":
            return {"bytes": moved + 2 * t * kv * d * 2 + bounds + before * kv * d * 2,
                    "flops": flops}
        return {"bytes": moved + bounds + 2 * full * kv * (page * d + 4) + 4 * before * kv * d
                + 4 * still * kv * d, "flops": flops + 6 * full * kv * page * d}
    if case["op"] == "read":
        return {"bytes": 2 * t * kv * d * (1 + 2) + meta, "flops": 2 * t * kv * d}
    pos, _ = _tokens(case)
    keys = sum((min(case["count"], p // page + 1) - 1) * page + p % page + 1 for p in pos)
    read, at = 0, 0
    for had, new in sequences(case):
        mine = sum((min(case["count"], p // page + 1) - 1) * page + p % page + 1
                   for p in pos[at:at + new])
        read += min(mine, had + new)
        at += new
    return {"bytes": 2 * t * h * d * 2 + t * h * 4 + t * kv * case["count"] * 4 + meta
            + read * kv * d * 2, "flops": keys * h * d * 4}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    h, kv, d, page, t, b = (case[x] for x in ("heads", "kv_heads", "dim", "page", "new", "seqs"))
    pos, seq = _tokens(case)
    had_new = sequences(case)
    s = {"op": case["op"], "page": page,
         "positions": torch.tensor(pos, dtype=torch.int32, device=DEV),
         "seq_ids": torch.tensor(seq, dtype=torch.int32, device=DEV)}
    # pages are taken from a shuffled pool, as a server that frees and reuses them has them
    need = [(a + n - 1) // page + 1 for a, n in had_new]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.full((b, max(need)), -1, dtype=torch.int32)
    first = 0
    for i, n in enumerate(need):
        table[i, :n] = order[first:first + n]
        first += n
    s["page_table"] = table.to(DEV)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)

    size = torch.exp(0.5 * normal(kv, 1, d))  # channels of unlike size, as a model's keys have them

    def rows(*shape):
        x = torch.empty(shape, dtype=dt, device=DEV)
        return x.normal_(generator=g)

    if case["op"] in ("append", "write"):
        # one projection's output, its queries, keys and values as views
        heads = rows(t, (h + 2 * kv) * d).view(t, h + 2 * kv, d)
        s["q"], s["k"], s["v"] = heads[:, :h], heads[:, h:h + kv], heads[:, h + kv:]
        s["interleaved"] = case["interleaved"]
        half = case["rot"] // 2
        freq = 10000.0 ** -(torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(max(pos) + 1, dtype=torch.float64)[:, None] * freq
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            s["q_weight"] = (1.0 + 0.2 * normal(d)).to(dt)
            s["k_weight"] = (1.0 + 0.2 * normal(d)).to(dt)
        s["bounds"] = torch.zeros((pool, kv, 2 * d), dtype=torch.int8, device=DEV)
        s["bound_scales"] = torch.zeros((pool, kv), device=DEV)
    if case["op"] == "append":
        s["k_cache"] = rows(pool, kv, page, d).mul_(size.to(dt))
        s["v_cache"] = rows(pool, kv, page, d)
        return s
    # codes as a block's quantisation leaves them: the largest near 127, a block in its own scale;
    # the block that a sequence has not filled has none (scales of 0) and lies in the open ones
    s["k_codes"] = torch.empty((pool, kv, page, d), dtype=torch.int8, device=DEV)
    s["v_codes"] = torch.empty((pool, kv, d, page), dtype=torch.int8, device=DEV)
    step = max(1, 2**27 // (kv * page * d))
    for i in range(0, pool, step):
        n = min(step, pool - i)
        x = normal(n, kv, page, d) * (size / size.amax() * 32.0)
        s["k_codes"][i:i + n] = x.round_().clamp_(-127, 127)
        s["v_codes"][i:i + n] = normal(n, kv, d, page).mul_(32.0).round_().clamp_(-127, 127)
    s["k_scales"] = (0.6 + 0.8 * torch.rand((pool, kv), generator=g, device=DEV)) * size.amax() / 32
    s["v_scales"] = (0.6 + 0.8 * torch.rand((pool, kv), generator=g, device=DEV)) / 32
    s["k_tail"] = rows(b, kv, page, d).mul_(size.to(dt))
    s["v_tail"] = rows(b, kv, d, page)
    for i, (had, new) in enumerate(had_new):
        end = had if case["op"] == "write" else had + new
        at = int(table[i, end // page]) if end % page else -1
        if at >= 0:
            s["k_scales"][at] = s["v_scales"][at] = 0.0
    if case["op"] != "attend":
        return s
    s["q"] = rows(t, h, d)
    # the choice: the forced blocks, the rest by scores that 32 neighbouring tokens mostly share
    n = max(need)
    last = (s["positions"] // page).long()[:, None, None]
    group = torch.arange(t, device=DEV) // 32
    score = normal(int(t + 31) // 32, kv, n)[group] + 0.5 * normal(t, kv, n)
    block = torch.arange(n, device=DEV)
    score = torch.where((block < 1) | (block > last - 2), math.inf, score)
    score = torch.where(block > last, -math.inf, score)
    best, at = score.topk(min(case["count"], n), dim=-1)
    at = torch.where(best == -math.inf, n, at).sort(-1).values
    blocks = torch.full((t, kv, case["count"]), -1, dtype=torch.int32, device=DEV)
    blocks[..., :at.shape[-1]] = torch.where(at == n, -1, at)
    s["blocks"] = blocks
    return s


# --- one pass ---------------------------------------------------------------------------------

CACHE = ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail")


def run(s):
    if own:
        from retrieve_amd import kv

        if s["op"] == "append":
            q = kv.append(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["seq_ids"],
                          s["page_table"], s["k_cache"], s["v_cache"], s["bounds"],
                          s["bound_scales"], s["interleaved"], s["q_weight"], s["k_weight"], EPS)
        elif s["op"] == "write":
            q = kv.append_int8(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["seq_ids"],
                               s["page_table"], *(s[x] for x in CACHE), s["bounds"],
                               s["bound_scales"], s["interleaved"], s["q_weight"], s["k_weight"],
                               EPS)
        elif s["op"] == "read":
            return kv.read_int8(*(s[x] for x in CACHE), s["positions"], s["seq_ids"],
                                s["page_table"])
        else:
            return kv.block_attention_int8(s["q"], *(s[x] for x in CACHE), s["blocks"],
                                           s["positions"], s["seq_ids"], s["page_table"])
    elif s["op"] == "append":
        q = plain_append(s)
    elif s["op"] == "write":
        q = plain_write(s)
    elif s["op"] == "read":
        return plain_read(s)
    else:
        return plain_attend(s)
    # the codes as the values they stand for, in the keys' type
    dt = q.dtype
    bounds = s["bounds"] * s["bound_scales"].to(dt)[..., None]
    if s["op"] == "append":
        return q, s["k_cache"], s["v_cache"], bounds
    return (q, s["k_codes"] * s["k_scales"].to(dt)[..., None, None],
            s["v_codes"] * s["v_scales"].to(dt)[..., None, None], s["k_tail"], s["v_tail"], bounds)


# --- the plain forms ----------------------------------------------------------------------------


def plain_quantize(x):
    """Codes of rows (the last channels), and their scales."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    codes = torch.round(x / top * 127.0).to(torch.int8)
    return codes, (top / torch.full_like(top, 127.0))[..., 0]


def plain_codes(x):
    """Codes of blocks (the last two dimensions), and their scales: ``127 x`` holds all of a 16-bit
    number in 32 bits, so a quotient halfway between two codes is seen as that."""
    top = x.abs().amax((-2, -1), keepdim=True).clamp(min=1e-8)
    codes = torch.round(x * 127.0 / top).to(torch.int8)
    return codes, (top / torch.full_like(top, 127.0))[..., 0, 0]


def plain_turn(x, weight, cos_sin, interleaved):
    """The heads' norm (its sum in 64 bits, the rest rounded step by step), then the rotation."""
    dt = x.dtype
    if weight is not None:
        r = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)
        x = x.float() * r.float() * weight.float()
    half = cos_sin.shape[-1] // 2
    x, c, n = x.float(), cos_sin[:, None, :half], cos_sin[:, None, half:]
    a = x[..., 0:2 * half:2] if interleaved else x[..., :half]
    b = x[..., 1:2 * half:2] if interleaved else x[..., half:2 * half]
    ab = (a * c - b * n, b * c + a * n)
    turned = torch.stack(ab, -1).flatten(-2) if interleaved else torch.cat(ab, -1)
    return torch.cat([turned, x[..., 2 * half:]], -1).to(dt)


def plain_heads(s):
    rows = s["cos_sin"][s["positions"].long()]
    return [plain_turn(s[x], s[x + "_weight"], rows, s["interleaved"]) for x in ("q", "k")]


def plain_bounds(s, full, stored):
    """Bounds of the pages ``full`` from their keys ``[n, kv, page, d]``."""
    low, high = stored.amin(2), stored.amax(2)
    row = torch.cat([(low + high) * 0.5, (high - low) * 0.5], -1)
    s["bounds"][full], s["bound_scales"][full] = plain_quantize(row)


def plain_append(s):
    page = s["page"]
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    q, k = plain_heads(s)
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    head = torch.arange(k.shape[1], device=k.device)
    s["k_cache"][at[:, None], head, slot[:, None]] = k
    s["v_cache"][at[:, None], head, slot[:, None]] = s["v"]
    full = at[slot == page - 1]
    plain_bounds(s, full, s["k_cache"][full].float())
    return q


def plain_write(s):
    page, dt = s["page"], s["q"].dtype
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    t = len(pos)
    q, k = plain_heads(s)
    v = s["v"]
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    # blocks that a token of this call completes: their tokens of this call, the rest as held so far
    end = torch.nonzero(slot == page - 1)[:, 0]
    row = end[:, None] - (page - 1) + torch.arange(page, device=pos.device)
    back = row.clamp(min=0)
    here = (row >= 0) & (seq[back] == seq[end][:, None]) & (
        pos[back] - pos[end][:, None] == row - end[:, None])
    full = at[end]

    def block(new, codes, scales, tail):  # [n, kv, page, d]
        held = s[codes][full].float() * s[scales][full][..., None, None]
        held = torch.where((s[scales][full] > 0)[..., None, None], held.to(dt), s[tail][seq[end]])
        held = held.transpose(2, 3) if codes == "v_codes" else held
        return torch.where(here[:, None, :, None], new[back].transpose(1, 2), held).float()

    kb, vb = block(k, "k_codes", "k_scales", "k_tail"), block(v, "v_codes", "v_scales", "v_tail")
    # the rest stays open
    to = torch.arange(t, device=pos.device) + (page - 1 - slot)
    there = to.clamp(max=t - 1)
    still = ~((to < t) & (seq[there] == seq) & (pos[there] - pos == page - 1 - slot))
    keep = torch.nonzero(still)[:, 0]
    head = torch.arange(k.shape[1], device=k.device)
    s["k_tail"][seq[keep][:, None], head, slot[keep][:, None]] = k[keep]
    s["v_tail"][seq[keep][:, None], head, :, slot[keep][:, None]] = v[keep]
    s["k_scales"][at[keep]] = 0.0
    s["v_scales"][at[keep]] = 0.0
    s["k_codes"][full], s["k_scales"][full] = plain_codes(kb)
    codes, s["v_scales"][full] = plain_codes(vb)
    s["v_codes"][full] = codes.transpose(2, 3)
    plain_bounds(s, full, kb)
    return q


def plain_read(s):
    page, dt = s["page"], s["k_tail"].dtype
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    at, slot = s["page_table"][seq, pos // page].long()[:, None], (pos % page)[:, None]
    head = torch.arange(s["k_codes"].shape[1], device=pos.device)
    out = []
    for codes, scales, tail, rows in ((s["k_codes"], s["k_scales"], s["k_tail"], (at, head, slot)),
                                      (s["v_codes"], s["v_scales"], s["v_tail"],
                                       (at, head, slice(None), slot))):
        scale = scales[at, head][..., None]
        value = (codes[rows].float() * scale).to(dt)
        out.append(torch.where(scale > 0, value, tail[(seq[:, None], *rows[1:])]))
    return out


def plain_attend(s):
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    t, h, d = s["q"].shape
    kv, page = s["k_codes"].shape[1:3]
    blocks = s["blocks"].long()
    at = s["page_table"].long()[seq[:, None, None], blocks.clamp(min=0)]
    head = torch.arange(kv, device=pos.device)[None, :, None]
    last = (pos // page)[:, None, None]
    open_ = (s["k_scales"][at, head] == 0.0)[..., None, None]

    def values(codes, scales, tail):
        x = s[codes][at, head].float() * s[scales][at, head][..., None, None]
        return torch.where(open_, s[tail][seq][:, :, None].float(), x)

    q = s["q"].float().view(t, kv, -1, d)
    k = values("k_codes", "k_scales", "k_tail").view(t, kv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    where = blocks[..., None] * page + torch.arange(page, device=pos.device)
    seen = ((blocks >= 0)[..., None] & (where <= pos[:, None, None, None]))
    seen &= ~open_[..., 0] | (blocks == last)[..., None]
    score = torch.where(seen.view(t, kv, 1, -1), score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    v = values("v_codes", "v_scales", "v_tail").transpose(3, 4).reshape(t, kv, -1, d)
    out = torch.matmul(weight / total, v)
    return out.reshape(t, h, d).to(s["q"].dtype), (top + torch.log(total)).reshape(t, h)


# --- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return exact_append(s)
    if case["op"] == "write":
        return exact_write(s)
    return exact_read(s) if case["op"] == "read" else exact_attend(s)


def exact_turn(s):
    """Norms, then the rotation as a complex product."""
    half = s["cos_sin"].shape[1] // 2
    turn = torch.complex(*s["cos_sin"].double()[s["positions"].long()].split(half, 1))[:, None]
    out = []
    for name in ("q", "k"):
        x = s[name].double()
        if s[name + "_weight"] is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s[name + "_weight"].double()
        pair = x[..., :2 * half]
        pair = (pair.unflatten(-1, (half, 2)) if s["interleaved"]
                else pair.unflatten(-1, (2, half)).transpose(-1, -2))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
        out.append(torch.cat([z, x[..., 2 * half:]], -1))
    return out


def exact_codes(x):
    """What is left of a block after its quantisation."""
    top = x.abs().flatten(1).amax(1).clamp(min=1e-8).view(-1, *[1] * (x.dim() - 1))
    return torch.round(x * 127 / top) * top / 127


def exact_bound(stored):
    """The bounds of a block's keys ``[kv, page, d]``."""
    top, low = stored.max(1).values, stored.min(1).values
    return exact_codes(torch.cat([(top + low) / 2, (top - low) / 2], 1))


def exact_append(s):
    dt, page = s["q"].dtype, s["page"]
    pos = s["positions"].long()
    q, k = exact_turn(s)
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    bound = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
    at = s["page_table"].long()[s["seq_ids"].long(), pos // page]
    kc.transpose(1, 2)[at, pos % page] = k
    vc.transpose(1, 2)[at, pos % page] = s["v"].double()
    for i in at[pos % page == page - 1].tolist():
        bound[i] = exact_bound(kc[i].to(dt).double())
    return q, kc, vc, bound


def exact_write(s):
    """Block by block: what a sequence holds of it, then the new tokens; codes once it is full."""
    dt, page = s["q"].dtype, s["page"]
    q, k = exact_turn(s)
    kc = s["k_codes"].double() * s["k_scales"].double()[..., None, None]
    vc = s["v_codes"].double() * s["v_scales"].double()[..., None, None]
    kt, vt = s["k_tail"].double(), s["v_tail"].double()
    bound = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
    table, v = s["page_table"].tolist(), s["v"].double()
    pos, seq = s["positions"].tolist(), s["seq_ids"].tolist()
    t = 0
    while t < len(pos):
        i, first = seq[t], pos[t] % page
        end = t
        while end < len(pos) and seq[end] == i and pos[end] // page == pos[t] // page:
            end += 1
        n, at = end - t, table[i][pos[t] // page]
        kb, vb = kt[i].clone(), vt[i].clone()
        kb[:, first:first + n] = k[t:end].transpose(0, 1)
        vb[:, :, first:first + n] = v[t:end].permute(1, 2, 0)
        if first + n == page:
            stored = kb.to(dt).double()
            kc[at], vc[at], bound[at] = exact_codes(stored), exact_codes(vb), exact_bound(stored)
        else:
            kt[i], vt[i], kc[at], vc[at] = kb, vb, 0.0, 0.0
        t = end
    return q, kc, vc, kt, vt, bound


def exact_read(s):
    page = s["page"]
    b, n = s["page_table"].shape
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    kv, d = s["k_codes"].shape[1], s["k_codes"].shape[3]
    k = torch.empty((len(pos), kv, d), dtype=torch.float64, device=DEV)
    v = torch.empty_like(k)
    for i in range(b):  # a sequence's blocks in a row
        mine = torch.nonzero(seq == i)[:, 0]
        where = pos[mine]
        blocks = s["page_table"][i][:int(where.max()) // page + 1].long()
        ks, vs = (s[x][blocks].double()[..., None, None] for x in ("k_scales", "v_scales"))
        kb = torch.where(ks > 0, s["k_codes"][blocks].double() * ks, s["k_tail"][i].double())
        vb = torch.where(vs > 0, s["v_codes"][blocks].double() * vs, s["v_tail"][i].double())
        k[mine] = kb.permute(0, 2, 1, 3).reshape(-1, kv, d)[where]
        v[mine] = vb.permute(0, 3, 1, 2).reshape(-1, kv, d)[where]
    return [k, v]


def exact_attend(s):
    """Some tokens at a time, softmax over the gathered keys in 64 bits."""
    t, h, d = s["q"].shape
    kv, page = s["k_codes"].shape[1:3]
    out = torch.empty((t, h, d), dtype=torch.float64, device=DEV)
    lse = torch.empty((t, h), dtype=torch.float64, device=DEV)
    step = max(1, 2**27 // (kv * s["blocks"].shape[2] * page * d))
    for i in range(0, t, step):
        m = slice(i, min(t, i + step))
        b = s["blocks"][m].long()
        p = s["positions"][m].long()
        sq = s["seq_ids"][m].long()
        phys = torch.gather(s["page_table"].long()[sq], 1, b.clamp(min=0).flatten(1)).view_as(b)
        flat = phys * kv + torch.arange(kv, device=DEV)[None, :, None]
        ks = s["k_scales"].flatten()[flat].double()[..., None, None]
        vs = s["v_scales"].flatten()[flat].double()[..., None, None]
        held = ks > 0
        k = s["k_codes"].flatten(0, 1)[flat].double() * ks  # [m, kv, n, page, d]
        k = torch.where(held, k, s["k_tail"][sq].double()[:, :, None])
        v = s["v_codes"].flatten(0, 1)[flat].double() * vs  # [m, kv, n, d, page]
        v = torch.where(held, v, s["v_tail"][sq].double()[:, :, None]).transpose(3, 4)
        q = s["q"][m].double().view(-1, kv, h // kv, d) / d**0.5
        x = torch.matmul(q, k.flatten(2, 3).transpose(2, 3))
        gone = (b < 0)[..., None] | (b[..., None] * page + torch.arange(page, device=DEV)
                                     > p[:, None, None, None])
        gone |= ~held[..., 0] & (b != (p // page)[:, None, None])[..., None]
        x.masked_fill_(gone.flatten(2)[:, :, None], -math.inf)
        lse[m] = torch.logsumexp(x, -1).flatten(1)
        out[m] = torch.matmul(torch.softmax(x, -1), v.reshape(*v.shape[:2], -1, d)).flatten(1, 2)
    return out, lse

"""Timed cases of the long-context cache: append with rotation, block selection, attention over blocks.

A language model served at long contexts keeps its keys and values in pages; each step it appends the
new tokens (rotated), scores every block's int8 bounds against the query, keeps the best blocks and
attends to those only. The cases are single calls of ``retrieve_amd.kv``'s three operators:

- ``append``: queries, keys and values of new tokens rotated, keys and values written to their pages,
  the bounds of the blocks that become full;
- ``select``: the best blocks of each token and key/value head by the bounds' score;
- ``attend``: softmax attention over chosen blocks.

Where ``own`` is false each is computed from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# --- the cases --------------------------------------------------------------------------------


def listed():
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 64}
    mha = {"heads": 14, "kv_heads": 14, "dim": 64, "page": 16}
    return [
        # one user's next token: launch latency
        {"name": "append_decode_b1", "op": "append", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 1000, "high": 1000, "rot": 128, "interleaved": False, "factor": 1.0},
        # a large decode batch of short ragged contexts, small pages, half of each head rotated
        {"name": "append_decode_b203", "op": "append", "dtype": "fp16", **mha, "seqs": 203,
         "new": 203, "low": 3, "high": 300, "rot": 32, "interleaved": True, "factor": 1.0},
        # ragged prompts over existing contexts, positions scaled for a longer range
        {"name": "append_prompt_9k", "op": "append", "dtype": "bf16", **gqa, "seqs": 3,
         "new": 9001, "low": 0, "high": 4099, "rot": 128, "interleaved": False, "factor": 8.0},
        # the largest prompt batch, wide heads and pages
        {"name": "append_prompt_32k_d256", "op": "append", "dtype": "fp16", "heads": 16,
         "kv_heads": 8, "dim": 256, "page": 128, "seqs": 8, "new": 32768, "low": 0, "high": 2000,
         "rot": 256, "interleaved": True, "factor": 4.0},
        # one user over a million tokens
        {"name": "select_decode_b1_1m", "op": "select", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 1000003, "high": 1000003, "count": 64, "sink": 1, "recent": 2},
        # a small decode batch over short contexts in small pages, no shared heads
        {"name": "select_decode_b7", "op": "select", "dtype": "fp16", **mha, "seqs": 7, "new": 7,
         "low": 500, "high": 9000, "count": 64, "sink": 2, "recent": 4},
        # a serving batch over long ragged contexts
        {"name": "select_decode_b64_128k", "op": "select", "dtype": "bf16", **gqa, "seqs": 64,
         "new": 64, "low": 16000, "high": 131000, "count": 64, "sink": 1, "recent": 2},
        # chunks of two prompts behind long contexts
        {"name": "select_prompt_4k", "op": "select", "dtype": "bf16", **gqa, "seqs": 2, "new": 4099,
         "low": 9000, "high": 30000, "count": 32, "sink": 1, "recent": 2},
        # one user's next token over few blocks
        {"name": "attend_decode_b1", "op": "attend", "dtype": "bf16", **gqa, "seqs": 1, "new": 1,
         "low": 30001, "high": 30001, "count": 32, "sink": 1, "recent": 2},
        # many small blocks, no shared heads
        {"name": "attend_decode_b48_p16", "op": "attend", "dtype": "fp16", **mha, "seqs": 48,
         "new": 48, "low": 100, "high": 12000, "count": 96, "sink": 2, "recent": 4},
        # a serving batch over long ragged contexts: the cache's bytes
        {"name": "attend_decode_b64", "op": "attend", "dtype": "bf16", **gqa, "seqs": 64, "new": 64,
         "low": 2000, "high": 40000, "count": 64, "sink": 1, "recent": 2},
        # chunks of two prompts, neighbouring tokens' choices alike
        {"name": "attend_prompt_2k", "op": "attend", "dtype": "bf16", **gqa, "seqs": 2, "new": 2053,
         "low": 3000, "high": 14000, "count": 16, "sink": 1, "recent": 2},
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
    small = (64, 96, 128, 128, 256)
    heads, kv, dims = rng.choice([(32, 8, (128, 128, 256)), (20, 20, small), (28, 4, small),
                                  (18, 6, small), (10, 2, small), (8, 1, small), (40, 10, small),
                                  (5, 5, small)])
    c = {"op": rng.choice(["append", "select", "attend"]), "dtype": rng.choice(["bf16", "fp16"]),
         "heads": heads, "kv_heads": kv, "dim": rng.choice(dims),
         "page": rng.choice([16, 32, 64, 64, 128])}
    prompt = rng.random() < 0.4
    row = (heads + 2 * kv) * c["dim"]
    if c["op"] == "append":
        c["seqs"] = _spread(rng, 1, 8) if prompt else _spread(rng, 1, 256)
        most = max(c["seqs"], 32768 * 8192 // row)
        c["new"] = _spread(rng, c["seqs"], min(32768, most)) if prompt else c["seqs"]
        c["low"] = 0 if rng.random() < 0.3 else _spread(rng, 1, 300)
        c["high"] = c["low"] + rng.randrange(0, 4000 if prompt else 300)
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 32, 20])
        c["interleaved"] = rng.random() < 0.5
        c["factor"] = rng.choice([1.0, 2.0, 8.0])
        return c
    if c["op"] == "select":
        # the longest context has twice the blocks that are kept, or more: else nothing is chosen
        c["count"] = rng.choice([8, 16, 32, 64, 100])
        few = 2 * c["count"] * c["page"]
        if prompt:
            c["seqs"] = _spread(rng, 1, 3)
            c["high"] = few + rng.randrange(0, 24000 * c["page"] // 64)
            c["low"] = rng.randrange(1, c["high"])
            blocks = c["high"] // c["page"]
            most = 4099 * 32 * 300 // (heads * blocks)  # scores of the whole chunk
            c["new"] = _spread(rng, max(c["seqs"], 2), max(c["seqs"], 2, min(4099, most)))
        else:
            c["seqs"] = c["new"] = _spread(rng, 1, 64)
            most = 73000 * 8 * 256 // (c["seqs"] * kv * 2 * c["dim"])  # blocks a sequence
            c["high"] = _spread(rng, few, max(few, c["page"] * min(15000, most)))
            c["low"] = rng.randrange(c["high"] // 4, c["high"] + 1)
    else:
        c["count"] = rng.choice([4, 16, 32, 64, 96])
        keys = c["count"] * c["page"]
        if prompt:
            c["seqs"] = _spread(rng, 1, 3)
            most = 2053 * 1024 * 128 // (keys * c["dim"] * max(kv / 8, heads / 32))
            c["new"] = _spread(rng, max(c["seqs"], 2), max(c["seqs"], 2, min(2053, int(most))))
            c["low"] = 0 if rng.random() < 0.2 else _spread(rng, 1, 8000)
            c["high"] = c["low"] + rng.randrange(0, 6000)
        else:
            most = 64 * 8 * 4096 * 128 // (kv * keys * c["dim"])
            c["seqs"] = c["new"] = _spread(rng, 1, max(1, min(64, most)))
            c["low"] = _spread(rng, 1, 4000)
            c["high"] = c["low"] + rng.randrange(0, 20000)
    c["sink"] = rng.choice([0, 1, 2])
    c["recent"] = rng.choice([1, 2])
    return c


# --- what a case holds, from its plain values ----------------------------------------------------


def sequences(case):
    """(tokens already in the cache, new tokens) of each sequence: spread over the case's range, the
    first at its upper end, and shares of the new tokens that differ by up to a factor of two."""
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
    pos, _ = _tokens(case)
    meta = 8 * t
    if case["op"] == "append":
        full = sum((had + new) // page - had // page for had, new in sequences(case))
        before = sum(had % page for had, new in sequences(case) if had // page < (had + new) // page)
        moved = 2 * t * (h + 2 * kv) * d * 2 + t * case["rot"] * 4 + 4 * t
        return {"bytes": moved + full * kv * (2 * d + 4) + before * kv * d * 2 + meta,
                "flops": t * (h + kv) * case["rot"] * 3 + 2 * full * kv * page * d}
    free = case["sink"] + case["recent"]
    if case["op"] == "select":
        rows = sum(max(0, (had + new - 1) // page + 1 - free) for had, new in sequences(case))
        scored = sum(max(0, p // page + 1 - free) for p in pos)
        return {"bytes": t * h * d * 2 + rows * (kv * (2 * d + 4) + 4) + t * kv * case["count"] * 4
                + meta, "flops": scored * h * 4 * d}
    keys = sum((min(case["count"], p // page + 1) - 1) * page + p % page + 1 for p in pos)
    read, at = 0, 0
    for had, new in sequences(case):
        mine = sum((min(case["count"], p // page + 1) - 1) * page + p % page + 1
                   for p in pos[at:at + new])
        read += min(mine, had + new)
        at += new
    return {"bytes": 2 * t * h * d * 2 + t * h * 4 + t * kv * case["count"] * 4 + meta
            + read * kv * d * 4, "flops": keys * h * d * 4}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    h, kv, d, page, t, b = (case[x] for x in ("heads", "kv_heads", "dim", "page", "new", "seqs"))
    pos, seq = _tokens(case)
    had_new = sequences(case)
    s = {"op": case["op"], "page": page, "longest": max(n for _, n in had_new),
         "positions": torch.tensor(pos, dtype=torch.int32, device=DEV),
         "seq_ids": torch.tensor(seq, dtype=torch.int32, device=DEV)}
    # pages are taken from a shuffled pool, as a server that frees and reuses them has them
    need = [(a + n - 1) // page + 1 for a, n in had_new]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, max(need)), -1, dtype=torch.int32)
    first, fill = 0, []
    for i, n in enumerate(need):
        fill.append((i, first, n))
        first += n
    order_host = order.cpu()
    for i, at, n in fill:
        table[i, :n] = order_host[at:at + n]
    s["page_table"] = table.to(DEV)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)

    def keys(*shape):  # channels of unlike size, as a model's keys have them
        size = torch.exp(0.5 * normal(kv, 1, d))
        x = torch.empty(shape, dtype=dt, device=DEV)
        x.normal_(generator=g)
        return x.mul_(size.to(dt))

    if case["op"] == "append":
        # one projection's output, its queries, keys and values as views
        qkv = (normal(t, (h + 2 * kv) * d)).to(dt)
        heads = qkv.view(t, h + 2 * kv, d)
        s["q"], s["k"], s["v"] = heads[:, :h], heads[:, h:h + kv], heads[:, h + kv:]
        s["interleaved"] = case["interleaved"]
        half = case["rot"] // 2
        freq = 10000.0 ** -(torch.arange(half, dtype=torch.float64) / half) / case["factor"]
        angle = torch.arange(max(pos) + 1, dtype=torch.float64)[:, None] * freq
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float().to(DEV)
        s["k_cache"], s["v_cache"] = keys(pool, kv, page, d), keys(pool, kv, page, d)
        s["bounds"] = torch.zeros((pool, kv, 2 * d), dtype=torch.int8, device=DEV)
        s["bound_scales"] = torch.zeros((pool, kv), device=DEV)
        return s
    s["q"] = normal(t, h, d).to(dt)
    if case["op"] == "select":
        # blocks' centres and half widths, quantised as append leaves them
        size = torch.exp(0.5 * normal(kv, d))
        mid = 0.5 * size * normal(pool, kv, d)
        half = size * (1.0 + 1.5 * torch.rand((pool, kv, d), generator=g, device=DEV))
        s["bounds"], s["bound_scales"] = plain_quantize(torch.cat([mid, half], -1))
        s.update(count=case["count"], sink=case["sink"], recent=case["recent"])
        return s
    s["k_cache"], s["v_cache"] = keys(pool, kv, page, d), keys(pool, kv, page, d)
    # the choice: the forced blocks, the rest by scores that 32 neighbouring tokens mostly share
    n = max(need)
    last = (s["positions"] // page).long()[:, None, None]
    group = torch.arange(t, device=DEV) // 32
    score = normal(int(t + 31) // 32, kv, n)[group] + 0.5 * normal(t, kv, n)
    block = torch.arange(n, device=DEV)
    score = torch.where((block < case["sink"]) | (block > last - case["recent"]), math.inf, score)
    score = torch.where(block > last, -math.inf, score)
    best, at = score.topk(min(case["count"], n), dim=-1)
    at = torch.where(best == -math.inf, n, at).sort(-1).values
    blocks = torch.full((t, kv, case["count"]), -1, dtype=torch.int32, device=DEV)
    blocks[..., :at.shape[-1]] = torch.where(at == n, -1, at)
    s["blocks"] = blocks
    return s


# --- one pass ---------------------------------------------------------------------------------


def run(s):
    if own:
        from retrieve_amd import kv

        if s["op"] == "append":
            q = kv.append(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["seq_ids"],
                          s["page_table"], s["k_cache"], s["v_cache"], s["bounds"],
                          s["bound_scales"], s["interleaved"])
        elif s["op"] == "select":
            return kv.select_blocks(s["q"], s["bounds"], s["bound_scales"], s["positions"],
                                    s["seq_ids"], s["page_table"], s["page"], s["count"],
                                    s["sink"], s["recent"])
        else:
            return kv.block_attention(s["q"], s["k_cache"], s["v_cache"], s["blocks"],
                                      s["positions"], s["seq_ids"], s["page_table"])
    elif s["op"] == "append":
        q = plain_append(s)
    elif s["op"] == "select":
        return plain_select(s)
    else:
        return plain_attend(s)
    # the bounds as the values their codes stand for
    return q, s["k_cache"], s["v_cache"], s["bounds"] * s["bound_scales"][..., None]


# --- the plain forms ----------------------------------------------------------------------------


def plain_quantize(x):
    """Rows of int8 codes and their scales."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=1e-8)
    codes = torch.round(x / top * 127.0).clamp(-128, 127).to(torch.int8)
    return codes, (top / torch.full_like(top, 127.0))[..., 0]


def plain_rotate(x, cos_sin, interleaved):
    half = cos_sin.shape[-1] // 2
    x, c, n = x.float(), cos_sin[:, None, :half], cos_sin[:, None, half:]
    a = x[..., 0:2 * half:2] if interleaved else x[..., :half]
    b = x[..., 1:2 * half:2] if interleaved else x[..., half:2 * half]
    ab = (a * c - b * n, b * c + a * n)
    turned = torch.stack(ab, -1).flatten(-2) if interleaved else torch.cat(ab, -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def plain_append(s):
    dt, page = s["q"].dtype, s["page"]
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    rows = s["cos_sin"][pos]
    q = plain_rotate(s["q"], rows, s["interleaved"]).to(dt)
    k = plain_rotate(s["k"], rows, s["interleaved"]).to(dt)
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    head = torch.arange(k.shape[1], device=k.device)
    s["k_cache"][at[:, None], head, slot[:, None]] = k
    s["v_cache"][at[:, None], head, slot[:, None]] = s["v"]
    full = at[slot == page - 1]
    stored = s["k_cache"][full].float()
    low, high = stored.amin(2), stored.amax(2)
    codes, scales = plain_quantize(torch.cat([(low + high) * 0.5, (high - low) * 0.5], -1))
    s["bounds"][full], s["bound_scales"][full] = codes, scales
    return q


def plain_select(s):
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    table = s["page_table"].long()
    t, h, d = s["q"].shape
    b, n = table.shape
    kv = s["bounds"].shape[1]
    codes, scale = plain_quantize(s["q"].float())
    codes = codes.float()
    both = torch.cat([codes, codes.abs()], -1)
    # tokens by sequence, so that a sequence's bounds are gathered once
    start = torch.searchsorted(s["seq_ids"], torch.arange(b, device=pos.device, dtype=torch.int32))
    slot = torch.arange(t, device=pos.device) - start[seq]
    padded = both.new_zeros((b, s["longest"], h, 2 * d))
    padded[seq, slot] = both
    left = padded.view(b, s["longest"], kv, -1, 2 * d).transpose(1, 2).reshape(b, kv, -1, 2 * d)
    at = table.clamp(min=0)
    right = s["bounds"][at].float().permute(0, 2, 3, 1).contiguous()  # [b, kv, 2d, n]
    dots = torch.matmul(left, right).view(b, kv, s["longest"], -1, n)  # whole numbers below 2^24
    dots = dots.transpose(1, 2)[seq, slot]  # [t, kv, g, n]
    score = (dots * scale.view(t, kv, -1, 1)).amax(2)
    score = score * s["bound_scales"][at].transpose(1, 2)[seq]
    block = torch.arange(n, device=pos.device)
    last = (pos // s["page"])[:, None, None]
    score = torch.where((block < s["sink"]) | (block > last - s["recent"]), math.inf, score)
    score = torch.where(block > last, -math.inf, score)
    score, order = torch.sort(score, dim=-1, descending=True, stable=True)
    chosen = torch.where(score == -math.inf, n, order)[..., :s["count"]].sort(-1).values
    out = torch.full((t, kv, s["count"]), -1, dtype=torch.int32, device=pos.device)
    out[..., :chosen.shape[-1]] = torch.where(chosen == n, -1, chosen)
    return out


def plain_attend(s):
    pos, seq = s["positions"].long(), s["seq_ids"].long()
    t, h, d = s["q"].shape
    kv, page = s["k_cache"].shape[1:3]
    blocks = s["blocks"].long()
    at = s["page_table"].long()[seq[:, None, None], blocks.clamp(min=0)]
    head = torch.arange(kv, device=pos.device)[None, :, None]
    q = s["q"].float().view(t, kv, -1, d)
    k = s["k_cache"][at, head].float().view(t, kv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    where = blocks[..., None] * page + torch.arange(page, device=pos.device)
    seen = ((blocks >= 0)[..., None] & (where <= pos[:, None, None, None])).view(t, kv, 1, -1)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    v = s["v_cache"][at, head].float().view(t, kv, -1, d)
    out = torch.matmul(weight / total, v)
    return out.reshape(t, h, d).to(s["q"].dtype), (top + torch.log(total)).reshape(t, h)


# --- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    return exact_append(s) if case["op"] == "append" else exact_attend(s)


def exact_append(s):
    """The rotation as a complex product; caches of 64-bit keys; bounds from the keys as stored."""
    dt, page = s["q"].dtype, s["page"]
    pos = s["positions"].long()
    half = s["cos_sin"].shape[1] // 2
    turn = torch.complex(*s["cos_sin"].double()[pos].split(half, 1))[:, None]

    def rotate(x):
        x = x.double()
        pair = x[..., :2 * half]
        pair = (pair.unflatten(-1, (half, 2)) if s["interleaved"]
                else pair.unflatten(-1, (2, half)).transpose(-1, -2))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, x[..., 2 * half:]], -1)

    q, k = rotate(s["q"]), rotate(s["k"])
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    bound = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
    at = s["page_table"].long()[s["seq_ids"].long(), pos // page]
    kc.transpose(1, 2)[at, pos % page] = k
    vc.transpose(1, 2)[at, pos % page] = s["v"].double()
    for i in at[pos % page == page - 1].tolist():
        stored = kc[i].to(dt).double()
        top, low = stored.max(1).values, stored.min(1).values
        row = torch.cat([(top + low) / 2, (top - low) / 2], 1)
        step = row.abs().max(1, keepdim=True).values.clamp(min=1e-8) / 127
        bound[i] = torch.round(row / step) * step
    return q, kc, vc, bound


def exact_attend(s):
    """Some tokens at a time, softmax over the gathered keys in 64 bits."""
    t, h, d = s["q"].shape
    kv, page = s["k_cache"].shape[1:3]
    out = torch.empty((t, h, d), dtype=torch.float64, device=DEV)
    lse = torch.empty((t, h), dtype=torch.float64, device=DEV)
    step = max(1, 2**28 // (kv * s["blocks"].shape[2] * page * d))
    for i in range(0, t, step):
        m = slice(i, min(t, i + step))
        b = s["blocks"][m].long()
        p = s["positions"][m].long()
        phys = torch.gather(s["page_table"].long()[s["seq_ids"][m].long()], 1,
                            b.clamp(min=0).flatten(1)).view_as(b)
        flat = phys * kv + torch.arange(kv, device=DEV)[None, :, None]
        k = s["k_cache"].flatten(0, 1)[flat].double()  # [m, kv, n, page, d]
        v = s["v_cache"].flatten(0, 1)[flat].double()
        q = s["q"][m].double().view(-1, kv, h // kv, d) / d**0.5
        x = torch.matmul(q, k.flatten(2, 3).transpose(2, 3))
        gone = (b < 0)[..., None] | (b[..., None] * page + torch.arange(page, device=DEV)
                                     > p[:, None, None, None])
        x.masked_fill_(gone.flatten(2)[:, :, None], -math.inf)
        lse[m] = torch.logsumexp(x, -1).flatten(1)
        out[m] = torch.matmul(torch.softmax(x, -1), v.flatten(2, 3)).flatten(1, 2)
    return out, lse

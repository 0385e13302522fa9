"""The 8-bit paged cache as a layer uses it: prompts and single tokens through all the calls together,
beside the 16-bit cache, captured, on another stream."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from oracle import kv_int8 as o8
from tests.kv_cases import KINDS, back, normal16, to
from tests.kv_int8_cases import NAMES, check_attention, same, weights

LENS = (260, 131)


def _cache(dev, kind, heads_kv, d, page, pages=80, sequences=2, max_pages=40):
    import torch

    from retrieve_amd import kv

    return kv.Int8PagedCache(pages, heads_kv, d, page, sequences, max_pages,
                             getattr(torch, KINDS[kind]), dev)


def _mirror(cache, kind):
    """The oracle's cache with the same contents."""
    c = o8.Cache(0, cache.k_codes.shape[0], cache.k_codes.shape[1], cache.page,
                 cache.k_codes.shape[3], cache.k_tail.shape[0], kind)
    for n, x in zip(NAMES, cache._tensors):
        setattr(c, n, back(x))
    c.bounds, c.bound_scales = back(cache.bounds), back(cache.bound_scales)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,normed",
                         [("bf16", 8, 2, 64, 16, True), ("fp16", 6, 1, 128, 64, False)])
def test_prompt_then_tokens(dev, kind, heads, heads_kv, d, page, normed):
    """Prompts in chunks, then decode steps, over pages that start as anything: every step held to
    the oracle on the oracle's own cache (what is held bit for bit, chosen blocks equal, outputs
    within the attention's tolerance), what is read back at the end as well. Sequence 1 is then cut
    back and goes on, sequence 0's pages are freed and taken by a new one."""
    from retrieve_amd import kv

    cache = _cache(dev, kind, heads_kv, d, page)
    cache.bound_scales.fill_(float("nan"))
    cache.k_tail.fill_(float("nan"))
    cache.v_tail.fill_(float("inf"))
    cs = kv.rotary_table(500, d, device=dev)
    angles = back(cs)
    c = _mirror(cache, kind)
    w = weights(40, d, kind) if normed else (None, None)
    gw = [None if x is None else to(dev, x, kind) for x in w]
    x = [normal16(200 + i, (500, heads + 2 * heads_kv, d), kind) for i in range(2)]
    at = [0, 0]

    def step(new, attend=True):
        rows, pos, seq = [], [], []
        for s, n in enumerate(new):
            cache.reserve(s, at[s] + n)
            rows.append(x[s][at[s]:at[s] + n])
            pos += range(at[s], at[s] + n)
            seq += [s] * n
            at[s] += n
        rows, pos, seq = np.concatenate(rows), np.array(pos, np.int32), np.array(seq, np.int32)
        tab = back(cache.page_table)
        g, gp, gs = to(dev, rows, kind), to(dev, pos), to(dev, seq)
        q = cache.append(g[:, :heads], g[:, heads:heads + heads_kv], g[:, heads + heads_kv:], cs, gp,
                         gs, False, *gw)
        want_q = c.append(rows[:, :heads], rows[:, heads:heads + heads_kv], rows[:, heads + heads_kv:],
                          angles, pos, seq, tab, False, *w)
        assert np.array_equal(back(q), want_q)
        same((cache._tensors, (cache.bounds, cache.bound_scales)), c)
        if not attend:
            return
        blocks = cache.select(q, gp, gs, 6, 1, 2)
        want = okv.select(want_q, c.bounds, c.bound_scales, pos, seq, tab, page, 6, 1, 2)
        assert np.array_equal(back(blocks), want)
        got = cache.attend(q, gp, gs, 6, 1, 2)
        check_attention([back(y) for y in got], c, want_q, want, pos, seq, tab)

    print(f"{kind} {heads}/{heads_kv} d={d} page={page}", flush=True)
    for new in [(200, 131), (60, 0)]:
        step(new, False)
    for new in [(1, 1)] * 20 + [(17, 0), (0, 13)]:
        step(new)
    pos = np.concatenate([np.arange(n) for n in at]).astype(np.int32)
    seq = np.repeat([0, 1], at).astype(np.int32)
    for got, want in zip(cache.read(to(dev, pos), to(dev, seq)),
                         c.read(pos, seq, back(cache.page_table))):
        assert np.array_equal(back(got), want)
    at[1] -= 2 * page + 3
    step((1, 1))
    cache.free(0)
    at[0] = 0
    step((page + 5, 1))
    step((1, 1))


@pytest.mark.gpu
def test_beside_the_cache_in_16_bits(dev):
    """The same layer over both caches, every block kept: each key and value is off by half a code's
    step at most (``top / 254`` of its block, 1/254 + 2^-9 of the largest), so a score by ``|q| . 1``
    times the keys' part of it, ``e``, and an output by ``exp(2 e) - 1`` of the weighted values' sizes
    plus the values' part. The bounds are the same bits; so are results while all tokens are in the
    open block but for the weights' rounding."""
    import torch

    from retrieve_amd import kv

    heads, heads_kv, d, page = 8, 2, 64, 16
    small = _cache(dev, "fp16", heads_kv, d, page)
    plain = kv.PagedCache(80, heads_kv, d, page, 2, 40, torch.float16, dev)
    rows = normal16(7, (sum(LENS), heads + 2 * heads_kv, d), "fp16")
    g = to(dev, rows, "fp16")
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device=dev) for n in LENS])
    seq = torch.repeat_interleave(torch.arange(2, dtype=torch.int32, device=dev),
                                  torch.tensor(LENS, device=dev)).int()
    cs = kv.rotary_table(400, d, device=dev)
    results = []
    for cache in (plain, small):
        for s, n in enumerate(LENS):
            cache.reserve(s, n)
        q = cache.append(g[:, :8], g[:, 8:10], g[:, 10:], cs, pos, seq)
        results.append([back(y) for y in (q, *cache.attend(q, pos, seq, 17, scale=0.125))])
    (q, out, lse), (q8, out8, lse8) = results
    assert np.array_equal(q, q8)
    full = [p for s, n in enumerate(LENS) for p in back(plain.page_table)[s][:n // page]]
    assert np.array_equal(back(plain.bounds)[full], back(small.bounds)[full])
    assert np.array_equal(back(plain.bound_scales)[full], back(small.bound_scales)[full])
    held = [np.nan_to_num(back(x)[full]) for x in (plain.k, plain.v)]
    top_k, top_v = (np.abs(x).max() for x in held)
    half = 1 / 254 + 2.0**-22
    e = np.abs(q).sum(-1, dtype=np.float64) * 0.125 * top_k * half + 2.0**-12
    assert (np.abs(lse - lse8) <= e).all()
    most = max(top_v, np.abs(rows[:, 10:]).max())
    # (and what either call rounds: weights to 16 bits, once, and the output)
    off = (np.exp(2 * e)[..., None] - 1 + 2 * 2.0**-11) * most + top_v * half
    off += 2 * 2.0**-11 * most
    assert (np.abs(out - out8) <= off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sequences,blocks,more", [(1, 300, 1), (2, 12, 1), (1, 60, 700)])
def test_graph_replays(dev, sequences, blocks, more):
    """Captured steps (single tokens over a split list and without; a prompt, whose workgroups join
    their lists), replayed with new inputs between eager work, and a second graph of the same cache in
    turn with the first: each replay gives what an eager step gives, over the same cache."""
    import torch

    from retrieve_amd import kv

    page, heads, heads_kv, d = 16, 8, 2, 64
    width = blocks + 2 + (more + page - 1) // page
    cache = kv.Int8PagedCache(sequences * width, heads_kv, d, page, sequences, width, device=dev)
    cs = kv.rotary_table(page * width, d, device=dev)
    for x in (cache.k_tail, cache.v_tail):
        x.zero_()  # (NaN would be unlike itself below)
    g = torch.Generator(device=dev).manual_seed(3)
    n = page * blocks - 3
    for s in range(sequences):
        cache.reserve(s, page * width)
        x = torch.randn((n, 12, d), generator=g, device=dev).to(torch.bfloat16)
        pos = torch.arange(n, dtype=torch.int32, device=dev)
        cache.append(x[:, :8], x[:, 8:10], x[:, 10:], cs, pos, torch.full_like(pos, s))
    start = [y.clone() for y in (*cache._tensors, cache.bounds, cache.bound_scales)]

    def graph_of(new):
        seq = torch.arange(sequences, dtype=torch.int32, device=dev).repeat_interleave(new)
        x = torch.zeros((sequences * new, 12, d), dtype=torch.bfloat16, device=dev)
        pos = (torch.arange(new, dtype=torch.int32, device=dev) + n).repeat(sequences)

        def step():
            q = cache.append(x[:, :8], x[:, 8:10], x[:, 10:], cs, pos, seq)
            return (q, *cache.attend(q, pos, seq, 40, 1, 2), *cache.read(pos, seq))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        return x, pos, step, graph, held

    print(f"{sequences} sequences of {blocks} blocks, {more} more tokens", flush=True)
    graphs = [graph_of(more), graph_of(more + 4)]
    for i in range(6):
        x, pos, step, graph, held = graphs[i % 2]
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        results = []
        for replay in (True, False):
            for y, z in zip((*cache._tensors, cache.bounds, cache.bound_scales), start):
                y.copy_(z)
            if replay:
                graph.replay()
            else:
                held = step()
            torch.cuda.synchronize()
            results.append([y.clone() for y in (*held, *cache._tensors, cache.bounds)])
        for k, (a, b) in enumerate(zip(*results)):
            assert torch.equal(a, b), (i, k)


@pytest.mark.gpu
def test_on_another_stream(dev):
    """Calls enqueue on the current stream: a step behind a long product on a side stream."""
    import torch

    from retrieve_amd import kv

    cache = _cache(dev, "bf16", 2, 64, 16)
    cache.reserve(0, 260)
    rows = to(dev, normal16(8, (260, 12, 64), "bf16"), "bf16")
    pos = torch.arange(260, dtype=torch.int32, device=dev)
    seq = torch.zeros_like(pos)
    cs = kv.rotary_table(260, 64, device=dev)

    def step(y):
        q = cache.append(y[:, :8], y[:, 8:10], y[:, 10:], cs, pos, seq)
        return q, *cache.attend(q, pos, seq, 5), *cache.read(pos, seq)

    want = step(rows)
    late = torch.zeros_like(rows)
    big = torch.randn((4096, 4096), device=dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(rows)
        got = step(late)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_sequences_share_full_pages(dev):
    """A prompt's full pages in two sequences' tables: each goes on by itself behind them, and gives
    what a sequence gives that holds the prompt alone."""
    import torch

    from retrieve_amd import kv

    page, d, shared = 16, 64, 6
    cache = _cache(dev, "bf16", 2, d, page, sequences=3)
    own = _cache(dev, "bf16", 2, d, page, sequences=3)
    x = [to(dev, normal16(60 + i, (shared * page + 30, 12, d), "bf16"), "bf16") for i in range(2)]
    x[1][:shared * page] = x[0][:shared * page]
    cs = kv.rotary_table(400, d, device=dev)

    def run(c, s, rows, pos):
        pos = torch.tensor(pos, dtype=torch.int32, device=dev)
        seq = torch.full_like(pos, s)
        q = c.append(rows[:, :8], rows[:, 8:10], rows[:, 10:], cs, pos, seq)
        return (q, *c.attend(q, pos, seq, 8), *c.read(pos, seq))

    for s in (0, 1):
        cache.reserve(s, len(x[s]))
        own.reserve(s, len(x[s]))
    cache.page_table[1, :shared] = cache.page_table[0, :shared]
    for s in (0, 1):
        run(own, s, x[s][:shared * page], range(shared * page))
    run(cache, 0, x[0][:shared * page], range(shared * page))
    at = shared * page
    for new in (1, 1, 17, 11):
        for s in (0, 1):
            got, want = (run(c, s, x[s][at:at + new], range(at, at + new)) for c in (cache, own))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (at, s)
        at += new


@pytest.mark.gpu
def test_idle_slots(dev):
    """``sequences`` chooses a kernel only: a prompt beside many idle rows of the table, said or not,
    is within the attention's tolerance, and rows that are not contiguous are read as they lie."""
    import torch

    heads, heads_kv, d, page = 8, 2, 128, 64
    cache = _cache(dev, "bf16", heads_kv, d, page, pages=30, sequences=500, max_pages=20)
    cache.k_tail.fill_(float("nan"))
    cache.v_tail.fill_(float("nan"))
    cache.reserve(311, 900)
    rows = to(dev, normal16(9, (900, heads + 2 * heads_kv, d), "bf16"), "bf16")
    pos = torch.arange(900, dtype=torch.int32, device=dev)
    seq = torch.full_like(pos, 311)
    cache.append(rows[:, :8], rows[:, 8:10], rows[:, 10:], None, pos, seq)
    q = rows[:, :8]
    assert not q.is_contiguous()
    c = _mirror(cache, "bf16")
    blocks = cache.select(q, pos, seq, 5, 1, 2)
    pick = np.r_[0:3, 60:70, 440, 899]
    case = [back(y)[pick] for y in (q, blocks, pos, seq)]
    for sequences in (None, 1, 500, 900):
        out, lse = cache.attend_to(q, blocks, pos, seq, None, sequences)
        check_attention((back(out)[pick], back(lse)[pick]), c, *case, back(cache.page_table))

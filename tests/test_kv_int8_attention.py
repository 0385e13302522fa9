"""Attention over chosen blocks of the 8-bit cache against softmax in 64 bits over what the codes
stand for (tolerances: ``kv_int8_cases.check_attention``)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv_int8 as o8
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to
from tests.kv_int8_cases import check_attention, on_gpu
from tests.test_kv_attention import _choose

SHAPES = [("bf16", 8, 2, 128, 64), ("fp16", 3, 3, 64, 16), ("bf16", 7, 1, 96, 32),
          ("fp16", 12, 2, 192, 16), ("bf16", 2, 1, 256, 128), ("fp16", 40, 2, 64, 64),
          ("bf16", 17, 1, 128, 16), ("fp16", 16, 1, 96, 128), ("bf16", 10, 5, 64, 32),
          ("fp16", 6, 2, 256, 16)]


def _case(seed, kind, heads, heads_kv, d, page, had_new, count, sparse=0.0, size=1.0):
    """A cache whose sequences have just taken their new tokens: the last block of each is open where
    it is not full."""
    print(f"attend int8 {kind} {heads}/{heads_kv} d={d} page={page} count={count}", flush=True)
    pos, seq, tab, pages = layout(seed, page, had_new)
    c = o8.Cache(seed + 1, pages, heads_kv, page, d, len(had_new), kind)
    for s, (had, new) in enumerate(had_new):
        if (had + new) % page:
            i = tab[s, (had + new) // page]
            c.ks[i] = c.vs[i] = 0.0
    q = normal16(seed + 2, (len(pos), heads, d), kind, size)
    return c, q, _choose(seed + 4, pos, heads_kv, page, count, sparse), pos, seq, tab


def _run(dev, c, q, blocks, pos, seq, tab, scale=None, sequences=None):
    from retrieve_amd import kv

    out, lse = kv.block_attention_int8(to(dev, q, c.kind), *on_gpu(dev, c)[0], to(dev, blocks),
                                       to(dev, pos), to(dev, seq), to(dev, tab), scale, sequences)
    return back(out), back(lse)


def _some(got, case, pick):
    c, q, blocks, pos, seq, tab = case
    return (got[0][pick], got[1][pick]), (c, q[pick], blocks[pick], pos[pick], seq[pick], tab)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", SHAPES)
def test_single_tokens(dev, kind, heads, heads_kv, d, page):
    """Contexts that end at the first and last slots of a block and of 16 keys: open blocks of every
    kind, full ones."""
    had = [0, 1, 14, 15, 16, 17, 31, 32, page - 1, page, 3 * page + 15, 5 * page + 16, 9 * page + 1,
           20 * page - 1, 37 * page + 33]
    case = _case(d + page, kind, heads, heads_kv, d, page, [(h, 1) for h in had], 11)
    check_attention(_run(dev, *case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", SHAPES)
def test_prompts(dev, kind, heads, heads_kv, d, page):
    """Tokens inside full blocks and in the open one, each with its own lists."""
    case = _case(d + page + 1, kind, heads, heads_kv, d, page,
                 [(0, page + 5), (6 * page + 3, 50), (2, 1)], 5, sparse=0.2)
    check_attention(_run(dev, *case), *case)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 2, 7, 64, 129, 600])
@pytest.mark.parametrize("tokens", [1, 3])
def test_few_rows_many_blocks(dev, tokens, count):
    """Long lists of few rows: the split over the list, and its join."""
    case = _case(count + tokens, "bf16", 4, 1, 64, 16,
                 [(16 * 700 + 3 * i, 1) for i in range(tokens)], count)
    check_attention(_run(dev, *case), *case)


MANY = [("bf16", 1, 1, 64, 16, 9), ("fp16", 2, 1, 128, 64, 5), ("bf16", 3, 1, 96, 32, 16),
        ("bf16", 7, 1, 64, 128, 4), ("fp16", 8, 1, 192, 64, 6), ("bf16", 12, 1, 128, 32, 5),
        ("fp16", 20, 1, 64, 64, 4), ("bf16", 4, 1, 256, 64, 70), ("fp16", 4, 1, 64, 16, 300),
        ("bf16", 8, 2, 128, 64, 16), ("fp16", 8, 8, 64, 16, 9), ("bf16", 16, 8, 128, 32, 5),
        ("fp16", 32, 8, 128, 64, 7)]


def _many(seed, kind, heads, heads_kv, d, page, count):
    """More rows than the GPU holds waves, of three sequences; neighbours choose alike in the first
    and last, by chance in the second."""
    had_new = [(3 * page + 5, 2000), (0, 5000 // heads_kv), (40, 7)]
    case = list(_case(seed, kind, heads, heads_kv, d, page, had_new, count, sparse=0.1))
    blocks, pos = case[2], case[3]
    for t in range(1, 2000):
        if t % 37:
            blocks[t] = blocks[t - 1]
            blocks[t, :, t % count] = pos[t] // page if t % 5 == 0 else blocks[t, :, t % count]
    own = np.sort(blocks, -1)  # (each block once a row)
    for t, h in np.argwhere((own[:, :, 1:] == own[:, :, :-1]).any(-1)):
        row = blocks[t, h]
        _, first = np.unique(row, return_index=True)
        row[np.setdiff1d(np.arange(count), first)] = -1
    return case


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count", MANY)
def test_many_rows(dev, kind, heads, heads_kv, d, page, count):
    case = _many(heads + count, kind, heads, heads_kv, d, page, count)
    got = _run(dev, *case)
    tokens = len(case[3])
    pick = np.r_[0:9, 31:45, 1990:2012, rng(5).integers(0, tokens, 60), tokens - 9:tokens]
    got, case = _some(got, case, pick)
    check_attention(got, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count,tokens",
                         [("bf16", 32, 8, 128, 64, 6, 230), ("fp16", 8, 8, 64, 16, 12, 430),
                          ("bf16", 6, 2, 256, 32, 5, 500), ("bf16", 24, 3, 96, 128, 3, 777),
                          ("bf16", 10, 10, 192, 16, 4, 201), ("fp16", 8, 4, 128, 16, 128, 410),
                          ("bf16", 4, 2, 256, 16, 96, 520)])
def test_hundreds_of_tokens(dev, kind, heads, heads_kv, d, page, count, tokens):
    """Prompts between few rows and many, short lists and long ones."""
    had_new = [(5 * page + 3, tokens - tokens // 3 - 9), (0, tokens // 3), (33, 9)]
    case = _case(tokens + d, kind, heads, heads_kv, d, page, had_new, count, sparse=0.1)
    got = _run(dev, *case, sequences=3)
    pick = np.r_[0:40, rng(6).integers(0, tokens, 60), tokens - 40:tokens]
    got, case = _some(got, case, pick)
    check_attention(got, *case)


@pytest.mark.gpu
def test_hundreds_of_sequences(dev):
    case = _case(600, "bf16", 16, 4, 64, 16, [(3 + 7 * i % 90, 1) for i in range(600)], 3)
    check_attention(_run(dev, *case), *case)


@pytest.mark.gpu
def test_rows_without_keys(dev):
    """All -1, padding tokens, blocks past the token's own, missing pages, blocks that were never
    filled: zeros and -inf."""
    case = list(_case(23, "bf16", 4, 2, 64, 16, [(100, 2), (50, 2), (30, 1), (3, 1)], 4))
    c, q, blocks, pos, seq, tab = case
    case[3:] = pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    blocks[0] = -1
    blocks[1, 0] = [50, 2**31 - 1, 7, -5]  # (7 is not yet begun at position 101)
    pos[2], seq[3] = -1, 9
    tab[2] = -1
    got = _run(dev, *case)
    check_attention(got, *case)
    assert np.isneginf(got[1][[0, 2, 3, 4]]).all() and np.isneginf(got[1][1, :2]).all()
    assert np.isfinite(got[1][1, 2:]).all() and np.isfinite(got[1][5]).all()
    # a block of the first sequence loses its codes: it counts no more; a few rows and many
    c.ks[tab[0, 2]] = c.vs[tab[0, 2]] = 0.0
    blocks[1, 0] = [2, 0, 6, -1]
    for n in (1, 900):
        many = [c, *(np.repeat(x, n, 0) for x in (q, blocks, pos, seq)), tab]
        got, small = _some(_run(dev, *many), many, np.r_[0:6 * n:n, n - 1:6 * n:n])
        check_attention(got, *small)


@pytest.mark.gpu
def test_no_list(dev):
    c, q, blocks, *rest = _case(25, "bf16", 4, 2, 64, 16, [(10, 2)], 1)
    out, lse = _run(dev, c, q, blocks[:, :, :0], *rest)
    assert (out == 0).all() and np.isneginf(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_open_slots_past_the_token_hold_anything(dev, kind, page, what):
    """NaN and infinities in the open block behind the tokens, single tokens and prompts."""
    had = [(0, 1), (page // 2, 1), (3 * page + 5, 1), (2 * page - 1, 1), (4 * page + page - 2, 1),
           (page + 2, page // 2)]
    c, q, blocks, pos, seq, tab = _case(29, kind, 4, 2, 64, page, had, 5)
    blocks[:, :, 0] = pos[:, None] // page  # (the own block is listed, once)
    for b in blocks.reshape(-1, 5):
        b[1:][b[1:] == b[0]] = -1
    clean = c.copy()
    for s, (a, n) in enumerate(had):
        c.kt[s, :, (a + n) % page:], c.vt[s, :, :, (a + n) % page:] = what, what
    clean.kt[~np.isfinite(clean.kt)] = 0
    check_attention(_run(dev, c, q, blocks, pos, seq, tab), clean, q, blocks, pos, seq, tab)
    n = 6000 // len(pos)
    case = [np.repeat(x, n, 0) for x in (q, blocks, pos, seq)]
    got, case = _some(_run(dev, c, *case, tab), (clean, *case, tab),
                      rng(4).integers(0, n * len(pos), 60))
    check_attention(got, *case)


@pytest.mark.gpu
def test_a_later_token_that_is_not_finite(dev):
    """A prompt's token in the open block with an infinite value and a NaN key: the tokens before it are
    as without it, the ones behind it not finite."""
    c, q, blocks, pos, seq, tab = _case(31, "bf16", 4, 1, 64, 64, [(64, 40)], 2)
    blocks[:] = [0, 1]
    clean = c.copy()
    c.vt[0, 0, 9, 20] = np.inf
    c.kt[0, 0, 30, 3] = np.nan
    for n in (1, 110):
        case = [np.repeat(x, n, 0) for x in (q, blocks, pos, seq)]
        out, lse = _run(dev, c, *case, tab)
        before = np.flatnonzero(case[2] < 64 + 20)[::n]
        got, small = _some((out, lse), (clean, *case, tab), before)
        check_attention(got, *small)
        middle, behind = (case[2] >= 84) & (case[2] < 94), case[2] >= 94
        assert np.isposinf(out[middle][:, :, 9]).all()
        assert np.isfinite(out[middle][:, :, :9]).all() and np.isfinite(lse[middle]).all()
        assert np.isnan(out[behind]).all() and np.isnan(lse[behind]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_large_scores(dev, kind):
    """Scores of hundreds to thousands, both signs; a scale of its own; queries of zeros."""
    case = _case(33, kind, 4, 2, 128, 16, [(400, 1), (37, 9), (16 * 40, 1)], 8, size=60.0)
    for scale in (None, 0.7, -0.4):
        check_attention(_run(dev, *case, scale), *case, scale)
    c, q, *rest = case
    check_attention(_run(dev, c, 0 * q, *rest), c, 0 * q, *rest)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_queries_of_unlike_size(dev, kind):
    """Channels from 2^-14 of the largest on (fp16: where its numbers are whole), rows that fp16 cannot
    hold, beside keys that make the small channels count."""
    c, q, *rest = _case(35, kind, 4, 2, 64, 16, [(200, 1), (90, 4)], 6)
    c.k[:, :, :, 0] = 0
    c.kt[:, :, :, 0] = 0
    q[:, :, 1:] *= np.float32(2.0**-12 if kind == "bf16" else 2.0**-4)
    q[:, :, 0] = 2.0**4
    check_attention(_run(dev, c, q, *rest, 500.0), c, q, *rest, 500.0)
    if kind == "bf16":
        for size, scale in ((2.0**100, 2.0**-90), (2.0**-100, 2.0**104)):
            x = q * np.float32(size)
            check_attention(_run(dev, c, x, *rest, scale), c, x, *rest, scale)


@pytest.mark.gpu
def test_scales_of_unlike_size(dev):
    """Blocks of values from nothing to the largest beside each other: each weighs as its scores say."""
    c, q, *rest = _case(37, "bf16", 4, 2, 64, 16, [(500, 1), (16 * 30, 3)], 20)
    g = rng(38)
    c.vs[:] = np.where(c.vs > 0, np.exp2(g.uniform(-30, 10, c.vs.shape)).astype(np.float32), 0)
    c.ks[:] = np.where(c.ks > 0, np.exp2(g.uniform(-30, -4, c.ks.shape)).astype(np.float32), 0)
    check_attention(_run(dev, c, q, *rest), c, q, *rest)
    c.vs[c.vs > 0] = np.float32(1e-8) / np.float32(127)
    check_attention(_run(dev, c, q, *rest), c, q, *rest)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_queries_that_are_not_finite(dev, kind):
    """Such a row is not a number, its neighbours are as without it; a row without keys stays empty."""
    c, q, blocks, pos, seq, tab = _case(39, kind, 8, 2, 64, 16, [(100, 3), (3, 1)], 4)
    blocks[2] = -1
    clean = _run(dev, c, q, blocks, pos, seq, tab)
    q[0, 1, 5], q[1, 6, 0], q[2, 0, 0] = np.inf, np.nan, np.nan
    out, lse = _run(dev, c, q, blocks, pos, seq, tab)
    assert np.isnan(out[0, 1]).all() and np.isnan(out[1, 6]).all()
    assert np.isnan(lse[0, 1]) and np.isnan(lse[1, 6])
    out[0, 1], out[1, 6], lse[0, 1], lse[1, 6] = clean[0][0, 1], clean[0][1, 6], *clean[1][[0, 1], [1, 6]]
    assert np.array_equal(out, clean[0]) and np.array_equal(lse, clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 1200])
def test_offsets_past_32_bits(dev, tokens):
    import torch

    from retrieve_amd import kv

    pages, page, d = 18400, 128, 128
    k = torch.zeros((pages, 8, page, d), dtype=torch.int8, device=dev)
    v = torch.zeros((pages, 8, d, page), dtype=torch.int8, device=dev)
    ks, vs = (torch.full((pages, 8), 0.03, device=dev) for _ in range(2))
    c = o8.Cache(41, 4, 8, page, d, 1, "bf16")
    c.ks[:] = c.vs[:] = np.float32(0.03)
    where = [0, pages // 2, pages - 2, pages - 1]
    k[where], v[where] = to(dev, c.k), to(dev, c.v)
    q = normal16(43, (tokens, 16, d), "bf16")
    pos = np.array([4 * page - 1, 3 * page + 9] * (tokens // 2), np.int32)
    seq = np.zeros(tokens, np.int32)
    blocks = np.ascontiguousarray(np.broadcast_to(np.arange(4, dtype=np.int32), (tokens, 8, 4)))
    got = kv.block_attention_int8(to(dev, q, "bf16"), k, v, ks, vs, to(dev, c.kt, "bf16"),
                                  to(dev, c.vt, "bf16"), to(dev, blocks), to(dev, pos),
                                  to(dev, seq), torch.tensor([where], dtype=torch.int32, device=dev))
    last = slice(-20, None)
    check_attention([back(x)[last] for x in got], c, q[last], blocks[last], pos[last], seq[last],
                    np.arange(4, dtype=np.int32)[None])


@pytest.mark.gpu
def test_the_same_bits_every_time(dev):
    for case in (_case(47, "bf16", 8, 2, 64, 16, [(9000, 1)], 200),
                 _case(47, "bf16", 8, 2, 64, 16, [(300, 400)], 6),
                 _many(48, "bf16", 4, 1, 64, 16, 9)):
        first = _run(dev, *case)
        for _ in range(3):
            again = _run(dev, *case)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])

"""Choosing blocks by their int8 bounds: every index equal to the oracle's, whose sums are
integers."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from oracle import quantize as oq
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to


def _bounds(seed, pages, heads_kv, d, ties=False):
    g = rng(seed)
    low = 0 if ties else -127
    codes = g.integers(low, 2 if ties else 128, (pages, heads_kv, 2 * d), dtype=np.int8)
    scales = np.ones((pages, heads_kv), np.float32) if ties else g.random(
        (pages, heads_kv), dtype=np.float32) + np.float32(0.1)
    return codes, scales


def _select(dev, q, kind, codes, scales, pos, seq, tab, *how):
    from retrieve_amd import kv

    return back(kv.select_blocks(to(dev, q, kind), to(dev, codes), to(dev, scales), to(dev, pos),
                                 to(dev, seq), to(dev, tab), *how))


def _check(dev, seed, kind, heads, heads_kv, d, page, had_new, how, ties=False, max_pages=None):
    print(f"select {kind} {heads}/{heads_kv} d={d} page={page} {how}", flush=True)
    pos, seq, tab, pages = layout(seed, page, had_new, max_pages=max_pages)
    q = normal16(seed + 1, (len(pos), heads, d), kind)
    codes, scales = _bounds(seed + 2, pages, heads_kv, d, ties)
    got = _select(dev, q, kind, codes, scales, pos, seq, tab, page, *how)
    want = okv.select(q, codes, scales, pos, seq, tab, page, *how)
    assert np.array_equal(got, want)
    return got


def test_selection_by_rationals():
    """The oracle's order is that of the exact scores (random scores are no fp32 rounding apart),
    and ties go to the lower block."""
    g = rng(31)
    q = normal16(32, (4, 64), "bf16")
    for ties in (False, True):
        codes, scales = _bounds(33, 40, 1, 64, ties)
        if ties:
            codes[20:] = codes[:20]
        pos = np.array([40 * 16 - 1], np.int32)
        tab = g.permutation(40).astype(np.int32)[None]
        got = okv.select(q[None], codes, scales, pos, np.zeros(1, np.int32), tab, 16, 9, 0, 1)[0, 0]
        qc, qs = oq.quantize_int8(q, divide=True)
        want = okv.blocks_by_bounds(qc, qs, codes[tab[0, :39], 0], scales[tab[0, :39], 0], 8)
        assert got.tolist() == want + [39]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", [
    ("bf16", 8, 2, 128, 64), ("fp16", 3, 3, 64, 16), ("bf16", 7, 1, 96, 32), ("fp16", 12, 2, 192, 16),
    ("bf16", 2, 1, 256, 128), ("fp16", 40, 2, 64, 16), ("bf16", 17, 1, 128, 16),
    ("bf16", 10, 5, 64, 64), ("bf16", 80, 1, 64, 16), ("fp16", 40, 1, 256, 32),
    ("bf16", 33, 1, 96, 64), ("fp16", 4, 1, 192, 64), ("bf16", 1, 1, 128, 16)])
def test_matches_the_oracle(dev, kind, heads, heads_kv, d, page):
    decode = [(n * page + r, 1) for n, r in [(0, 0), (0, page - 1), (1, 0), (3, 5), (9, 0), (20, 7),
                                              (63, 1), (64, page - 1), (65, 0), (130, 3)]]
    _check(dev, d, kind, heads, heads_kv, d, page, decode, (12, 1, 2))
    _check(dev, d + 7, kind, heads, heads_kv, d, page, decode, (64, 2, 1))
    prompts = [(0, 2 * page + 3), (17 * page, 21), (40 * page + 3, page), (5, 1)]
    if heads * d <= 1024:
        _check(dev, d + 9, kind, heads, heads_kv, d, page, prompts, (8, 0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("how", [(1, 0, 1), (3, 1, 2), (2, 0, 1), (16, 5, 5), (200, 1, 1),
                                 (1024, 0, 1), (33, 32, 1)])
def test_counts_and_forced_blocks(dev, how):
    had_new = [(16 * n + 3, 1) for n in (0, 1, 2, 3, 15, 16, 17, 199, 200, 201, 300)]
    got = _check(dev, 41, "bf16", 4, 2, 64, 16, had_new, how)
    count, sink, recent = how
    for row, (at, _) in zip(got, had_new):
        last = at // 16
        assert set(range(max(0, last - recent + 1), last + 1)) <= set(row[0])
        assert set(range(min(sink, last + 1))) <= set(row[1])
        assert (row >= 0).sum(1).tolist() == [min(count, last + 1)] * 2


@pytest.mark.gpu
def test_ties_go_to_the_lower_block(dev):
    """Scores that mostly tie, over one wave's blocks and over many workgroups' of them."""
    g = rng(51)
    for blocks in (50, 700, 9000):
        pos = np.array([16 * blocks - 1], np.int32)
        tab = g.permutation(blocks).astype(np.int32)[None]
        codes = np.zeros((blocks, 1, 128), np.int8)
        codes[:, 0, 0] = g.integers(0, 3, blocks)
        scales = np.ones((blocks, 1), np.float32)
        q = np.ones((1, 2, 64), np.float32)
        how = (16, 20 + blocks // 40, 2, 3)
        got = _select(dev, q, "fp16", codes, scales, pos, np.zeros(1, np.int32), tab, *how)
        assert np.array_equal(got, okv.select(q, codes, scales, pos, np.zeros(1, np.int32), tab, *how))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,d,blocks,count", [
    (4, 64, 511, 64), (4, 64, 513, 64), (4, 64, 2047, 64), (4, 96, 2048, 260), (4, 64, 4095, 250),
    (4, 64, 4096, 100), (40, 64, 4200, 300), (20, 256, 5000, 64), (4, 128, 20000, 64),
    (4, 64, 70001, 1000)])
def test_long_contexts(dev, heads, d, blocks, count):
    """Single tokens around the sizes where the kernels change: one launch up to 4096 blocks, keys
    in registers or read again."""
    had = [(16 * blocks - 5, 1), (16 * 333, 1)]
    _check(dev, blocks, "bf16", heads, 1, d, 16, had, (count, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,d,blocks,count", [(4, 64, 200, 30), (2, 128, 900, 30), (2, 64, 1000, 60),
                                                  (1, 96, 1100, 64), (8, 64, 3000, 300),
                                                  (16, 64, 4500, 64), (3, 192, 300, 20)])
def test_prompts_behind_long_contexts(dev, heads, d, blocks, count):
    """A few tokens of each sequence, over blocks that take a wave's registers, four waves' or
    more."""
    had = [(16 * blocks + 9, 9), (16 * (blocks // 2), 3), (40, 5)]
    _check(dev, blocks + 1, "fp16", heads, 1, d, 16, had, (count, 1, 2))


@pytest.mark.gpu
def test_scores_close_together(dev):
    """Keys that agree in their high bits: a narrow range of scores around a large common one, and a
    range where all but a few scores are far below."""
    g = rng(61)
    blocks, d = 3000, 64
    pos = np.array([16 * blocks + 1], np.int32)
    tab = np.arange(blocks + 1, dtype=np.int32)[None]
    q = np.ones((1, 1, d), np.float32)
    codes = np.full((blocks + 1, 1, 2 * d), 127, np.int8)
    codes[:, 0, :4] -= g.integers(0, 3, (blocks + 1, 4)).astype(np.int8)
    far = codes.copy()
    far[50:, 0] = -126
    far[50:, 0, :9] += g.integers(0, 2, (blocks - 49, 9)).astype(np.int8)
    scales = np.ones((blocks + 1, 1), np.float32)
    near = scales * (1 + g.integers(0, 4, (blocks + 1, 1)).astype(np.float32) * np.float32(2**-23))
    for c, s in ((codes, scales), (codes, near), (far, scales), (far, near)):
        how = (16, 128, 1, 1)
        got = _select(dev, q, "bf16", c, s, pos, np.zeros(1, np.int32), tab, *how)
        assert np.array_equal(got, okv.select(q, c, s, pos, np.zeros(1, np.int32), tab, *how))


@pytest.mark.gpu
def test_padding_and_missing_pages(dev):
    pos, seq, tab, pages = layout(71, 16, [(500, 1), (300, 1), (100, 20), (40, 1), (0, 1)])
    pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    pos[4], seq[5], seq[6], pos[7] = -1, -1, 5, 2**31 - 1
    tab[0, 3], tab[0, 9:20], tab[1, 5], tab[2, 2] = -1, pages, 2**31 - 1, -7
    q = normal16(72, (len(pos), 4, 64), "bf16")
    codes, scales = _bounds(73, pages, 2, 64)
    got = _select(dev, q, "bf16", codes, scales, pos, seq, tab, 16, 10, 1, 2)
    assert np.array_equal(got, okv.select(q, codes, scales, pos, seq, tab, 16, 10, 1, 2))
    assert (got[4:8] == -1).all()


@pytest.mark.gpu
def test_scores_that_are_not_numbers_rank_last(dev):
    pos, seq, tab, pages = layout(81, 16, [(16 * 30, 1)])
    q = normal16(82, (1, 2, 64), "bf16")
    codes, scales = _bounds(83, pages, 1, 64)
    scales[tab[0, 4]], scales[tab[0, 7]] = np.nan, -np.inf
    got = _select(dev, q, "bf16", codes, scales, pos, seq, tab, 16, 29, 0, 1)
    assert np.array_equal(got, okv.select(q, codes, scales, pos, seq, tab, 16, 29, 0, 1))
    assert len(set(range(31)) - set(got[0, 0])) == 2
    q[:] = np.nan
    got = _select(dev, q, "bf16", codes, scales, pos, seq, tab, 16, 29, 0, 1)[0, 0]
    assert len(set(got)) == 29 and got[-1] == 30 and (np.diff(got) > 0).all()


@pytest.mark.gpu
def test_all_zero_queries(dev):
    """Every score zero: the lowest blocks."""
    pos, seq, tab, pages = layout(91, 16, [(16 * 100, 1)])
    codes, scales = _bounds(92, pages, 1, 64)
    got = _select(dev, np.zeros((1, 4, 64), np.float32), "fp16", codes, scales, pos, seq, tab, 16, 12,
                  2, 3)[0, 0]
    assert got.tolist() == list(range(9)) + [98, 99, 100]


@pytest.mark.gpu
def test_strided_queries(dev):
    from retrieve_amd import kv

    pos, seq, tab, pages = layout(101, 16, [(900, 3), (77, 1)])
    q = normal16(102, (4, 6, 64), "bf16")
    codes, scales = _bounds(103, pages, 2, 64)
    x = to(dev, np.concatenate([q, q * 2], 1), "bf16")
    got = back(kv.select_blocks(x[:, :6], to(dev, codes), to(dev, scales), to(dev, pos),
                                to(dev, seq), to(dev, tab), 16, 9))
    assert np.array_equal(got, okv.select(q, codes, scales, pos, seq, tab, 16, 9))


@pytest.mark.gpu
def test_refusals(dev):
    from retrieve_amd import kv

    pos, seq, tab, pages = layout(111, 16, [(100, 2)])
    codes, scales = _bounds(112, pages, 2, 64)
    q = to(dev, normal16(113, (2, 4, 64), "bf16"), "bf16")
    good = dict(q=q, bounds=to(dev, codes), bound_scales=to(dev, scales), positions=to(dev, pos),
                seq_ids=to(dev, seq), page_table=to(dev, tab), page_size=16, count=4)
    assert kv.select_blocks(**good).shape == (2, 2, 4)
    assert kv.select_blocks(**{**good, "q": q[:0], "positions": good["positions"][:0],
                               "seq_ids": good["seq_ids"][:0]}).shape == (0, 2, 4)
    for error, wrong in [
        (ValueError, {"q": q[0]}), (TypeError, {"q": q.float()}), (ValueError, {"q": q[:, :3]}),
        (ValueError, {"bounds": good["bounds"][..., :64].contiguous()}),
        (TypeError, {"bound_scales": good["bound_scales"].double()}),
        (ValueError, {"bound_scales": good["bound_scales"][:1]}),
        (ValueError, {"page_size": 24}), (ValueError, {"count": 0}), (ValueError, {"count": 1025}),
        (ValueError, {"sink": -1}), (ValueError, {"recent": 0}), (ValueError, {"sink": 3, "recent": 2}),
        (TypeError, {"seq_ids": good["seq_ids"].long()}), (ValueError, {"seq_ids": good["seq_ids"][:1]}),
        (ValueError, {"page_table": good["page_table"].cpu()}),
    ]:
        with pytest.raises(error):
            kv.select_blocks(**{**good, **wrong})


def test_codes_by_reciprocal():
    """The kernels' quotient (reciprocal, product, one correction) is the division's, rounded to
    nearest, for every pair of bf16 significands, a spread of fp16's, and the floor: codes equal bit
    for bit. (The correction's product and sum are exact in 64 bits up to their last rounding.)"""
    def quotient(x, top):
        r = (np.float32(1) / top).astype(np.float32)
        q = (x * r).astype(np.float32)
        rest = (x.astype(np.float64) - q.astype(np.float64) * top).astype(np.float32)
        return (rest.astype(np.float64) * r + q).astype(np.float32)

    for bits, step in ((8, 1), (11, 13)):
        m = np.arange(1 << (bits - 1), 1 << bits, dtype=np.float32)
        for top in m[::step]:
            for e in range(9):
                x = (m * 2.0**-e).astype(np.float32)
                x = x[x <= top]
                assert np.array_equal(quotient(x, np.float32(top)), x / np.float32(top))
    x = (np.arange(0, 129, dtype=np.float32) * np.float32(2.0**-34)).astype(np.float32)
    x = x[x <= np.float32(1e-8)]
    assert np.array_equal(quotient(x, np.float32(1e-8)), x / np.float32(1e-8))


@pytest.mark.gpu
def test_queries_of_extreme_sizes(dev):
    """Largest magnitudes from below the floor to the ends of bf16's range."""
    pos, seq, tab, pages = layout(121, 16, [(16 * 60, 1)] * 8)
    q = normal16(122, (8, 4, 64), "bf16")
    q *= np.float32(2.0)**np.array([-120, -40, -27, -20, 0, 60, 101, 120], np.float32)[:, None, None]
    q[7, 2] = 0.0
    codes, scales = _bounds(123, pages, 1, 64)
    got = _select(dev, q, "bf16", codes, scales, pos, seq, tab, 16, 12, 1, 2)
    assert np.array_equal(got, okv.select(q, codes, scales, pos, seq, tab, 16, 12, 1, 2))
    prompt = [np.repeat(x, 5, 0) for x in (q, pos, seq)]
    got = _select(dev, prompt[0], "bf16", codes, scales, prompt[1], prompt[2], tab, 16, 12, 1, 2)
    assert np.array_equal(got[::5], okv.select(q, codes, scales, pos, seq, tab, 16, 12, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,blocks", [(1, 40), (9, 40), (2, 5000)])
def test_a_cache_without_pages(dev, tokens, blocks):
    """One launch, prompts and long page tables: the forced blocks only."""
    print(f"no pages, {tokens} tokens, {blocks} blocks", flush=True)
    pos = np.arange(16 * blocks - tokens, 16 * blocks, dtype=np.int32)
    seq, tab = np.zeros(tokens, np.int32), np.full((1, blocks), -1, np.int32)
    tab[0, ::3] = 0
    codes, scales = _bounds(131, 0, 2, 64)
    got = _select(dev, normal16(132, (tokens, 4, 64), "bf16"), "bf16", codes, scales, pos, seq, tab,
                  16, 10, 1, 2)
    forced = [[0, p // 16 - 1, p // 16] + [-1] * 7 for p in pos]
    assert np.array_equal(got, np.repeat(np.array(forced, np.int32)[:, None], 2, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("max_pages", [200, 2000])
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", [
    ("bf16", 2, 2, 64, 16), ("fp16", 4, 2, 128, 64), ("bf16", 6, 2, 96, 32), ("fp16", 8, 2, 128, 16),
    ("bf16", 14, 2, 256, 32), ("fp16", 16, 2, 64, 128), ("bf16", 24, 2, 192, 16),
    ("fp16", 40, 2, 96, 16)])
def test_prompts_by_the_table_s_width(dev, kind, heads, heads_kv, d, page, max_pages):
    """The same ragged prompts as few keys (scored as single tokens are) and as many."""
    had_new = [(90 * page + 3, 37), (0, 2 * page + 1), (150 * page, 11)]
    _check(dev, heads + d, kind, heads, heads_kv, d, page, had_new, (24, 1, 2), max_pages=max_pages)

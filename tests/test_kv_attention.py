"""Attention over chosen blocks against softmax in 64 bits.

Tolerances, from the arithmetic: with ``u`` the 16-bit type's unit roundoff, an output is rounded
once (``u |out|``) and every weight once before its product with ``v`` (``u`` relative; for fp16
also its least step, 2^-25 of a weight of 1), so a sum moves by ``u sum w |v|``; scores are fp32
sums of ``D`` exact products, off by ``(D + 8) 2^-24 scale sum |q k|`` at most, which moves a weight
by twice that, relative, and the log-sum by once.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to

UNIT = {"bf16": 2.0**-8, "fp16": 2.0**-11}


def _choose(seed, pos, heads_kv, page, count, sparse=0.0):
    """Distinct blocks of each row up to the token's own, in any order, -1 among them."""
    g = rng(seed)
    out = np.full((len(pos), heads_kv, count), -1, np.int32)
    for t, p in enumerate(pos):
        for h in range(heads_kv):
            n = min(count, p // page + 1)
            pick = g.permutation(p // page + 1)[:n]
            pick[g.random(n) < sparse] = -1
            out[t, h, g.permutation(count)[:n]] = pick
    return out


def _run(dev, kind, q, kc, vc, blocks, pos, seq, tab, scale=None):
    from retrieve_amd import kv

    out, lse = kv.block_attention(to(dev, q, kind), to(dev, kc, kind), to(dev, vc, kind),
                                  to(dev, blocks), to(dev, pos), to(dev, seq), to(dev, tab), scale)
    return back(out), back(lse)


def _check(got, kind, q, kc, vc, blocks, pos, seq, tab, scale=None):
    d = q.shape[2]
    scale = 1 / np.sqrt(d) if scale is None else scale
    out, lse, spread, slack = okv.attention(q, kc, vc, blocks, pos, seq, tab, scale)
    u = UNIT[kind]
    off = (d + 8) * 2.0**-24 * slack
    least = 2.0**-25 * kc.shape[2] * blocks.shape[2] * np.abs(vc).max() if kind == "fp16" else 0.0
    tol = u * np.abs(out) + (u + 2 * off[..., None] + 2.0**-18) * spread * (1 + u) + least + 2.0**-25
    bad = ~(np.abs(got[0] - out) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[0][bad][:5], out[bad][:5], tol[bad][:5])
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got[1]), empty) and (got[0][empty] == 0).all()
    with np.errstate(invalid="ignore"):
        assert (empty | (np.abs(got[1] - lse) <= off + 2.0**-20 * np.maximum(1, np.abs(lse)))).all()


def _case(seed, kind, heads, heads_kv, d, page, had_new, count, sparse=0.0, size=1.0):
    print(f"attend {kind} {heads}/{heads_kv} d={d} page={page} count={count}", flush=True)
    pos, seq, tab, pages = layout(seed, page, had_new)
    q = normal16(seed + 1, (len(pos), heads, d), kind, size)
    kc = normal16(seed + 2, (pages, heads_kv, page, d), kind)
    vc = normal16(seed + 3, (pages, heads_kv, page, d), kind)
    blocks = _choose(seed + 4, pos, heads_kv, page, count, sparse)
    return q, kc, vc, blocks, pos, seq, tab


SHAPES = [("bf16", 8, 2, 128, 64), ("fp16", 3, 3, 64, 16), ("bf16", 7, 1, 96, 32),
          ("fp16", 12, 2, 192, 16), ("bf16", 2, 1, 256, 128), ("fp16", 40, 2, 64, 64),
          ("bf16", 17, 1, 128, 16), ("fp16", 16, 1, 96, 128), ("bf16", 10, 5, 64, 32),
          ("fp16", 6, 2, 256, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", SHAPES)
def test_single_tokens(dev, kind, heads, heads_kv, d, page):
    """Contexts that end at the first and last slots of a block and of a tile of 16 and 32 keys."""
    had = [0, 1, 14, 15, 16, 17, 31, 32, page - 1, page, 3 * page + 15, 5 * page + 16, 9 * page + 1,
           20 * page - 1, 37 * page + 33]
    case = _case(d + page, kind, heads, heads_kv, d, page, [(h, 1) for h in had], 11)
    _check(_run(dev, kind, *case), kind, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page", SHAPES)
def test_prompts(dev, kind, heads, heads_kv, d, page):
    """Many tokens a sequence, each with its own blocks (and some with fewer)."""
    case = _case(d + page + 1, kind, heads, heads_kv, d, page,
                 [(0, page + 5), (6 * page + 3, 50), (2, 1)], 5, sparse=0.2)
    _check(_run(dev, kind, *case), kind, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 2, 3, 7, 64, 129, 600])
@pytest.mark.parametrize("tokens", [1, 3])
def test_few_rows_many_blocks(dev, tokens, count):
    """Long lists of few rows: the split over the list, and its join."""
    case = _case(count + tokens, "bf16", 4, 1, 64, 16, [(16 * 700 + 3 * i, 1) for i in range(tokens)],
                 count)
    _check(_run(dev, "bf16", *case), "bf16", *case)


MANY = [("bf16", 1, 1, 64, 16, 9), ("fp16", 2, 1, 128, 64, 5), ("bf16", 3, 1, 96, 32, 16),
        ("fp16", 4, 1, 128, 16, 7), ("bf16", 7, 1, 64, 128, 4), ("fp16", 8, 1, 192, 64, 6),
        ("bf16", 12, 1, 128, 32, 5), ("fp16", 20, 1, 64, 64, 4), ("bf16", 4, 1, 256, 64, 70),
        ("fp16", 4, 1, 64, 16, 300), ("bf16", 8, 2, 128, 64, 16), ("fp16", 8, 8, 64, 16, 9),
        ("bf16", 16, 8, 128, 32, 5), ("fp16", 32, 8, 128, 64, 7), ("bf16", 8, 4, 256, 16, 6)]


def _many(seed, kind, heads, heads_kv, d, page, count):
    """More rows than the GPU holds waves (a wave then takes a row, or several tokens at once), of
    three sequences; neighbours choose alike in the first and last, by chance in the second."""
    had_new = [(3 * page + 5, 2000), (0, 5000 // heads_kv), (40, 7)]
    case = list(_case(seed, kind, heads, heads_kv, d, page, had_new, count, sparse=0.1))
    blocks, pos = case[3], case[4]
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


def _some(got, case, pick):
    q, kc, vc, blocks, pos, seq, tab = case
    return (got[0][pick], got[1][pick]), (q[pick], kc, vc, blocks[pick], pos[pick], seq[pick], tab)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count", MANY)
def test_many_rows(dev, kind, heads, heads_kv, d, page, count):
    case = _many(heads + count, kind, heads, heads_kv, d, page, count)
    got = _run(dev, kind, *case)
    tokens = len(case[4])
    assert tokens * heads_kv >= 4096 and tokens * heads_kv * d >= 400 << 10
    pick = np.r_[0:9, 31:45, 1990:2012, rng(5).integers(0, tokens, 60), tokens - 9:tokens]
    got, case = _some(got, case, pick)
    _check(got, kind, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count,tokens",
                         [("bf16", 32, 8, 128, 64, 6, 230), ("fp16", 8, 8, 64, 16, 12, 430),
                          ("bf16", 6, 2, 256, 32, 5, 500), ("fp16", 8, 8, 128, 16, 20, 300),
                          ("bf16", 24, 3, 96, 128, 3, 777), ("bf16", 10, 10, 192, 16, 4, 201)])
def test_hundreds_of_tokens(dev, kind, heads, heads_kv, d, page, count, tokens):
    """Prompts between few rows and many: a wave joins fewer tokens than its columns would hold."""
    had_new = [(5 * page + 3, tokens - tokens // 3 - 9), (0, tokens // 3), (33, 9)]
    case = _case(tokens + d, kind, heads, heads_kv, d, page, had_new, count, sparse=0.1)
    _check(_run(dev, kind, *case), kind, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [600, 1100])
def test_hundreds_of_sequences(dev, sequences):
    """Single tokens of many sequences."""
    case = _case(sequences, "bf16", 16, 4, 64, 16, [(3 + 7 * i % 90, 1) for i in range(sequences)],
                 3)
    _check(_run(dev, "bf16", *case), "bf16", *case)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 4, 8, 16])
def test_many_rows_and_values_that_are_not_finite(dev, heads):
    """Neighbours that choose different blocks: a NaN key or an infinite value reaches the tokens
    whose lists hold it, and no other; slots past every token's are NaN; padding among the
    tokens."""
    page, tokens = 16, 6700
    q, kc, vc, blocks, pos, seq, tab = _case(71, "bf16", heads, 1, 64, page, [(16 * 7 + 3, 1)], 4)
    q = normal16(72, (tokens, heads, 64), "bf16")
    pos, seq = np.full(tokens, 16 * 7 + 3, np.int32), np.zeros(tokens, np.int32)
    odd = np.arange(tokens) % 2 == 1
    blocks = np.where(odd[:, None, None], [[[6, 5, -1, 7]]], [[[0, 1, 2, 7]]]).astype(np.int32)
    pos[::50], blocks[::70] = -1, -1
    kc[tab[0, 7], 0, 4:], vc[tab[0, 7], 0, 4:] = np.nan, np.nan
    clean = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    kc0, vc0 = np.nan_to_num(kc), np.nan_to_num(vc)
    pick = np.r_[0:80, 6600:6700]
    got, case = _some(clean, (q, kc0, vc0, blocks, pos, seq, tab), pick)
    _check(got, "bf16", *case)
    kc[tab[0, 1], 0, 3, 5], vc[tab[0, 6], 0, 2, 9] = np.nan, np.inf
    out, lse = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    full = (pos >= 0) & (blocks[:, 0, 0] >= 0)
    assert np.isnan(out[full & ~odd]).all() and np.isnan(lse[full & ~odd]).all()
    assert np.isposinf(out[full & odd][:, :, 9]).all()
    out[full & odd, :, 9] = clean[0][full & odd, :, 9]
    rest = pick[(odd | ~full)[pick]]
    got, case = _some((out, lse), (q, kc0, vc0, blocks, pos, seq, tab), rest)
    _check(got, "bf16", *case)


@pytest.mark.gpu
def test_rows_without_keys(dev):
    """All -1, padding tokens, blocks past the token's own, pages that are missing: zeros and
    -inf."""
    q, kc, vc, blocks, pos, seq, tab = _case(23, "bf16", 4, 2, 64, 16,
                                             [(100, 2), (50, 2), (30, 1), (3, 1)], 4)
    pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    blocks[0] = -1
    blocks[1, 0] = [50, 2**31 - 1, 7, -5]  # (7 is not yet begun at position 101)
    pos[2], seq[3] = -1, 9
    tab[2] = -1
    got = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    _check(got, "bf16", q, kc, vc, blocks, pos, seq, tab)
    assert np.isneginf(got[1][[0, 2, 3, 4]]).all() and np.isneginf(got[1][1, :2]).all()
    assert np.isfinite(got[1][1, 2:]).all() and np.isfinite(got[1][5]).all()


@pytest.mark.gpu
def test_no_list(dev):
    q, kc, vc, blocks, pos, seq, tab = _case(25, "bf16", 4, 2, 64, 16, [(10, 2)], 1)
    out, lse = _run(dev, "bf16", q, kc, vc, blocks[:, :, :0], pos, seq, tab)
    assert (out == 0).all() and np.isneginf(lse).all()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_slots_past_the_token_hold_anything(dev, page, what):
    """Recycled pages: NaN and infinities in the slots after the token's own, in keys and values."""
    had = [(0, 1), (page // 2, 1), (3 * page + 5, 1), (2 * page - 1, 1), (4 * page + page - 2, 1)]
    q, kc, vc, blocks, pos, seq, tab = _case(29, "bf16", 4, 2, 64, page, had, 5)
    clean = kc.copy(), vc.copy()
    for p, row in zip(pos, tab):
        kc[row[p // page], :, p % page + 1:] = what
        vc[row[p // page], :, p % page + 1:] = what
    got = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    _check(got, "bf16", q, *clean, blocks, pos, seq, tab)
    q, blocks, pos, seq = (np.repeat(x, 500, 0) for x in (q, blocks, pos, seq))
    many = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    got, case = _some(many, (q, *clean, blocks, pos, seq, tab), np.r_[0:2500:250, 498:503, 2499])
    _check(got, "bf16", *case)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_large_scores(dev, kind):
    """Scores of hundreds to thousands, both signs: the running maximum jumps; a scale of its own;
    equal keys; zero queries."""
    case = _case(33, kind, 4, 2, 128, 16, [(400, 1), (37, 9), (16 * 40, 1)], 8, size=60.0)
    _check(_run(dev, kind, *case), kind, *case)
    _check(_run(dev, kind, *case, 3.7), kind, *case, 3.7)
    _check(_run(dev, kind, *case, -0.4), kind, *case, -0.4)
    q, kc, vc, *rest = case
    same = np.broadcast_to(kc[:1, :, :1], kc.shape)
    _check(_run(dev, kind, q, same, vc, *rest), kind, q, same, vc, *rest)
    _check(_run(dev, kind, 0 * q, kc, vc, *rest), kind, 0 * q, kc, vc, *rest)


@pytest.mark.gpu
def test_values_that_are_not_finite_reach_their_rows_only(dev):
    """A NaN key or value of one block: the rows that list it are NaN, the others as without it."""
    q, kc, vc, blocks, pos, seq, tab = _case(37, "bf16", 4, 2, 64, 16, [(90, 1), (95, 1), (60, 1)], 3)
    blocks[0, :, :], blocks[1, :, :] = [0, 1, 2], [3, 4, 5]
    clean = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    kc[tab[0, 1], 0, 3, 5] = np.nan
    vc[tab[1, 4], 1, 2, 9] = np.inf
    out, lse = _run(dev, "bf16", q, kc, vc, blocks, pos, seq, tab)
    assert np.isnan(out[0, :2]).all() and np.isnan(lse[0, :2]).all()
    assert np.isposinf(out[1, 2:, 9]).all()
    out[0, :2], lse[0, :2], out[1, 2:, 9] = clean[0][0, :2], clean[1][0, :2], clean[0][1, 2:, 9]
    assert np.array_equal(out, clean[0]) and np.array_equal(lse, clean[1])


@pytest.mark.gpu
def test_keys_of_minus_infinity_weigh_nothing(dev):
    """q . k of -inf for some keys, and for all of a row's: no NaN, the second zeros and -inf."""
    q, kc, vc, blocks, pos, seq, tab = _case(39, "fp16", 2, 1, 64, 16, [(47, 1), (47, 1)], 3)
    q[:, :, 0] = np.abs(q[:, :, 0]) + 1
    kc[tab[0, 1], :, :7, 0] = -np.inf
    kc[tab[1], :, :, 0] = -np.inf
    got = _run(dev, "fp16", q, kc, vc, blocks, pos, seq, tab)
    finite = kc.copy()
    finite[tab[0, 1], :, :7, 0] = -30000.0
    _check((got[0][:1], got[1][:1]), "fp16", q[:1], finite, vc, blocks[:1], pos[:1], seq[:1], tab)
    assert (got[0][1] == 0).all() and np.isneginf(got[1][1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 600])
def test_offsets_past_32_bits(dev, tokens):
    """Caches of 2.4 G elements: blocks on their first and last pages, few rows and many."""
    import torch

    from retrieve_amd import kv

    pages, page, d = 18400, 128, 128
    kc = torch.zeros((pages, 8, page, d), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    small_k = normal16(41, (4, 8, page, d), "bf16")
    small_v = normal16(42, (4, 8, page, d), "bf16")
    where = [0, pages // 2, pages - 2, pages - 1]
    kc[where], vc[where] = to(dev, small_k, "bf16"), to(dev, small_v, "bf16")
    q = normal16(43, (tokens, 16, d), "bf16")
    pos = np.array([4 * page - 1, 3 * page + 9] * (tokens // 2), np.int32)
    seq = np.zeros(tokens, np.int32)
    blocks = np.broadcast_to(np.arange(4, dtype=np.int32), (tokens, 8, 4))
    got = kv.block_attention(to(dev, q, "bf16"), kc, vc, to(dev, blocks), to(dev, pos), to(dev, seq),
                             torch.tensor([where], dtype=torch.int32, device=dev))
    last = slice(-20, None)
    _check([back(x)[last] for x in got], "bf16", q[last], small_k, small_v, blocks[last], pos[last],
           seq[last], np.arange(4, dtype=np.int32)[None])


@pytest.mark.gpu
def test_strided_queries(dev):
    import torch

    from retrieve_amd import kv

    q, kc, vc, blocks, pos, seq, tab = _case(45, "bf16", 4, 2, 64, 16, [(60, 5), (9, 1)], 3)
    x = torch.zeros((6, 4, 71), dtype=torch.bfloat16, device=dev)
    x[..., 7:] = to(dev, q, "bf16")
    wide = torch.cat([to(dev, q, "bf16"), to(dev, q, "bf16")], 1)
    for view in (x[..., 7:], wide[:, 4:], to(dev, q.transpose(1, 0, 2), "bf16").transpose(0, 1)):
        got = kv.block_attention(view, to(dev, kc, "bf16"), to(dev, vc, "bf16"), to(dev, blocks),
                                 to(dev, pos), to(dev, seq), to(dev, tab))
        _check([back(y) for y in got], "bf16", q, kc, vc, blocks, pos, seq, tab)


@pytest.mark.gpu
def test_the_same_bits_every_time(dev):
    """No order that changes from call to call: few rows (split and joined) and many."""
    for case in (_case(47, "bf16", 8, 2, 64, 16, [(9000, 1)], 200),
                 _case(47, "bf16", 8, 2, 64, 16, [(300, 400)], 6),
                 _many(48, "bf16", 4, 1, 64, 16, 9)):
        first = _run(dev, "bf16", *case)
        for _ in range(3):
            again = _run(dev, "bf16", *case)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.gpu
def test_refusals(dev):
    from retrieve_amd import kv

    q, kc, vc, blocks, pos, seq, tab = _case(49, "bf16", 4, 2, 64, 16, [(60, 2)], 3)
    good = dict(q=to(dev, q, "bf16"), k_cache=to(dev, kc, "bf16"), v_cache=to(dev, vc, "bf16"),
                blocks=to(dev, blocks), positions=to(dev, pos), seq_ids=to(dev, seq),
                page_table=to(dev, tab))
    kv.block_attention(**good)
    for error, wrong in [
        (ValueError, {"q": good["q"][:, :3]}), (TypeError, {"q": good["q"].half()}),
        (ValueError, {"q": good["q"][..., :32]}), (ValueError, {"blocks": good["blocks"][:1]}),
        (ValueError, {"blocks": good["blocks"][:, :1]}), (TypeError, {"blocks": good["blocks"].long()}),
        (ValueError, {"blocks": good["blocks"].transpose(1, 2)}),
        (ValueError, {"v_cache": good["v_cache"][1:]}), (TypeError, {"v_cache": good["v_cache"].half()}),
        (ValueError, {"k_cache": good["k_cache"].transpose(2, 3)}),
        (ValueError, {"positions": good["positions"][:1]}),
        (TypeError, {"positions": good["positions"].long()}),
        (ValueError, {"seq_ids": good["seq_ids"].cpu()}),
    ]:
        with pytest.raises(error):
            kv.block_attention(**{**good, **wrong})


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_scales_that_are_not_finite_are_refused(dev, scale):
    """(3e38 is not finite in the kernels' powers of two.)"""
    from retrieve_amd import kv

    q, kc, vc, blocks, pos, seq, tab = _case(51, "bf16", 4, 2, 64, 16, [(60, 2)], 3)
    with pytest.raises(ValueError, match="scale"):
        kv.block_attention(to(dev, q, "bf16"), to(dev, kc, "bf16"), to(dev, vc, "bf16"),
                           to(dev, blocks), to(dev, pos), to(dev, seq), to(dev, tab), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count,tokens",
                         [("fp16", 8, 4, 128, 16, 128, 410), ("bf16", 14, 7, 96, 32, 65, 460),
                          ("bf16", 4, 2, 256, 16, 96, 520), ("fp16", 8, 8, 64, 16, 129, 420),
                          ("bf16", 32, 8, 128, 16, 256, 211), ("fp16", 16, 8, 192, 64, 70, 150)])
def test_prompts_of_long_lists(dev, kind, heads, heads_kv, d, page, count, tokens):
    """A workgroup's lists are joined though few of its tokens' fit."""
    had_new = [(150 * page + 3, tokens - tokens // 3 - 9), (0, tokens // 3), (300 * page, 9)]
    case = _case(tokens + d, kind, heads, heads_kv, d, page, had_new, count, sparse=0.1)
    got = _run(dev, kind, *case)
    pick = np.r_[0:12, rng(7).integers(0, tokens, 40), tokens - 12:tokens]
    got, case = _some(got, case, pick)
    _check(got, kind, *case)

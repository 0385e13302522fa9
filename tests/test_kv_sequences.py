"""Calls over page tables with more rows than their tokens have sequences."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to
from tests.test_kv_attention import _check

SLOTS = 700


def _case(seed, had_new, heads, heads_kv, d, page, count, kind="bf16"):
    """Some of a table's slots hold sequences, spread over its rows."""
    pos, seq, few, pages = layout(seed, page, had_new)
    rows = np.sort(rng(seed + 1).permutation(SLOTS)[:len(had_new)])
    tab = np.full((SLOTS, few.shape[1]), -1, np.int32)
    tab[rows] = few
    seq = rows[seq].astype(np.int32)
    q = normal16(seed + 2, (len(pos), heads, d), kind)
    codes = rng(seed + 3).integers(-127, 128, (pages, heads_kv, 2 * d), dtype=np.int8)
    scales = rng(seed + 4).random((pages, heads_kv), dtype=np.float32) + np.float32(0.1)
    kc = normal16(seed + 5, (pages, heads_kv, page, d), kind)
    vc = normal16(seed + 6, (pages, heads_kv, page, d), kind)
    print(f"{len(pos)} tokens, {heads}/{heads_kv} heads of {d}, pages of {page}", flush=True)
    return q, codes, scales, kc, vc, pos, seq, tab, count


CASES = [([(16 * 40, 500)], 16, 8, 128, 16, 12), ([(5, 300), (900, 260)], 8, 4, 64, 16, 9),
         ([(64 * 30, 90)], 32, 8, 128, 64, 16), ([(400 + i, 1) for i in range(30)] + [(32 * 20, 450)],
                                                 8, 8, 96, 32, 6)]


@pytest.mark.gpu
@pytest.mark.parametrize("had_new,heads,heads_kv,d,page,count", CASES)
@pytest.mark.parametrize("sequences", [None, 1, "known", 10**6])
def test_the_results_do_not_depend_on_the_number(dev, sequences, had_new, heads, heads_kv, d, page,
                                                 count):
    """Unsaid, right, too small and too large: the blocks are the oracle's, the outputs within the
    roundings."""
    from retrieve_amd import kv

    q, codes, scales, kc, vc, pos, seq, tab, count = _case(31 + count, had_new, heads, heads_kv, d,
                                                           page, count)
    n = len(had_new) if sequences == "known" else sequences
    where = [to(dev, x) for x in (pos, seq, tab)]
    g = to(dev, q, "bf16")
    blocks = kv.select_blocks(g, to(dev, codes), to(dev, scales), *where, page, count, 1, 2, n)
    out, lse = kv.block_attention(g, to(dev, kc, "bf16"), to(dev, vc, "bf16"), blocks, *where,
                                  sequences=n)
    pick = np.unique(np.r_[0:5, rng(3).integers(0, len(pos), 25), len(pos) - 4:len(pos)])
    want = okv.select(q[pick], codes, scales, pos[pick], seq[pick], tab, page, count, 1, 2)
    assert np.array_equal(back(blocks)[pick], want)
    _check((back(out)[pick], back(lse)[pick]), "bf16", q[pick], kc, vc, want, pos[pick], seq[pick],
           tab)


@pytest.mark.gpu
@pytest.mark.parametrize("sequences", [0, -1])
def test_numbers_below_one_are_refused(dev, sequences):
    from retrieve_amd import kv

    q, codes, scales, kc, vc, pos, seq, tab, count = _case(41, [(40, 3)], 4, 2, 64, 16, 4)
    where = [to(dev, x) for x in (pos, seq, tab)]
    g, blocks = to(dev, q, "bf16"), to(dev, np.zeros((3, 2, 1), np.int32))
    with pytest.raises(ValueError, match="sequences"):
        kv.select_blocks(g, to(dev, codes), to(dev, scales), *where, 16, 4, sequences=sequences)
    with pytest.raises(ValueError, match="sequences"):
        kv.block_attention(g, to(dev, kc, "bf16"), to(dev, vc, "bf16"), blocks, *where,
                           sequences=sequences)


def test_the_workspace_follows_the_number():
    """512 tokens of one sequence in a table of 700 rows take the prompts' two launches, 512 single
    tokens one."""
    import torch  # noqa: F401

    from retrieve_amd import _native as nat

    lib = nat.lib()
    assert lib.rt_kv_select_workspace(512, 8, 1, 500, 32, 1, 2) == 512 * 8 * 512 * 4
    assert lib.rt_kv_select_workspace(512, 8, SLOTS, 500, 32, 1, 2) == 0


def test_the_cache_knows_its_sequences(monkeypatch):
    """The slots that hold pages, unless the caller says how many."""
    import torch

    from retrieve_amd import kv

    seen = []
    monkeypatch.setattr(kv, "select_blocks", lambda *a: seen.append(a[-1]))
    monkeypatch.setattr(kv, "block_attention", lambda *a: seen.append(a[-1]))
    c = kv.PagedCache(pages=40, heads=1, dim=64, page=16, sequences=8, device="cpu")
    q, i = torch.zeros((1, 1, 64), dtype=torch.bfloat16), torch.zeros((1,), dtype=torch.int32)
    c.attend(q, i, i, 4)
    for s, tokens in ((0, 5), (3, 0), (5, 40), (0, 30), (6, 1)):
        c.reserve(s, tokens)
    c.attend(q, i, i, 4)
    c.free(5)
    c.free(5)
    c.select(q, i, i, 4)
    c.attend(q, i, i, 4, sequences=1)
    assert seen == [None, None, 3, 3, 2, 1, 1]

"""Choosing blocks through page tables wider than the contexts."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to


def _call(dev, seed, kind, heads, heads_kv, d, had_new, how, max_pages):
    """The call's choice, and a function that gives the oracle's for some of its tokens."""
    from retrieve_amd import kv

    print(f"select {kind} {heads}/{heads_kv} d={d} {how} of {max_pages} columns", flush=True)
    pos, seq, tab, pages = layout(seed, 16, had_new, max_pages=max_pages)
    q = normal16(seed + 1, (len(pos), heads, d), kind)
    codes = rng(seed + 2).integers(-127, 128, (pages, heads_kv, 2 * d), dtype=np.int8)
    scales = rng(seed + 3).random((pages, heads_kv), dtype=np.float32) + np.float32(0.1)
    got = back(kv.select_blocks(to(dev, q, kind), to(dev, codes), to(dev, scales), to(dev, pos),
                                to(dev, seq), to(dev, tab), 16, *how))

    def want(pick):
        return okv.select(q[pick], codes, scales, pos[pick], seq[pick], tab, 16, *how)

    return got, want


def _some(tokens, *near):
    return np.unique(np.r_[0:4, [x for n in near for x in range(n - 3, n + 3)],
                           rng(9).integers(0, tokens, 25), tokens - 4:tokens])


@pytest.mark.gpu
@pytest.mark.parametrize("max_pages,count", [(1500, 24), (3000, 200), (5000, 64), (17000, 64)])
def test_short_and_long_rows_of_a_wide_table(dev, max_pages, count):
    """Many rows, each cut by its own number of candidates: none, a few, about 1024, more."""
    had_new = [(0, 700), (16 * 300, 900), (16 * 1024 - 400, 800), (16 * 1400, 90)]
    got, want = _call(dev, 3, "bf16", 2, 1, 64, had_new, (count, 1, 2), max_pages)
    at = 1600 + 400  # (the token whose own block is the 1025th)
    pick = _some(len(got), 700, 1600, at, at + 48, at + 64, 2400)
    assert np.array_equal(got[pick], want(pick))


def test_the_workspace_is_bounded():
    """However many tokens, however wide the table: at most 512 MiB, or a single token's keys."""
    import torch  # noqa: F401

    from retrieve_amd import _native as nat

    def need(t, heads_kv, max_pages):
        return nat.lib().rt_kv_select_workspace(t, heads_kv, 2, max_pages, 64, 1, 2)

    most = 512 << 20
    for t, heads_kv, max_pages in [(8192, 8, 2048), (32768, 8, 4096), (4099, 8, 16384), (2**20, 8, 700),
                                   (32768, 8, 16384), (5000, 1, 10**6), (2**30, 128, 65)]:
        assert 0 < need(t, heads_kv, max_pages) <= most, (t, heads_kv, max_pages)
    assert need(3, 1024, 2**20) == 4 * 1024 * 2**20
    assert need(400, 8, 1000) == 4 * 400 * 8 * 1024  # (one slab)


@pytest.mark.gpu
def test_prompts_in_slabs(dev):
    """1400 tokens of which 576 are taken at a time (a table of 29056 columns, 8 heads): the pieces'
    first and last tokens, and of the last, short one."""
    from retrieve_amd import _native as nat

    heads_kv, columns = 8, 29056
    had_new = [(16 * 200, 700), (16 * 90 + 5, 650), (3, 50)]
    assert nat.lib().rt_kv_select_workspace(1400, heads_kv, 3, columns, 24, 1, 2) \
        == 576 * 4 * heads_kv * columns
    got, want = _call(dev, 5, "fp16", 16, heads_kv, 64, had_new, (24, 1, 2), columns)
    pick = _some(len(got), 576, 700, 1152, 1350)
    assert np.array_equal(got[pick], want(pick))


@pytest.mark.gpu
def test_single_tokens_in_slabs(dev):
    """150 sequences' tokens, 63 at a time (a table of 266240 columns, 8 heads)."""
    from retrieve_amd import _native as nat

    heads_kv, columns = 8, 266240
    had_new = [(16 * (7 * i % 300) + i % 16, 1) for i in range(150)]
    assert nat.lib().rt_kv_select_workspace(150, heads_kv, 150, columns, 24, 1, 2) \
        == 63 * 4 * heads_kv * columns
    got, want = _call(dev, 7, "bf16", 16, heads_kv, 64, had_new, (24, 1, 2), columns)
    pick = np.r_[0:5, 58:68, 120:150]
    assert np.array_equal(got[pick], want(pick))

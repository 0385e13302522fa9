"""Sequences that share pages of a prefix: full for one, still partly past another's tokens."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, normal16, to
from tests.test_kv_attention import _check

PAGE = 16


def _shared(tokens, shift):
    """Tokens of three sequences in turn over one pool: B holds 20 blocks; A's first ten are B's, and
    its tokens are inside the ninth and tenth of them; C holds B's blocks 3 to 12 as its own blocks
    ``shift`` lower, and ends inside the last."""
    pages = 40
    order = rng(1).permutation(pages).astype(np.int32)
    tab = np.full((3, 24), -1, np.int32)
    tab[1, :20] = order[:20]
    tab[0, :10] = tab[1, :10]
    tab[2, :3 - shift] = order[20:23 - shift]
    tab[2, 3 - shift:13 - shift] = tab[1, 3:13]
    seq = np.arange(tokens, dtype=np.int32) % 3
    step = np.arange(tokens) // 3
    pos = np.where(seq == 0, 8 * PAGE + step % (2 * PAGE), 0)
    pos = np.where(seq == 1, 19 * PAGE + step % PAGE, pos)
    pos = np.where(seq == 2, (12 - shift) * PAGE + step % PAGE, pos).astype(np.int32)
    return pos, seq, tab, pages


def _lists(seed, pos, heads_kv, count):
    """Some blocks of each row, the token's own and a shared one always among them."""
    out = np.full((len(pos), heads_kv, count), -1, np.int32)
    g = rng(seed)
    for t, p in enumerate(pos):
        own = p // PAGE
        for h in range(heads_kv):
            rest = g.permutation([b for b in range(own) if b != min(8, own - 1)])[:count - 2]
            row = np.r_[own, min(8, own - 1), rest]
            out[t, h, :len(row)] = g.permutation(row)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 2])
@pytest.mark.parametrize("kind,heads,heads_kv,d,tokens,count", [
    ("bf16", 8, 2, 128, 6, 5), ("bf16", 8, 2, 128, 900, 5), ("fp16", 4, 4, 64, 1200, 7),
    ("fp16", 14, 2, 256, 600, 11), ("bf16", 24, 2, 64, 2100, 6), ("bf16", 8, 8, 128, 500, 90)])
def test_attention_over_shared_pages(dev, kind, heads, heads_kv, d, tokens, count, shift):
    """Few rows, joined ones, a wave a row: each token counts a shared page's keys up to its own
    position, whatever its neighbours count; slots past every token are NaN."""
    from retrieve_amd import kv

    print(f"{kind} {heads}/{heads_kv} d={d} {tokens} tokens, {count} blocks", flush=True)
    pos, seq, tab, pages = _shared(tokens, shift)
    q = normal16(2, (tokens, heads, d), kind)
    kc, vc = (normal16(i, (pages, heads_kv, PAGE, d), kind) for i in (3, 4))
    blocks = _lists(5, pos, heads_kv, count)
    last = tab[1, 19]
    dirty = kc.copy(), vc.copy()
    for x in dirty:
        x[last, :, pos[seq == 1].max() % PAGE + 1:] = np.nan
    got = kv.block_attention(to(dev, q, kind), to(dev, dirty[0], kind), to(dev, dirty[1], kind),
                             to(dev, blocks), to(dev, pos), to(dev, seq), to(dev, tab), sequences=3)
    pick = np.unique(np.r_[0:6, rng(6).integers(0, tokens, 40), tokens - 6:tokens])
    _check((back(got[0])[pick], back(got[1])[pick]), kind, q[pick], kc, vc, blocks[pick], pos[pick],
           seq[pick], tab)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 600])
def test_selection_over_shared_pages(dev, tokens):
    from retrieve_amd import kv

    pos, seq, tab, pages = _shared(tokens, 2)
    q = normal16(7, (tokens, 4, 64), "bf16")
    codes = rng(8).integers(-127, 128, (pages, 2, 128), dtype=np.int8)
    scales = rng(9).random((pages, 2), dtype=np.float32) + np.float32(0.1)
    got = back(kv.select_blocks(to(dev, q, "bf16"), to(dev, codes), to(dev, scales), to(dev, pos),
                                to(dev, seq), to(dev, tab), PAGE, 6, 1, 2, sequences=3))
    assert np.array_equal(got, okv.select(q, codes, scales, pos, seq, tab, PAGE, 6, 1, 2))

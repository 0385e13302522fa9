"""Choosing blocks by scores at the ends of the range: infinite queries, scores of either zero."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, to

FORMS = [1, 400]  # tokens of one sequence: scored as single tokens, as a prompt


def _order(score, want):
    """The blocks that are kept of one row's scores, by (score desc, block asc), not a number
    last."""
    least = np.where(np.isnan(score), -np.inf, score)
    return sorted(np.lexsort((np.arange(len(score)), -least))[:want])


def _run(dev, q, codes, scales, tab, blocks, count, tokens):
    """One token's query at the end of ``blocks`` blocks of 16, ``tokens`` times; the rows are one
    another's copies."""
    from retrieve_amd import kv

    pos = np.full(tokens, 16 * blocks - 1, np.int32)
    got = back(kv.select_blocks(to(dev, np.repeat(q, tokens, 0), "bf16"), to(dev, codes),
                                to(dev, scales), to(dev, pos), to(dev, np.zeros_like(pos)),
                                to(dev, tab), 16, count, 0, 1))
    assert (got == got[:1]).all()
    return got[0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", FORMS)
@pytest.mark.parametrize("d", [64, 96])
def test_infinite_queries(dev, tokens, d):
    """A row that holds an infinity has codes 0 where it is finite (a number over infinity) and -127
    where it is not (not a number): only the infinite channels' bounds are in the sum, whose sign
    alone is left; a sum of 0 is not a number."""
    blocks, heads = 60, 3
    _, _, tab, pages = layout(1, 16, [(16 * blocks - 1, 1)])
    codes = rng(2).integers(-2, 3, (pages, 1, 2 * d), dtype=np.int8)
    scales = rng(3).random((pages, 1), dtype=np.float32) + np.float32(0.1)
    rows = codes[tab[0, :blocks - 1], 0].astype(np.int64)
    for where in ([5], [0, d - 1], [7, 9, 33]):
        q = normal16(4, (1, heads, d), "bf16")
        q[:, :, where] = np.array([np.inf, -np.inf, np.inf], np.float32)[:len(where)]
        c = np.zeros(d, np.int64)
        c[where] = -127
        with np.errstate(invalid="ignore"):
            score = (rows @ np.concatenate([c, np.abs(c)])).astype(np.float32) * np.float32(np.inf)
        assert len(set(np.sign(score[~np.isnan(score)]))) == 2 and np.isnan(score).any()
        got = _run(dev, q, codes, scales, tab, blocks, 20, tokens)
        assert got.tolist() == _order(score, 19) + [blocks - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", FORMS)
@pytest.mark.parametrize("blocks", [60, 5000])
def test_either_zero_is_one_score(dev, tokens, blocks):
    """Blocks of scale 0 score zero whichever the sign of their sums: ties, to the lower block."""
    _, _, tab, pages = layout(11, 16, [(16 * blocks - 1, 1)])
    q = normal16(12, (1, 2, 64), "bf16")
    codes = rng(13).integers(-127, 128, (pages, 1, 128), dtype=np.int8)
    scales = np.zeros((pages, 1), np.float32)
    best = [11, 29, blocks - 3]
    codes[tab[0, best]] = 0
    codes[tab[0, best], :, 64:] = 1
    scales[tab[0, best]] = 1.0
    got = _run(dev, q, codes, scales, tab, blocks, 20, tokens)
    assert got.tolist() == sorted(set(range(17)) | set(best)) + [blocks - 1]
